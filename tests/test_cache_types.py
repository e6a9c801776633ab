"""Caches of the passes hold bf16: what the projections give and the append kernels write."""
import pytest
import torch


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_the_cache_of_trees_is_bf16(dtype):
    from fitllm_b200.verify import TreeKVCache
    with pytest.raises(ValueError, match="bf16"):
        TreeKVCache(1, 2, 1, 64, 16, "cpu", dtype=dtype)
    assert TreeKVCache(1, 2, 1, 64, 16, "cpu", dtype=torch.bfloat16).k[0].dtype == torch.bfloat16
