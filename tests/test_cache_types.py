"""Caches of the passes hold bf16: what the projections give and the append kernels write."""
import pytest
import torch


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_the_cache_of_trees_is_bf16(dtype):
    from fitllm_b200.verify import TreeKVCache
    with pytest.raises(ValueError, match="bf16"):
        TreeKVCache(1, 2, 1, 64, 16, "cpu", dtype=dtype)
    assert TreeKVCache(1, 2, 1, 64, 16, "cpu", dtype=torch.bfloat16).k[0].dtype == torch.bfloat16


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_the_append_of_a_pass_refuses_other_caches(dtype):
    from fitllm_b200.layer_ops import rope_kv_append
    q, k = torch.zeros(2, 3, 256, dtype=torch.bfloat16), torch.zeros(2, 3, 64, dtype=torch.bfloat16)
    cos = torch.zeros(3, 32)
    good, bad = torch.zeros(2, 1, 16, 64, dtype=torch.bfloat16), torch.zeros(2, 1, 16, 64, dtype=dtype)
    for args in ((q, k, k, bad, bad), (q, k, k, good, bad), (q, k, k, bad, good), (q.to(dtype), k, k, good, good),
                 (q, k.to(dtype), k, good, good)):
        with pytest.raises(ValueError, match="bf16"):
            rope_kv_append(*args[:3], cos, cos, *args[3:], 0, 4, 1)
