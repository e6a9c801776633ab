"""fp16 prompts' roles hand over by parity, tiles of one step each: many calls of every number of steps,
one row tile and two, beside another stream's work, end without a wait run out and give the same bits."""
import pytest
import torch

from tests.test_gpu_kv4 import FP, _attend, _case, _check_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("count", [17, 61])
def test_many_fp16_rows_end_under_every_schedule(cuda_dev, d, count):
    from fitllm_b200 import ops
    c = _case([64 * i for i in range(12)], [count] * 12, 32, 8, d, 128, FP, cuda_dev, ragged=False)
    want = _attend(c)
    _check_attention(c, want)
    side, x = torch.cuda.Stream(cuda_dev), torch.randn(4096, 4096, device=cuda_dev)
    for _ in range(40):
        with torch.cuda.stream(side):
            y = x.sin()
        got = [_attend(c) for _ in range(5)]
        assert all(torch.equal(g, want) for g in got)
    side.synchronize()
    assert y.isfinite().all() and ops.device_status() == 0
