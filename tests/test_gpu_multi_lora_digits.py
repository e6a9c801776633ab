"""The adapters' delta alone (y_add = 0), at the contraction lengths of the served layers: its digits by norms
(tests/multi_lora_digits.py), in the kernels of few tokens and in the tcgen05 product of prompts."""
import pytest
import torch

from tests import multi_lora_digits as digits
from tests import tree_ref as ref

pytestmark = pytest.mark.gpu

CASES = [
    # tokens of each sequence, K, N, R
    ([1] * 64, 5120, 1024, 16),
    ([3], 27648, 8192, 64),
    ([16, 1, 9], 27648, 1024, 32),
    ([300, 129], 27648, 512, 64),
    ([17] * 160, 27648, 256, 64),   # a CTA sums all of K
    ([64] * 150, 13824, 128, 32),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("news,k,n,r", CASES)
def test_digits_of_the_delta(cuda_dev, news, k, n, r, dtype):
    from fitllm_b200 import ops
    g = torch.Generator(device=cuda_dev).manual_seed(k + len(news))
    tokens, batch = sum(news), len(news)
    x = torch.randn(tokens, k, device=cuda_dev, generator=g).to(dtype)
    a = (torch.randn(3, r, k, device=cuda_dev, generator=g) / k ** 0.5).to(dtype)
    b = torch.randn(3, n, r, device=cuda_dev, generator=g).to(dtype)
    scale = torch.tensor([0.7, 1.0, 1.9], device=cuda_dev)
    adapter = (torch.arange(batch, device=cuda_dev) % 3).int()
    starts = [0]
    for c in news:
        starts.append(starts[-1] + c)
    at = torch.tensor(starts, dtype=torch.int32, device=cuda_dev)
    zero = torch.zeros(tokens, n, device=cuda_dev, dtype=dtype)
    got = ops.multi_lora(x, a, b, scale, adapter, zero, q_start=at)
    assert ops.device_status() == 0
    delta = ref.multi_lora(x, a, b, scale, adapter, zero, starts)
    error, limit = (got.double() - delta).norm().item(), digits.bound(delta, k, dtype)
    print(f"error {error / digits.rounding(delta, dtype):.4f} of the rounding's, bound {limit / digits.rounding(delta, dtype):.4f}")
    assert error <= limit
