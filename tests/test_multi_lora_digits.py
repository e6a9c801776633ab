"""The bound of tests/multi_lora_digits.py sees what it is for: mistakes planted in the restatement (no GPU needed)."""
import pytest
import torch

from tests import multi_lora_digits as digits


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("k,r", [(512, 16), (5120, 32), (27648, 64)])
def test_a_lost_half_is_seen(dtype, k, r):
    g = torch.Generator().manual_seed(k)
    x, a = torch.randn(96, k, generator=g).to(dtype).double(), (torch.randn(r, k, generator=g) / k ** 0.5).to(dtype).double()
    b, scale = torch.randn(512, r, generator=g).to(dtype).double(), 0.7
    t = x @ a.T
    delta = scale * (t @ b.T)

    def error(t):
        return ((scale * (t @ b.T)).to(dtype).double() - delta).norm().item()

    limit = digits.bound(delta, k, dtype)
    assert error(digits.parts(t, dtype, 2)) < limit
    assert error(digits.parts(t, dtype, 1)) > 1.05 * limit  # lo lost
    assert error(t * (1 - 2.0 ** -24 * k / 16 / 2)) < limit  # sums that lose half a step of a third of the last sum
    assert error(t * (1 + torch.finfo(dtype).eps / 2)) > 1.05 * limit
