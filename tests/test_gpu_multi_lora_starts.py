"""Packed starts of multi_lora that fall, lie before the first token or behind the last: they are recorded,
sequences are clamped to the tokens, and a token that several name is one's of them or left as it is."""
import pytest
import torch

from tests import tree_ref as ref

pytestmark = pytest.mark.gpu


def _state(dev, tokens, batch, k=128, n=136, r=16, dtype=torch.bfloat16, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    x, y = torch.randn(tokens, k, device=dev, generator=g).to(dtype), torch.randn(tokens, n, device=dev, generator=g).to(dtype)
    a = (torch.randn(batch, r, k, device=dev, generator=g) / k ** 0.5).to(dtype)
    b = torch.randn(batch, n, r, device=dev, generator=g).to(dtype)
    return x, y, a, b, torch.rand(batch, device=dev, generator=g) + 0.5, torch.arange(batch, device=dev, dtype=torch.int32)


def _clamped(starts, tokens):
    return [(max(s, 0), min(e, tokens)) for s, e in zip(starts, starts[1:])]


SKEWED = [  # tokens, starts of sequences that share none
    (9, [-4, 2, 5, 9]), (9, [0, 3, 6, 40]), (9, [-(1 << 31), 3, 6, (1 << 31) - 1]), (300, [-7, 150, 290, 1000]),
]


@pytest.mark.parametrize("tokens,starts", SKEWED)
def test_starts_outside_the_tokens(cuda_dev, tokens, starts):
    from fitllm_b200 import ops
    x, y, a, b, scale, adapter = _state(cuda_dev, tokens, len(starts) - 1)
    at = torch.tensor(starts, dtype=torch.int32, device=cuda_dev)
    got = ops.multi_lora(x, a, b, scale, adapter, y, q_start=at)
    assert ops.device_status() == 1
    own = _clamped(starts, tokens)
    flat = [s for s, _ in own] + [own[-1][1]]
    want = ops.multi_lora(x, a, b, scale, adapter, y, q_start=torch.tensor(flat, dtype=torch.int32, device=cuda_dev))
    assert ops.device_status() == 0 and torch.equal(got, want)
    exact = ref.multi_lora(x, a, b, scale, adapter, y, flat)
    assert ((want.double() - exact).abs() <= ref.multi_lora_bound(x, a, b, scale, adapter, y, flat, x.dtype)).all()


@pytest.mark.parametrize("tokens,starts", [
    (9, [0, 6, 3, 9]), (9, [0, 9, 3, 3]), (9, [5, 2, 7, 9]), (700, [0, 600, 90, 333, 333, 20, 700]),
    (500, [7 * i % 31 * 16 for i in range(41)]), (12, [0, 12, 0, 12, 0, 12]),
])
def test_starts_that_fall(cuda_dev, tokens, starts):
    from fitllm_b200 import ops
    batch = len(starts) - 1
    x, y, a, b, scale, adapter = _state(cuda_dev, tokens, batch, seed=tokens)
    at = torch.tensor(starts, dtype=torch.int32, device=cuda_dev)
    got = ops.multi_lora(x, a, b, scale, adapter, y, q_start=at, out=y.clone())
    assert ops.device_status() == 1
    for _ in range(3):  # in place, as the passes call it: the same again
        assert torch.equal(ops.multi_lora(x, a, b, scale, adapter, y, q_start=at, out=y.clone()), got)
        assert ops.device_status() == 1
    fits = (got == y).all(1)
    for s, (lo, hi) in enumerate(_clamped(starts, tokens)):
        if lo < hi:
            one = torch.tensor([0, hi - lo], dtype=torch.int32, device=cuda_dev)
            rows = ops.multi_lora(x[lo:hi], a, b, scale, adapter[s:s + 1].contiguous(), y[lo:hi], q_start=one)
            fits[lo:hi] |= ((got[lo:hi] - rows).abs() <= 0.02 * rows.abs() + 0.02).all(1)
    assert fits.all() and not torch.equal(got, y)
    # a later call is as ever
    even = torch.tensor([0] + [tokens] * batch, dtype=torch.int32, device=cuda_dev)
    ops.multi_lora(x, a, b, scale, adapter, y, q_start=even)
    assert ops.device_status() == 0


def test_many_sequences_of_a_token(cuda_dev):
    """Searches over several levels; empty sequences between."""
    from fitllm_b200 import ops
    batch, tokens = 2500, 1700
    g = torch.Generator().manual_seed(3)
    cuts = torch.randint(0, tokens + 1, (batch - 1,), generator=g).sort().values.tolist()
    starts = [0] + cuts + [tokens]
    x, y, a, b, scale, _ = _state(cuda_dev, tokens, 7, seed=2)
    adapter = torch.randint(-1, 7, (batch,), generator=g).int().to(cuda_dev)
    at = torch.tensor(starts, dtype=torch.int32, device=cuda_dev)
    got = ops.multi_lora(x, a, b, scale, adapter, y, q_start=at)
    assert ops.device_status() == 0
    exact = ref.multi_lora(x, a, b, scale, adapter, y, starts)
    assert ((got.double() - exact).abs() <= ref.multi_lora_bound(x, a, b, scale, adapter, y, starts, x.dtype)).all()
