"""Adapters of many requests beside a shared projection, against the definition in 64
bits; the tolerance is derived in tests/tree_ref.py."""
import pytest
import torch

from tests import tree_ref as ref

pytestmark = pytest.mark.gpu


def _state(dev, news, k, n, r, adapters, dtype, seed=0, lead=0, tail=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    starts = [lead]
    for c in news:
        starts.append(starts[-1] + c)
    tokens = starts[-1] + tail
    x, y = torch.randn(tokens, k, device=dev, generator=g).to(dtype), torch.randn(tokens, n, device=dev, generator=g).to(dtype)
    a = (torch.randn(adapters, r, k, device=dev, generator=g) / k ** 0.5).to(dtype)
    b = torch.randn(adapters, n, r, device=dev, generator=g).to(dtype)
    scale = torch.rand(adapters, device=dev, generator=g) * 3 - 1
    adapter = torch.randint(-1, adapters, (len(news),), device=dev, generator=g).int()
    return x, y, a, b, scale, adapter, starts


def _check(x, y, a, b, scale, adapter, starts, got):
    exact = ref.multi_lora(x, a, b, scale, adapter, y, starts)
    bound = ref.multi_lora_bound(x, a, b, scale, adapter, y, starts, x.dtype)
    worst = ((got.double() - exact).abs() / bound).max().item()
    assert worst <= 1.0, f"error {worst:.2f} times the bound"


CASES = [
    # new tokens of each sequence, K, N, R, adapters, dtype
    ([1], 8, 8, 16, 1, torch.bfloat16),
    ([1], 5120, 5120, 16, 4, torch.bfloat16),
    ([1] * 64, 1024, 1048, 16, 64, torch.float16),
    ([5] * 8, 512, 264, 32, 3, torch.bfloat16),
    ([1, 0, 17, 3, 200, 0, 64], 776, 520, 48, 4, torch.float16),
    ([300, 1, 1, 129], 2048, 1000, 64, 2, torch.bfloat16),
    ([15, 16, 17, 31, 32, 33], 264, 136, 64, 6, torch.float16),
    ([0, 0, 7], 5128, 1544, 16, 9, torch.bfloat16),
    ([2] * 130, 520, 2056, 16, 5, torch.bfloat16),
    ([1000], 1024, 512, 32, 1, torch.float16),
    ([3], 27648, 128, 64, 2, torch.float16),
]


@pytest.mark.parametrize("news,k,n,r,adapters,dtype", CASES)
def test_multi_lora(cuda_dev, news, k, n, r, adapters, dtype):
    from fitllm_b200 import ops
    x, y, a, b, scale, adapter, starts = _state(cuda_dev, news, k, n, r, adapters, dtype)
    start = torch.tensor(starts, dtype=torch.int32, device=cuda_dev)
    got = ops.multi_lora(x, a, b, scale, adapter, y, q_start=start)
    assert ops.device_status() == 0
    _check(x, y, a, b, scale, adapter, starts, got)
    assert torch.equal(got, ops.multi_lora(x, a, b, scale, adapter, y, q_start=start))
    none = torch.full_like(adapter, -1)
    assert torch.equal(ops.multi_lora(x, a, b, scale, none, y, q_start=start), y)
    if len(set(news)) == 1:
        assert torch.equal(ops.multi_lora(x, a, b, scale, adapter, y), got)


def test_rows_of_no_sequence_stay(cuda_dev):
    from fitllm_b200 import ops
    x, y, a, b, scale, adapter, starts = _state(cuda_dev, [4, 0, 30], 256, 264, 16, 2, torch.bfloat16, lead=3, tail=21)
    adapter[2] = 1
    start = torch.tensor(starts, dtype=torch.int32, device=cuda_dev)
    out = torch.full_like(y, 7.0)
    got = ops.multi_lora(x, a, b, scale, adapter, y, q_start=start, out=out)
    assert got is out and got[:3].eq(7).all() and got[starts[-1]:].eq(7).all()
    rows = slice(3, starts[-1])
    own = [s - 3 for s in starts]
    _check(x[rows], y[rows], a, b, scale, adapter, own, got[rows])
    # what stands in the other rows reaches nobody
    x[:3], x[starts[-1]:] = float("nan"), float("inf")
    assert torch.equal(ops.multi_lora(x, a, b, scale, adapter, y, q_start=start, out=out.clone())[rows], got[rows])


@pytest.mark.parametrize("k,r,dtype", [(1032, 64, torch.bfloat16), (8, 16, torch.float16), (2120, 48, torch.float16),
                                       (264, 32, torch.bfloat16)])
def test_prompts_beside_one_another(cuda_dev, k, r, dtype):
    """Slots that are full, nearly so and not, in parts of K some of which are short or empty: rows of other
    sequences that hold no numbers stand in the same copies and reach nobody."""
    from fitllm_b200 import ops
    news = [100, 20, 128, 97, 96, 31, 260, 17, 16, 1]
    x, y, a, b, scale, adapter, starts = _state(cuda_dev, news, k, 136, r, 3, dtype, seed=k)
    adapter.copy_(torch.tensor([0, -1, 2, -1, 1, 0, -1, 2, 1, -1]))
    start = torch.tensor(starts, dtype=torch.int32, device=cuda_dev)
    clean = ops.multi_lora(x, a, b, scale, adapter, y, q_start=start)
    _check(x, y, a, b, scale, adapter, starts, clean)
    for s, l in enumerate(adapter.tolist()):
        if l < 0:
            x[starts[s]:starts[s + 1]] = float("nan")
    assert torch.equal(ops.multi_lora(x, a, b, scale, adapter, y, q_start=start), clean)
    wide = torch.full((x.shape[0], k + 24), float("inf"), device=cuda_dev).to(dtype)
    wide[:, 16:16 + k] = x
    assert torch.equal(ops.multi_lora(wide[:, 16:16 + k], a, b, scale, adapter, y, q_start=start), clean)
    # equal lengths, told or not
    even = torch.arange(0, 601, 100, dtype=torch.int32, device=cuda_dev)
    x, y, adapter = x[:600].nan_to_num(0.5), y[:600], adapter[:6].clamp(min=0)
    assert torch.equal(ops.multi_lora(x, a, b, scale, adapter, y, q_start=even), ops.multi_lora(x, a, b, scale, adapter, y))
    assert ops.device_status() == 0


def test_in_place_and_strided(cuda_dev):
    from fitllm_b200 import ops
    x, y, a, b, scale, adapter, starts = _state(cuda_dev, [9, 40], 128, 136, 32, 3, torch.float16)
    start = torch.tensor(starts, dtype=torch.int32, device=cuda_dev)
    want = ops.multi_lora(x, a, b, scale, adapter, y, q_start=start)
    wide_x, wide_y = torch.randn(49, 200, device=cuda_dev).half(), torch.randn(49, 160, device=cuda_dev).half()
    wide_x[:, 8:136], wide_y[:, 16:152] = x, y
    assert torch.equal(ops.multi_lora(wide_x[:, 8:136], a, b, scale, adapter, wide_y[:, 16:152], q_start=start), want)
    wide_x[:, 3:131], wide_y[:, 1:137] = x.clone(), y.clone()  # rows that are not aligned are copied
    assert torch.equal(ops.multi_lora(wide_x[:, 3:131], a, b, scale, adapter, wide_y[:, 1:137], q_start=start), want)
    assert ops.multi_lora(x, a, b, scale, adapter, y, q_start=start, out=y) is y and torch.equal(y, want)


def test_adapters_that_are_not_there(cuda_dev):
    from fitllm_b200 import ops
    x, y, a, b, scale, adapter, starts = _state(cuda_dev, [2, 2, 2], 128, 128, 16, 2, torch.bfloat16)
    adapter.copy_(torch.tensor([2, 1, -2]))
    got = ops.multi_lora(x, a, b, scale, adapter, y)
    assert ops.device_status() == 1
    assert torch.equal(got[:2], y[:2]) and torch.equal(got[4:], y[4:]) and not torch.equal(got[2:4], y[2:4])
    # an adapter that holds no numbers reaches its own request alone
    adapter.copy_(torch.tensor([0, 1, -1]))
    clean = ops.multi_lora(x, a, b, scale, adapter, y)
    a[0] = float("nan")
    got = ops.multi_lora(x, a, b, scale, adapter, y)
    assert got[:2].isnan().all() and torch.equal(got[2:], clean[2:]) and ops.device_status() == 0


@pytest.mark.parametrize("starts", [[0, 6, 3, 9], [-4, 2, 5, 9], [0, 3, 6, 40]])
def test_bad_starts_lead_nowhere(cuda_dev, starts):
    """Starts that fall, lie before the first token or behind the last: rows in bounds are read."""
    from fitllm_b200 import ops
    x, y, a, b, scale, adapter, _ = _state(cuda_dev, [3, 3, 3], 128, 128, 16, 2, torch.bfloat16)
    got = ops.multi_lora(x, a, b, scale, adapter, y, q_start=torch.tensor(starts, dtype=torch.int32, device=cuda_dev), out=y.clone())
    assert got.shape == y.shape and ops.device_status() in (0, 1)


def test_refusals(cuda_dev):
    from fitllm_b200 import ops
    x, y, a, b, scale, adapter, _ = _state(cuda_dev, [2, 2], 128, 128, 16, 2, torch.bfloat16)
    for args in ((x.half(), a, b, scale, adapter, y), (x, a[:, :, :120], b, scale, adapter, y), (x, a, b, scale[:1], adapter, y),
                 (x, a, b, scale, adapter.long(), y), (x, a, b, scale, adapter.cpu(), y), (x, a, b.transpose(1, 2), scale, adapter, y)):
        with pytest.raises(ValueError):
            ops.multi_lora(*args)
    with pytest.raises(NotImplementedError):
        ops.multi_lora(x.requires_grad_(), a, b, scale, adapter, y)
    with pytest.raises(ops._lib.FitqError):
        ops.multi_lora(x.detach()[:3], a, b, scale, adapter, y[:3])  # 3 tokens do not divide over 2 sequences
