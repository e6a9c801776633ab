"""Token log probabilities, entropies, top alternatives and their gradient against
64 bits.

Bounds.  A row's sums are joined from at most 2^6 fp32 terms in a row and a tree
of 2^5 more, each off by 2^-24, over exponentials off by 2^-21 (the approximate
base-2 exponential, its argument rounded once): log S is off by at most
(96 / 8 + 1) 2^-21 < 2^-17.  logp adds two roundings of values up to |logp| (2^-23
|logp|); the entropy adds the same relative error of a mean of |z - M|, taken as
2^-17 (1 + H).  A gradient is g p (...) with p off by the error of its logarithm,
below 2^-15 at these sizes, and is rounded to the logits' type: half a step, u.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25, torch.float32: 0.0}  # half a subnormal step
BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32


def _logits(rows, vocab, dtype, dev, seed=0, stride=None, offset=0, std=3.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    stride = stride or vocab
    flat = torch.full((rows * stride + offset + 8,), 50.0, dtype=dtype, device=dev)
    z = flat[offset:offset + rows * stride].view(rows, stride)[:, :vocab]
    z.copy_(torch.randn(rows, vocab, generator=g, device=dev) * std)
    ids = torch.randint(0, vocab, (rows,), generator=g, device=dev)
    return z, ids


def _want(z, ids, top):
    z = z.detach().double()
    lp = torch.log_softmax(z, -1)
    ent = -torch.nansum(lp.exp() * lp, -1)
    ok = (ids >= 0) & (ids < z.shape[1])
    logp = torch.where(ok, lp.gather(1, ids.clamp(0, z.shape[1] - 1)[:, None])[:, 0], 0.0)
    order = torch.sort(z, dim=-1, descending=True, stable=True).indices[:, :top]
    return lp, logp, ent, lp.gather(1, order), order


def _check(r, z, ids, top):
    lp, logp, ent, top_lp, order = _want(z, ids, top)
    assert bool(((r.logp.double() - logp).abs() <= 2.0 ** -17 + 2.0 ** -23 * logp.abs()).all())
    assert bool(((r.entropy.double() - ent).abs() <= 2.0 ** -17 * (1 + ent)).all())
    assert torch.equal(r.top_ids, order)
    fine = top_lp.isfinite()
    assert torch.equal(r.top_logp.isfinite(), fine)
    assert bool(((r.top_logp.double() - top_lp).abs()[fine] <= (2.0 ** -17 + 2.0 ** -23 * top_lp.abs())[fine]).all())


CASES = [
    # rows, vocab, dtype, top, stride, offset
    (1, 1, F32, 1, None, 0), (3, 7, BF, 7, None, 1), (5, 64, FP, 64, 71, 3), (2, 1000, BF, 20, None, 0),
    (7, 4099, FP, 5, None, 0), (1, 32001, F32, 64, None, 1), (300, 8191, BF, 3, 8200, 5), (4, 152064, BF, 20, None, 0),
    (600, 152064, BF, 1, None, 0), (1, 152064, F32, 20, None, 0), (3, 151665, FP, 8, 152064, 0), (2, 500009, F32, 5, None, 0),
    (2, 1000003, BF, 64, None, 0), (149, 50257, BF, 0, None, 0), (37, 20000, F32, 64, None, 0),
    # many rows: CTAs of 256 threads
    (600, 30001, FP, 0, None, 1), (700, 24000, BF, 0, 24008, 3), (592, 12289, F32, 0, None, 0),
]


@pytest.mark.parametrize("rows,vocab,dtype,top,stride,offset", CASES)
def test_forward_matches_64_bits(cuda_dev, rows, vocab, dtype, top, stride, offset):
    from fitllm_b200.lm_head import token_logprobs
    z, ids = _logits(rows, vocab, dtype, cuda_dev, seed=rows + vocab, stride=stride, offset=offset)
    r = token_logprobs(z, ids, top=top)
    assert r.top_logp.shape == (rows, top) and r.top_ids.dtype == torch.int64
    _check(r, z, ids, top)
    again = token_logprobs(z, ids, top=top)
    for a, b in zip(r, again):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("vocab", [4000, 152064])
def test_ties_rank_by_index(cuda_dev, dtype, vocab):
    from fitllm_b200.lm_head import token_logprobs
    rows = 6
    z = torch.zeros(rows, vocab, dtype=dtype, device=cuda_dev)
    z[1] = float("-inf")
    z[1, 7] = z[1, vocab - 1] = 1.0       # two finite logits, then -inf from index 0 on
    z[2, 1::2] = -0.0                      # equal to 0
    z[3] = torch.arange(vocab, device=cuda_dev) // 50 * -1.0  # runs of fifty equal ones
    z[4, 100:3000] = 5.0
    z[5] = torch.finfo(dtype).min
    ids = torch.arange(rows, device=cuda_dev)
    r = token_logprobs(z, ids, top=20)
    _, _, _, top_lp, order = _want(z, ids, 20)
    assert torch.equal(r.top_ids, order)
    live = [0, 1, 2, 3, 4, 5]
    fine = top_lp.isfinite()
    assert torch.equal(r.top_logp.isfinite()[live], fine[live])


def test_masked_nan_and_infinite_logits(cuda_dev):
    from fitllm_b200.lm_head import token_logprobs
    z, ids = _logits(6, 5000, F32, cuda_dev, seed=5)
    z = z.clone()
    z[0, 1000:] = float("-inf")
    z[1] = float("-inf")                   # nothing left
    z[2, 17] = float("nan")
    z[3, 9] = float("inf")
    z[4, 10:] = torch.finfo(F32).min       # masks of the type's lowest value
    ids = torch.tensor([3, 0, 1, 2, 4, 4999], device=cuda_dev)
    z.requires_grad_(True)
    r = token_logprobs(z, ids, top=4)
    (r.logp.sum() + 0.3 * r.entropy.sum()).backward()
    keep = [0, 4, 5]
    lp, logp, ent, _, _ = _want(z, ids, 4)
    assert bool(((r.logp.double() - logp).abs()[keep] <= 1e-5).all())
    assert bool(((r.entropy.double() - ent).abs()[keep] <= 2.0 ** -17 * (1 + ent[keep])).all())
    for row in (1, 2, 3):
        assert bool(r.logp[row].isnan()) and bool(r.entropy[row].isnan()) and bool(z.grad[row].isnan().any())
    assert bool(z.grad[keep].isfinite().all())
    assert bool((z.grad[0, 1000:] == 0).all()) and bool((z.grad[4, 10:] == 0).all())
    assert int(r.top_ids[2, 0]) == 17 and int(r.top_ids[3, 0]) == 9
    assert r.top_ids[1].tolist() == [0, 1, 2, 3]


@pytest.mark.parametrize("dtype,vocab", [(BF, 30000), (FP, 30001), (F32, 12345)])
@pytest.mark.parametrize("top", [20, 0])
def test_ties_masks_and_nans_in_streamed_rows(cuda_dev, dtype, vocab, top):
    """More rows than find room as clusters: a row's candidates overflow their list, or hold a NaN."""
    from fitllm_b200.lm_head import token_logprobs
    rows, kinds = 700, 7
    z, ids = _logits(rows, vocab, dtype, cuda_dev, seed=vocab)
    z[0::kinds] = 0.0
    z[1::kinds] = float("-inf")
    z[1::kinds, 7] = z[1::kinds, vocab - 1] = 1.0
    z[2::kinds] = (torch.arange(vocab, device=cuda_dev) // 50 * -1.0).to(dtype).clamp(min=torch.finfo(dtype).min)
    z[3::kinds] = torch.finfo(dtype).min
    z[4::kinds, vocab // 2] = float("nan")
    z[5::kinds, 20:] = torch.finfo(dtype).min
    ids[1::kinds] = 7
    r = token_logprobs(z, ids, top=top)
    keep = torch.arange(rows, device=cuda_dev) % kinds != 4
    lp, logp, ent, top_lp, order = _want(z[keep], ids[keep], top)
    assert bool(((r.logp.double()[keep] - logp).abs() <= 2.0 ** -17 + 2.0 ** -23 * logp.abs()).all())
    assert bool(((r.entropy.double()[keep] - ent).abs() <= 2.0 ** -17 * (1 + ent)).all())
    assert bool(r.logp[~keep].isnan().all()) and bool(r.entropy[~keep].isnan().all())
    assert torch.equal(r.top_ids[keep], order)
    if top:
        assert bool((r.top_ids[~keep, 0] == vocab // 2).all())


@pytest.mark.parametrize("rows,vocab,dtype,top,stride,offset",
                         [(1, 1, F32, 1, None, 0), (3, 77, BF, 4, None, 1), (5, 4099, FP, 9, None, 0),
                          (4, 32001, BF, 3, 32004, 2), (2, 152064, F32, 0, None, 0), (130, 20000, BF, 0, None, 0)])
def test_backward_matches_the_formula(cuda_dev, rows, vocab, dtype, top, stride, offset):
    from fitllm_b200.lm_head import token_logprobs
    z, ids = _logits(rows, vocab, dtype, cuda_dev, seed=3 * rows + vocab, stride=stride, offset=offset)
    ids[rows // 2] = -100 if rows > 1 else ids[0]
    if rows > 2:
        ids[2] = z[2].argmax()             # the given token is an alternative too
    leaf = z.detach().requires_grad_(True)
    g = torch.Generator(device=cuda_dev).manual_seed(1)
    a, h, t = (torch.randn(s, generator=g, device=cuda_dev) for s in ((rows,), (rows,), (rows, top)))
    r = token_logprobs(leaf, ids, top=top)
    got, = torch.autograd.grad([r.logp, r.entropy, r.top_logp], leaf, [a, h, t])
    assert got.dtype == dtype and got.shape == z.shape
    zz = z.detach().double().requires_grad_(True)
    lp = torch.log_softmax(zz, -1)
    ok = ids >= 0
    order = _want(z, ids, top)[4]
    loss = (torch.where(ok, lp.gather(1, ids.clamp(min=0)[:, None])[:, 0], 0.0) * a.double()).sum()
    loss = loss - ((lp.exp() * lp).sum(-1) * h.double()).sum() + (lp.gather(1, order) * t.double()).sum()
    want, = torch.autograd.grad(loss, zz)
    p = lp.detach().exp()
    mass = a.abs()[:, None] + t.abs().sum(-1, keepdim=True) + h.abs()[:, None] * (lp.detach().abs() + 12)
    bound = U[dtype] * want.abs() + TINY[dtype] + 2.0 ** -15 * p * mass + 2.0 ** -22 * want.abs()
    assert bool(((got.double() - want).abs() <= bound + 1e-30).all())
    # one upstream gradient at a time, and through a masked middle
    for i, (up, fn) in enumerate(((a, "logp"), (h, "entropy"))):
        r = token_logprobs(leaf, ids, top=top)
        one, = torch.autograd.grad(getattr(r, fn), leaf, up)
        zeros = [torch.zeros_like(a), torch.zeros_like(h), torch.zeros_like(t)]
        zeros[i] = up
        r = token_logprobs(leaf, ids, top=top)
        all3, = torch.autograd.grad([r.logp, r.entropy, r.top_logp], leaf, zeros)
        assert torch.equal(one, all3)


def test_backward_matches_differences(cuda_dev):
    from fitllm_b200.lm_head import token_logprobs
    z, ids = _logits(3, 40, F32, cuda_dev, seed=11, std=1.0)
    ids[1] = 40  # no such token
    w = torch.tensor([0.7, -1.3, 0.4], device=cuda_dev)

    def loss(x):
        r = token_logprobs(x, ids, top=3)
        return (w * r.logp).sum() + (w * w * r.entropy).sum() - 0.5 * r.top_logp.sum()

    leaf = z.detach().requires_grad_(True)
    g, = torch.autograd.grad(loss(leaf), leaf)
    step = 2.0 ** -6
    for r in range(3):
        for c in range(0, 40, 3):
            d = torch.zeros_like(z)
            d[r, c] = step
            if not torch.equal(token_logprobs(z + d, ids, top=3).top_ids, token_logprobs(z - d, ids, top=3).top_ids):
                continue  # the order of the alternatives changes within the step
            num = float((loss(z + d) - loss(z - d)).double() / (2 * step))
            # fp32 losses near 10 over a step of 2^-5, and the third derivative's step^2 / 6
            assert abs(num - float(g[r, c])) < 4 * 10 * 2.0 ** -23 * 2 ** 5 + 4 * step ** 2


def test_leading_dimensions_other_types_of_ids_and_empty_batches(cuda_dev):
    from fitllm_b200.lm_head import token_logprobs
    z, ids = _logits(6, 333, BF, cuda_dev, seed=2)
    flat = token_logprobs(z, ids, top=2)
    cube = token_logprobs(z.view(2, 3, 333), ids.view(2, 3).int(), top=2)
    assert cube.logp.shape == (2, 3) and cube.top_ids.shape == (2, 3, 2)
    for a, b in zip(flat, cube):
        assert torch.equal(a, b.reshape(a.shape))
    turned = token_logprobs(z.t().contiguous().t(), ids, top=2)
    assert torch.equal(turned.logp, flat.logp)
    leaf = z.view(2, 3, 333).detach().requires_grad_(True)
    token_logprobs(leaf, ids.view(2, 3)).logp.sum().backward()
    assert leaf.grad.shape == (2, 3, 333)
    none = token_logprobs(z[:0].requires_grad_(True), ids[:0], top=2)
    assert none.logp.shape == (0,) and none.top_ids.shape == (0, 2)
    one = z[:1].expand(4, 333)  # a row stride of 0
    assert torch.equal(token_logprobs(one, ids[:1].expand(4)).logp, flat.logp[:1].expand(4))


def test_forward_and_backward_in_a_captured_graph_and_on_another_stream(cuda_dev):
    from fitllm_b200.lm_head import token_logprobs
    z, ids = _logits(9, 5003, BF, cuda_dev, seed=4)
    up = torch.ones(9, device=cuda_dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    static = z.detach().clone().requires_grad_(True)
    with torch.cuda.stream(side):
        for _ in range(2):
            r = token_logprobs(static, ids, top=3)
            torch.autograd.grad(r.logp, static, up)
    del r
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr, stream=side):
        r = token_logprobs(static, ids, top=3)
        grad, = torch.autograd.grad(r.logp, static, up)
    for seed in (8, 9):
        fresh, _ = _logits(9, 5003, BF, cuda_dev, seed=seed)
        with torch.no_grad():
            static.copy_(fresh)
        gr.replay()
        torch.cuda.synchronize()
        leaf = fresh.detach().requires_grad_(True)
        e = token_logprobs(leaf, ids, top=3)
        want, = torch.autograd.grad(e.logp, leaf, up)
        assert torch.equal(r.logp, e.logp) and torch.equal(r.top_ids, e.top_ids) and torch.equal(grad, want)


def test_a_second_derivative_is_refused(cuda_dev):
    from fitllm_b200.lm_head import token_logprobs
    z = torch.randn(3, 50, device=cuda_dev, requires_grad=True)
    r = token_logprobs(z, torch.tensor([1, 2, 3], device=cuda_dev))
    (g,) = torch.autograd.grad(r.logp.sum(), z, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
