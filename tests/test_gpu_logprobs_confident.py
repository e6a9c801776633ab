"""Rows of a confident model: one likely token, whose log probability and entropy are what the others,
far below it, add up to.

The sums are of all elements but one that is the maximum, S' and E' = sum exp(d) d with d = z - M, and
  H = log1p(S') + |E'| / (1 + S'),  log p(M) = -log1p(S'),
so nothing cancels.  Each term is off by its exponent's rounding, 2^-24 |d| log2 e, and the exponential's own,
below 2^-19 for the terms that count; E' adds d's rounding: 2^-17 of H covers both.  S' besides loses the last
bits of what is added next to the maximum's 1 in one batch of a thread's loads, at most 32 additions of
2^-25 on average, spread evenly: 2^-20 covers four deviations.
The gradient -p (h (log p + H) + a) + marks: H as above; log p = (z - M) - log1p(S') is off by two roundings and
its product with log2 e by one, so that p is off by 3 * 2^-24 |log p| <= 2^-22 |log p| of itself, and by the
exponential's 2^-22; the few roundings of the rest are another 2^-22, of the marks 2^-22 too."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32

CASES = [
    # rows, vocabulary, dtype, alternatives, spread, likely token above: small CTAs, large ones, clusters
    (600, 152064, F32, 0, 1.0, 17.0), (600, 152064, F32, 0, 1.0, 19.0), (600, 152064, BF, 0, 2.5, 26.0),
    (600, 50257, FP, 0, 1.0, 20.0), (400, 152064, F32, 0, 1.0, 18.0), (400, 152064, BF, 5, 1.0, 18.0),
    (300, 152063, F32, 20, 2.5, 25.0), (2, 152064, F32, 0, 1.0, 17.0), (1, 152064, BF, 20, 1.0, 18.0),
    (40, 152064, F32, 5, 1.0, 18.0), (70, 32001, FP, 0, 1.0, 16.0), (5, 40, F32, 3, 1.0, 12.0),
]


def _logits(rows, vocab, dtype, spread, above, dev):
    g = torch.Generator(device=dev).manual_seed(rows + vocab)
    z = torch.randn(rows, vocab, generator=g, device=dev) * spread
    likely = torch.randint(0, vocab, (rows,), generator=g, device=dev)
    likely[0], likely[-1] = 0, vocab - 1
    z[torch.arange(rows, device=dev), likely] += above
    return z.to(dtype), likely, g


@pytest.mark.parametrize("rows,vocab,dtype,top,spread,above", CASES)
def test_likely_tokens_and_their_entropies_keep_their_digits(cuda_dev, rows, vocab, dtype, top, spread, above):
    from fitllm_b200.lm_head import token_logprobs
    z, likely, _ = _logits(rows, vocab, dtype, spread, above, cuda_dev)
    r = token_logprobs(z, likely, top=top)
    for a in range(0, rows, 100):
        w = torch.log_softmax(z[a:a + 100].double(), -1)
        h = -(w.exp() * w).sum(-1)
        logp = w.gather(1, likely[a:a + 100, None])[:, 0]
        assert bool(((r.entropy[a:a + 100].double() - h).abs() <= 2.0 ** -17 * h + 2.0 ** -20).all())
        assert bool(((r.logp[a:a + 100].double() - logp).abs() <= 2.0 ** -17 * logp.abs() + 2.0 ** -20).all())
        if top:
            assert torch.equal(r.top_ids[a:a + 100, 0], w.argmax(-1))


@pytest.mark.parametrize("rows,vocab,top", [(600, 50257, 0), (300, 152064, 3), (2, 152064, 0), (40, 32001, 5)])
def test_gradients_of_confident_rows(cuda_dev, rows, vocab, top):
    from fitllm_b200.lm_head import token_logprobs
    z, likely, g = _logits(rows, vocab, F32, 1.0, 17.0, cuda_dev)
    z.requires_grad_(True)
    r = token_logprobs(z, likely, top=top)
    ups = [torch.randn(rows, generator=g, device=cuda_dev), torch.randn(rows, generator=g, device=cuda_dev)]
    ups += [torch.randn(rows, top, generator=g, device=cuda_dev)] if top else []
    got = torch.autograd.grad([r.logp, r.entropy] + ([r.top_logp] if top else []), z, ups)[0]
    for a in range(0, rows, 100):
        rr = slice(a, a + 100)
        w = torch.log_softmax(z.detach()[rr].double(), -1)
        p = w.exp()
        h = -(p * w).sum(-1, keepdim=True)
        mark = torch.zeros_like(w)
        mark.scatter_add_(1, likely[rr, None], ups[0][rr, None].double())
        size = mark.abs()
        if top:
            mark.scatter_add_(1, r.top_ids[rr], ups[2][rr].double())
            size.scatter_add_(1, r.top_ids[rr], ups[2][rr].double().abs())
        all_marks, u = mark.sum(-1, keepdim=True), ups[1][rr, None].double()
        want = mark - p * all_marks - u * p * (w + h)
        terms = p * (size.sum(-1, keepdim=True) + u.abs() * (w.abs() + h))
        bound = 2.0 ** -22 * size + (2.0 ** -21 + 2.0 ** -22 * w.abs()) * terms
        bound += u.abs() * p * (2.0 ** -17 * h + 2.0 ** -20)
        assert bool(((got[rr].double() - want).abs() <= bound).all())


@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("rows,vocab", [(700, 30000), (200, 152064), (3, 152064), (4, 9)])
def test_rows_that_rise_and_rows_of_few_values(cuda_dev, dtype, rows, vocab):
    """Every granule of a row above the one before it; ties of the maximum; one finite logit; the type's
    lowest value throughout."""
    from fitllm_b200.lm_head import token_logprobs
    z = torch.zeros(rows, vocab, device=cuda_dev)
    z[0] = torch.linspace(-300, 300, vocab, device=cuda_dev)
    z[1] = float("-inf")
    z[1, vocab // 2] = 3.0
    z[2, ::max(1, vocab // 7)] = 11.0
    if rows > 3:
        z[3] = torch.finfo(dtype).min
        z[4:] = torch.linspace(0, 40, vocab, device=cuda_dev).flip(0) if rows > 4 else 0
    z = z.to(dtype)
    ids = torch.full((rows,), vocab // 2, device=cuda_dev)
    r = token_logprobs(z, ids)
    for a in range(0, rows, 100):
        w = torch.log_softmax(z[a:a + 100].double(), -1)
        h = -torch.nansum(w.exp() * w, -1)
        logp = w[:, vocab // 2]
        assert bool(((r.entropy[a:a + 100].double() - h).abs() <= 2.0 ** -17 * h + 2.0 ** -20).all())
        assert bool(((r.logp[a:a + 100].double() - logp).abs() <= 2.0 ** -17 * logp.abs() + 2.0 ** -20).all())
