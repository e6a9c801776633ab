"""Accuracy of attention over the 4-bit cache, held per token and head to the rounding that the
kernels state, so that the bound shrinks with the output it is for.

Errors of a row o = sum_p w_p v_p / sum_p w_p (norms over the head's D elements), with r = 2^-11 half a
step of fp16 and each rounding's error spread evenly over its half steps (standard deviation 1/sqrt(3) of it):
* the result is rounded once to its type: at most u |o| (u: bf16 2^-8, fp16 2^-11), and for an fp16
  element below 2^-14, whose steps are 2^-24 however small it is, half of that: 2^-25 sqrt(D) over a row;
* up to 64 rows: a weight is rounded to fp16, and its product with the group's scale once more; more
  rows: the weight and the value are.  Either way two roundings of terms not larger than
  w_p a_p, a_p^2 = sum_d v_pd^2 + (8 s_pd)^2 (codes enter the products less eight);
* more rows: keys are rounded too, which moves a score by r q.k element by element, and so a
  weight by kappa_p, kappa_p^2 = sum_d q_d^2 (k_pd^2 + tiny^2) / D, and the row by w_p kappa_p |v_p - o|;
* below fp16's normal range a rounding is 2^-25 at most: of weights, and of weights times scales, whose
  largest lies at 2^7 / max(1, s) or above; of halved keys and values and of their halved lows
  (2^-23 of a value in all: `tiny` is that over r).
The errors of different positions are independent: they add up in squares.  Three standard deviations
cover a row (one rounding alone reaches sqrt(3) of its own).  fp32 sums and exponentials are far below.
"""
import math

import pytest
import torch

from tests import kv4_ref as ref
from tests.test_gpu_kv4 import ATTEND, BF, FP, U, _attend, _case

pytestmark = pytest.mark.gpu
R = 2.0 ** -11
TINY = 2.0 ** -23


def _params(pool, d):
    """(scale, low) pairs of a pool as a view [pages, KVH, blocks, 16, key / value, D / 64, 2] fp16."""
    return pool[..., 16 * d:].view(torch.float16).view(*pool.shape[:3], 16, 2, d // 64, 2)


def _scales(pool, table_row, length):
    """The values' scales float64 [KVH, length, D] behind one row of a page table."""
    d = pool.shape[3] // 18
    ps = pool.shape[2] * 16
    rows = table_row[:-(-length // ps)].long()
    s = _params(pool, d)[rows][..., 1, :, 0].double()  # [n, KVH, blocks, 16, G]
    s = s.permute(1, 0, 2, 3, 4).reshape(pool.shape[1], -1, d // 64)[:, :length]
    return s.repeat_interleave(64, -1)


def _rows(q, k, v, s, pre, i0, dtype):
    """(want, bound) of queries q [n, D] (tokens i0, i0 + 1, ... behind `pre`) over k, v [N, D]."""
    n, d = q.shape
    q = q.double()
    at = torch.arange(k.shape[0], device=q.device)[None]
    hidden = at > pre + i0 + torch.arange(n, device=q.device)[:, None]
    p = torch.softmax((q @ k.T / math.sqrt(d)).masked_fill(hidden, float("-inf")), -1)
    want = p @ v
    p2, seen = p.square(), (~hidden).double()
    a2 = (v.square() + (8 * s).square()).sum(-1)
    kappa2 = q.square() @ (k.square() + (TINY / R) ** 2).T / d
    away2 = (v.square().sum(-1)[None] - 2 * want @ v.T + want.square().sum(-1)[:, None]).clamp(min=0)
    wide = 2.0 ** max(0, math.ceil(math.log2(float(s.max().clamp(min=1.0)))))
    low = p.amax(-1) * 2.0 ** -32 * wide * (seen @ (a2 + 64.0 * d)).sqrt()
    spread = (p2 @ (2 * a2) + (p2 * kappa2 * away2).sum(-1)).sqrt() * R
    tiny = TINY * (d * p2.sum(-1)).sqrt()
    step = 2.0 ** -25 * math.sqrt(d) if dtype == FP else 0.0
    return want, U[dtype] * want.norm(dim=-1) + step + 3 / math.sqrt(3) * (spread + low + tiny)


def _check(c, o, rows=None):
    """Every row of o, or tokens `rows` of every sequence; returns the largest |o| and the worst ratio."""
    h, d = c["q"].shape[1:]
    kvh = c["pool"].shape[1]
    worst, norms = 0.0, []
    for b, (pre, a, n) in enumerate(zip(c["prefix"], c["starts"], c["counts"])):
        if n == 0:
            continue
        k, v = ref.read_sequence(c["pool"], c["table"][b], pre + n)
        s = _scales(c["pool"], c["table"][b], pre + n)
        for i in range(h):
            kv = i // (h // kvh)
            for t in ([slice(0, n)] if rows is None else [slice(r, r + 1) for r in rows]):
                want, bound = _rows(c["q"][a:a + n][t, i], k[kv], v[kv], s[kv], pre, t.start, c["q"].dtype)
                err = (o[a:a + n][t, i].double() - want).norm(dim=-1)
                worst = max(worst, float((err / bound).max()))
                norms.append((want.norm(dim=-1) / bound).min())
    assert worst <= 1, f"worst {worst:.2f} of the bound"
    assert float(min(norms)) > 2, "an output of zeros would pass"


@pytest.mark.parametrize("prefix,counts,h,kvh,d,ps,dtype", ATTEND)
def test_rows_are_as_near_as_their_roundings(cuda_dev, prefix, counts, h, kvh, d, ps, dtype):
    from fitllm_b200 import ops
    c = _case(prefix, counts, h, kvh, d, ps, dtype, cuda_dev, seed=2 * h + d + prefix[0], head=1, tail=2)
    o = _attend(c)
    assert ops.device_status() == 0
    _check(c, o)


LONG = [([131071], [1], 2, 2, 128, 128, BF), ([131071], [1], 5, 1, 64, 64, FP), ([65000, 40000], [5, 5], 8, 2, 128, 64, FP),
        ([60000], [70], 2, 1, 128, 128, BF), ([60000, 33333], [40, 40], 16, 8, 64, 64, FP)]


@pytest.mark.parametrize("prefix,counts,h,kvh,d,ps,dtype", LONG)
def test_long_contexts_lose_no_part(cuda_dev, prefix, counts, h, kvh, d, ps, dtype):
    c = _case(prefix, counts, h, kvh, d, ps, dtype, cuda_dev, seed=3)
    _check(c, _attend(c))


def test_rows_of_a_long_prompt_of_many_heads(cuda_dev):
    """More than 2^20 rows in one call."""
    from fitllm_b200 import ops
    n, h, d, ps = 131072, 8, 64, 128
    g = torch.Generator(device=cuda_dev).manual_seed(6)
    table, pages = ref.page_table([n], ps, g, cuda_dev)
    pool = ref.random_pool(pages, 1, ps, d, g, cuda_dev)
    q = torch.randn(n, h, d, generator=g, device=cuda_dev, dtype=BF)
    o = ops.kv4_attention(q, pool, table, torch.zeros(1, dtype=torch.int32, device=cuda_dev))
    assert ops.device_status() == 0
    c = dict(q=q, pool=pool, table=table, prefix=[0], starts=[0], counts=[n])
    _check(c, o, rows=(0, 1, 127, 128, 5000, 65535, 100001, n - 1))


FORMS = [([900, 3000, 64], [1, 1, 1], 40, 8), ([3000] * 9, [1] * 9, 40, 8), ([500, 2000], [5, 3], 10, 2),
         ([700, 40], [60, 90], 8, 4), ([200], [120], 160, 160)]


@pytest.mark.parametrize("prefix,counts,h,kvh", FORMS)
@pytest.mark.parametrize("d,dtype", [(128, BF), (128, FP), (64, BF), (64, FP)])
def test_peaked_rows_of_queries_with_outlier_channels(cuda_dev, prefix, counts, h, kvh, d, dtype):
    c = _case(prefix, counts, h, kvh, d, 64, dtype, cuda_dev, seed=d)
    c["q"] = c["q"] * 3
    c["q"][..., [3, d - 5]] *= 12
    c["q"][..., 9] *= 1e-3
    _check(c, _attend(c))


@pytest.mark.parametrize("prefix,counts,h,kvh", FORMS)
@pytest.mark.parametrize("d,dtype", [(128, BF), (128, FP), (64, BF), (64, FP)])
@pytest.mark.parametrize("factor", [4000.0, 30.0, 2.0 ** -9, 2.0 ** -14])
def test_values_of_every_size(cuda_dev, prefix, counts, h, kvh, d, dtype, factor):
    """Value scales from 0.3 x 4,000 (fp16's end) down to 2^-17 (a few steps of fp16's subnormals); every
    third position keeps a tenth of it, and one sequence meets its largest only late."""
    c = _case(prefix, counts, h, kvh, d, 64, dtype, cuda_dev, seed=d + 1)
    par = _params(c["pool"], d)
    v = par[..., 1, :, :].float() * factor
    v[:, :, :, ::3] *= 0.1
    par[..., 1, :, :] = v.half()
    if factor > 1:  # the pages of the first half of sequence 0 hold small ones
        early = c["table"][0, :(c["prefix"][0] // 64 + 1) // 2].long()
        par[early, ..., 1, :, :] = (v[early] / factor).half()
    _check(c, _attend(c))


@pytest.mark.parametrize("n", [32768, 131072])
@pytest.mark.parametrize("batch,count", [(1, 1), (40, 1), (2, 70), (80, 70)])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_what_stands_behind_a_strong_first_position(cuda_dev, n, batch, count, dtype):
    """The first position holds 99.9% of a row's mass and a value of zero; the result is what the rest
    adds up to.  Sequences share the pages.  One token of one sequence and of many, tiles whose
    positions are split over CTAs and tiles whose positions are not."""
    d, ps = 128, 128
    g = torch.Generator(device=cuda_dev).manual_seed(n)
    pool = ref.random_pool(n // ps, 1, ps, d, g, cuda_dev)
    par = _params(pool, d)
    par[..., 1, :, 1] += 1.0          # values around one
    par[0, 0, 0, 0, 1] = 0.0          # the first position's are zeros
    table = torch.arange(n // ps, dtype=torch.int32, device=cuda_dev).expand(batch, -1).contiguous()
    k, v = (x[0] for x in ref.read_sequence(pool, table[0], n))
    # q along the first key, so long that its score stands at log(999 * the others' sum)
    dirn = k[0] / k[0].norm()
    lo, hi = 0.0, 400.0
    for _ in range(60):
        mid = (lo + hi) / 2
        s = k @ dirn * mid / math.sqrt(d)
        lo, hi = (mid, hi) if float(s[0] - torch.logsumexp(s[1:], 0)) < math.log(999.0) else (lo, mid)
    q = (dirn * hi + 0.01 * torch.randn(batch * count, 1, d, generator=g, device=cuda_dev)).to(dtype)
    pre = n - count
    c = dict(q=q, pool=pool, table=table, prefix=[pre] * batch, starts=[i * count for i in range(batch)],
             counts=[count] * batch, pre=torch.full((batch,), pre, dtype=torch.int32, device=cuda_dev), q_start=None,
             max_new=count, max_len=n)
    o = _attend(c)
    few = dict(c, prefix=c["prefix"][:2], starts=c["starts"][:2], counts=c["counts"][:2])
    _check(few, o)
    # the sequences differ in their queries' small part only
    assert float((o.double().mean(-1) / o.double().mean() - 1).abs().max()) < 0.2


# ---- long sums, over all heads together: the outputs' own rounding and one of the weights.
# A rounding to nearest is off by u / m of a value with mantissa m in [1, 2) at most, evenly: its variance
# is u^2 / 3 E[1 / m^2] of the value's square, 3 / (8 ln 2) u^2 / 3 = 0.18 u^2 where mantissas spread as
# logarithms do.  The results' own is taken from the results.  Sums in the tensor cores round towards zero at
# the accumulator's size, at most 2^-23 of it each:
# * up to 64 rows: of 16 positions each and at most 32 blocks of codes less eight (fp16 results of more than
#   2^15 positions: 8) before they are joined in fp32, that is 2^-23 * 32 * 8 s w_p per position on average over
#   the blocks; the halves that cancel (codes against eights, scales against lows) bring 2 of that;
# * more rows: 2^14 / 16 (bf16: 2^16 / 16) of them before they join the row's sums in fp32, of the output itself.
# A quarter more for the statistics of a few hundred values.

def _long(dev, n, d, dtype, h, new, batch, mean):
    g = torch.Generator(device=dev).manual_seed(n + d + batch)
    pool = ref.random_pool(n // 128, 1, 128, d, g, dev)
    _params(pool, d)[..., 1, :, 1] += mean
    q = torch.randn(new, h, d, generator=g, device=dev).to(dtype)
    table = torch.randperm(n // 128, generator=g, device=dev).int().expand(batch, -1).contiguous()
    return dict(q=q.repeat(batch, 1, 1), pool=pool, table=table, q_start=None, max_new=new, max_len=n,
                pre=torch.full((batch,), n - new, dtype=torch.int32, device=dev))


def _long_bound(c, o, n, new, few):
    """(error, bound) of the last sequence's first eight tokens, norms over all of their heads."""
    h, d = c["q"].shape[1:]
    dtype = c["q"].dtype
    k, v = (x[0] for x in ref.read_sequence(c["pool"], c["table"][-1], n))
    s = _scales(c["pool"], c["table"][-1], n)[0]
    rows = c["table"][-1].long()
    low = _params(c["pool"], d)[rows][..., 1, :, 1].double().permute(1, 0, 2, 3, 4).reshape(n, -1).repeat_interleave(64, -1)
    mid = low + 8 * s
    terms = ((v - mid).square() + mid.square()).sum(-1) if few else (v.square() if dtype == FP else 3 * v.square()).sum(-1)
    err2 = want2 = out2 = weights2 = sums2 = 0.0
    for i in range(min(new, 8)):
        seen = n - new + i + 1
        p = torch.softmax(c["q"][i].double() @ k[:seen].T / math.sqrt(d), -1)
        want = p @ v[:seen]
        err2 += float((o[i - new].double() - want).square().sum())
        want2 += float(want.square().sum())
        out2 += float((want.to(dtype).double() - want).square().sum())
        weights2 += float((p.square() @ terms[:seen]).sum()) * 0.18 * R ** 2
        window = 8 if dtype == FP and n > 1 << 15 else 32
        sums = 2 * window * 8 * (p @ s[:seen]) if few else want * ((1 << 14 if dtype == FP else 1 << 16) / 16)
        sums2 += float(sums.square().sum()) * 2.0 ** -46
    return math.sqrt(err2), 1.25 * math.sqrt(out2 + weights2) + math.sqrt(sums2), math.sqrt(want2)


@pytest.mark.parametrize("n,batch,new", [(65536, 1, 1), (131072, 64, 3), (131072, 640, 1), (1 << 20, 1, 4), (1 << 20, 16, 3)])
@pytest.mark.parametrize("d,dtype", [(128, BF), (128, FP), (64, BF), (64, FP)])
def test_few_rows_keep_their_digits_over_long_contexts(cuda_dev, n, batch, new, d, dtype):
    c = _long(cuda_dev, n, d, dtype, 5, new, batch, 0.0)
    err, bound, norm = _long_bound(c, _attend(c), n, new, True)
    assert err <= bound, f"{err / norm:.2e} of the output, the bound {bound / norm:.2e}"
    assert bound < norm / 20


@pytest.mark.parametrize("prefix,counts,h,kvh", [([0, 700], [333, 200], 8, 4), ([3000], [130], 2, 1), ([300] * 80, [70] * 80, 1, 1)])
@pytest.mark.parametrize("d", [64, 128])
def test_fp16_rows_of_prompts_show_their_weights_rounding_only(cuda_dev, prefix, counts, h, kvh, d):
    """Keys and values lose nothing: the result's own rounding and one of the weights are all there is (with
    keys and values rounded to fp16 as well the error is 1.4 times that)."""
    c = _case(prefix, counts, h, kvh, d, 64, FP, cuda_dev, seed=d)
    o = _attend(c)
    err2 = expect2 = 0.0
    for b, (pre, a, n) in enumerate(zip(prefix, c["starts"], counts)):
        k, v = ref.read_sequence(c["pool"], c["table"][b], pre + n)
        hidden = torch.arange(pre + n, device=cuda_dev)[None] > torch.arange(pre, pre + n, device=cuda_dev)[:, None]
        for i in range(h):
            kv = i // (h // kvh)
            s = c["q"][a:a + n, i].double() @ k[kv].T / math.sqrt(d)
            p = torch.softmax(s.masked_fill(hidden, float("-inf")), -1)
            want = p @ v[kv]
            err2 += float((o[a:a + n, i].double() - want).square().sum())
            expect2 += float((want.half().double() - want).square().sum())
            expect2 += float((p.square() @ v[kv].square().sum(-1)).sum()) * 0.18 * R ** 2
    assert err2 <= 1.15 ** 2 * expect2, f"{math.sqrt(err2 / expect2):.2f} of what two roundings give"


@pytest.mark.parametrize("n,batch,new", [(65536, 80, 65), (131072, 80, 70), (1 << 20, 80, 66), (1 << 20, 1, 66)])
@pytest.mark.parametrize("d,dtype", [(128, BF), (128, FP), (64, BF), (64, FP)])
@pytest.mark.parametrize("mean", [0.0, 1.0])
def test_many_rows_keep_their_digits_over_long_contexts(cuda_dev, n, batch, new, d, dtype, mean):
    """Calls whose positions are split over CTAs, and calls whose are not."""
    c = _long(cuda_dev, n, d, dtype, 1, new, batch, mean)
    err, bound, norm = _long_bound(c, _attend(c), n, new, False)
    assert err <= bound, f"{err / norm:.2e} of the output, the bound {bound / norm:.2e}"
    assert bound < norm / 20


def test_a_long_call_of_many_rows_comes_in_several_launches(cuda_dev):
    """Rows whose sums exceed the scratch of a launch, of sequences of every length under one hint."""
    from fitllm_b200 import _lib, ops
    n, d, ps, batch = 1 << 17, 128, 128, 6
    g = torch.Generator(device=cuda_dev).manual_seed(9)
    pool = ref.random_pool(n // ps, 1, ps, d, g, cuda_dev)
    table = torch.arange(n // ps, dtype=torch.int32, device=cuda_dev).expand(batch, -1).contiguous()
    prefix, counts = [n - 7300, 0, 70000, 16383, 16000, 5], [7300, 1, 0, 600, 1200, 130]
    starts = [sum(counts[:i]) for i in range(batch)]
    for dtype in (FP, BF):
        q = torch.randn(sum(counts) + 3, 12, d, generator=g, device=cuda_dev).to(dtype)
        c = dict(q=q, pool=pool, table=table, prefix=prefix, starts=starts, counts=counts, max_new=7300, max_len=n,
                 pre=torch.tensor(prefix, dtype=torch.int32, device=cuda_dev),
                 q_start=torch.tensor(starts + [sum(counts)], dtype=torch.int32, device=cuda_dev))
        out = torch.full_like(q, 7.0)
        before = _lib.load().fitq_launch_count()
        o = _attend(c, out=out)
        assert _lib.load().fitq_launch_count() - before == 2
        assert ops.device_status() == 0 and bool((o[sum(counts):] == 7).all())
        few = dict(c, counts=[130, 1, 0, 90, 130, 130])
        few["starts"] = [s + n - m for s, n, m in zip(starts, counts, few["counts"])]
        few["prefix"] = [p + n - m for p, n, m in zip(prefix, counts, few["counts"])]
        _check(few, o)
        assert torch.equal(o, _attend(c, out=torch.full_like(q, 7.0)))
        c["max_len"] = 4096  # a hint that is too small: no sums apart, the same result within its roundings
        _check(few, _attend(c))


@pytest.mark.parametrize("d,dtype", [(128, BF), (128, FP), (64, BF), (64, FP)])
def test_few_rows_keep_their_digits_where_max_len_is_too_small(cuda_dev, d, dtype):
    """A captured call goes on as clusters of few tiles when its sequences have grown long."""
    n = 1 << 19
    c = _long(cuda_dev, n, d, dtype, 5, 1, 2, 0.0)
    c["max_len"] = 1000
    err, bound, norm = _long_bound(c, _attend(c), n, 1, True)
    assert err <= bound, f"{err / norm:.2e} of the output, the bound {bound / norm:.2e}"
