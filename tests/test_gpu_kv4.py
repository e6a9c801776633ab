"""The 4-bit paged key/value cache: append with rotation, read back, attention.

Append and read-back are held to the stated arithmetic bit for bit (every step
of the coding is a single fp32 rounding).  Attention is compared with 64-bit
attention over the values the cache stands for.  Its bound per element: with u
half a step of the type (bf16 2^-8, fp16 2^-11) the scaled weights w s enter the
tensor cores rounded, off by at most u of a term s |code - 8| <= 8 s, and the
output is rounded once (u |o|); weights rounded to fp16 before (2^-11) and the fp32
rounding of the scores' sums (below 2^-11 in the exponent at these sizes) move a
weighted mean of values within [-vmax, vmax] by at most 2^-10 * 2 vmax.
"""
import pytest
import torch

from tests import kv4_ref as ref

pytestmark = pytest.mark.gpu
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
BF, FP = torch.bfloat16, torch.float16


def _case(prefix, counts, h, kvh, d, ps, dtype, dev, seed=0, ragged=True, head=0, tail=0):
    """Inputs of a call; head / tail packed rows belong to no sequence."""
    g = torch.Generator(device=dev).manual_seed(seed)
    starts = [head]
    for n in counts:
        starts.append(starts[-1] + n)
    tokens = starts[-1] + tail
    lengths = [p + n for p, n in zip(prefix, counts)]
    table, pages = ref.page_table(lengths, ps, g, dev)
    c = dict(prefix=prefix, counts=counts, starts=starts[:-1], table=table,
             pool=ref.random_pool(pages, kvh, ps, d, g, dev),
             pre=torch.tensor(prefix, dtype=torch.int32, device=dev),
             q_start=torch.tensor(starts, dtype=torch.int32, device=dev) if ragged else None,
             q=torch.randn(tokens, h, d, generator=g, device=dev).to(dtype),
             k=(torch.randn(tokens, kvh, d, generator=g, device=dev) * 2 + 1).to(dtype),
             v=torch.randn(tokens, kvh, d, generator=g, device=dev).to(dtype),
             max_new=max(counts), max_len=max(lengths))
    return c


def _attend(c, **kw):
    from fitllm_b200 import ops
    return ops.kv4_attention(c["q"], c["pool"], c["table"], c["pre"], c["max_len"], q_start=c["q_start"],
                             max_new=c["max_new"], **kw)


def _check_attention(c, o):
    want = ref.attention(c["q"], c["pool"], c["table"], c["prefix"], c["starts"], c["counts"])
    par = c["pool"][..., 16 * c["q"].shape[2]:].contiguous().view(torch.float16).float()
    smax = float(par[..., 0::2].nan_to_num(0).clamp(max=1.0).max())
    u = U[c["q"].dtype]
    rows = ~want.isnan().any(-1).any(-1)
    bound = u * (8 * smax + want[rows].abs()) + 2.0 ** -10 * 2 * (8 * smax + 1)
    err = (o.double()[rows] - want[rows]).abs()
    assert bool((err <= bound).all()), f"worst {float((err / bound).max()):.2f} of the bound"
    return rows


APPEND = [
    ([0], [1], 8, 1, 128, 16, BF), ([15, 16, 17], [1, 1, 1], 40, 8, 128, 16, BF),
    ([0, 63, 5], [70, 1, 33], 4, 4, 64, 32, FP), ([5, 0, 2000], [900, 511, 2], 3, 1, 128, 16, BF),
    ([0, 31], [1201, 40], 20, 4, 64, 64, FP), ([1000, 0], [5, 300], 14, 2, 128, 64, FP),
    ([7, 3, 0, 100], [3, 0, 129, 1], 28, 4, 64, 128, BF),
]


@pytest.mark.parametrize("prefix,counts,h,kvh,d,ps,dtype", APPEND)
def test_append_and_gather_are_the_stated_arithmetic(cuda_dev, prefix, counts, h, kvh, d, ps, dtype):
    from fitllm_b200 import ops
    c = _case(prefix, counts, h, kvh, d, ps, dtype, cuda_dev, seed=sum(counts) + d, head=2, tail=3)
    before = c["pool"].clone()
    cos, sin = ref.tables(max(p + n for p, n in zip(prefix, counts)), d, cuda_dev)
    q_out = torch.full_like(c["q"], 7.0)
    got = ops.kv4_append(c["q"], c["k"], c["v"], c["pool"], c["table"], c["pre"], cos, sin, q_start=c["q_start"],
                         q_out=q_out)
    assert got is q_out
    k, v = ops.kv4_gather(c["pool"], c["table"], c["pre"], c["q"].shape[0], q_start=c["q_start"], dtype=dtype)
    assert ops.device_status() == 0
    pos = torch.cat([torch.arange(p, p + n) for p, n in zip(prefix, counts)]).to(cuda_dev)
    live = slice(2, 2 + sum(counts))
    assert torch.equal(got[live], ref.rotate(c["q"][live], cos[pos], sin[pos]).to(dtype))
    assert torch.equal(k[live], ref.coded_values(ref.rotate(c["k"][live], cos[pos], sin[pos])).to(dtype))
    assert torch.equal(v[live], ref.coded_values(c["v"][live].float()).to(dtype))
    # rows of no sequence, and every block position that was not appended, are as they were
    assert bool((got[:2] == 7).all()) and bool((got[2 + sum(counts):] == 7).all())
    for b, (p, n) in enumerate(zip(prefix, counts)):
        if p:
            for x, y in zip(ref.read_sequence(c["pool"], c["table"][b], p), ref.read_sequence(before, c["table"][b], p)):
                assert torch.equal(x, y)
        if n:
            kk, vv = ref.read_sequence(c["pool"], c["table"][b], p + n)
            rows = slice(c["starts"][b], c["starts"][b] + n)
            assert torch.equal(kk[:, p:].transpose(0, 1).to(dtype), k[rows])
            assert torch.equal(vv[:, p:].transpose(0, 1).to(dtype), v[rows])
    used = torch.zeros(c["pool"].shape[0], dtype=torch.bool, device=cuda_dev)
    used[c["table"][c["table"] >= 0].long()] = True
    assert torch.equal(c["pool"][~used], before[~used])


@pytest.mark.parametrize("dtype,d", [(BF, 128), (FP, 64)])
def test_append_reads_slices_of_a_fused_projection_and_rotates_in_place(cuda_dev, dtype, d):
    from fitllm_b200 import ops
    c = _case([9, 40], [6, 6], 6, 2, d, 16, dtype, cuda_dev, ragged=False)
    cos, sin = ref.tables(64, d, cuda_dev)
    fused = torch.cat([c["q"].flatten(1), c["k"].flatten(1), c["v"].flatten(1)], dim=1)
    q, k, v = (t.unflatten(1, (-1, d)) for t in fused.split([6 * d, 2 * d, 2 * d], dim=1))
    assert not q.is_contiguous()
    plain, strided = c["pool"].clone(), c["pool"].clone()
    a = ops.kv4_append(c["q"], c["k"], c["v"], plain, c["table"], c["pre"], cos, sin)
    b = ops.kv4_append(q, k, v, strided, c["table"], c["pre"], cos, sin)
    assert torch.equal(a, b) and torch.equal(plain, strided)
    own = c["q"].clone()
    assert torch.equal(ops.kv4_append(own, c["k"], c["v"], plain, c["table"], c["pre"], cos, sin, q_out=own), a)
    assert torch.equal(plain, strided)
    oddly = torch.empty(c["q"].numel() + 1, dtype=dtype, device=cuda_dev)[1:].view_as(c["q"]).copy_(c["q"])
    assert torch.equal(ops.kv4_append(oddly, c["k"], c["v"], plain, c["table"], c["pre"], cos, sin), a)


def test_append_codes_constant_huge_and_non_finite_groups(cuda_dev):
    from fitllm_b200 import ops
    d = 128
    v = torch.zeros(5, 1, d, dtype=BF, device=cuda_dev)
    v[0, 0, :64], v[0, 0, 64:] = 3.25, -0.0
    v[1, 0, 7], v[1, 0, 100] = float("nan"), 1.0
    v[2, 0, 70] = float("inf")
    v[3, 0, 1] = -1.0e30
    v[4, 0, 5] = 60000.0
    c = _case([0], [5], 1, 1, d, 16, BF, cuda_dev, ragged=False)
    cos, sin = ref.tables(8, d, cuda_dev)
    ops.kv4_append(c["q"], c["k"], v, c["pool"], c["table"], c["pre"], cos, sin)
    _, got = ops.kv4_gather(c["pool"], c["table"], c["pre"], 5)
    got = got[:, 0].float()
    assert bool((got[0, :64] == 3.25).all()) and bool((got[0, 64:] == 0).all())
    assert bool(got[1, :64].isnan().all()) and bool(got[1, 64:].isfinite().all())
    assert bool(got[2, 64:].isnan().all()) and bool(got[2, :64].isfinite().all())
    assert bool(got[3, :64].isnan().all())
    assert bool(got[4].isfinite().all())


ATTEND = [
    # one token at every position of a block and around tile and page ends
    *[([p], [1], 8, 1, 128, 16, BF) for p in (0, 1, 14, 15, 16, 17, 62, 63, 64, 65, 255, 256)],
    ([1, 700, 64, 0], [1, 1, 1, 1], 40, 8, 128, 64, BF), ([33, 2000], [1, 1], 5, 1, 64, 32, FP),
    # drafts: one, two and four column tiles, an odd group
    ([100, 5], [2, 2], 16, 4, 128, 32, FP), ([511, 64, 3], [3, 3, 3], 40, 8, 128, 128, BF),
    ([300], [5], 40, 8, 128, 16, FP), ([77, 1024], [6, 2], 10, 2, 64, 64, BF), ([4095], [32], 4, 4, 128, 64, BF),
    # more pairs than clusters take: runs of the list, cut pairs joined behind them
    ([3, 200, 1400, 64, 0, 777], [1] * 6, 40, 8, 128, 64, BF), ([90, 2500, 1, 511, 300], [2, 3, 1, 0, 2], 40, 8, 128, 16, FP),
    ([1000 + 37 * i for i in range(9)], [1] * 9, 8, 8, 64, 32, BF), ([9000], [1], 2, 2, 128, 128, BF),
    ([20000], [5], 5, 1, 128, 64, FP),
    # several row tiles, prompts with and without a prefix, empty sequences
    ([0], [200], 8, 2, 128, 64, BF), ([130, 0, 9], [40, 0, 97], 12, 4, 64, 16, FP), ([31], [65], 7, 1, 128, 16, FP),
    # few row tiles over many positions: their parts joined behind the kernel
    ([3000], [40], 8, 1, 128, 64, BF), ([5000, 900, 0], [30, 17, 20], 16, 4, 64, 32, FP), ([2300], [130], 4, 2, 128, 128, FP),
    ([0, 1, 700], [333, 17, 64], 40, 8, 128, 128, BF), ([0, 3], [129, 128], 16, 16, 64, 32, BF),
]


@pytest.mark.parametrize("prefix,counts,h,kvh,d,ps,dtype", ATTEND)
def test_attention_matches_64_bits(cuda_dev, prefix, counts, h, kvh, d, ps, dtype):
    from fitllm_b200 import ops
    c = _case(prefix, counts, h, kvh, d, ps, dtype, cuda_dev, seed=h + d + prefix[0], head=1, tail=2)
    out = torch.full_like(c["q"], 7.0)
    o = _attend(c, out=out)
    assert o is out and ops.device_status() == 0
    rows = _check_attention(c, o)
    assert bool((o[~rows] == 7).all())  # rows of no sequence are left as they are


@pytest.mark.parametrize("dtype", [BF, FP])
def test_attention_is_deterministic_and_ignores_the_hint(cuda_dev, dtype):
    c = _case([900, 3, 5000], [1, 1, 1], 40, 8, 128, 64, dtype, cuda_dev, ragged=False)
    a = _attend(c)
    assert torch.equal(a, _attend(c))
    c["max_len"] = 1  # a wrong hint makes the grid small, not the result wrong
    _check_attention(c, _attend(c))
    c["max_len"] = None
    _check_attention(c, _attend(c))


@pytest.mark.parametrize("prefix,counts,h,kvh", [([900], [1], 40, 8), ([900, 3, 5000] * 3, [1] * 9, 40, 8),
                                                 ([400, 30, 900, 0] * 2, [5, 2, 1, 3] * 2, 40, 8), ([3, 500], [60, 41], 8, 2),
                                                 ([4000], [70], 8, 2)])
def test_attention_may_write_over_its_queries(cuda_dev, prefix, counts, h, kvh):
    c = _case(prefix, counts, h, kvh, 128, 64, BF, cuda_dev, seed=8)
    want = _attend(c)
    assert torch.equal(_attend(c, out=c["q"]), want)


@pytest.mark.parametrize("d,steps", [(64, 0), (64, 1), (128, 0), (128, 1)])
def test_many_rows_end_under_every_schedule(cuda_dev, d, steps):
    """The tensor-memory kernel's roles hand over by parity: many calls whose last tile has one
    step of positions or two, beside another stream's work, end without a wait run out."""
    from fitllm_b200 import ops
    c = _case([128 * (3 + 7 * i) + 64 * steps for i in range(10)], [61] * 10, 32, 8, d, 128, BF, cuda_dev, ragged=False)
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


@pytest.mark.parametrize("counts", [[1, 1], [40, 3]])
def test_attention_never_reads_what_is_hidden(cuda_dev, counts):
    """Positions behind a sequence hold NaN codes' parameters and huge scales."""
    c = _case([70, 33], counts, 8, 2, 128, 32, BF, cuda_dev, ragged=True)
    a = _attend(c)
    for b in range(2):
        for p in range(c["prefix"][b] + counts[b], c["table"].shape[1] * 32):
            page = int(c["table"][b, p // 32])
            if page < 0:
                break
            c["pool"][page, :, (p % 32) // 16, 16 * 128 + (p % 16) * 16:16 * 128 + (p % 16) * 16 + 16] = 255
    assert torch.equal(a, _attend(c))


def test_attention_gives_nan_only_where_a_nan_is_seen(cuda_dev):
    c = _case([0], [40], 4, 2, 128, 16, BF, cuda_dev, ragged=False)
    page, blk = int(c["table"][0, 1]), 0
    c["pool"][page, 1, blk, 16 * 128 + 4 * 16 + 8:16 * 128 + 5 * 16] = 255  # values of position 20, KV head 1
    o = _attend(c)
    assert bool(o[:, :2].isfinite().all()) and bool(o[:20].isfinite().all())
    assert bool(o[20:, 2:].isnan().all())


@pytest.mark.parametrize("prefix,counts,h,kvh,d,ps,dtype", [
    ([40, 20], [1, 1], 8, 2, 128, 16, BF), ([30, 200, 1400, 64, 0, 777], [1] * 6, 40, 8, 128, 64, BF),
    ([90, 2500, 60, 511, 300], [2, 3, 1, 4, 2], 40, 8, 128, 16, FP), ([300, 40], [5, 5], 10, 2, 64, 64, BF),
    ([70, 33], [40, 3], 8, 2, 128, 32, BF)])
@pytest.mark.parametrize("bits", [0x7c00, 0xfe00])
def test_a_value_group_without_numbers_spoils_its_own_elements_only(cuda_dev, prefix, counts, h, kvh, d, ps, dtype,
                                                                    bits):
    """An infinite or NaN scale of one group: inside the cache, and at the last new token."""
    c = _case(prefix, counts, h, kvh, d, ps, dtype, cuda_dev, seed=5)
    want = ref.attention(c["q"], c["pool"], c["table"], c["prefix"], c["starts"], c["counts"])
    spoilt = torch.zeros(want.shape, dtype=torch.bool, device=cuda_dev)
    for b, pos, kv, gr in ((0, 17, 0, 0), (1, prefix[1] + counts[1] - 1, kvh - 1, d // 64 - 1)):
        at = 16 * d + ((pos % 16) * 2 * (d // 64) + d // 64 + gr) * 4
        block = c["pool"][int(c["table"][b, pos // ps]), kv, pos % ps // 16]
        block[at], block[at + 1] = bits & 255, bits >> 8
        for i in range(counts[b]):
            if pos <= prefix[b] + i:
                spoilt[c["starts"][b] + i, kv * (h // kvh):(kv + 1) * (h // kvh), 64 * gr:64 * gr + 64] = True
    o = _attend(c).double()
    assert not bool(o[spoilt].isfinite().any())
    bound = U[dtype] * (8 * 0.3 + want.abs()) + 2.0 ** -10 * 2 * (8 * 0.3 + 1)
    assert bool(((o - want).abs() <= bound)[~spoilt].all())


def test_bad_pages_positions_and_prefixes_are_recorded_and_left_out(cuda_dev):
    from fitllm_b200 import ops
    cos, sin = ref.tables(64, 128, cuda_dev)
    FITQ_ERR_ARG = 1
    for what in ("page", "negative page", "table end", "prefix", "rotary"):
        c = _case([40, 20], [1, 1], 8, 2, 128, 16, BF, cuda_dev, ragged=False)
        before = c["pool"].clone()
        if what == "page":
            c["table"][1, 1] = c["pool"].shape[0]
        if what == "negative page":
            c["table"][1, 1] = -7
        if what == "table end":
            c["pre"][1] = 16 * c["table"].shape[1]
        if what == "prefix":
            c["pre"][1] = -1
        if what == "rotary":
            cos, sin = ref.tables(20, 128, cuda_dev)
            c["pre"][0] = 19
        q = ops.kv4_append(c["q"], c["k"], c["v"], c["pool"], c["table"], c["pre"], cos, sin)
        assert ops.device_status() == FITQ_ERR_ARG and ops.device_status() == 0
        assert bool((q[1] == 0).all()) and bool((q[0] != 0).any())
        keep = c["table"][1][c["table"][1] >= 0].long()
        keep = keep[keep < before.shape[0]]
        assert torch.equal(c["pool"][keep], before[keep])
        if what == "rotary":
            continue
        k, _ = ops.kv4_gather(c["pool"], c["table"], c["pre"], 2)
        assert ops.device_status() == FITQ_ERR_ARG and bool((k[1] == 0).all())
        o = _attend(c)
        assert ops.device_status() == FITQ_ERR_ARG
        assert bool(o.isfinite().all())
        if what in ("page", "negative page"):  # what is left: the first page's 16 positions
            kk, vv = ref.read_sequence(c["pool"], c["table"][1], 16)
            s = torch.softmax(c["q"][1, 0].double() @ kk[0].T / 128 ** 0.5, -1) @ vv[0]
            assert float((o[1, 0].double() - s).abs().max()) < 2.0 ** -8 * (8 * 0.3 + float(s.abs().max())) + 0.01
        if what == "prefix":
            assert bool((o[1] == 0).all())


def test_more_new_tokens_than_max_new_are_recorded(cuda_dev):
    from fitllm_b200 import ops
    c = _case([5, 5], [1, 30], 8, 1, 128, 16, BF, cuda_dev)
    c["max_new"] = 1
    out = torch.zeros_like(c["q"])
    _attend(c, out=out)
    assert ops.device_status() == 1
    assert bool((out[2:] == 0).all())


def test_long_pools_and_many_sequences(cuda_dev):
    """Block offsets beyond 2^32 bytes; more sequences than a CTA has threads."""
    from fitllm_b200 import ops
    ps, kvh, d = 128, 8, 128
    pages = (1 << 32) // (kvh * ps * 144) + 600
    big = torch.empty(pages, kvh, ps // 16, 18 * d, dtype=torch.uint8, device=cuda_dev)
    g = torch.Generator(device=cuda_dev).manual_seed(3)
    n = 300
    big[-n:] = ref.random_pool(n, kvh, ps, d, g, cuda_dev)
    counts, prefix = [1] * n, [(7 * i) % 127 for i in range(n)]
    c = _case(prefix, counts, 16, kvh, d, ps, BF, cuda_dev, ragged=False)
    c["pool"] = big
    c["table"] = (pages - 1 - torch.arange(n, dtype=torch.int32, device=cuda_dev)).view(n, 1).contiguous()
    cos, sin = ref.tables(128, d, cuda_dev)
    ops.kv4_append(c["q"], c["k"], c["v"], big, c["table"], c["pre"], cos, sin)
    k, _ = ops.kv4_gather(big, c["table"], c["pre"], n)
    assert torch.equal(k, ref.coded_values(ref.rotate(c["k"], cos[c["pre"].long()], sin[c["pre"].long()])).bfloat16())
    o = _attend(c)
    assert ops.device_status() == 0
    small = dict(c, pool=big[-n:], table=(c["table"] - (pages - n)).contiguous())
    assert torch.equal(o, _attend(small))
    _check_attention(small, o)


def test_a_long_prompt_of_many_heads(cuda_dev):
    """More than 2^20 rows in one call."""
    n, h, d, ps = 131072, 8, 64, 128
    g = torch.Generator(device=cuda_dev).manual_seed(6)
    table, pages = ref.page_table([n], ps, g, cuda_dev)
    pool = ref.random_pool(pages, 1, ps, d, g, cuda_dev)
    q = torch.randn(n, h, d, generator=g, device=cuda_dev, dtype=BF)
    from fitllm_b200 import ops
    o = ops.kv4_attention(q, pool, table, torch.zeros(1, dtype=torch.int32, device=cuda_dev))
    k, v = (x[0] for x in ref.read_sequence(pool, table[0], n))
    for i in (0, 1, 127, 128, 5000, 65535, 100001, n - 1):
        want = torch.softmax(q[i].double() @ k[:i + 1].T / d ** 0.5, -1) @ v[:i + 1]
        bound = U[BF] * (8 * 0.3 + want.abs()) + 2.0 ** -10 * 2 * (8 * 0.3 + 1)
        assert bool(((o[i].double() - want).abs() <= bound).all())
    assert ops.device_status() == 0


def test_captured_calls_follow_lengths_on_another_stream(cuda_dev):
    from fitllm_b200 import ops
    c = _case([500, 100], [1, 1], 40, 8, 128, 64, BF, cuda_dev, ragged=False)
    cos, sin = ref.tables(1024, 128, cuda_dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())

    def step():
        q = ops.kv4_append(c["q"], c["k"], c["v"], c["pool"], c["table"], c["pre"], cos, sin)
        return q, ops.kv4_attention(q, c["pool"], c["table"], c["pre"], 512)

    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):  # two graphs, each with scratch of its own
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=side):
            outs = step()
        graphs.append((gr, outs))
    for pre in ([500, 100], [3, 511], [0, 0]):
        c["pre"].copy_(torch.tensor(pre, dtype=torch.int32))
        c["q"].normal_()
        torch.cuda.synchronize()
        for gr, _ in graphs:
            gr.replay()
        torch.cuda.synchronize()
        q, o = step()
        for _, (gq, go) in graphs:
            assert torch.equal(q, gq) and torch.equal(o, go)
        # sequence 1 has pages for 128 positions: the second round leads behind them
        assert ops.device_status() == (1 if pre[1] > 127 else 0)


def test_two_threads_on_two_streams(cuda_dev):
    """Calls at once share nothing but the pool they read."""
    import threading
    from fitllm_b200.lm_head import token_logprobs
    a = _case([900, 3, 5000], [1, 1, 1], 40, 8, 128, 64, BF, cuda_dev, ragged=False)
    b = _case([700, 90], [60, 41], 8, 2, 128, 64, FP, cuda_dev)
    z = torch.randn(40, 32001, device=cuda_dev)
    ids = torch.arange(40, device=cuda_dev)
    jobs = [lambda: _attend(a), lambda: _attend(b), lambda: token_logprobs(z, ids, top=8).top_logp]
    want = [f() for f in jobs]
    torch.cuda.synchronize()
    bad = []

    def work(order):
        with torch.cuda.stream(torch.cuda.Stream(cuda_dev)):
            for _ in range(30):
                got = [(i, jobs[i]()) for i in order]
                torch.cuda.current_stream().synchronize()
                bad.extend(i for i, g in got if not torch.equal(g, want[i]))

    threads = [threading.Thread(target=work, args=(o,)) for o in ([0, 1, 2], [2, 0, 1])]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad
