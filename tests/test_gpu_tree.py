"""Trees of drafted tokens on the GPU: append, attention, verification and keep against
plain restatements in 64 bits.

Tolerance of the attention.  With weights w (sum 1) and values v, a result's element has
one rounding, eps |o|; the weights enter the second product in the values' type, each off
by eps w at most, and the sum of weights is fp32: eps sum w |v|.  Scores are fp32 sums of D
products of q and k, whose error of at most (D + 2) 2^-24 |q| |k| / sqrt D changes a weight by
as much of itself, twice (its own and the sum's): a factor of 2 (D + 2) 2^-24 S on sum w |v|,
S the largest |q| |k| / sqrt D; ex2 and the accumulation add 2^-20.  bf16 may keep weights in
two parts, which only lowers the error."""
import math

import pytest
import torch

from tests import tree_ref as ref

pytestmark = pytest.mark.gpu


def _bound(q, k_cache, v_cache, prefix, parents, exact):
    """sum w |v| per element by the restatement itself, on |v|."""
    eps = ref.EPS[q.dtype]
    d = q.shape[-1]
    mag = ref.attention(q, k_cache, v_cache.abs(), prefix, parents)
    n = int(max(int(p) for p in prefix)) + q.shape[1]
    top = float(q.double().norm(dim=-1).max() * k_cache[:, :, :n].double().norm(dim=-1).nan_to_num().max()) / math.sqrt(d)
    return eps * exact.abs() * 1.001 + mag * (eps + 2 * (d + 2) * 2.0 ** -24 * top + 2.0 ** -20) + 6e-8


def _tree(g, t, shape):
    if shape == "chain":
        return list(range(-1, t - 1))
    if shape == "star":
        return [-1] + [0] * (t - 1)
    if shape == "forest":  # several tokens right behind the cache
        return [-1 if i % 3 == 0 else i - 1 for i in range(t)]
    up = [-1]
    for i in range(1, t):
        up.append(int(torch.randint(-2 if shape == "holes" else 0, i, (1,), generator=g)))
    if shape == "holes":
        up[0] = -1
    return up


def _state(dev, b, t, h, kvh, d, dtype, ctx, shape, cap=None, seed=0):
    g = torch.Generator().manual_seed(seed)
    parents = [_tree(g, t, shape) for _ in range(b)]
    cap = cap or max(ctx) + t + 5
    k, v = (torch.randn(b, kvh, cap, d, generator=g).to(dev, dtype) for _ in range(2))
    q = torch.randn(b, t, h, d, generator=g).to(dev, dtype)
    return q, k, v, torch.tensor(ctx, dtype=torch.int32, device=dev), parents


def _check(q, k, v, prefix, parents, got):
    exact = ref.attention(q, k, v, prefix, parents)
    err = (got.double() - exact).abs()
    bound = _bound(q, k, v, prefix, parents, exact)
    assert torch.isfinite(got).all()
    worst = (err / bound).max().item()
    assert worst <= 1.0, f"error {worst:.2f} times the bound"
    for s, up in enumerate(parents):
        for i in set(range(q.shape[1])) - set(ref.lineage(up)):
            assert got[s, i].eq(0).all()


CASES = [
    # b, t, h, kvh, d, dtype, cached positions, shape
    (1, 1, 1, 1, 128, torch.bfloat16, [0], "chain"),
    (1, 1, 8, 1, 64, torch.float16, [1], "chain"),
    (2, 5, 40, 8, 128, torch.bfloat16, [127, 130], "chain"),
    (3, 7, 8, 2, 128, torch.float16, [0, 63, 64], "tree"),
    (2, 64, 10, 2, 128, torch.bfloat16, [100, 65], "tree"),
    (1, 64, 40, 8, 64, torch.float16, [321], "star"),
    (4, 13, 28, 4, 128, torch.bfloat16, [0, 1, 500, 255], "holes"),
    (2, 33, 16, 16, 64, torch.bfloat16, [191, 192], "forest"),
    (1, 26, 5, 1, 128, torch.float16, [1000], "tree"),       # 130 rows: a second row tile of two
    (1, 52, 5, 1, 128, torch.bfloat16, [700], "holes"),      # 260 rows: a second pair of row tiles
    (1, 9, 64, 1, 128, torch.bfloat16, [383], "tree"),       # 576 rows of one KV head
    (65, 3, 4, 2, 64, torch.bfloat16, [(37 * i) % 200 for i in range(65)], "chain"),
    (3, 4, 8, 1, 128, torch.float16, [2049, 0, 4100], "tree"),
    (150, 1, 1, 1, 128, torch.bfloat16, [255] * 150, "chain"),   # several tiles of a pair per CTA
    (8, 32, 40, 8, 128, torch.bfloat16, [600 + i for i in range(8)], "tree"),
    (64, 8, 40, 8, 128, torch.bfloat16, [(97 * i) % 800 for i in range(64)], "tree"),  # several pairs per CTA
    (64, 7, 20, 4, 64, torch.float16, [(197 * i) % 1800 for i in range(64)], "holes"),
    (5, 64, 40, 8, 128, torch.float16, [(997 * i) % 3800 for i in range(5)], "tree"),
]


@pytest.mark.parametrize("b,t,h,kvh,d,dtype,ctx,shape", CASES)
def test_attention(cuda_dev, b, t, h, kvh, d, dtype, ctx, shape):
    from fitllm_b200 import ops
    q, k, v, prefix, parents = _state(cuda_dev, b, t, h, kvh, d, dtype, ctx, shape)
    up = torch.tensor(parents, dtype=torch.int32, device=cuda_dev)
    got = ops.tree_attention(q, k, v, prefix, up)
    again = ops.tree_attention(q, k, v, prefix, up)
    assert ops.device_status() == 0
    assert torch.equal(got, again)
    _check(q, k, v, prefix, parents, got)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_attention_of_large_scores_and_a_dominant_position(cuda_dev, dtype):
    """Scores that differ by hundreds, and one position with almost all the weight first."""
    from fitllm_b200 import ops
    q, k, v, prefix, parents = _state(cuda_dev, 2, 6, 8, 2, 128, dtype, [700, 300], "tree", seed=3)
    q[0] *= 12
    k[1, :, 0] = q[1, 0, 0] * 1.5
    k[1, :, 250] = q[1, 1, 3] * 2
    got = ops.tree_attention(q, k, v, prefix, torch.tensor(parents, dtype=torch.int32, device=cuda_dev))
    _check(q, k, v, prefix, parents, got)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf"), "lowest"])
def test_what_no_token_sees_changes_nothing(cuda_dev, bad):
    """Slots behind the tree, absent tokens' slots, and each token's unseen relatives."""
    from fitllm_b200 import ops
    for d, dtype in ((128, torch.bfloat16), (64, torch.float16)):
        value = -torch.finfo(dtype).max if bad == "lowest" else bad
        q, k, v, prefix, _ = _state(cuda_dev, 3, 6, 8, 2, d, dtype, [126, 0, 250], "tree", cap=300)
        parents = [[-1, 0, 0, 1, -2, 2]] * 3
        up = torch.tensor(parents[0], dtype=torch.int32, device=cuda_dev)
        clean = ops.tree_attention(q, k, v, prefix, up)
        for s in range(3):
            n = int(prefix[s])
            k[s, :, n + 4], v[s, :, n + 4] = value, value
            k[s, :, n + 6:], v[s, :, n + 6:] = value, value
        got = ops.tree_attention(q, k, v, prefix, up)
        assert torch.equal(clean, got)
        # token 3's key and value: seen by token 3 alone
        for s in range(3):
            k[s, :, int(prefix[s]) + 3], v[s, :, int(prefix[s]) + 3] = 0.5, value
        got = ops.tree_attention(q, k, v, prefix, up)
        others = [0, 1, 2, 4, 5]
        assert torch.equal(clean[:, others], got[:, others])
        if bad != "lowest":
            assert not torch.isfinite(got[:, 3]).any()
    assert ops.device_status() == 0


def test_one_element_that_is_not_finite_stays_in_its_column(cuda_dev):
    from fitllm_b200 import ops
    q, k, v, prefix, _ = _state(cuda_dev, 1, 5, 8, 2, 128, torch.bfloat16, [200], "tree")
    up = torch.tensor([-1, 0, 1, 0, 3], dtype=torch.int32, device=cuda_dev)
    clean = ops.tree_attention(q, k, v, prefix, up)
    v[0, 0, 203, 17] = float("inf")   # token 3: seen by tokens 3 and 4, heads 0-3
    v[0, 1, 202, 100] = float("nan")  # token 2: seen by itself, heads 4-7
    got = ops.tree_attention(q, k, v, prefix, up)
    bad = torch.zeros_like(got, dtype=torch.bool)
    bad[0, 3:5, :4, 17] = True
    bad[0, 2, 4:, 100] = True
    assert got[0, 3:5, :4, 17].eq(float("inf")).all() and got[0, 2, 4:, 100].isnan().all()
    assert torch.isfinite(got[~bad]).all()
    # the column's own weight aside, the others' sums are what they were
    keep = ~bad
    keep[0, 3:5, :4], keep[0, 2, 4:] = False, False
    assert torch.equal(clean[keep], got[keep])


def test_attention_takes_strides_and_one_tree_for_all(cuda_dev):
    from fitllm_b200 import ops
    b, t, h, kvh, d = 2, 7, 8, 2, 64
    q, k, v, prefix, parents = _state(cuda_dev, b, t, h, kvh, d, torch.bfloat16, [70, 129], "tree", cap=160)
    up = torch.tensor(parents[0], dtype=torch.int32, device=cuda_dev)
    want = ops.tree_attention(q, k, v, prefix, up)
    wide = torch.randn(b, t, h + 2 * kvh, d, device=cuda_dev).bfloat16()
    wide[:, :, :h] = q
    kt, vt = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (k, v))  # [B, cap, KVH, D] in memory
    big = [torch.randn(b + 1, kvh + 1, 170, d, device=cuda_dev).bfloat16() for _ in range(2)]
    for x, src in zip(big, (k, v)):
        x[1:, 1:, :160] = src
    views = [x[1:, 1:, :160] for x in big]
    rows = up.expand(b, t).contiguous()
    odd = torch.full((b, t + 3), 9, dtype=torch.int32, device=cuda_dev)
    odd[:, :t] = rows
    for args in ((wide[:, :, :h], k, v, prefix, up), (q, kt, vt, prefix, rows), (q, *views, prefix, odd[:, :t]),
                 (q.transpose(0, 1).contiguous().transpose(0, 1), k, v, prefix, up)):
        assert torch.equal(ops.tree_attention(*args), want)
    out = q.clone()
    assert ops.tree_attention(out, k, v, prefix, up, out=out) is out and torch.equal(out, want)


def test_attention_of_a_long_cache(cuda_dev):
    """Offsets behind 2^31 elements, sums over 100,000 positions."""
    from fitllm_b200 import ops
    b, t, h, kvh, d, n = 2, 5, 16, 8, 128, 1_050_000
    k, v = (torch.empty(b, kvh, n + 8, d, device=cuda_dev, dtype=torch.bfloat16) for _ in range(2))
    g = torch.Generator(device=cuda_dev).manual_seed(1)
    k.normal_(generator=g)
    v.normal_(generator=g)
    v += 1.0
    q = torch.randn(b, t, h, d, device=cuda_dev, generator=g).bfloat16()
    prefix = torch.tensor([n, 100_000], dtype=torch.int32, device=cuda_dev)
    up = torch.tensor([-1, 0, 0, 1, 2], dtype=torch.int32, device=cuda_dev)
    got = ops.tree_attention(q, k, v, prefix, up)
    for s, i, hd in ((0, 4, 15), (1, 0, 0), (0, 0, 3)):
        m = int(prefix[s])
        line = ref.lineage(up.tolist())[i][0]
        at = torch.cat([torch.arange(m), torch.tensor([m + j for j in line])]).to(cuda_dev)
        kk, vv = k[s, hd // 2, at].double(), v[s, hd // 2, at].double()
        w = torch.softmax(kk @ q[s, i, hd].double() / math.sqrt(d), 0)
        exact = w @ vv
        # values around one: eps of the result, eps of the weights (their sum is held by the same
        # factors, so that it enters once more), and tensor-core sums that round towards zero
        tol = 3 * ref.EPS[torch.bfloat16] * (w @ vv.abs())
        assert ((got[s, i, hd].double() - exact).abs() <= tol).all()


def test_attention_of_long_runs_in_fp16(cuda_dev):
    """More steps of a unit than its sums are kept in tensor memory for, many pairs at once."""
    from fitllm_b200 import ops
    b, t, h, kvh, d, n = 19, 3, 8, 8, 64, 40_000
    g = torch.Generator(device=cuda_dev).manual_seed(2)
    k, v = (torch.empty(b, kvh, n + 8, d, device=cuda_dev, dtype=torch.float16).normal_(generator=g) for _ in range(2))
    q = torch.randn(b, t, h, d, device=cuda_dev, generator=g).half()
    q[:, 1] *= 4
    prefix = torch.full((b,), n, dtype=torch.int32, device=cuda_dev)
    parents = [[-1, 0, 0]] * b
    got = ops.tree_attention(q, k, v, prefix, torch.tensor(parents[0], dtype=torch.int32, device=cuda_dev))
    for s in (0, 7, 18):
        one = q[s:s + 1], k[s:s + 1], v[s:s + 1], prefix[s:s + 1], parents[:1]
        exact = ref.attention(*one)
        err, size = (got[s:s + 1].double() - exact).norm(dim=-1), exact.norm(dim=-1)
        # the result's rounding and the weights', each at most eps, seldom near it in all 64 elements
        assert (err <= 2 * ref.EPS[torch.float16] * size + 1e-6).all(), (err / size).max()


@pytest.mark.parametrize("dtype,d,shape", [(torch.bfloat16, 128, "tree"), (torch.float16, 64, "holes"),
                                           (torch.bfloat16, 64, "chain"), (torch.float16, 128, "forest")])
def test_append_and_keep(cuda_dev, dtype, d, shape):
    from fitllm_b200 import ops
    from fitllm_b200.layer import rotary_tables
    b, t, h, kvh, layers = 4, 11, 6, 2, 70
    q, _, _, prefix, parents = _state(cuda_dev, b, t, h, kvh, d, dtype, [0, 9, 33, 5], shape, seed=5)
    g = torch.Generator(device=cuda_dev).manual_seed(7)
    kn, vn = (torch.randn(b, t, kvh, d, device=cuda_dev, generator=g).to(dtype) for _ in range(2))
    ks, vs = ([torch.randn(b, kvh, 50, d, device=cuda_dev, generator=g).to(dtype) for _ in range(layers)] for _ in range(2))
    cos, sin = rotary_tables(64, d, 1e4, cuda_dev)
    up = torch.tensor(parents, dtype=torch.int32, device=cuda_dev)
    before = [x.clone() for x in ks + vs]
    turned = ops.tree_append(q, kn, vn, ks[0], vs[0], prefix, up, cos, sin)
    eps = ref.EPS[dtype]
    want_k, want_v = before[0].clone(), before[layers].clone()
    for s, tree in enumerate(parents):
        line = ref.lineage(tree)
        for i in range(t):
            if i not in line:
                assert turned[s, i].eq(0).all()
                continue
            pos, slot = int(prefix[s]) + line[i][1], int(prefix[s]) + i
            exact = ref.rotate(q[s, i], cos[pos], sin[pos])
            # one rounding of the result; products and their sum in fp32
            tol = eps * exact.abs() * 1.001 + 3 * 2.0 ** -24 * 2 * q[s, i].double().abs().max() + 6e-8
            assert ((turned[s, i].double() - exact).abs() <= tol).all()
            exact = ref.rotate(kn[s, i], cos[pos], sin[pos])
            tol = eps * exact.abs() * 1.001 + 3 * 2.0 ** -24 * 2 * kn[s, i].double().abs().max() + 6e-8
            assert ((ks[0][s, :, slot].double() - exact).abs() <= tol).all()
            want_k[s, :, slot], want_v[s, :, slot] = ks[0][s, :, slot], vn[s, i]
    assert torch.equal(ks[0], want_k) and torch.equal(vs[0], want_v)
    out = q.clone()
    assert torch.equal(ops.tree_append(out, kn, vn, ks[0], vs[0], prefix, up, cos, sin, q_out=out), turned)
    # ---- keep
    path = torch.tensor([[0, 2, 3, 10] + [-1] * 7, [0] + [-1] * 10, [-1] * 11, list(range(11))], dtype=torch.int32, device=cuda_dev)
    accepted = torch.tensor([3, 0, -1, 10], device=cuda_dev)
    had = [x.clone() for x in ks + vs]
    lengths = ops.tree_keep(ks, vs, prefix, path, accepted)
    assert lengths.tolist() == [4, 10, 33, 16] and prefix.tolist() == [0, 9, 33, 5]
    for old, new in zip(had, ks + vs):
        old[0, :, [1, 2, 3]] = old[0, :, [2, 3, 10]].clone()
        assert torch.equal(old, new)
    assert ops.tree_keep(ks, vs, prefix, torch.full_like(path, -1), torch.full_like(accepted, -1), lengths=prefix) is prefix
    assert prefix.tolist() == [0, 9, 33, 5] and ops.device_status() == 0


def test_lengths_are_written_over_the_old_ones(cuda_dev):
    """Every cache of every layer moves by the lengths that were, also where the new ones replace them."""
    from fitllm_b200 import ops
    b, t, layers, cap = 300, 6, 70, 24
    g = torch.Generator(device=cuda_dev).manual_seed(9)
    old = [torch.randn(b, 2, cap, 64, device=cuda_dev, generator=g).half() for _ in range(2 * layers)]
    new = [x.clone() for x in old]
    prefix = torch.randint(0, cap - t, (b,), device=cuda_dev, generator=g).int()
    path = torch.tensor([0, 2, 4, 5, -1, -1], dtype=torch.int32, device=cuda_dev).expand(b, t).contiguous()
    accepted = torch.full((b,), 3, device=cuda_dev)
    before = prefix.clone()
    for _ in range(3):  # three steps in a row, on the lengths that each leaves
        at = prefix.clone().clamp(max=cap - t)
        prefix.copy_(at)
        ops.tree_keep(new[:layers], new[layers:], prefix, path, accepted, lengths=prefix)
        assert torch.equal(prefix, at + 4)
        rows = torch.arange(b, device=cuda_dev)[:, None]
        for x in old:
            x[rows, :, (at[:, None] + torch.arange(4, device=cuda_dev)).long()] = x[rows, :, (at[:, None] + path[:, :4]).long()]
    assert not torch.equal(before, prefix) and all(torch.equal(x, y) for x, y in zip(old, new)) and ops.device_status() == 0


def test_what_the_device_refuses(cuda_dev):
    """Bad parents, prefixes and paths are recorded, touch nothing and leave the others as they are."""
    from fitllm_b200 import ops
    from fitllm_b200.layer import rotary_tables
    b, t, h, kvh, d = 5, 4, 4, 2, 64
    q, k, v, _, _ = _state(cuda_dev, b, t, h, kvh, d, torch.bfloat16, [10] * 5, "chain", cap=20)
    cos, sin = rotary_tables(16, d, 1e4, cuda_dev)
    prefix = torch.tensor([10, -1, 18, 10, 30], dtype=torch.int32, device=cuda_dev)
    up = torch.tensor([[-1, 0, 1, 2], [-1, 0, 1, 2], [-1, 0, 1, 2], [-1, 0, 2, 99], [-1, 0, 1, 2]], dtype=torch.int32, device=cuda_dev)
    before = k.clone(), v.clone()
    turned = ops.tree_append(q, q[:, :, :kvh], q[:, :, :kvh], k, v, prefix, up, cos, sin)
    assert ops.device_status() == 1
    same = torch.ones_like(k, dtype=torch.bool)
    same[0, :, 10:14] = False                       # all of it, positions 10 .. 13
    same[3, :, 10:12] = False                       # tokens 2 and 3 have no parent
    assert torch.equal(k[same], before[0][same]) and torch.equal(v[same], before[1][same])
    assert torch.equal(v[0, :, 10:14], q[0, :, :kvh].transpose(0, 1)) and not torch.equal(k[0, :, 11], before[0][0, :, 11])
    assert turned[1].eq(0).all() and turned[2].eq(0).all() and turned[3, 2:].eq(0).all() and turned[4].eq(0).all()
    got = ops.tree_attention(q, k, v, prefix, up)
    assert ops.device_status() == 1 and torch.isfinite(got).all()
    assert got[1].eq(0).all() and got[2, 2:].eq(0).all() and got[3, 2:].eq(0).all() and got[4].eq(0).all()
    _check(q[:1], k[:1], v[:1], prefix[:1], [[-1, 0, 1, 2]], got[:1])
    _check(q[2:4], k[2:4], v[2:4], prefix[2:4], [[-1, 0, -2, -2], [-1, 0, -2, -2]], got[2:4])
    path = torch.tensor([[0, 2, 1, -1], [0, 1, -1, -1], [0, 1, 2, 3], [1, 3, 9, -1], [0, 1, 2, 3]], dtype=torch.int32, device=cuda_dev)
    accepted = torch.tensor([2, 1, 3, 2, 7], device=cuda_dev)
    before = k.clone(), v.clone()
    lengths = ops.tree_keep([k], [v], prefix, path, accepted)
    assert ops.device_status() == 1 and lengths.tolist() == prefix.tolist()
    assert torch.equal(k, before[0]) and torch.equal(v, before[1])


def _logits(dev, b, t, v, dtype, seed, spread=2.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    z = torch.randn(b, t, v, device=dev, generator=g) * spread
    z[..., v // 3] += 6
    return z.to(dtype), g


VERIFY = [
    # b, t, v, dtype, shape, with a drafting distribution, temperature
    (1, 1, 1, torch.float32, "chain", False, 1.0),
    (1, 1, 17, torch.bfloat16, "chain", False, 0.7),
    (3, 5, 1000, torch.bfloat16, "chain", True, 0.8),
    (3, 9, 1001, torch.float16, "tree", True, 1.3),
    (2, 64, 777, torch.float32, "star", True, 1.0),
    (2, 64, 2053, torch.bfloat16, "star", False, 1.0),
    (4, 20, 32001, torch.float16, "tree", False, 0.5),
    (2, 6, 152064, torch.bfloat16, "chain", True, 1.0),
    (70, 4, 5003, torch.float32, "chain", True, 0.3),
    (200, 3, 3001, torch.bfloat16, "chain", False, 1.0),
    (5, 12, 1500, torch.bfloat16, "holes", False, 0.0),
    (3, 7, 1500, torch.float32, "tree", True, 0.0),
]


@pytest.mark.parametrize("b,t,v,dtype,shape,with_q,temp", VERIFY)
def test_verify(cuda_dev, b, t, v, dtype, shape, with_q, temp):
    from fitllm_b200 import ops
    from fitllm_b200.verify import verify_tree
    z, g = _logits(cuda_dev, b, t, v, dtype, seed=b * 100 + t)
    cg = torch.Generator().manual_seed(t)
    parents = [_tree(cg, t, shape) for _ in range(b)]
    u = torch.rand(b, t, device=cuda_dev, generator=g)
    q = None
    p = torch.softmax(z.float() / max(temp, 0.5), -1)
    rows = torch.tensor(parents, device=cuda_dev).clamp(min=0)
    if with_q:
        q = torch.softmax(torch.log(p + 1e-9) * 0.7 + torch.randn(p.shape, device=cuda_dev, generator=g), -1)[:, :max(t - 1, 1)]
    draft = torch.multinomial((q if with_q else p).gather(1, rows.clamp(max=max(t - 2, 0))[..., None].expand(b, t, v)).view(b * t, v), 1,
                              generator=g).view(b, t)
    if b > 2:
        draft[2, -1] = v + 3  # an id that no row has
    up = torch.tensor(parents, dtype=torch.int32, device=cuda_dev)
    r = verify_tree(z, draft, up, u, draft_probs=q, temperature=temp)
    assert ops.device_status() == 0
    for s in range(b):
        path, acc, nxt = ref.verify(z[s], draft[s].tolist(), parents[s], u[s], None if q is None else q[s], temp)
        assert r.path[s].tolist() == path + [-1] * (t - len(path)) and int(r.accepted[s]) == acc, (s, path)
        assert int(r.next_token[s]) == nxt, s
    temps = torch.full((b,), temp, device=cuda_dev)
    same = verify_tree(z, draft.int(), up, u, draft_probs=q, temperature=temps)
    assert all(torch.equal(x, y) for x, y in zip(r, same))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_verify_takes_masked_rows_and_odd_numbers(cuda_dev, dtype):
    from fitllm_b200 import ops
    from fitllm_b200.verify import verify_tree
    b, t, v = 9, 3, 515
    z, g = _logits(cuda_dev, b, t, v, dtype, seed=4)
    u = torch.full((b, t), 0.5, device=cuda_dev)
    up = torch.tensor([[-1, 0, 1]] * b, dtype=torch.int32, device=cuda_dev)
    draft = z.argmax(-1).roll(1, 1)
    ninf = float("-inf")
    z[0, 0] = ninf                       # no token is allowed
    z[1, 0, 7] = float("nan")
    z[2, 0] = ninf
    z[2, 0, 300] = -5.0                  # one token alone, which is drafted
    draft[2, 1] = 300
    z[3, 0] = ninf
    z[3, 0, 200] = 1.0                   # one token alone, and another one drafted
    z[4, 0] = torch.finfo(dtype).min     # a uniform row
    u[4] = 0.0
    z[5, 0, 100] = float("inf")
    u[6, 0] = 1.0                        # one or more: the last token that has weight
    u[7, 0] = -1.0
    up[8, 0] = -2
    draft[6:8, 1] = -100
    r = verify_tree(z, draft, up, u)
    assert ops.device_status() == 0
    for s in range(b):
        path, acc, nxt = ref.verify(z[s], draft[s].tolist(), up[s].tolist(), u[s], None, 1.0)
        assert (r.path[s].tolist(), int(r.accepted[s]), int(r.next_token[s])) == (path + [-1] * (t - len(path)), acc, nxt), s
    greedy = verify_tree(z, draft, up, u, temperature=0.0)
    for s in range(b):
        path, acc, nxt = ref.verify(z[s], draft[s].tolist(), up[s].tolist(), u[s], None, 0.0)
        assert (greedy.path[s].tolist(), int(greedy.accepted[s]), int(greedy.next_token[s])) == (path + [-1] * (t - len(path)), acc, nxt), s
    bad = verify_tree(z, draft, up, u, temperature=torch.tensor([-1.0] + [1.0] * (b - 1), device=cuda_dev))
    assert ops.device_status() == 1 and int(bad.next_token[0]) == -1 and torch.equal(bad.path[1:], r.path[1:])


def test_verify_of_refused_children_that_hold_all_the_weight(cuda_dev):
    """Every token of the row drafted and refused in turn, and the same id twice."""
    from fitllm_b200.verify import verify_tree
    v = 6
    z = torch.zeros(1, 8, v, device=cuda_dev)
    up = torch.tensor([-1] + [0] * 7, dtype=torch.int32, device=cuda_dev)
    u = torch.full((1, 8), 0.999999, device=cuda_dev)
    draft = torch.tensor([[0, 0, 0, 1, 2, 3, 4, 4]], device=cuda_dev)
    r = verify_tree(z, draft, up, u)
    assert r.path[0].tolist() == [0] + [-1] * 7 and int(r.next_token) == 5
    u[0, 1:] = 1.0  # never below a probability
    draft = torch.tensor([[0, 0, 1, 2, 3, 4, 5, 5]], device=cuda_dev)
    assert int(verify_tree(z, draft, up, u).next_token) == 0  # no weight is left: the largest logit
    q = torch.full((1, 7, v), 1 / v, device=cuda_dev)
    assert int(verify_tree(z, draft, up, u, draft_probs=q).next_token) in range(v)


@pytest.mark.parametrize("v,spread,temp", [(20_000, 2.0, 1.0), (9_000, 0.0, 1.0), (700, 2.0, 0.7), (20_000, 30.0, 0.05)])
def test_verify_draws_next_to_a_border(cuda_dev, v, spread, temp):
    """Few tokens allowed, the first of them drafted and refused, and random numbers that fall on a border
    of the cumulated weights: the next token is always one that has weight."""
    from fitllm_b200.verify import verify_tree
    b, t, n = 96, 3, 40
    g = torch.Generator(device=cuda_dev).manual_seed(v)
    z = torch.full((b, t, v), float("-inf"), device=cuda_dev)
    allowed = torch.stack([torch.randperm(min(v, 2500), device=cuda_dev, generator=g)[:n].sort().values for _ in range(b)])
    some = torch.randn(b, n, device=cuda_dev, generator=g) * spread
    z[:, 0] = z[:, 0].scatter(1, allowed, some)
    z = z.bfloat16()
    # exp(-707), 2^-1020, of the largest weighs nothing (exp(-746) is the last fp64 that is not 0); at the
    # fourth case's temperature that is 35.35 below the largest, where bf16 logits are multiples of 1/8
    weighed = z.clone()
    weighed[z.double() < z.double().amax(-1, keepdim=True) - 707 * temp] = float("-inf")
    draft = torch.zeros(b, t, dtype=torch.int64, device=cuda_dev)
    draft[:, 1:] = allowed[:, :2]
    up = torch.tensor([-1, 0, 0], dtype=torch.int32, device=cuda_dev)
    for first in (0.0, 1 - 2.0 ** -24, 1.0):
        u = torch.full((b, t), 1 - 2.0 ** -24, device=cuda_dev)
        u[:, 0] = first
        r = verify_tree(z, draft, up, u, temperature=temp)
        for s in range(b):
            path, acc, nxt = ref.verify(weighed[s], draft[s].tolist(), [-1, 0, 0], u[s], None, temp)
            assert (int(r.accepted[s]), int(r.next_token[s])) == (acc, nxt), (first, s)
    if spread == 0.0:  # equal weights: a random number on each border of the 38 that are left
        u = torch.full((b, t), 1 - 2.0 ** -24, device=cuda_dev)
        u[:, 0] = torch.arange(b, device=cuda_dev) % 38 / 38
        r = verify_tree(z, draft, up, u)
        at = torch.arange(b, device=cuda_dev)[:, None] % 38 + torch.tensor([1, 2], device=cuda_dev)  # either side of it
        assert (r.next_token[:, None] == allowed.gather(1, at)).any(1).all() and not (r.next_token[:, None] == draft[:, 1:]).any()


def test_verify_is_a_sample_of_the_model(cuda_dev):
    """First accepted-or-next tokens follow p, whatever was drafted: 40,000 sequences of one draft
    of a distribution far from p; chi-square over 8 tokens below its 1 - 1e-6 quantile (40.5 for 7)."""
    from fitllm_b200.verify import verify_tree
    n, v = 40_000, 8
    g = torch.Generator(device=cuda_dev).manual_seed(11)
    z = torch.tensor([0.0, 1.0, 2.0, -1.0, 0.5, -2.0, 1.5, 0.2], device=cuda_dev)
    q = torch.softmax(-z, -1)
    draft = torch.zeros(n, 3, dtype=torch.int64, device=cuda_dev)
    draft[:, 1:] = torch.multinomial(q.expand(n, v), 2, replacement=True, generator=g)
    up = torch.tensor([-1, 0, 0], dtype=torch.int32, device=cuda_dev)
    r = verify_tree(z.expand(n, 3, v), draft, up, torch.rand(n, 3, device=cuda_dev, generator=g), draft_probs=q.expand(n, 2, v))
    first = torch.where(r.accepted > 0, draft.gather(1, r.path[:, 1:2].long().clamp(min=0))[:, 0], r.next_token)
    seen = torch.bincount(first, minlength=v).double()
    want = torch.softmax(z.double(), -1) * n
    assert float(((seen - want) ** 2 / want).sum()) < 40.5


def test_strided_logits_and_drafts(cuda_dev):
    from fitllm_b200.verify import verify_tree
    b, t, v = 3, 5, 999
    z, g = _logits(cuda_dev, b, t, v + 30, torch.bfloat16, seed=8)
    u = torch.rand(b, t, device=cuda_dev, generator=g)
    q = torch.softmax(torch.randn(b, t, v + 2, device=cuda_dev, generator=g), -1)
    draft = z[..., 1:v + 1].float().argmax(-1).roll(1, 1)
    up = torch.tensor([-1, 0, 1, 1, 3], dtype=torch.int32, device=cuda_dev)
    a = verify_tree(z[..., 1:v + 1], draft, up, u, draft_probs=q[..., 1:v + 1])
    c = verify_tree(z[..., 1:v + 1].contiguous(), draft, up, u, draft_probs=q[..., 1:v + 1].contiguous())
    assert all(torch.equal(x, y) for x, y in zip(a, c))
