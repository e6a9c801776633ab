"""Tensors that lie over one another in the calls on trees of drafted tokens and of the adapters
of many requests: refused by the C entry points before any device call (no GPU needed)."""
import ctypes
import itertools

import pytest
import torch

from fitllm_b200 import _lib

ARG, NO_DEVICE = 1, 8
P = 0x10000
FAR = P + (1 << 32)


@pytest.fixture(scope="module")
def L():
    from fitllm_b200 import build
    build.build()
    return _lib.load()


def _tree(batch=3, heads=2, cap=20, strides=None, d=64, tokens=4):
    sb, sh, sp = strides or (heads * cap * d, cap * d, d)
    return _lib.TreeC(P, P, 0, cap, sb, sh, sp, batch, tokens, heads, d, 0)


def _append(L, c, kc, vc, q=FAR, out=2 * FAR):
    return L.fitq_tree_append(c, q, c.kv_heads * c.head_dim, FAR, c.kv_heads * c.head_dim, FAR, c.kv_heads * c.head_dim, out, kc, vc,
                              P, P, 64, c.kv_heads, None)


def _keep(L, c, ks, vs):
    n = len(ks)
    return L.fitq_tree_keep(c, (ctypes.c_void_p * n)(*ks), (ctypes.c_void_p * n)(*vs), n, P, P, P, None)


def _good(code):
    """The call was not refused: it went on to the device, which is not here (or was not asked on one)."""
    return code == NO_DEVICE


LAYOUTS = [  # batch, heads, slots, strides of sequences, heads and slots, in elements
    (3, 2, 20, (2 * 20 * 64, 20 * 64, 64)),           # dense
    (3, 2, 20, (2 * 2 * 20 * 64, 20 * 64, 64)),       # room for another cache between sequences
    (3, 2, 20, (2 * 20 * 128, 20 * 128, 128)),        # keys and values of a slot side by side
    (3, 2, 20, (20 * 2 * 64, 64, 2 * 64)),            # slots before heads
    (3, 2, 20, (20 * 4 * 64, 64, 4 * 64)),            # [batch, slots, keys and values, heads, 64]
    (1, 3, 7, (64, 7 * 72, 72)),                      # padded slots, one sequence
    (2, 1, 5, (5 * 64 + 8, 64, 64)),                  # padded sequences
]


@pytest.mark.skipif(torch.cuda.is_available(), reason="addresses that are nothing's")
@pytest.mark.parametrize("batch,heads,cap,strides", LAYOUTS)
def test_caches_over_one_another(L, batch, heads, cap, strides):
    """By counting every element: caches that share one are refused, others at any distance are not."""
    c = _tree(batch, heads, cap, strides)
    pieces = {sum(i * s for i, s in zip(at, strides)) // 8 + y for at in itertools.product(range(batch), range(heads), range(cap))
              for y in range(8)}  # of eight elements
    base = FAR + (1 << 24)
    tried = {False: 0, True: 0}
    for off in range(0, 8 * max(pieces) + 80, 8):
        meets = not pieces.isdisjoint({x + off // 8 for x in pieces})
        for kc, vc in ((base, base + 2 * off), (base + 2 * off, base)):
            assert (_append(L, c, kc, vc) == ARG) == meets, off
            assert _good(_append(L, c, kc, vc)) == (not meets)
        if off % 24 == 0:
            assert (_keep(L, c, [base, base + (1 << 20)], [base - (1 << 20), base + 2 * off]) == ARG) == meets, off
        tried[meets] += 1
    assert tried[1] and tried[0]


@pytest.mark.skipif(torch.cuda.is_available(), reason="addresses that are nothing's")
def test_many_layers_in_one_storage(L):
    layers, cap, d = 60, 20, 64
    # [batch, layers, 2, heads, slots, d]: every cache lies between the others'
    c = _tree(strides=(layers * 2 * 2 * cap * d, cap * d, d))
    at = [FAR + i * 2 * cap * d * 2 for i in range(2 * layers)]
    assert _good(_keep(L, c, at[::2], at[1::2]))
    at[77] -= 2 * d
    assert _keep(L, c, at[::2], at[1::2]) == ARG


@pytest.mark.skipif(torch.cuda.is_available(), reason="addresses that are nothing's")
def test_the_largest_strides(L):
    """Reaches that 64 bits do not hold."""
    big = (1 << 38) - 8
    c = _tree(batch=1, heads=1, cap=1 << 30, strides=(big, big, big))
    assert _good(_append(L, c, FAR, FAR + 64 * 2)) and _append(L, c, FAR, FAR + 32 * 2) == ARG
    assert _append(L, c, FAR, FAR + 2 * big) == ARG
    # sequences, heads and slots that lie over one another: such a cache shares elements with any beside it
    c = _tree(batch=65535, heads=2, cap=1 << 30, strides=(big, big, big))
    assert _append(L, c, FAR, FAR + 64 * 2) == ARG


@pytest.mark.skipif(torch.cuda.is_available(), reason="addresses that are nothing's")
def test_results_over_the_caches(L):
    c = _tree(tokens=5)
    caches, row, size, out = (FAR + (1 << 24), FAR + (2 << 24)), 128, 3 * 2 * 20 * 64 * 2, 3 * 5 * 128 * 2

    def attend(at):
        return L.fitq_tree_attention(c, FAR, row, caches[0], caches[1], at, 2, P, 1 << 40, None)

    for call in (attend, lambda at: _append(L, c, *caches, out=at)):
        for cache in caches:
            for at in (cache - out + 16, cache, cache + 4096, cache + size - 16):
                assert call(at) == ARG
            assert _good(call(cache - out)) and _good(call(cache + size))


def test_results_in_place_over_the_caches(monkeypatch):
    """The wrappers look at results that are q, too."""
    from fitllm_b200 import ops
    from fitllm_b200.ops import _result_beside
    store = torch.zeros(3, 2, 20, 64, dtype=torch.bfloat16)
    k, v = store, torch.zeros_like(store)
    inside, beside = store.view(-1)[:1920].view(3, 5, 2, 64), torch.zeros(3, 5, 2, 64, dtype=torch.bfloat16)
    for caches in ((k, v), (v, k)):
        with pytest.raises(ValueError, match="overlaps"):
            _result_beside("tree_attention", "out", inside, *caches)
        _result_beside("tree_attention", "out", beside, *caches)


@pytest.mark.skipif(torch.cuda.is_available(), reason="addresses that are nothing's")
@pytest.mark.parametrize("batch,heads,cap,strides", LAYOUTS)
def test_results_between_the_caches_parts(L, batch, heads, cap, strides):
    """By counting every element: results that share one with a cache are refused, others are not."""
    from fitllm_b200.ops import _holds
    c = _tree(batch, heads, cap, strides, tokens=1)
    pieces = {sum(i * s for i, s in zip(at, strides)) // 8 + y for at in itertools.product(range(batch), range(heads), range(cap))
              for y in range(8)}  # of eight elements
    n, base = batch * heads * 64, FAR + (1 << 24)
    view = torch.empty(8 * max(pieces) + 8, dtype=torch.bfloat16).as_strided((batch, heads, cap, 64), (*strides, 1))
    tried = {False: 0, True: 0}
    for off in range(-n - 16, 8 * max(pieces) + 32, 8):
        meets = any(off // 8 + i in pieces for i in range(n // 8))
        for caches in ((base, FAR << 1), (FAR << 1, base)):
            assert (L.fitq_tree_attention(c, FAR, heads * 64, *caches, base + 2 * off, heads, P, 1 << 40, None) == ARG) == meets, off
            assert (_append(L, c, *caches, out=base + 2 * off) == ARG) == meets, off
        assert _holds(view, 2 * off, 2 * (off + n)) == meets, off
        tried[meets] += 1
    assert tried[True] and tried[False]


@pytest.mark.skipif(torch.cuda.is_available(), reason="addresses that are nothing's")
@pytest.mark.parametrize("start", [None, FAR + (6 << 24)])
def test_results_over_the_adapters(L, start):
    tokens, k, n, r, adapters, batch = 6, 256, 128, 16, 2, 3
    at = {name: FAR + (i << 24) for i, name in enumerate(("x", "a", "b", "scale", "adapter", "ws"))}
    sizes = dict(a=adapters * r * k * 2, b=adapters * n * r * 2, scale=adapters * 4, adapter=batch * 4, ws=tokens * r * 4)
    if start is not None:
        at["q_start"], sizes["q_start"] = start, (batch + 1) * 4
    y = FAR + (8 << 24)

    def call(out, add=y):
        return L.fitq_multi_lora(at["x"], k, tokens, k, n, at["a"], at["b"], r, adapters, at["scale"], at["adapter"], start, batch,
                                 add, n, out, 0, at["ws"], sizes["ws"], None)

    size = tokens * n * 2
    assert _good(call(y)) and _good(call(y + size))
    for name, nbytes in sizes.items():
        first, last = at[name] // 16 * 16, (at[name] + nbytes - 1) // 16 * 16
        for out in (first - size + 16, first, last):
            assert call(out) == ARG and call(out, add=out) == ARG, name
        assert _good(call(first - size)) and _good(call(last + 16)), name
