"""Refusals of the calls on trees of drafted tokens and of the adapters of many
requests, before any device call (no GPU needed), and their host-side logic."""
import ctypes

import pytest
import torch

from fitllm_b200 import _lib, ops
from tests import tree_ref as ref

ARG, SHAPE, ALIGN, UNSUPPORTED, NO_DEVICE = 1, 2, 3, 4, 8
P = 0x10000  # an aligned address that no refused call reads
FAR = P + (1 << 30)


@pytest.fixture(scope="module")
def L():
    from fitllm_b200 import build
    build.build()
    return _lib.load()


def _tree(**kw):
    c = dict(parents=P, prefix=P, parents_stride=8, capacity=100, stride_b=2 * 100 * 128, stride_h=100 * 128, stride_p=128,
             batch=3, tokens=8, kv_heads=2, head_dim=128, dtype=0)
    c.update(kw)
    return _lib.TreeC(**c)


def _append(L, c, q=P, k=FAR, v=FAR, out=2 * FAR, kc=P, vc=3 * FAR, cos=P, rope=64, heads=8, qs=1024, ks=256):
    return L.fitq_tree_append(c, q, qs, k, ks, v, ks, out, kc, vc, cos, P, rope, heads, None)


def _attend(L, c, q=P, qs=1024, kc=P, out=FAR, heads=8, ws=P, size=1 << 40):
    return L.fitq_tree_attention(c, q, qs, kc, P, out, heads, ws, size, None)


def _keep(L, c, layers=1, ptr=P, path=P, acc=P, lengths=P, values=FAR):
    k, v = ((ctypes.c_void_p * max(layers, 1))(*[x and x + i * (1 << 24) for i in range(max(layers, 1))]) for x in (ptr, values))
    return L.fitq_tree_keep(c, k, v, layers, path, acc, lengths, None)


BAD_TREES = [
    (dict(parents=None), ARG), (dict(prefix=None), ARG), (dict(head_dim=96), UNSUPPORTED), (dict(dtype=2), UNSUPPORTED),
    (dict(tokens=0), UNSUPPORTED), (dict(tokens=65), UNSUPPORTED), (dict(batch=0), SHAPE), (dict(kv_heads=3), SHAPE),
    (dict(capacity=0), SHAPE), (dict(capacity=(1 << 30) + 1), SHAPE), (dict(parents_stride=7), SHAPE),
    (dict(stride_p=120), SHAPE), (dict(stride_b=0), SHAPE), (dict(stride_h=0), SHAPE), (dict(stride_h=12801), SHAPE), (dict(stride_b=-8), SHAPE), (dict(stride_b=1 << 40), SHAPE),
    (dict(parents=P + 2), ALIGN), (dict(prefix=P + 1), ALIGN),
]


@pytest.mark.parametrize("bad,code", BAD_TREES)
def test_bad_trees_are_refused_by_every_call(L, bad, code):
    c = _tree(**bad)
    assert _append(L, c) == code and _attend(L, c) == code
    if bad != dict(kv_heads=3):
        assert _keep(L, c) == code
    assert L.fitq_tree_attention_workspace(c, 8) == 0
    assert L.fitq_last_error().decode()


def test_append_refusals(L):
    c = _tree()
    assert L.fitq_tree_append(None, P, 1024, P, 256, P, 256, P, P, P, P, P, 64, 8, None) == ARG
    assert _append(L, c, q=None) == ARG and _append(L, c, kc=None) == ARG and _append(L, c, cos=None) == ARG
    assert _append(L, c, rope=0) == SHAPE and _append(L, c, heads=7) == SHAPE
    assert _append(L, c, qs=1000) == SHAPE and _append(L, c, qs=1028) == SHAPE and _append(L, c, ks=248) == SHAPE
    assert _append(L, c, q=P + 2) == ALIGN and _append(L, c, kc=P + 8) == ALIGN and _append(L, c, cos=P + 4) == ALIGN
    assert _append(L, c, out=P, qs=2048) == ARG and _append(L, c, out=P + 2048) == ARG and _append(L, c, k=2 * FAR) == ARG
    assert _append(L, c, vc=P) == ARG  # keys and values in one cache
    if not torch.cuda.is_available():
        assert _append(L, c) == NO_DEVICE and _append(L, c, out=P) == NO_DEVICE


def test_attention_refusals(L):
    c = _tree()
    assert _attend(L, c, out=None) == ARG and _attend(L, c, ws=None) == ARG and _attend(L, c, kc=None) == ARG
    assert _attend(L, c, qs=1000) == SHAPE and _attend(L, c, qs=1028) == SHAPE and _attend(L, c, heads=7) == SHAPE
    assert _attend(L, c, q=P + 8) == ALIGN and _attend(L, c, kc=P + 4) == ALIGN
    assert _attend(L, c, out=P + 2048) == ARG and _attend(L, c, out=P, qs=2048) == ARG  # out over q
    wide = _tree(batch=65535, capacity=1 << 30)
    assert _attend(L, wide) == SHAPE and L.fitq_tree_attention_workspace(wide, 8) == 0
    assert L.fitq_tree_attention_workspace(c, 8) > 0 and L.fitq_tree_attention_workspace(c, 7) == 0
    if not torch.cuda.is_available():
        assert _attend(L, c) == NO_DEVICE and _attend(L, c, out=P) == NO_DEVICE


def test_keep_refusals(L):
    c = _tree()
    assert _keep(L, c, ptr=None) == ARG and _keep(L, c, path=None) == ARG and _keep(L, c, lengths=None) == ARG
    assert _keep(L, c, layers=0) == SHAPE
    assert _keep(L, c, values=P) == ARG and _keep(L, c, layers=3, values=P + (2 << 24)) == ARG  # a cache twice
    assert _keep(L, c, lengths=P + 4) == ARG  # over the prefix, other than being it
    assert _keep(L, c, ptr=P + 8) == ALIGN and _keep(L, c, acc=P + 4) == ALIGN and _keep(L, c, path=P + 2) == ALIGN


def test_verify_refusals(L):
    def call(z=P, dtype=0, sb=800, st=100, batch=2, tokens=8, vocab=100, ids=P, parents=P, ps=8, u=P, q=P, qb=700, qt=100,
             temps=None, temp=1.0, path=P):
        return L.fitq_tree_verify(z, dtype, sb, st, batch, tokens, vocab, ids, parents, ps, u, q, qb, qt, temps, temp, path,
                                  P, P, None)

    assert call(z=None) == ARG and call(ids=None) == ARG and call(u=None) == ARG and call(path=None) == ARG
    assert call(temp=-0.5) == ARG and call(temp=float("nan")) == ARG and call(temp=float("inf")) == ARG
    assert call(dtype=3) == UNSUPPORTED and call(tokens=0) == UNSUPPORTED and call(tokens=65) == UNSUPPORTED
    assert call(batch=0) == SHAPE and call(vocab=0) == SHAPE and call(vocab=1 << 24, st=1 << 24, qt=1 << 24) == SHAPE
    assert call(st=99) == SHAPE and call(ps=7) == SHAPE and call(qt=99) == SHAPE and call(qb=-1) == SHAPE
    assert call(z=P + 1) == ALIGN and call(dtype=2, z=P + 2) == ALIGN and call(ids=P + 4) == ALIGN and call(q=P + 2) == ALIGN
    if not torch.cuda.is_available():
        assert call() == NO_DEVICE and call(q=None) == NO_DEVICE and call(temps=P, temp=-1.0) == NO_DEVICE


def test_multi_lora_refusals(L):
    def call(x=P, xs=256, tokens=6, k=256, n=128, a=P, b=P, rank=16, adapters=2, scale=P, adapter=P, start=None, batch=3,
             y=FAR, ys=128, out=2 * FAR, dtype=0, ws=P, size=1 << 30):
        return L.fitq_multi_lora(x, xs, tokens, k, n, a, b, rank, adapters, scale, adapter, start, batch, y, ys, out, dtype, ws,
                                 size, None)

    assert call(x=None) == ARG and call(adapter=None) == ARG and call(ws=None) == ARG and call(out=None) == ARG
    assert call(rank=8) == UNSUPPORTED and call(rank=80) == UNSUPPORTED and call(dtype=2) == UNSUPPORTED
    assert call(k=252, xs=256) == SHAPE and call(n=100, ys=104) == SHAPE and call(tokens=-1) == SHAPE and call(adapters=0) == SHAPE
    assert call(batch=(1 << 20) + 1, start=P) == SHAPE and call(n=(1 << 24) - 8, ys=1 << 24, tokens=1 << 27, start=P) == SHAPE
    assert call(xs=248) == SHAPE and call(ys=132) == SHAPE and call(tokens=7) == SHAPE and call(batch=0) == SHAPE
    assert call(a=P + 8) == ALIGN and call(scale=P + 2) == ALIGN and call(start=P + 1) == ALIGN
    assert call(out=FAR + 256) == ARG and call(out=FAR, ys=136) == ARG and call(out=P) == ARG  # over y, over x
    assert call(tokens=0) == 0
    assert L.fitq_multi_lora_workspace(6, 256, 128, 16, 3) > 0 and L.fitq_multi_lora_workspace(6, 256, 128, 8, 3) == 0
    if not torch.cuda.is_available():
        assert call() == NO_DEVICE and call(out=FAR) == NO_DEVICE and call(tokens=7, start=P) == NO_DEVICE


def test_struct_layout_matches_the_header():
    assert ctypes.sizeof(_lib.TreeC) == 2 * 8 + 5 * 8 + 5 * 4 + 4


def test_python_refusals():
    from fitllm_b200.verify import verify_tree
    k = torch.zeros(2, 1, 16, 64, dtype=torch.bfloat16)
    q, prefix, parents = torch.zeros(2, 3, 4, 64, dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        ops.tree_attention(q, k, k, prefix, parents)
    with pytest.raises(ValueError, match="CUDA"):
        verify_tree(torch.zeros(2, 3, 8), torch.zeros(2, 3, dtype=torch.int64), parents, torch.zeros(2, 3))
    with pytest.raises(ValueError, match="CUDA"):
        ops.multi_lora(q.view(6, 256), k.view(1, 16, 128).repeat(1, 1, 2), k.view(1, 128, 16)[:, :64], torch.zeros(1), prefix,
                       torch.zeros(6, 64).bfloat16())
    with pytest.raises(NotImplementedError, match="gradient"):
        ops.tree_attention(q.requires_grad_(), k, k, prefix, parents)
    with pytest.raises(ValueError, match="0 key"):
        ops.tree_keep([], [], prefix, parents, prefix)


def test_the_cache_of_trees_refuses_other_layers():
    from types import SimpleNamespace
    from fitllm_b200.verify import TreeKVCache, chain_parents, tree_pass
    with pytest.raises(ValueError, match="head_dim"):
        TreeKVCache(1, 2, 1, 96, 16, "cpu")
    cache = TreeKVCache(1, 2, 1, 64, 16, "cpu")
    assert cache.batch == 2 and cache.prefix.tolist() == [0, 0] and cache.tables[0].shape == (16, 32)
    h = torch.zeros(2, 3, 64)
    layer = SimpleNamespace(cfg=SimpleNamespace(rope_theta=1e4))
    with pytest.raises(ValueError, match="rope_theta"):
        tree_pass([layer], h, cache, chain_parents(3, "cpu"))
    with pytest.raises(ValueError, match="sequences"):
        tree_pass([layer], h[:1], cache, chain_parents(3, "cpu"))
    assert chain_parents(3, "cpu").tolist() == [-1, 0, 1]
    cache.set_lengths([3, 16])
    assert cache.prefix.tolist() == [3, 16]
    for bad in ([3], [17, 0], [-1, 0]):
        with pytest.raises(ValueError, match="set_lengths"):
            cache.set_lengths(bad)
    cache.release(1)
    assert cache.prefix.tolist() == [3, 0]


def test_adapters_are_loaded_by_name_and_padded():
    from fitllm_b200.lora import MultiLoRAManager
    from fitllm_b200.qlora import Linear4bit
    model = torch.nn.Module()
    model.q_proj, model.v_proj, model.other = Linear4bit(64, 64), Linear4bit(64, 32), Linear4bit(64, 64)
    m = MultiLoRAManager(3, 16, ("q_proj", "v_proj"))
    m.apply(model)
    assert set(m.layers) == {"q_proj", "v_proj"} and isinstance(model.other, Linear4bit)
    assert not [n for n, _ in model.named_parameters() if "lora" in n]
    state = {"base.q_proj.lora_A.weight": torch.ones(8, 64), "base.q_proj.lora_B.weight": torch.full((64, 8), 2.0)}
    assert m.load(1, state, alpha=16.0) == 1
    q, v = m.layers["q_proj"], m.layers["v_proj"]
    assert q.scaling.tolist() == [0.0, 2.0, 0.0] and q.lora_A[1, :8].eq(1).all() and q.lora_A[1, 8:].eq(0).all()
    assert q.lora_B[1, :, :8].eq(2).all() and q.lora_B[1, :, 8:].eq(0).all() and v.scaling.tolist() == [0.0] * 3
    for bad in ({"base.x.lora_A.weight": torch.ones(8, 64)}, {"q_proj.lora_A.weight": torch.ones(8, 64)},
                {"q_proj.lora_A.weight": torch.ones(32, 64), "q_proj.lora_B.weight": torch.ones(64, 32)}):
        with pytest.raises(ValueError):
            m.load(0, bad, alpha=1.0)
    with pytest.raises(IndexError):
        q.load(3, torch.ones(8, 64), torch.ones(64, 8), 1.0)
    m.unload(1)
    assert q.scaling.eq(0).all() and q.lora_B.eq(0).all()
    with pytest.raises(ValueError, match="int32"):
        m.route(torch.zeros(2))


def test_the_restatement_walks_trees():
    line = ref.lineage([-1, 0, 0, 1, -2, 4, -1])
    assert line == {0: ([0], 0), 1: ([0, 1], 1), 2: ([0, 2], 1), 3: ([0, 1, 3], 2), 6: ([6], 0)}
    logits = torch.log(torch.tensor([[0.5, 0.3, 0.2]] * 3))
    # child 1 (id 0) is refused by its number, child 2 (id 1) accepted against 0.3 / 0.5
    assert ref.verify(logits, [9, 0, 1], [-1, 0, 0], [0.0, 0.6, 0.55], None, 1.0) == ([0, 2], 1, 0)
    assert ref.verify(logits, [9, 0, 1], [-1, 0, 0], [0.9, 0.6, 0.65], None, 1.0) == ([0], 0, 2)
    assert ref.verify(logits, [9, 0, 1], [-1, 0, 1], [0.0, 0.0, 0.0], None, 0.0) == ([0, 1], 1, 0)
