"""Refusals of the 4-bit cache and log-probability calls, before any device call
(no GPU needed), and the plain restatement the GPU tests compare with."""
import ctypes

import pytest
import torch

from fitllm_b200 import _lib, ops
from fitllm_b200.lm_head import token_logprobs
from tests import kv4_ref as ref

ARG, SHAPE, ALIGN, UNSUPPORTED, WORKSPACE, NO_DEVICE = 1, 2, 3, 4, 5, 8
P = 0x10000  # an aligned address that no refused call reads


@pytest.fixture(scope="module")
def L():
    from fitllm_b200 import build
    build.build()
    return _lib.load()


def _cache(**kw):
    c = dict(pool=P, page_table=P, prefix=P, q_start=None, tokens=8, num_pages=4, batch=4, kv_heads=2, head_dim=128,
             page_size=64, max_pages=3)
    c.update(kw)
    return _lib.Kv4C(**c)


def _append(L, c, q=P, k=P, v=P, out=P + 4096, cos=P, sin=P, rope=64, heads=8, dtype=0, qs=None, ks=None):
    qs = heads * c.head_dim if qs is None else qs
    ks = c.kv_heads * c.head_dim if ks is None else ks
    return L.fitq_kv4_append(c, q, qs, k, ks, v, c.kv_heads * c.head_dim, out, cos, sin, rope, heads, dtype, None)


BAD_CACHES = [
    (dict(pool=None), ARG), (dict(page_table=None), ARG), (dict(prefix=None), ARG), (dict(head_dim=96), UNSUPPORTED),
    (dict(head_dim=0), UNSUPPORTED), (dict(page_size=8), UNSUPPORTED), (dict(page_size=48), UNSUPPORTED),
    (dict(page_size=2048), UNSUPPORTED), (dict(page_size=0), UNSUPPORTED), (dict(batch=0), SHAPE),
    (dict(kv_heads=3), SHAPE), (dict(kv_heads=0), SHAPE), (dict(tokens=7), SHAPE), (dict(tokens=-4), SHAPE),
    (dict(tokens=1 << 31), SHAPE), (dict(num_pages=0), SHAPE), (dict(max_pages=0), SHAPE),
    (dict(max_pages=1 << 25), SHAPE), (dict(max_pages=(1 << 24) + 1), SHAPE), (dict(pool=P + 8), ALIGN), (dict(prefix=P + 2), ALIGN),
]


@pytest.mark.parametrize("bad,code", BAD_CACHES)
def test_bad_caches_are_refused_by_every_call(L, bad, code):
    c = _cache(**bad)
    assert _append(L, c) == code
    assert L.fitq_kv4_attention(c, P, 8 * 128, P, 8, 0, 2, 192, P, 1 << 30, None) == code
    if "kv_heads" not in bad or bad["kv_heads"] == 0:
        assert L.fitq_kv4_gather(c, P, P, 0, None) == code
    assert L.fitq_last_error().decode()


def test_append_refusals(L):
    c = _cache()
    assert _append(L, c, q=None) == ARG and _append(L, c, sin=None) == ARG
    assert L.fitq_kv4_append(None, P, 1024, P, 256, P, 256, P, P, P, 64, 8, 0, None) == ARG
    assert _append(L, c, dtype=2) == UNSUPPORTED
    assert _append(L, c, rope=0) == SHAPE
    assert _append(L, c, qs=1000) == SHAPE and _append(L, c, qs=1028) == SHAPE and _append(L, c, ks=248) == SHAPE
    assert _append(L, c, q=P, out=P, qs=2048) == ARG
    far = P + (1 << 20)
    assert _append(L, c, q=P, out=P + 2048, k=far, v=far) == ARG and _append(L, c, q=far, out=P + 16, k=far) == ARG
    assert _append(L, c, q=P + 2) == ALIGN and _append(L, c, cos=P + 4) == ALIGN
    assert _append(L, _cache(tokens=0)) == 0


def test_attention_refusals(L):
    def call(c, q=P, stride=1024, out=P, heads=8, dtype=0, max_new=2, max_len=192, ws=P, size=1 << 30):
        return L.fitq_kv4_attention(c, q, stride, out, heads, dtype, max_new, max_len, ws, size, None)

    c = _cache()
    assert call(c, out=None) == ARG and call(c, ws=None) == ARG
    assert call(c, dtype=2) == UNSUPPORTED
    assert call(c, max_new=0) == SHAPE and call(c, max_new=9) == SHAPE and call(c, max_new=1) == SHAPE
    assert call(c, max_len=0) == SHAPE and call(c, heads=7) == SHAPE
    assert call(c, stride=1020) == SHAPE and call(c, stride=512) == SHAPE
    assert call(c, q=P + 8) == ALIGN
    assert call(c, stride=1032) == ARG and call(c, out=P + 2048) == ARG and call(c, q=P + 2048) == ARG  # out over q
    assert call(_cache(tokens=0)) == 0
    wide = dict(tokens=1 << 28, batch=1, max_pages=1 << 20)
    assert call(_cache(**wide, kv_heads=8), heads=8 * 4096, stride=8 * 4096 * 128, max_new=1 << 28) == SHAPE
    if not torch.cuda.is_available():
        assert call(c, out=P + 65536) == NO_DEVICE
        assert call(_cache(**dict(wide, tokens=131072), kv_heads=1), max_new=131072, out=P + (1 << 30)) == NO_DEVICE
    assert L.fitq_kv4_attention_workspace(c, 8, 2, 192) > 0
    assert L.fitq_kv4_attention_workspace(c, 7, 2, 192) == 0
    assert L.fitq_kv4_attention_workspace(c, 8, 0, 192) == 0


def test_logprob_refusals(L):
    def fwd(z=P, dtype=0, ids=P, rows=4, vocab=100, stride=100, top=5, out=P):
        return L.fitq_token_logprobs(z, dtype, ids, rows, vocab, stride, top, out, P, P, P, P, None)

    def bwd(z=P, dtype=0, rows=4, vocab=100, stride=100, top=5, stats=P, g_top=P, top_ids=P, d=P + 4096):
        return L.fitq_token_logprobs_bwd(z, dtype, P, rows, vocab, stride, top, stats, P, top_ids, P, P, g_top, d, None)

    assert fwd(z=None) == ARG and fwd(ids=None) == ARG and fwd(out=None) == ARG
    assert fwd(dtype=3) == UNSUPPORTED and fwd(top=65) == UNSUPPORTED and fwd(top=-1) == UNSUPPORTED
    assert fwd(vocab=3, stride=3, top=4) == UNSUPPORTED
    assert fwd(rows=-1) == SHAPE and fwd(vocab=0) == SHAPE and fwd(stride=99) == SHAPE and fwd(vocab=1 << 24, stride=1 << 24) == SHAPE
    assert fwd(z=P + 1) == ALIGN and fwd(dtype=2, z=P + 2) == ALIGN and fwd(ids=P + 4) == ALIGN
    assert fwd(rows=0) == 0 and bwd(rows=0) == 0
    assert bwd(stats=None) == ARG and bwd(d=None) == ARG and bwd(top_ids=None) == ARG
    assert bwd(d=P) == ARG and bwd(d=P + 4 * 100 * 2 - 16) == ARG  # over the logits
    assert bwd(stride=104, d=P + 3 * 104 * 2) == ARG
    assert bwd(stride=128, d=P) == ARG and bwd(d=P + 4104) == ALIGN


def test_python_refusals():
    pool = torch.zeros(2, 1, 4, 18 * 128, dtype=torch.uint8)
    table, prefix = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    q = torch.zeros(1, 4, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="pool"):
        ops.kv4_attention(q, pool, table, prefix)
    with pytest.raises(ValueError, match="CUDA"):
        token_logprobs(torch.zeros(2, 8), torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="do not match"):
        token_logprobs(torch.zeros(2, 8), torch.zeros(3, dtype=torch.int64))


def test_struct_layout_matches_the_header(L):
    # five pointers and two int64 and five int32, as include/fitq.h declares them
    assert ctypes.sizeof(_lib.Kv4C) == 4 * 8 + 2 * 8 + 5 * 4 + 4


@pytest.mark.parametrize("dim", [64, 128])
def test_reference_layout_covers_a_block_once(dim):
    kb, vb, sh, pb = ref.offsets(dim)
    nibbles = torch.cat([(2 * kb + sh // 4).flatten(), (2 * vb + sh // 4).flatten()])
    assert torch.equal(nibbles.sort().values, torch.arange(32 * dim))
    params = torch.cat([pb.flatten(), pb.flatten() + dim // 64 * 4]).unique()
    assert torch.equal(params, torch.arange(16 * dim, 18 * dim, 4))


def test_reference_coding_rounds_half_to_even_and_keeps_constants():
    x = torch.zeros(1, 64)
    x[0, 0], x[0, 1], x[0, 2], x[0, 3] = 15.0, 0.5, 1.5, 2.5
    c, s, low = ref.code_group(x)
    assert float(s) == 1.0 and float(low) == 0.0 and c[0, :4].tolist() == [15, 0, 2, 2]
    assert torch.equal(ref.coded_values(torch.full((1, 64), 3.25)), torch.full((1, 64), 3.25))
