"""Functional ops over the C ABI: the QLoRA linear forward/backward, the NF4
GEMV, the raw tcgen05 GEMM and the LoRA optimizer step.  Device tensors in,
device tensors out; every call is asynchronous on the current CUDA stream.
"""
from __future__ import annotations

import contextlib
import ctypes
import functools
from typing import List, Optional, Sequence, Tuple

import torch
from torch.autograd import forward_ad

from . import _lib
from .nf4 import Nf4WeightCRef, QuantState


def _stream(dev) -> int:
    return torch.cuda.current_stream(dev).cuda_stream


def _raw_stream(index: int) -> int:
    """Handle of a device's current stream, without a Stream object (looked up at the
    call: torch builds without CUDA lack it)."""
    return torch._C._cuda_getCurrentRawStream(index)


def _bf16_2d(t: torch.Tensor, cols: int) -> torch.Tensor:
    t = t.reshape(-1, cols)
    if t.dtype != torch.bfloat16:
        t = t.to(torch.bfloat16)
    return t.contiguous()


def _workspace(nbytes: int, dev) -> torch.Tensor:
    return torch.empty(max(int(nbytes), 1), dtype=torch.uint8, device=dev)


def qlora_forward(x2: torch.Tensor, w: Nf4WeightCRef, lora_a: Optional[torch.Tensor],
                  lora_b: Optional[torch.Tensor], scale: float, y_add: Optional[torch.Tensor] = None,
                  want_t: bool = False, gemv: bool = False,
                  bias: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """y[M,N] = x.W^T + scale.(x.A^T).B^T (+ bias) (+ y_add).  x2: bf16 [M, K] contiguous.

    Returns (y, T) with T = x.A^T (bf16 [M, r]) when want_t."""
    L = _lib.load()
    m = x2.shape[0]
    n, k = w.c.n_out, w.c.k_in
    rank = 0 if lora_a is None else int(lora_a.shape[0])
    dev = x2.device
    y = torch.empty(m, n, dtype=torch.bfloat16, device=dev)
    t = torch.empty(m, rank, dtype=torch.bfloat16, device=dev) if (want_t and rank) else None
    a = None if lora_a is None else lora_a.detach().to(torch.float32).contiguous()
    b = None if lora_b is None else lora_b.detach().to(torch.float32).contiguous()
    if y_add is not None:
        y_add = _bf16_2d(y_add, n)
    if bias is not None:
        bias = bias.detach().to(torch.bfloat16).contiguous()
    with torch.cuda.device(dev):
        if gemv:
            nbytes = L.fitq_nf4_gemv_workspace(m, n, k, rank)
            ws = _workspace(nbytes, dev)
            _lib.check(L.fitq_nf4_gemv(w.ref, x2.data_ptr(), m, _lib.ptr(a), _lib.ptr(b), rank,
                                       float(scale), _lib.ptr(bias), y.data_ptr(), _lib.ptr(y_add),
                                       ws.data_ptr(),
                                       nbytes, _stream(dev)), "fitq_nf4_gemv")
        else:
            nbytes = L.fitq_qlora_fwd_workspace(m, n, k, rank)
            ws = _workspace(nbytes, dev)
            _lib.check(L.fitq_qlora_fwd(w.ref, x2.data_ptr(), m, _lib.ptr(a), _lib.ptr(b), rank,
                                        float(scale), _lib.ptr(bias), y.data_ptr(), _lib.ptr(y_add),
                                        _lib.ptr(t),
                                        ws.data_ptr(), nbytes, _stream(dev)), "fitq_qlora_fwd")
    return y, t


def qlora_backward(x2: Optional[torch.Tensor], dy2: torch.Tensor, w: Nf4WeightCRef,
                   lora_a: Optional[torch.Tensor], lora_b: Optional[torch.Tensor], scale: float,
                   t_saved: Optional[torch.Tensor] = None, need_dx: bool = True,
                   dx: Optional[torch.Tensor] = None, grad_a: Optional[torch.Tensor] = None,
                   grad_b: Optional[torch.Tensor] = None, grad_accumulate: bool = False):
    """(dx, grad_a, grad_b) of the QLoRA linear for upstream dy2 [M, N] bf16.

    dx: bf16 [M, K] (accumulated into when passed in); grads fp32 in the PEFT
    layouts [r, K] and [N, r] (accumulated into when grad_accumulate)."""
    L = _lib.load()
    m = dy2.shape[0]
    n, k = w.c.n_out, w.c.k_in
    rank = 0 if lora_a is None else int(lora_a.shape[0])
    dev = dy2.device
    dx_acc = dx is not None
    if need_dx and dx is None:
        dx = torch.empty(m, k, dtype=torch.bfloat16, device=dev)
    a = b = None
    if rank:
        a = lora_a.detach().to(torch.float32).contiguous()
        b = lora_b.detach().to(torch.float32).contiguous()
        if grad_a is None:
            grad_a = torch.empty(rank, k, dtype=torch.float32, device=dev)
            grad_b = torch.empty(n, rank, dtype=torch.float32, device=dev)
            grad_accumulate = False
    nbytes = L.fitq_qlora_bwd_workspace(m, n, k, rank)
    ws = _workspace(nbytes, dev)
    with torch.cuda.device(dev):
        _lib.check(L.fitq_qlora_bwd(w.ref, _lib.ptr(x2), dy2.data_ptr(), m, _lib.ptr(a), _lib.ptr(b),
                                    rank, float(scale), _lib.ptr(t_saved),
                                    _lib.ptr(dx) if need_dx else None, int(dx_acc),
                                    _lib.ptr(grad_a), _lib.ptr(grad_b), int(grad_accumulate),
                                    ws.data_ptr(), nbytes, _stream(dev)), "fitq_qlora_bwd")
    return (dx if need_dx else None), grad_a, grad_b


def _gemv_jobs(x2: torch.Tensor, jobs, with_y: bool):
    """The fitq_gemv_job array of (wref, lora_a, lora_b, scale, bias, y_add)
    tuples, the tensors it points at (kept alive by the caller) and, with
    with_y, the bf16 [M, N] outputs it writes."""
    m = x2.shape[0]
    dev = x2.device
    arr = (_lib.GemvJobC * len(jobs))()
    keep, outs = [], []
    for i, (wref, lora_a, lora_b, scale, bias, y_add) in enumerate(jobs):
        n = wref.c.n_out
        y = torch.empty(m, n, dtype=torch.bfloat16, device=dev) if with_y else None
        a = None if lora_a is None else lora_a.detach().to(torch.float32).contiguous()
        b = None if lora_b is None else lora_b.detach().to(torch.float32).contiguous()
        bb = None if bias is None else bias.detach().to(torch.bfloat16).contiguous()
        ya = None if y_add is None else _bf16_2d(y_add, n)
        keep += [a, b, bb, ya]
        arr[i].w = ctypes.pointer(wref.c)
        arr[i].lora_a, arr[i].lora_b = _lib.ptr(a), _lib.ptr(b)
        arr[i].rank = 0 if a is None else int(a.shape[0])
        arr[i].scale = float(scale)
        arr[i].bias, arr[i].y, arr[i].y_add = _lib.ptr(bb), _lib.ptr(y), _lib.ptr(ya)
        outs.append(y)
    return arr, keep, outs


def nf4_gemv_grouped(x2: torch.Tensor, jobs) -> List[torch.Tensor]:
    """Up to three projections of the same x2 [M, K] bf16 in one call
    (fitq_nf4_gemv_grouped).  jobs: (wref, lora_a, lora_b, scale, bias,
    y_add) per projection (None for absent parts).  Returns the bf16 [M, N]
    outputs, each fitq_nf4_gemv's result."""
    L = _lib.load()
    m = x2.shape[0]
    dev = x2.device
    arr, keep, outs = _gemv_jobs(x2, jobs, True)
    with torch.cuda.device(dev):
        nbytes = L.fitq_nf4_gemv_grouped_workspace(arr, len(jobs), m)
        ws = _workspace(nbytes, dev)
        _lib.check(L.fitq_nf4_gemv_grouped(arr, len(jobs), x2.data_ptr(), m, ws.data_ptr(), nbytes,
                                           _stream(dev)), "fitq_nf4_gemv_grouped")
    del keep
    return outs


def nf4_gemv_swiglu(x2: torch.Tensor, gate_job, up_job) -> torch.Tensor:
    """SiLU(x2.Wg^T) * (x2.Wu^T) as bf16 [M, N] (fitq_nf4_gemv_swiglu): the
    gate and up projections (rank 0) and the SwiGLU of their bf16 results."""
    L = _lib.load()
    m = x2.shape[0]
    dev = x2.device
    arr, keep, _ = _gemv_jobs(x2, [gate_job, up_job], False)
    act = torch.empty(m, gate_job[0].c.n_out, dtype=torch.bfloat16, device=dev)
    with torch.cuda.device(dev):
        nbytes = L.fitq_nf4_gemv_swiglu_workspace(arr, m)
        ws = _workspace(nbytes, dev)
        _lib.check(L.fitq_nf4_gemv_swiglu(arr, x2.data_ptr(), m, act.data_ptr(), ws.data_ptr(), nbytes,
                                          _stream(dev)), "fitq_nf4_gemv_swiglu")
    del keep
    return act


def nf4_gateup_swiglu(x2: torch.Tensor, w_gate: Nf4WeightCRef, w_up: Nf4WeightCRef,
                      keep_gate_up: bool = False):
    """act = silu(x.Wg^T) * (x.Wu^T) as ONE tcgen05 GEMM over both NF4 weights
    (fitq_nf4_gateup_swiglu).  x2: bf16 [M, K].  Returns (act, gate, up), bf16
    [M, N]; gate / up only with keep_gate_up (for the backward), else None."""
    L = _lib.load()
    m = x2.shape[0]
    n, k = w_gate.c.n_out, w_gate.c.k_in
    dev = x2.device
    act = torch.empty(m, n, dtype=torch.bfloat16, device=dev)
    gate = torch.empty_like(act) if keep_gate_up else None
    up = torch.empty_like(act) if keep_gate_up else None
    with torch.cuda.device(dev):
        nbytes = L.fitq_nf4_gateup_swiglu_workspace(m, n, k)
        ws = _workspace(nbytes, dev)
        _lib.check(L.fitq_nf4_gateup_swiglu(w_gate.ref, w_up.ref, x2.data_ptr(), m, act.data_ptr(),
                                            _lib.ptr(gate), _lib.ptr(up), ws.data_ptr(), nbytes,
                                            _stream(dev)), "fitq_nf4_gateup_swiglu")
    return act, gate, up


def nf4_down_dswiglu(dy2: torch.Tensor, w_down: Nf4WeightCRef, gate: torch.Tensor,
                     up: torch.Tensor):
    """(d_gate, d_up) of act = silu(gate) * up through down_proj: the dX GEMM of
    down_proj with the SwiGLU backward in its epilogue (fitq_nf4_down_dswiglu)."""
    L = _lib.load()
    m = dy2.shape[0]
    k = w_down.c.k_in
    dev = dy2.device
    d_gate = torch.empty(m, k, dtype=torch.bfloat16, device=dev)
    d_up = torch.empty_like(d_gate)
    with torch.cuda.device(dev):
        nbytes = L.fitq_nf4_down_dswiglu_workspace(m, w_down.c.n_out, k)
        ws = _workspace(nbytes, dev)
        _lib.check(L.fitq_nf4_down_dswiglu(w_down.ref, dy2.data_ptr(), m, gate.data_ptr(),
                                           up.data_ptr(), d_gate.data_ptr(), d_up.data_ptr(),
                                           ws.data_ptr(), nbytes, _stream(dev)),
                   "fitq_nf4_down_dswiglu")
    return d_gate, d_up


def verify_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                     prefix: int) -> torch.Tensor:
    """Attention of T new tokens over a KV cache (fitq_verify_attention).

    q: [B, T, H, D] bf16 (post-RoPE); k_cache, v_cache: [B, KVH, cap, D] bf16 with
    the new tokens' keys/values at [prefix, prefix + T).  Returns [B, T, H, D]
    bf16; token i attends to positions <= prefix + i."""
    L = _lib.load()
    b, t, h, d = q.shape
    kvh, cap = int(k_cache.shape[1]), int(k_cache.shape[2])
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError("verify_attention: caches must be contiguous [B, KVH, cap, D]")
    q = q.contiguous()
    out = torch.empty_like(q)
    dev = q.device
    with torch.cuda.device(dev):
        nbytes = L.fitq_verify_attention_workspace(b, h, kvh, t, prefix)
        ws = _workspace(nbytes, dev)
        _lib.check(L.fitq_verify_attention(q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
                                           out.data_ptr(), b, h, kvh, t, prefix, cap, d,
                                           ws.data_ptr(), nbytes, _stream(dev)),
                   "fitq_verify_attention")
    return out


_KV4_DTYPES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16}


def _kv4_cache(what: str, pool: torch.Tensor, page_table: torch.Tensor, prefix: torch.Tensor,
               q_start: Optional[torch.Tensor], tokens: int) -> _lib.Kv4C:
    """The fitq_kv4 descriptor of a call (its pointers live as long as the tensors)."""
    dev, shape, table = pool.device, pool.shape, page_table.shape
    if pool.dtype != torch.uint8 or len(shape) != 4 or not pool.is_contiguous() or not pool.is_cuda:
        raise ValueError(f"{what}: pool must be a contiguous uint8 CUDA tensor [pages, kv_heads, page_size / 16, "
                         "18 * head_dim]")
    pages, kv_heads, per_page, block = shape
    if block % 18:
        raise ValueError(f"{what}: pool blocks have {block} bytes, not 18 * head_dim")
    if page_table.dtype != torch.int32 or len(table) != 2 or not page_table.is_contiguous():
        raise ValueError(f"{what}: page_table must be contiguous int32 [batch, max_pages]")
    batch, max_pages = table
    if prefix.dtype != torch.int32 or prefix.shape != (batch,) or not prefix.is_contiguous():
        raise ValueError(f"{what}: prefix must be contiguous int32 [batch]")
    if page_table.device != dev or prefix.device != dev:
        raise ValueError(f"{what}: page_table is on {page_table.device}, prefix on {prefix.device}, the pool on {dev}")
    start = None
    if q_start is not None:
        if q_start.dtype != torch.int32 or q_start.shape != (batch + 1,) or not q_start.is_contiguous():
            raise ValueError(f"{what}: q_start must be contiguous int32 [batch + 1]")
        if q_start.device != dev:
            raise ValueError(f"{what}: q_start is on {q_start.device}, the pool on {dev}")
        start = q_start.data_ptr()
    return _lib.Kv4C(pool.data_ptr(), page_table.data_ptr(), prefix.data_ptr(), start, tokens, pages, batch, kv_heads,
                     block // 18, per_page * 16, max_pages)


def _kv4_tokens(what: str, name: str, t: torch.Tensor, heads: Optional[int], dim: int, like: torch.Tensor,
                dev) -> torch.Tensor:
    """t as [tokens, heads, dim] whose heads and elements are dense (tokens may be strided)."""
    shape = t.shape
    if len(shape) != 3 or shape[2] != dim or shape[0] != like.shape[0] or (heads is not None and shape[1] != heads):
        raise ValueError(f"{what}: {name} has shape {tuple(shape)}")
    if t.dtype not in _KV4_DTYPES or t.dtype != like.dtype:
        raise ValueError(f"{what}: {name} must be bf16 or fp16, all of one dtype (got {t.dtype})")
    if t.device != dev:
        raise ValueError(f"{what}: {name} is on {t.device}, the pool on {dev}")
    s0, s1, s2 = t.stride()
    if s2 != 1 or s1 != dim or s0 % 8 or s0 < shape[1] * dim or t.data_ptr() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
    return t


def _kv4_out(what: str, name: str, out: Optional[torch.Tensor], like: torch.Tensor) -> torch.Tensor:
    if out is None:
        return torch.empty_like(like, memory_format=torch.contiguous_format)
    if out.shape != like.shape or out.dtype != like.dtype or out.device != like.device or not out.is_contiguous():
        raise ValueError(f"{what}: {name} must be a contiguous {like.dtype} tensor {tuple(like.shape)} on {like.device}")
    return out


def _on(dev: torch.device):
    """torch.cuda.device(dev), or nothing where dev is current already (a decode
    step's calls are bound by the host)."""
    return _HERE if torch.cuda.current_device() == dev.index else torch.cuda.device(dev)


_HERE = contextlib.nullcontext()


def kv4_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, pool: torch.Tensor, page_table: torch.Tensor,
               prefix: torch.Tensor, cos_half: torch.Tensor, sin_half: torch.Tensor,
               q_start: Optional[torch.Tensor] = None, q_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rotate the new tokens' q and k and append k and v to a 4-bit paged cache
    (fitq_kv4_append).

    q [tokens, heads, D], k, v [tokens, kv_heads, D] bf16 or fp16 (the token
    stride is free); cos_half, sin_half fp32 [positions, D / 2], row = position.
    Returns the rotated q (into q_out when given; rows of no sequence are left
    as they are)."""
    L = _lib.load()
    dev = pool.device
    c = _kv4_cache("kv4_append", pool, page_table, prefix, q_start, q.shape[0])
    d, kvh = c.head_dim, c.kv_heads
    q = _kv4_tokens("kv4_append", "q", q, None, d, q, dev)
    k = _kv4_tokens("kv4_append", "k", k, kvh, d, q, dev)
    v = _kv4_tokens("kv4_append", "v", v, kvh, d, q, dev)
    rows = cos_half.shape
    if len(rows) != 2 or rows[1] * 2 != d or sin_half.shape != rows:
        raise ValueError(f"kv4_append: cos_half and sin_half must be of one shape [positions, {d // 2}]")
    for name, t in (("cos_half", cos_half), ("sin_half", sin_half)):
        if t.dtype != torch.float32 or not t.is_contiguous() or t.device != dev:
            raise ValueError(f"kv4_append: {name} must be contiguous fp32 on {dev}")
    out = _kv4_out("kv4_append", "q_out", q_out, q)
    with _on(dev):
        _lib.check(L.fitq_kv4_append(c, q.data_ptr(), q.stride(0), k.data_ptr(), k.stride(0), v.data_ptr(),
                                     v.stride(0), out.data_ptr(), cos_half.data_ptr(), sin_half.data_ptr(),
                                     rows[0], q.shape[1], _KV4_DTYPES[q.dtype], _raw_stream(dev.index)),
                   "fitq_kv4_append")
    return out


def kv4_gather(pool: torch.Tensor, page_table: torch.Tensor, prefix: torch.Tensor, tokens: int,
               q_start: Optional[torch.Tensor] = None,
               dtype: torch.dtype = torch.bfloat16) -> Tuple[torch.Tensor, torch.Tensor]:
    """(k, v) [tokens, kv_heads, D]: what a 4-bit paged cache holds at the positions
    kv4_append writes for the same prefix, tokens and q_start (fitq_kv4_gather)."""
    L = _lib.load()
    dev = pool.device
    c = _kv4_cache("kv4_gather", pool, page_table, prefix, q_start, int(tokens))
    if dtype not in _KV4_DTYPES:
        raise ValueError(f"kv4_gather: dtype must be bf16 or fp16 (got {dtype})")
    k = torch.empty(int(tokens), c.kv_heads, c.head_dim, dtype=dtype, device=dev)
    v = torch.empty_like(k)
    with _on(dev):
        _lib.check(L.fitq_kv4_gather(c, k.data_ptr(), v.data_ptr(), _KV4_DTYPES[dtype], _raw_stream(dev.index)),
                   "fitq_kv4_gather")
    return k, v


def kv4_attention(q: torch.Tensor, pool: torch.Tensor, page_table: torch.Tensor, prefix: torch.Tensor,
                  max_len: Optional[int] = None, q_start: Optional[torch.Tensor] = None,
                  max_new: Optional[int] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of the new tokens over a 4-bit paged cache (fitq_kv4_attention).

    q [tokens, heads, D] bf16 or fp16, rotated, its keys and values appended:
    token i of a sequence sees positions <= prefix + i.  max_new: the most new
    tokens of one sequence (needed with q_start); max_len: the most positions of
    one sequence, a hint for the grid and the scratch.  Returns [tokens, heads, D] (into out when
    given; rows of no sequence are left as they are)."""
    L = _lib.load()
    dev = pool.device
    c = _kv4_cache("kv4_attention", pool, page_table, prefix, q_start, q.shape[0])
    q = _kv4_tokens("kv4_attention", "q", q, None, c.head_dim, q, dev)
    if max_new is None:
        if q_start is not None:
            raise ValueError("kv4_attention: pass max_new with q_start")
        max_new = max(1, q.shape[0] // max(1, c.batch))
    if max_len is None:
        max_len = c.max_pages * c.page_size
    out = _kv4_out("kv4_attention", "out", out, q)
    with _on(dev):
        nbytes = L.fitq_kv4_attention_workspace(c, q.shape[1], max_new, max_len)
        ws = pool.new_empty(max(nbytes, 1))
        _lib.check(L.fitq_kv4_attention(c, q.data_ptr(), q.stride(0), out.data_ptr(), q.shape[1],
                                        _KV4_DTYPES[q.dtype], max_new, max_len, ws.data_ptr(), nbytes,
                                        _raw_stream(dev.index)), "fitq_kv4_attention")
    return out


def _serving_only(what: str) -> None:
    """Refuses a call that would lose its inputs' gradient."""
    raise NotImplementedError(f"{what}: an input requires a gradient, which this call does not have "
                              "(use torch.no_grad())")


def _refuse_tangents(what: str, *inputs: Optional[torch.Tensor]) -> None:
    """Refuses, inside a forward_ad.dual_level, inputs whose tangent a call would lose."""
    if any(x is not None and forward_ad.unpack_dual(x).tangent is not None for x in inputs):
        raise NotImplementedError(f"{what}: an input carries a tangent (there is no forward-mode derivative)")


@functools.lru_cache(maxsize=256)
def _tree_attention_workspace(cap: int, batch: int, t: int, kv_heads: int, d: int, heads: int, device: int) -> int:
    """fitq_tree_attention_workspace of the sizes, on a device's SMs."""
    c = _lib.TreeC(1 << 16, 1 << 16, 0, cap, d, d, d, batch, t, kv_heads, d, _lib.DTYPE_BF16)
    return _lib.load().fitq_tree_attention_workspace(c, heads)


def _tree_parents(what: str, parents: torch.Tensor, batch: int, t: int, dev) -> int:
    """Entries from sequence to sequence of parents int32 [batch, t], or 0 of [t]."""
    shape, strides = parents.shape, parents.stride()
    if parents.dtype != torch.int32 or (shape != (batch, t) and shape != (t,)) or (t > 1 and strides[-1] != 1):
        raise ValueError(f"{what}: parents must be int32 [{batch}, {t}] or [{t}] with dense rows (got {parents.dtype} "
                         f"{tuple(shape)})")
    if parents.device != dev:
        raise ValueError(f"{what}: parents is on {parents.device}, not on {dev}")
    if len(strides) == 1 or batch == 1:
        return 0
    if 0 < strides[0] < t:
        raise ValueError(f"{what}: rows of parents overlap")
    return strides[0]


def _tree_cache(what: str, k_cache: torch.Tensor, v_cache: torch.Tensor, prefix: torch.Tensor, parents: torch.Tensor,
                t: int) -> _lib.TreeC:
    """The fitq_tree descriptor of a call (its pointers live as long as the tensors)."""
    dev, shape, strides, dtype = k_cache.device, k_cache.shape, k_cache.stride(), _KV4_DTYPES.get(k_cache.dtype)
    if dtype is None or len(shape) != 4 or dev.type != "cuda":
        raise ValueError(f"{what}: caches must be bf16 or fp16 CUDA tensors [batch, kv_heads, capacity, head_dim]")
    if v_cache.shape != shape or v_cache.dtype != k_cache.dtype or v_cache.device != dev:
        raise ValueError(f"{what}: k_cache and v_cache differ in shape, dtype or device")
    batch, kv_heads, cap, d = shape
    if v_cache.stride() != strides:
        raise ValueError(f"{what}: k_cache and v_cache differ in strides")
    sb, sh, sp, one = strides
    if batch <= 1:
        sb = 0
    if kv_heads <= 1:
        sh = 0
    if cap <= 1:
        sp = d
    if one != 1 or sp < d or (sb | sh | sp) % 8 or (sb == 0 and batch > 1) or (sh == 0 and kv_heads > 1) \
            or (k_cache.data_ptr() | v_cache.data_ptr()) % 16:
        raise ValueError(f"{what}: caches need dense heads, strides in multiples of 8 elements and 16-byte alignment "
                         f"(got strides {strides})")
    if prefix.dtype != torch.int32 or prefix.shape != (batch,) or not prefix.is_contiguous() or prefix.device != dev:
        raise ValueError(f"{what}: prefix must be contiguous int32 [{batch}] on {dev}")
    ps = _tree_parents(what, parents, batch, t, dev)
    return _lib.TreeC(parents.data_ptr(), prefix.data_ptr(), ps, cap, sb, sh, sp, batch, t, kv_heads, d, dtype)


def _tree_tokens(what: str, name: str, x: torch.Tensor, heads: Optional[int], c: _lib.TreeC,
                 cache: torch.Tensor) -> Tuple[torch.Tensor, int]:
    """x [batch, t, heads, head_dim] whose tokens follow one another at one stride, heads dense, and
    that stride."""
    shape, d, t = x.shape, c.head_dim, c.tokens
    if len(shape) != 4 or shape[0] != c.batch or shape[1] != t or shape[3] != d or shape[2] == 0 \
            or (heads is not None and shape[2] != heads):
        raise ValueError(f"{what}: {name} has shape {tuple(shape)}")
    if x.dtype != cache.dtype or x.device != cache.device:
        raise ValueError(f"{what}: {name} must be {cache.dtype} on {cache.device} like the caches (got {x.dtype} on "
                         f"{x.device})")
    row = shape[2] * d
    if x.is_contiguous() and x.data_ptr() % 16 == 0:
        return x, row
    s0, s1, s2, s3 = x.stride()
    if t == 1:
        s1 = s0 if shape[0] > 1 else row
    if s3 != 1 or s2 != d or s1 % 8 or s1 < row or (shape[0] > 1 and s0 != t * s1) or x.data_ptr() % 16:
        return x.clone(memory_format=torch.contiguous_format), row
    return x, s1


def _holds(x: torch.Tensor, lo: int, hi: int) -> bool:
    """Whether bytes [lo, hi) from a tensor's first element on hold one of its own."""
    size = x.element_size()
    dims = sorted(((s * size, n) for n, s in zip(x.shape, x.stride()) if n > 1), reverse=True)
    inner = [size]
    for s, n in reversed(dims):
        inner.append(inner[-1] + (n - 1) * s)
    inner.reverse()

    def meets(lo, hi, i):
        if hi <= 0 or lo >= inner[i]:
            return False
        if i == len(dims):
            return True
        s, n = dims[i]
        first, last = max(0, -(-(lo - inner[i + 1] + 1) // s)), min((hi - 1) // s, n - 1)
        return last - first > 64 or any(meets(lo - d * s, hi - d * s, i + 1) for d in range(first, last + 1))

    return meets(lo, hi, 0)


def _result_beside(what: str, name: str, out: torch.Tensor, *inputs: torch.Tensor) -> None:
    """Raises where a contiguous result lies over an input that other rows still read."""
    nbytes = out.numel() * out.element_size()
    for x in inputs:
        at = out.data_ptr() - x.data_ptr()
        if _holds(x, at, at + nbytes):
            raise ValueError(f"{what}: {name} overlaps an input")


def tree_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                prefix: torch.Tensor, parents: torch.Tensor, cos_half: torch.Tensor, sin_half: torch.Tensor,
                q_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rotate a tree's q and k and write its k and v to the cache (fitq_tree_append).

    q [B, T, heads, D], k, v [B, T, kv_heads, D] and the caches [B, kv_heads, capacity, D]
    of one dtype (bf16 or fp16; tokens and caches may be strided); prefix int32 [B]: cached
    positions; parents int32 [B, T] or [T]: a token's parent, -1 for one right behind the
    cached positions, -2 for no token.  Token i goes to slot prefix + i and is rotated at
    position prefix + depth with row prefix + depth of cos_half, sin_half fp32 [positions,
    D / 2].  Returns the rotated q [B, T, heads, D] (into q_out when given; absent tokens: zeros)."""
    L = _lib.load()
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or k_cache.requires_grad
                                    or v_cache.requires_grad):
        _serving_only("tree_append")
    if forward_ad._current_level >= 0:
        _refuse_tangents("tree_append", q, k, v, k_cache, v_cache)
    c = _tree_cache("tree_append", k_cache, v_cache, prefix, parents, q.shape[1] if q.dim() == 4 else 0)
    dev = k_cache.device
    q, qs = _tree_tokens("tree_append", "q", q, None, c, k_cache)
    k, ks = _tree_tokens("tree_append", "k", k, c.kv_heads, c, k_cache)
    v, vs = _tree_tokens("tree_append", "v", v, c.kv_heads, c, k_cache)
    rows = cos_half.shape
    if len(rows) != 2 or rows[1] * 2 != c.head_dim or sin_half.shape != rows:
        raise ValueError(f"tree_append: cos_half and sin_half must be of one shape [positions, {c.head_dim // 2}]")
    if cos_half.dtype != torch.float32 or sin_half.dtype != torch.float32 or cos_half.device != dev \
            or sin_half.device != dev or not cos_half.is_contiguous() or not sin_half.is_contiguous() \
            or (cos_half.data_ptr() | sin_half.data_ptr()) % 16:
        raise ValueError(f"tree_append: cos_half and sin_half must be contiguous, 16-byte aligned fp32 on {dev}")
    out = q.new_empty(q.shape) if q_out is None else _kv4_out("tree_append", "q_out", q_out, q)
    if q_out is not None:
        _result_beside("tree_append", "q_out", out, k_cache, v_cache)
    with _on(dev):
        _lib.check(L.fitq_tree_append(c, q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs, out.data_ptr(),
                                      k_cache.data_ptr(), v_cache.data_ptr(), cos_half.data_ptr(), sin_half.data_ptr(), rows[0], q.shape[2],
                                      _raw_stream(dev.index)), "fitq_tree_append")
    return out


def tree_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, prefix: torch.Tensor,
                   parents: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of a tree of drafted tokens over a cache (fitq_tree_attention).

    q [B, T, heads, D], rotated, the tree's keys and values in the cache's slots
    [prefix, prefix + T) (tree_append; arguments as there): token i sees the cached
    positions, its ancestors and itself.  Returns [B, T, heads, D] (into out when given;
    absent tokens: zeros)."""
    L = _lib.load()
    if torch.is_grad_enabled() and (q.requires_grad or k_cache.requires_grad or v_cache.requires_grad):
        _serving_only("tree_attention")
    if forward_ad._current_level >= 0:
        _refuse_tangents("tree_attention", q, k_cache, v_cache)
    c = _tree_cache("tree_attention", k_cache, v_cache, prefix, parents, q.shape[1] if q.dim() == 4 else 0)
    dev = k_cache.device
    q, qs = _tree_tokens("tree_attention", "q", q, None, c, k_cache)
    if out is None:
        out = q.new_empty(q.shape)
    else:
        _result_beside("tree_attention", "out", _kv4_out("tree_attention", "out", out, q), k_cache, v_cache)
    heads = q.shape[2]
    with _on(dev):
        nbytes = _tree_attention_workspace(c.capacity, c.batch, c.tokens, c.kv_heads, c.head_dim, heads, dev.index)
        ws = prefix.new_empty(nbytes // 4 + 1)
        _lib.check(L.fitq_tree_attention(c, q.data_ptr(), qs, k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(),
                                         heads, ws.data_ptr(), nbytes, _raw_stream(dev.index)), "fitq_tree_attention")
    return out


def tree_keep(k_caches: Sequence[torch.Tensor], v_caches: Sequence[torch.Tensor], prefix: torch.Tensor,
              path: torch.Tensor, accepted: torch.Tensor, lengths: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The accepted path of a tree stays in the caches of all layers (fitq_tree_keep): slot
    prefix + path[b, i] moves to prefix + i for i <= accepted[b].  path int32 [B, T], accepted
    int64 [B] as verify.verify_tree gives them.  Returns prefix + accepted + 1 as int32 [B] (into
    lengths when given, which may be prefix)."""
    L = _lib.load()
    if not k_caches or len(k_caches) != len(v_caches):
        raise ValueError(f"tree_keep: {len(k_caches)} key and {len(v_caches)} value caches")
    if torch.is_grad_enabled() and any(x.requires_grad for x in (*k_caches, *v_caches)):
        _serving_only("tree_keep")
    if forward_ad._current_level >= 0:
        _refuse_tangents("tree_keep", *k_caches, *v_caches)
    first = k_caches[0]
    if path.dim() != 2 or path.dtype != torch.int32 or not path.is_contiguous() or path.device != first.device \
            or path.shape[0] != first.shape[0]:
        raise ValueError("tree_keep: path must be contiguous int32 [batch, T] on the caches' device")
    batch, t = path.shape
    if accepted.dtype != torch.int64 or accepted.shape != (batch,) or not accepted.is_contiguous() \
            or accepted.device != first.device:
        raise ValueError(f"tree_keep: accepted must be contiguous int64 [{batch}] on the caches' device")
    c = _tree_cache("tree_keep", first, v_caches[0], prefix, path, t)
    shape, strides, dtype, dev = first.shape, first.stride(), first.dtype, first.device
    for x in (*k_caches, *v_caches):
        if x.shape != shape or x.stride() != strides or x.dtype != dtype or x.device != dev:
            raise ValueError("tree_keep: the layers' caches must be of one shape, stride, dtype and device")
    if lengths is None:
        lengths = torch.empty_like(prefix)
    elif lengths.dtype != torch.int32 or lengths.shape != (batch,) or not lengths.is_contiguous() \
            or lengths.device != first.device:
        raise ValueError(f"tree_keep: lengths must be contiguous int32 [{batch}] on the caches' device")
    n = len(k_caches)
    array = ctypes.c_void_p * n
    with _on(first.device):
        _lib.check(L.fitq_tree_keep(c, array(*[x.data_ptr() for x in k_caches]), array(*[x.data_ptr() for x in v_caches]),
                                    n, path.data_ptr(), accepted.data_ptr(), lengths.data_ptr(),
                                    _raw_stream(first.device.index)), "fitq_tree_keep")
    return lengths


def _lora_rows(x: torch.Tensor, rows: int, cols: int) -> Tuple[torch.Tensor, int]:
    """x [rows, cols] with dense, aligned rows (the row stride is free), and that stride."""
    s0, s1 = x.stride()
    if rows <= 1:
        s0 = cols
    if s1 != 1 or s0 % 8 or s0 < cols or x.data_ptr() % 16:
        return x.clone(memory_format=torch.contiguous_format), cols
    return x, s0


def multi_lora(x: torch.Tensor, lora_a: torch.Tensor, lora_b: torch.Tensor, scale: torch.Tensor, adapter: torch.Tensor,
               y: torch.Tensor, q_start: Optional[torch.Tensor] = None,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Adapters of many requests beside a shared projection (fitq_multi_lora):
    y[n] + scale[l] (x[n].A_l^T).B_l^T with l = adapter[sequence of token n].

    x [tokens, K], y [tokens, N] (the shared projection of x; rows may be strided), lora_a
    [adapters, R, K], lora_b [adapters, N, R], all bf16 or all fp16, R 16, 32, 48 or 64;
    scale fp32 [adapters]; adapter int32 [batch], -1 for none; q_start int32 [batch + 1]
    (sequence b has the tokens [q_start[b], q_start[b + 1])), or None for tokens / batch
    each.  Returns [tokens, N] (into out when given, which may be y; rows of no sequence
    are left as they are there)."""
    L = _lib.load()
    if torch.is_grad_enabled() and (x.requires_grad or y.requires_grad or lora_a.requires_grad or lora_b.requires_grad
                                    or scale.requires_grad):
        _serving_only("multi_lora")
    if forward_ad._current_level >= 0:
        _refuse_tangents("multi_lora", x, y, lora_a, lora_b, scale)
    xs, ys, sa, sb = x.shape, y.shape, lora_a.shape, lora_b.shape
    if len(xs) != 2 or len(ys) != 2 or len(sa) != 3 or len(sb) != 3:
        raise ValueError("multi_lora: x and y are [tokens, .], lora_a and lora_b [adapters, ., .]")
    tokens, k = xs
    n, dev, dtype = ys[1], x.device, x.dtype
    n_ad, r, _ = sa
    if sa[2] != k or sb[0] != n_ad or sb[1] != n or sb[2] != r or ys[0] != tokens:
        raise ValueError(f"multi_lora: x {tuple(xs)}, y {tuple(ys)}, lora_a {tuple(sa)} and lora_b {tuple(sb)} do not match")
    code = _KV4_DTYPES.get(dtype)
    if code is None or dev.type != "cuda":
        raise ValueError("multi_lora: x must be a bf16 or fp16 CUDA tensor")
    if y.dtype != dtype or lora_a.dtype != dtype or lora_b.dtype != dtype or y.device != dev or lora_a.device != dev \
            or lora_b.device != dev:
        raise ValueError(f"multi_lora: y, lora_a and lora_b must be {dtype} on {dev} (got {y.dtype}, {lora_a.dtype}, "
                         f"{lora_b.dtype} on {y.device}, {lora_a.device}, {lora_b.device})")
    if not (lora_a.is_contiguous() and lora_b.is_contiguous()):
        raise ValueError("multi_lora: lora_a and lora_b must be contiguous")
    if scale.dtype != torch.float32 or scale.shape != (n_ad,) or not scale.is_contiguous() or scale.device != dev:
        raise ValueError(f"multi_lora: scale must be contiguous fp32 [{n_ad}] on {dev}")
    ad = adapter.shape
    if adapter.dtype != torch.int32 or len(ad) != 1 or not adapter.is_contiguous() or adapter.device != dev:
        raise ValueError(f"multi_lora: adapter must be contiguous int32 [batch] on {dev}")
    batch, start = ad[0], None
    if q_start is not None:
        if q_start.dtype != torch.int32 or q_start.shape != (batch + 1,) or not q_start.is_contiguous() \
                or q_start.device != dev:
            raise ValueError(f"multi_lora: q_start must be contiguous int32 [{batch + 1}] on {dev}")
        start = q_start.data_ptr()
    if out is None:
        out = x.new_empty((tokens, n))
    elif out.shape != (tokens, n) or out.dtype != dtype or out.device != dev or not out.is_contiguous():
        raise ValueError(f"multi_lora: out must be a contiguous {dtype} tensor {(tokens, n)} on {dev}")
    x, x_stride = _lora_rows(x, tokens, k)
    y, y_stride = _lora_rows(y, tokens, n)
    with _on(dev):
        ws = scale.new_empty(tokens * r)  # fitq_multi_lora_workspace: x.A^T
        _lib.check(L.fitq_multi_lora(x.data_ptr(), x_stride, tokens, k, n, lora_a.data_ptr(), lora_b.data_ptr(), r, n_ad,
                                     scale.data_ptr(), adapter.data_ptr(), start, batch, y.data_ptr(), y_stride,
                                     out.data_ptr(), code, ws.data_ptr(), tokens * r * 4, _raw_stream(dev.index)),
                   "fitq_multi_lora")
    return out


def gemm_bf16_tn(a: torch.Tensor, b: torch.Tensor, c_add: Optional[torch.Tensor] = None) -> torch.Tensor:
    """c = a.b^T (+ c_add) on the tcgen05 tensor cores (bf16 in/out, fp32 accumulate)."""
    L = _lib.load()
    a = a.contiguous()
    b = b.contiguous()
    m, k = a.shape
    n = b.shape[0]
    c = torch.empty(m, n, dtype=torch.bfloat16, device=a.device)
    with torch.cuda.device(a.device):
        _lib.check(L.fitq_gemm_bf16_tn(a.data_ptr(), b.data_ptr(), c.data_ptr(),
                                       _lib.ptr(None if c_add is None else c_add.contiguous()),
                                       m, n, k, _stream(a.device)), "fitq_gemm_bf16_tn")
    return c


def adamw_step(param: torch.Tensor, grad: torch.Tensor, exp_avg: torch.Tensor,
               exp_avg_sq: torch.Tensor, step: int, lr: float, beta1: float, beta2: float,
               eps: float, weight_decay: float, clip: Optional[torch.Tensor] = None) -> None:
    """In-place AdamW on flat fp32 CUDA buffers (fitllm/optimizer.py:206-231 order)."""
    L = _lib.load()
    with torch.cuda.device(param.device):
        _lib.check(L.fitq_adamw_step(param.data_ptr(), grad.data_ptr(), exp_avg.data_ptr(),
                                     exp_avg_sq.data_ptr(), param.numel(), lr, beta1, beta2, eps,
                                     weight_decay, int(step), _lib.ptr(clip),
                                     _stream(param.device)), "fitq_adamw_step")


def grad_clip_coef(flat_grads: torch.Tensor, max_norm: float) -> torch.Tensor:
    """Device fp32 [2] = (global L2 norm, clip coefficient) of a flat fp32 buffer."""
    L = _lib.load()
    out = torch.empty(2, dtype=torch.float32, device=flat_grads.device)
    nbytes = L.fitq_grad_norm_workspace(flat_grads.numel())
    ws = _workspace(nbytes, flat_grads.device)
    with torch.cuda.device(flat_grads.device):
        _lib.check(L.fitq_grad_clip_coef(flat_grads.data_ptr(), flat_grads.numel(), float(max_norm),
                                         out.data_ptr(), ws.data_ptr(), nbytes,
                                         _stream(flat_grads.device)), "fitq_grad_clip_coef")
    return out


def device_status(reset: bool = True) -> int:
    """Synchronise the current stream and return the library's device status word."""
    L = _lib.load()
    return int(L.fitq_get_device_status(int(reset), torch.cuda.current_stream().cuda_stream))
