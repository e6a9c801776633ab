"""KV-cached speculative-verify forward over NF4 QLoRA layers.

FitLLM verifies draft tokens by re-running the full prefix through the model
(fitllm/inference.py:380-397, the prefill path of fitllm/forward.py:547-655).
This module runs the same layers over a key/value cache instead: each verify
step feeds only the draft + 1 new tokens of every sequence (batch B, T tokens
each), so every projection is a skinny NF4 GEMM with M = B * T rows (the
decode kernels of this library), attention reads the cached prefix, and the
new keys/values are written into the cache at positions [P, P + T).

The layer arithmetic is DecoderLayer's (fitllm_b200/layer.py): RMSNorm, q/k/v
with bias, rotary embedding at the tokens' absolute positions, grouped-query
attention (causal within the new tokens, full over the prefix), o_proj with
the residual fused, RMSNorm, SwiGLU MLP with the residual fused.

Attention runs on the library's split-KV kernel (fitq_verify_attention) when
head_dim is 128 and (heads / kv_heads) * T <= 32 -- every verify step of the
Qwen2.5 shapes; other shapes (e.g. filling a cache with a long prompt) use
torch's scaled_dot_product_attention with the prefix + causal mask.

``PagedKVCache`` is the same step over a cache in 4 bits and in pages: 4.5 bits
an element instead of 16, sequences of different lengths in one batch, pages
handed out as sequences grow.  ``verify_pass`` takes either cache; with a paged
one the rotation, the coding and the append are one launch (fitq_kv4_append)
and attention reads the codes (fitq_kv4_attention) for single tokens, drafts and
prompts alike.  ``score_drafts`` turns the pass's hidden states into the drafts'
log probabilities, the model's alternatives and the number of drafts it accepts.

``TreeKVCache`` is the step for trees of drafted tokens: a bf16 cache whose lengths
live on the device.  ``tree_pass`` runs the layers over a tree per sequence (ops.tree_append,
ops.tree_attention), ``verify_tree`` accepts drafts against the model's probabilities by
given random numbers, and ``TreeKVCache.keep`` leaves the accepted path in the cache.
"""
from __future__ import annotations

from typing import List, NamedTuple, Optional, Sequence, Tuple

import torch
import torch.nn.functional as F

from . import _lib, ops
from .layer import DecoderLayer, rotary_tables
from .layer_ops import rope_kv_append, swiglu
from .lm_head import _LOGIT_DTYPES, LMHeadLoss, token_logprobs
from .qlora import Linear4bit, grouped_forward, swiglu_forward


class KVCache:
    """Per-layer key/value cache [B, kv_heads, capacity, head_dim] (bf16)."""

    def __init__(self, num_layers: int, batch: int, kv_heads: int, head_dim: int, capacity: int,
                 device, dtype=torch.bfloat16):
        shape = (batch, kv_heads, capacity, head_dim)
        self.k = [torch.zeros(shape, device=device, dtype=dtype) for _ in range(num_layers)]
        self.v = [torch.zeros(shape, device=device, dtype=dtype) for _ in range(num_layers)]
        self.capacity = capacity

    def fill_random_(self, length: int, seed: int = 0) -> None:
        """Seeded N(0, 1) prefix of `length` positions (a synthetic context)."""
        g = torch.Generator(device=self.k[0].device).manual_seed(seed)
        for k, v in zip(self.k, self.v):
            k[:, :, :length].normal_(generator=g)
            v[:, :, :length].normal_(generator=g)

    def bytes_read(self, length: int) -> int:
        """K and V bytes one verify pass reads over `length` cached positions."""
        b, h, _, d = self.k[0].shape
        return 2 * len(self.k) * b * h * length * d * self.k[0].element_size()


class PagedKVCache:
    """Per-layer key/value cache in 4 bits and in pages (the layout of
    include/fitq.h's fitq_kv4): pools [num_pages, kv_heads, page_size / 16,
    18 * head_dim] uint8, one page table for all layers.

    The host keeps the sequences' lengths and hands pages out (``reserve``); the
    device sees them as ``page_table`` and ``prefix``.  ``verify_pass`` writes the
    new tokens behind ``lengths`` without moving it: ``advance`` accepts them,
    so that rejected drafts are overwritten by the next pass.  Positions are accepted
    as far as they were reserved, by a pass or, for passes that are captured and
    replayed, by ``reserve`` beforehand.  capacity: the most
    positions of one sequence; num_pages: pages shared by all sequences (default:
    enough for every sequence at capacity); rope_theta: the layers' rotary base (a
    pass refuses layers of another one, whose rotation is not the tables')."""

    def __init__(self, num_layers: int, batch: int, kv_heads: int, head_dim: int, capacity: int, device,
                 page_size: int = 64, num_pages: Optional[int] = None, rope_theta: float = 1e6):
        if head_dim not in (64, 128):
            raise ValueError(f"PagedKVCache: head_dim must be 64 or 128 (got {head_dim})")
        if page_size not in (16, 32, 64, 128, 256, 512, 1024):
            raise ValueError(f"PagedKVCache: page_size must be a power of two in 16..1024 (got {page_size})")
        self.page_size, self.capacity, self.rope_theta = page_size, capacity, rope_theta
        max_pages = -(-capacity // page_size)
        num_pages = batch * max_pages if num_pages is None else num_pages
        shape = (num_pages, kv_heads, page_size // 16, 18 * head_dim)
        self.pools = [torch.zeros(shape, dtype=torch.uint8, device=device) for _ in range(num_layers)]
        self.page_table = torch.full((batch, max_pages), -1, dtype=torch.int32, device=device)
        self.prefix = torch.zeros(batch, dtype=torch.int32, device=device)
        self.tables = rotary_tables(max_pages * page_size, head_dim, rope_theta, device)
        self.lengths = [0] * batch
        self._reserved = [0] * batch  # positions of each sequence that advance may accept
        self._pages: List[List[int]] = [[] for _ in range(batch)]
        self._free = list(range(num_pages - 1, -1, -1))

    @property
    def batch(self) -> int:
        return len(self.lengths)

    def check_rotary(self, layer: DecoderLayer) -> None:
        """Raises where the layer rotates with another base than the cache's tables."""
        if layer.cfg.rope_theta != self.rope_theta:
            raise ValueError(f"PagedKVCache: the layer's rope_theta is {layer.cfg.rope_theta:g}, the cache's "
                             f"{self.rope_theta:g}")

    def reserve(self, counts: Sequence[int]) -> None:
        """Pages for counts[b] more positions of every sequence; raises, and changes
        nothing, where the capacity or the pages do not suffice."""
        if len(counts) != self.batch:
            raise ValueError(f"reserve: {len(counts)} counts for {self.batch} sequences")
        need = []
        for b, (n, c) in enumerate(zip(self.lengths, counts)):
            if c < 0 or n + c > self.capacity:
                raise ValueError(f"reserve: sequence {b} has {n} positions, {c} more exceed its capacity "
                                 f"{self.capacity}")
            need.append(max(0, -(-(n + c) // self.page_size) - len(self._pages[b])))
        if sum(need) > len(self._free):
            raise RuntimeError(f"reserve: {sum(need)} pages needed, {len(self._free)} free")
        for b, n in enumerate(need):
            self._reserved[b] = max(self._reserved[b], self.lengths[b] + int(counts[b]))
            if n:
                fresh = [self._free.pop() for _ in range(n)]
                at = len(self._pages[b])
                self._pages[b] += fresh
                self.page_table[b, at:at + n] = torch.tensor(fresh, dtype=torch.int32)

    def advance(self, counts: Sequence[int]) -> None:
        """The first counts[b] positions written behind sequence b's length stay; raises, and
        changes nothing, where they were not reserved."""
        if len(counts) != self.batch:
            raise ValueError(f"advance: {len(counts)} counts for {self.batch} sequences")
        for b, c in enumerate(counts):
            if c < 0 or self.lengths[b] + c > self._reserved[b]:
                raise ValueError(f"advance: sequence {b} has no {c} positions behind {self.lengths[b]}")
        self.lengths = [n + int(c) for n, c in zip(self.lengths, counts)]
        self.prefix.copy_(torch.tensor(self.lengths, dtype=torch.int32))

    def release(self, b: int) -> None:
        """Sequence b is done: its pages are free, its length 0."""
        self._free += reversed(self._pages[b])
        self._pages[b] = []
        self.page_table[b].fill_(-1)
        self.lengths[b] = self._reserved[b] = 0
        self.prefix[b] = 0

    def read(self, layer: int, b: int) -> Tuple[torch.Tensor, torch.Tensor]:
        """(k, v) bf16 [lengths[b], kv_heads, head_dim]: what the cache holds of a sequence."""
        n = self.lengths[b]
        zero = torch.zeros(1, dtype=torch.int32, device=self.prefix.device)
        return ops.kv4_gather(self.pools[layer], self.page_table[b:b + 1], zero, n)

    def bytes_read(self, length: int) -> int:
        """K and V bytes one verify pass reads over `length` cached positions of every sequence."""
        _, h, _, block = self.pools[0].shape
        return len(self.pools) * self.batch * h * length * block // 16


def verify_mask(prefix: int, t: int, device) -> torch.Tensor:
    """[t, prefix + t] boolean: new token i sees the prefix and new tokens <= i."""
    cols = torch.arange(prefix + t, device=device)
    rows = torch.arange(t, device=device)
    return cols[None, :] <= (prefix + rows)[:, None]


def kernel_attention_ok(cfg, t: int) -> bool:
    """Shapes fitq_verify_attention covers: head_dim 128, (heads / kv_heads) * t <= 32."""
    return cfg.head_dim == 128 and (cfg.heads // cfg.kv_heads) * t <= 32


def _layer_forward(layer: DecoderLayer, h: torch.Tensor, attend) -> torch.Tensor:
    """One layer over the new tokens h [B, T, hidden]; attend maps the q, k and v
    projections to the attention output [B, T, heads * head_dim]."""
    b, t, _ = h.shape
    attn = layer.self_attn
    x = layer.input_layernorm(h)
    grouped = b * t <= 64  # the skinny GEMM path: q/k/v (and gate/up) as one launch each
    if grouped:
        q_raw, k_raw, v_raw = grouped_forward([attn.q_proj, attn.k_proj, attn.v_proj], x)
    else:
        q_raw, k_raw, v_raw = attn.q_proj(x), attn.k_proj(x), attn.v_proj(x)
    h1 = attn.o_proj(attend(q_raw, k_raw, v_raw), residual=h)
    mlp = layer.mlp
    x2 = layer.post_attention_layernorm(h1)
    if grouped and isinstance(mlp.gate_proj, Linear4bit) and isinstance(mlp.up_proj, Linear4bit):
        act = swiglu_forward(mlp.gate_proj, mlp.up_proj, x2)  # gate/up/SwiGLU, one GEMM + one finish
    else:
        gate, up = grouped_forward([mlp.gate_proj, mlp.up_proj], x2) if grouped else (
            mlp.gate_proj(x2), mlp.up_proj(x2))
        act = swiglu(gate, up)
    return mlp.down_proj(act, residual=h1)


def verify_layer_forward(layer: DecoderLayer, h: torch.Tensor, k_cache: torch.Tensor,
                         v_cache: torch.Tensor, prefix: int, tables: Tuple[torch.Tensor, torch.Tensor],
                         mask: torch.Tensor) -> torch.Tensor:
    """One layer over the T new tokens of each sequence.  h: [B, T, hidden]
    bf16; tables: fp32 rotary (cos, sin) half tables of positions
    [prefix, prefix + T); writes K/V of the new tokens into the caches."""
    cfg = layer.cfg
    b, t, _ = h.shape
    cos, sin = tables

    def attend(q_raw, k_raw, v_raw):
        # rotary embedding of q and k and the append of k, v to the caches: one launch
        q = rope_kv_append(q_raw, k_raw, v_raw, cos, sin, k_cache, v_cache, prefix, cfg.heads,
                           cfg.kv_heads)
        if kernel_attention_ok(cfg, t):
            o = ops.verify_attention(q, k_cache, v_cache, prefix)
        else:
            o = F.scaled_dot_product_attention(q.transpose(1, 2), k_cache[:, :, :prefix + t],
                                               v_cache[:, :, :prefix + t], attn_mask=mask,
                                               enable_gqa=True).transpose(1, 2)
        return o.reshape(b, t, cfg.heads * cfg.head_dim)

    return _layer_forward(layer, h, attend)


def paged_layer_forward(layer: DecoderLayer, h: torch.Tensor, pool: torch.Tensor, cache: PagedKVCache,
                        max_len: int, q_start: Optional[torch.Tensor] = None,
                        max_new: Optional[int] = None) -> torch.Tensor:
    """One layer over new tokens behind a paged cache: h [B, T, hidden] (T tokens of
    every sequence) or, with q_start int32 [batch + 1], [1, tokens, hidden] packed."""
    cache.check_rotary(layer)
    cfg = layer.cfg
    cos, sin = cache.tables

    def attend(q_raw, k_raw, v_raw):
        q, k, v = (x.reshape(-1, n, cfg.head_dim) for x, n in ((q_raw, cfg.heads), (k_raw, cfg.kv_heads),
                                                               (v_raw, cfg.kv_heads)))
        q = ops.kv4_append(q, k, v, pool, cache.page_table, cache.prefix, cos, sin, q_start=q_start)
        o = ops.kv4_attention(q, pool, cache.page_table, cache.prefix, max_len, q_start=q_start, max_new=max_new)
        return o.view(*h.shape[:2], cfg.heads * cfg.head_dim)

    return _layer_forward(layer, h, attend)


@torch.no_grad()
def paged_verify_pass(layers: List[DecoderLayer], h: torch.Tensor, cache: PagedKVCache,
                      counts: Optional[Sequence[int]] = None) -> torch.Tensor:
    """All layers over the new tokens behind ``cache.lengths``; returns the final hidden
    states.  h [B, T, hidden], or [1, sum(counts), hidden]: the sequences' new tokens one
    behind the other, counts[b] of sequence b.  Pages are reserved; lengths stay until
    ``cache.advance``."""
    if counts is None:
        if h.shape[0] != cache.batch:
            raise ValueError(f"paged_verify_pass: {h.shape[0]} sequences, the cache has {cache.batch}")
        news, q_start = [h.shape[1]] * cache.batch, None
    else:
        news = [int(c) for c in counts]
        if len(news) != cache.batch or h.shape[0] != 1 or h.shape[1] != sum(news):
            raise ValueError("paged_verify_pass: counts must name every sequence's tokens of h [1, tokens, hidden]")
        starts = [0]
        for c in news:
            starts.append(starts[-1] + c)
        q_start = torch.tensor(starts, dtype=torch.int32, device=h.device)
    if max(news) == 0:
        return h
    for layer in layers:
        cache.check_rotary(layer)
    cache.reserve(news)
    max_len = max(n + c for n, c in zip(cache.lengths, news))
    for i, layer in enumerate(layers):
        h = paged_layer_forward(layer, h, cache.pools[i], cache, max_len, q_start, max(news))
    return h


@torch.no_grad()
def verify_pass(layers: List[DecoderLayer], h: torch.Tensor, cache, prefix: Optional[int] = None) -> torch.Tensor:
    """All layers over the new tokens; returns the final hidden states.  cache: a
    KVCache with `prefix` positions, or a PagedKVCache, which knows its lengths."""
    if isinstance(cache, PagedKVCache):
        return paged_verify_pass(layers, h, cache)
    cfg = layers[0].cfg
    t = h.shape[1]
    pos = torch.arange(prefix, prefix + t, device=h.device)
    tables = rotary_tables(t, cfg.head_dim, cfg.rope_theta, h.device, position_ids=pos)
    mask = None if kernel_attention_ok(cfg, t) else verify_mask(prefix, t, h.device)
    for i, layer in enumerate(layers):
        h = verify_layer_forward(layer, h, cache.k[i], cache.v[i], prefix, tables, mask)
    return h


class DraftScores(NamedTuple):
    """Of T - 1 drafts per sequence: logp [B, T - 1] of each, entropy [B, T], top_logp and
    top_ids [B, T, top] of every row, accepted [B] (leading drafts that are the model's
    first choice) and next_token [B], its first choice behind them."""
    logp: torch.Tensor
    entropy: torch.Tensor
    top_logp: torch.Tensor
    top_ids: torch.Tensor
    accepted: torch.Tensor
    next_token: torch.Tensor


@torch.no_grad()
def score_drafts(head: LMHeadLoss, h: torch.Tensor, drafts: torch.Tensor, top: int = 1) -> DraftScores:
    """What a verify pass says about its drafts (the comparison of
    fitllm/inference.py:380-397, there a loop over the argmax of every position).

    h [B, T, hidden]: the pass's final hidden states, row i behind draft i - 1; drafts
    [B, T - 1] token ids.  One read of the logits gives everything."""
    b, t, _ = h.shape
    if drafts.shape != (b, t - 1):
        raise ValueError(f"score_drafts: drafts {tuple(drafts.shape)} do not match h {tuple(h.shape)}")
    ids = torch.cat([drafts.to(torch.int64), torch.full((b, 1), -1, dtype=torch.int64, device=h.device)], dim=1)
    r = token_logprobs(head.logits(h), ids, top=max(1, top))
    first = r.top_ids[..., 0]
    accepted = (first[:, :-1] == ids[:, :-1]).long().cumprod(dim=1).sum(dim=1)
    return DraftScores(r.logp[:, :-1], r.entropy, r.top_logp, r.top_ids, accepted,
                       first.gather(1, accepted[:, None])[:, 0])


class TreeVerdict(NamedTuple):
    """path int32 [B, T] (token 0 and the accepted drafts in order, then -1), accepted int64 [B]
    (how many drafts; -1 for a sequence without a token) and next_token int64 [B]."""
    path: torch.Tensor
    accepted: torch.Tensor
    next_token: torch.Tensor


def verify_tree(logits: torch.Tensor, tokens: torch.Tensor, parents: torch.Tensor, uniforms: torch.Tensor,
                draft_probs: Optional[torch.Tensor] = None, temperature=1.0) -> TreeVerdict:
    """Drafted tokens against the model's probabilities, from given random numbers
    (fitq_tree_verify): accepted and next tokens are a sample of softmax(logits /
    temperature), whatever was drafted.

    logits [B, T, V] bf16, fp16 or fp32 (rows may be strided), row i behind token i; tokens
    [B, T] integers; parents int32 [B, T] or [T] as in ops.tree_append (a chain: chain_parents);
    token 0, with parent -1, is the last one that is certain.  uniforms fp32 [B, T] in [0, 1).
    draft_probs [B, T - 1 or more, V]: row i the distribution that token i's children were
    drawn from; None where they are a model's choice.  temperature: a number, or fp32 [B]; 0
    takes the largest logit."""
    L = _lib.load()
    if logits.dim() != 3 or logits.dtype not in _LOGIT_DTYPES or not logits.is_cuda:
        raise ValueError("verify_tree: logits must be a bf16, fp16 or fp32 CUDA tensor [batch, T, vocab]")
    b, t, vocab = logits.shape
    dev = logits.device
    if tokens.shape != (b, t) or tokens.dtype.is_floating_point or tokens.dtype == torch.bool or tokens.device != dev:
        raise ValueError(f"verify_tree: tokens must be integers [{b}, {t}] on {dev}")
    if uniforms.shape != (b, t) or uniforms.dtype != torch.float32 or uniforms.device != dev:
        raise ValueError(f"verify_tree: uniforms must be fp32 [{b}, {t}] on {dev}")
    ps = ops._tree_parents("verify_tree", parents, b, t, dev)
    if (vocab > 1 and logits.stride(2) != 1) or (t > 1 and logits.stride(1) < vocab):
        logits = logits.contiguous()
    tokens, uniforms = tokens.to(torch.int64).contiguous(), uniforms.contiguous()
    q, qb, qt = None, 0, vocab
    if draft_probs is not None:
        shape = draft_probs.shape
        if len(shape) != 3 or shape[0] != b or shape[1] < t - 1 or shape[2] != vocab or draft_probs.device != dev \
                or not draft_probs.dtype.is_floating_point:
            raise ValueError(f"verify_tree: draft_probs must be [{b}, {t - 1}, {vocab}] on {dev}")
        q = draft_probs.detach().float()
        if (vocab > 1 and q.stride(2) != 1) or (shape[1] > 1 and q.stride(1) < vocab):
            q = q.contiguous()
        qb, qt = (q.stride(0) if b > 1 else 0), (q.stride(1) if shape[1] > 1 else vocab)
    temps, temp = None, 0.0
    if isinstance(temperature, torch.Tensor):
        if temperature.shape != (b,) or temperature.dtype != torch.float32 or temperature.device != dev:
            raise ValueError(f"verify_tree: temperature must be a number or fp32 [{b}] on {dev}")
        temps = temperature.contiguous()
    else:
        temp = float(temperature)
    r = TreeVerdict(parents.new_empty((b, t)), tokens.new_empty(b), tokens.new_empty(b))
    with ops._on(dev):
        _lib.check(L.fitq_tree_verify(logits.data_ptr(), _LOGIT_DTYPES[logits.dtype], logits.stride(0) if b > 1 else 0,
                                      logits.stride(1) if t > 1 else vocab, b, t, vocab, tokens.data_ptr(),
                                      parents.data_ptr(), ps, uniforms.data_ptr(), _lib.ptr(q), qb, qt, _lib.ptr(temps),
                                      temp, r.path.data_ptr(), r.accepted.data_ptr(), r.next_token.data_ptr(),
                                      ops._raw_stream(dev.index)), "fitq_tree_verify")
    return r


def chain_parents(t: int, device) -> torch.Tensor:
    """The tree of T tokens in a row: int32 [t], each the child of the one before."""
    return torch.arange(-1, t - 1, dtype=torch.int32, device=device)


class TreeKVCache(KVCache):
    """A KVCache (bf16) whose sequences have lengths of their own, on the device (``prefix`` int32
    [B]), for passes over trees of drafted tokens: ``tree_pass`` writes a tree's tokens behind
    the lengths without moving them, ``keep`` accepts a path (no copy to the host: a step of
    both can be captured and replayed).  rope_theta: the layers' rotary base (a pass refuses
    layers of another one)."""

    def __init__(self, num_layers: int, batch: int, kv_heads: int, head_dim: int, capacity: int, device,
                 dtype=torch.bfloat16, rope_theta: float = 1e6):
        if head_dim not in (64, 128):
            raise ValueError(f"TreeKVCache: head_dim must be 64 or 128 (got {head_dim})")
        if dtype != torch.bfloat16:  # what the layers' projections give, for prompts and trees alike
            raise ValueError(f"TreeKVCache: the passes write bf16 (got {dtype})")
        super().__init__(num_layers, batch, kv_heads, head_dim, capacity, device, dtype)
        self.rope_theta = rope_theta
        self.prefix = torch.zeros(batch, dtype=torch.int32, device=device)
        self.tables = rotary_tables(capacity, head_dim, rope_theta, device)

    @property
    def batch(self) -> int:
        return self.prefix.shape[0]

    def set_lengths(self, lengths: Sequence[int]) -> None:
        """The sequences' cached positions, e.g. behind a prompt that ``verify_pass`` wrote."""
        if len(lengths) != self.batch or any(not 0 <= n <= self.capacity for n in lengths):
            raise ValueError(f"set_lengths: {list(lengths)} for {self.batch} sequences of {self.capacity} positions")
        self.prefix.copy_(torch.tensor(lengths, dtype=torch.int32))

    def keep(self, verdict: TreeVerdict) -> None:
        """The verdict's path stays behind each sequence's length, in all layers."""
        ops.tree_keep(self.k, self.v, self.prefix, verdict.path, verdict.accepted, lengths=self.prefix)

    def release(self, b: int) -> None:
        """Sequence b is done: its length is 0."""
        self.prefix[b] = 0


@torch.no_grad()
def tree_pass(layers: List[DecoderLayer], h: torch.Tensor, cache: TreeKVCache, parents: torch.Tensor) -> torch.Tensor:
    """All layers over the trees h [B, T, hidden] behind the cache's lengths; returns the final
    hidden states.  parents int32 [B, T] or [T]; layers whose projections carry adapters of many
    requests (lora.MultiLoRAManager) take each sequence's own."""
    b, t, _ = h.shape
    if b != cache.batch or len(layers) != len(cache.k):
        raise ValueError(f"tree_pass: {b} sequences and {len(layers)} layers, the cache has {cache.batch} and {len(cache.k)}")
    for layer in layers:
        if layer.cfg.rope_theta != cache.rope_theta:
            raise ValueError(f"tree_pass: the layer's rope_theta is {layer.cfg.rope_theta:g}, the cache's "
                             f"{cache.rope_theta:g}")
    cos, sin = cache.tables
    for layer, k_cache, v_cache in zip(layers, cache.k, cache.v):
        cfg = layer.cfg

        def attend(q_raw, k_raw, v_raw):
            q, k, v = (x.view(b, t, n, cfg.head_dim) for x, n in ((q_raw, cfg.heads), (k_raw, cfg.kv_heads),
                                                                  (v_raw, cfg.kv_heads)))
            q = ops.tree_append(q, k, v, k_cache, v_cache, cache.prefix, parents, cos, sin)
            o = ops.tree_attention(q, k_cache, v_cache, cache.prefix, parents)
            return o.view(b, t, cfg.heads * cfg.head_dim)

        h = _layer_forward(layer, h, attend)
    return h
