"""Serving and scoring operators of the verify step: what they compute, in
elementary torch operations, and the calls that run them on the library.

* ``append``   -- new keys and values of a ragged batch go into a paged cache
                  held in 4 bits, the rotary embedding applied on the way (and
                  to the queries); the appended positions read back as the
                  values they stand for.
* ``attend``   -- attention of the new tokens over that cache (grouped-query,
                  causal among the new tokens): single-token decode, draft
                  verification, prompts.
* ``logprobs`` -- log probabilities of given tokens with the entropy of each
                  row and the top alternatives, and their gradient.

The cache format.  A pool is uint8 [pages, kv_heads, page_size / 16, 18 D]: one
block per 16 positions and KV head, D = head_dim in {64, 128}.  The D values of
a key or value are coded in groups of 64 as value = scale * code + low with
code in 0..15 and scale, low fp16.  Block bytes, G = D / 64 groups, element j of
eight in nibble j (low nibble first) of a 4-byte word:
  keys    [16 positions][4][G][2][4 B]: word (c, g, w) = elements 64 g + 16 c + 8 w + (0..7);
  values  [2][8][4][2][G][4 B]: word (h, e, q, o, g) = elements 64 g + 8 e + (0..7)
          of position 8 h + 2 q + o;
  params  [16 positions][2: key, value][G][2: scale, low] fp16.
Coding a group x: low = fp16(min x); scale = fp16((max x - low) / 15);
code = round_half_even((x - low) * (1 / scale)) clamped to 0..15, 0 where scale
is 0; differences, products and the reciprocal each rounded to fp32.  Keys are
coded from the fp32 rotated values a c - b s and b c + a s (each product and sum
rounded to fp32).
"""
import math

import torch

own = False

NEG = float("-inf")
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------ cases
def listed():
    a = dict(kind="append", heads=40, kv_heads=8, dim=128, page=64, dtype="bf16", ragged=False)
    t = dict(a, kind="attend")
    p = dict(kind="logprobs", vocab=152064, pad=0, top=0, dtype="bf16", grad=False)
    return [
        # one sequence decodes one token: the call's latency
        dict(a, name="append_decode_1", batch=1, new=1, ctx_lo=4095, ctx_hi=4095),
        # a decode step of a full batch, every sequence at its own length
        dict(a, name="append_decode_64", batch=64, new=1, ctx_lo=1, ctx_hi=8191),
        # three prompts of different lengths enter an fp16 cache with small pages
        dict(a, name="append_prompts", batch=3, new=4001, ctx_lo=0, ctx_hi=777, page=16, dtype="fp16", ragged=True),
        # one short sequence decodes one token: latency
        dict(t, name="attend_decode_1", batch=1, new=1, ctx_lo=1023, ctx_hi=1023),
        # a decode step of a full ragged batch: bandwidth
        dict(t, name="attend_decode_64", batch=64, new=1, ctx_lo=100, ctx_hi=8191),
        # one long document: the cache of one sequence over the whole card
        dict(t, name="attend_long", batch=1, new=1, ctx_lo=131071, ctx_hi=131071, page=128),
        # four drafts and the token before them for eight sequences, fp16
        dict(t, name="attend_verify", batch=8, new=5, ctx_lo=3500, ctx_hi=4099, dtype="fp16"),
        # prompts behind a cached prefix
        dict(t, name="attend_prompts", batch=2, new=2048, ctx_lo=0, ctx_hi=513, ragged=True),
        # the next-token row of one sequence, with alternatives for the user: latency
        dict(p, name="logprobs_decode", rows=1, top=20),
        # the rows of a verify step in fp32, columns behind the tokenizer's last token masked
        dict(p, name="logprobs_verify", rows=40, top=5, dtype="fp32", pad=399),
        # a training micro-batch: policy log probabilities and entropies with their gradient
        dict(p, name="logprobs_train", rows=2048, grad=True),
        # an odd vocabulary in fp16: rows at odd offsets, alternatives in the loss too
        dict(p, name="logprobs_odd", rows=257, vocab=32001, top=8, dtype="fp16", grad=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "attend", "attend", "logprobs"])
    if kind == "logprobs":
        vocab = _log_int(rng, 1000, 152064)
        grad = rng.random() < 0.5
        rows = _log_int(rng, 1, max(2, min(2048, 2048 * 152064 // vocab // (2 if grad else 1))))
        top = rng.choice([0, 1, 5, 20])
        if top:
            rows = max(1, min(rows, 300_000_000 // (4 * vocab)))
        dtype = rng.choice(["bf16", "fp16", "fp32"])
        if dtype == "fp32":
            rows = max(1, rows // 2)
        return dict(kind=kind, rows=rows, vocab=vocab, pad=rng.choice([0, 0, 17]), top=top, dtype=dtype, grad=grad)
    heads, kv_heads = rng.choice([(40, 8), (32, 8), (32, 4), (28, 4), (16, 16), (8, 1)])
    batch = _log_int(rng, 1, 64)
    shape = rng.choice(["decode", "verify", "prompt"])
    new = 1 if shape == "decode" else rng.randint(2, 8) if shape == "verify" else _log_int(rng, 9, max(10, 4096 // batch))
    ctx_hi = _log_int(rng, 1, max(2, min(131072, 500_000 // batch)))
    if kind == "attend":
        while batch * new * (ctx_hi + new) * heads > 300_000_000 and ctx_hi > 1:
            ctx_hi //= 2
    return dict(kind=kind, heads=heads, kv_heads=kv_heads, dim=rng.choice([64, 128, 128]),
                page=rng.choice([16, 32, 64, 128]), dtype=rng.choice(["bf16", "fp16"]), batch=batch, new=new,
                ctx_lo=rng.randint(0, ctx_hi), ctx_hi=ctx_hi, ragged=new > 1 and rng.random() < 0.5)


def _spread(lo, hi, n):
    """n whole numbers spread over lo..hi in a fixed scrambled order, the last one hi."""
    return [lo + int((hi - lo) * ((0.6180339887 * (i + 1)) % 1.0)) for i in range(n - 1)] + [hi]


def _lengths(c):
    """(cached positions, new tokens) of each sequence."""
    ctx = _spread(c["ctx_lo"], c["ctx_hi"], c["batch"])
    new = _spread(max(1, c["new"] // 3), c["new"], c["batch"]) if c["ragged"] else [c["new"]] * c["batch"]
    return ctx, new


def work(c):
    size = 4 if c["dtype"] == "fp32" else 2
    if c["kind"] == "logprobs":
        n = c["rows"] * c["vocab"]
        passes = 3 if c["grad"] else 1  # logits read; read again and the gradient written
        return {"bytes": n * size * passes + c["rows"] * (24 + 12 * c["top"]), "flops": n * (12 if c["grad"] else 6)}
    ctx, new = _lengths(c)
    h, kvh, d = c["heads"], c["kv_heads"], c["dim"]
    tokens, position = sum(new), kvh * 18 * d // 16
    if c["kind"] == "append":  # q, k, v in; q, the coded position and its values out; the tables' rows
        moved = tokens * ((2 * h + 4 * kvh) * d * size + 2 * position) + 4 * d * tokens
        return {"bytes": moved, "flops": tokens * d * (3 * h + 11 * kvh)}
    seen = sum(n * p + n * (n + 1) // 2 for p, n in zip(ctx, new))
    return {"bytes": sum(p + n for p, n in zip(ctx, new)) * position + 2 * tokens * h * d * size, "flops": 4 * h * d * seen}


# ------------------------------------------------------------------ inputs
def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[c["dtype"]]

    def randn(*shape, dtype=dt):
        return torch.randn(*shape, generator=g, device="cuda", dtype=dtype)

    if c["kind"] == "logprobs":
        rows, vocab, top = c["rows"], c["vocab"], c["top"]
        logits = randn(rows, vocab).mul_(2.5)
        ids = torch.randint(0, vocab - c["pad"], (rows,), generator=g, device="cuda")
        logits[torch.arange(rows, device="cuda"), ids] += 9.0  # most tokens were likely ones
        if c["pad"]:
            logits[:, vocab - c["pad"]:] = NEG
        s = {"case": c, "logits": logits, "ids": ids}
        if c["grad"]:
            ids[3::7] = -100  # prompt tokens carry no loss
            s["logits"].requires_grad_(True)
            s["ups"] = (randn(rows, dtype=torch.float32), randn(rows, dtype=torch.float32) * 0.1)
            if top:
                s["ups"] += (randn(rows, top, dtype=torch.float32),)
        return s
    ctx, new = _lengths(c)
    h, kvh, d, ps = c["heads"], c["kv_heads"], c["dim"], c["page"]
    max_len = max(p + n for p, n in zip(ctx, new))
    need = [-(-(p + n) // ps) for p, n in zip(ctx, new)]
    order = torch.randperm(sum(need) + 3, generator=g, device="cuda")[:sum(need)].int()
    table = torch.full((c["batch"], max(need)), -1, dtype=torch.int32, device="cuda")
    filled = torch.arange(max(need), device="cuda")[None, :] < torch.tensor(need, device="cuda")[:, None]
    table[filled] = order
    groups = d // 64
    pool = torch.randint(0, 256, (sum(need) + 3, kvh, ps // 16, 18 * d), generator=g, device="cuda", dtype=torch.uint8)
    params = pool[..., 16 * d:].view(torch.float16).view(*pool.shape[:3], 16, 2, groups, 2)
    scale = torch.rand(params.shape[:-1], generator=g, device="cuda") * 0.2 + 0.1
    params[..., 0] = scale.half()
    params[..., 1] = (torch.randn(scale.shape, generator=g, device="cuda") * 0.1 - 7.5 * scale).half()
    tokens = sum(new)
    starts = torch.tensor([0] + list(torch.tensor(new).cumsum(0)), dtype=torch.int32, device="cuda")
    s = {"case": c, "pool": pool, "table": table, "q": randn(tokens, h, d), "max_len": max_len, "max_new": max(new),
         "prefix": torch.tensor(ctx, dtype=torch.int32, device="cuda"), "q_start": starts if c["ragged"] else None}
    if c["kind"] == "append":
        s["k"], s["v"] = randn(tokens, kvh, d), randn(tokens, kvh, d)
        # keys carry a few strong channels, as trained models' do
        s["k"] += (torch.randn(kvh, d, generator=g, device="cuda") * 2.0).to(dt)
        inv = 1.0 / (1e6 ** (torch.arange(0, d, 2, device="cuda", dtype=torch.float64) / d))
        angle = torch.outer(torch.arange(max_len, device="cuda", dtype=torch.float64), inv)
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
    return s


# ------------------------------------------------------------------ the operators
def run(s):
    c = s["case"]
    if own:
        return {"append": _own_append, "attend": _own_attend, "logprobs": _own_logprobs}[c["kind"]](s)
    return {"append": _append, "attend": _attend, "logprobs": _logprobs}[c["kind"]](s)


def _own_append(s):
    from fitllm_b200 import ops
    q = ops.kv4_append(s["q"], s["k"], s["v"], s["pool"], s["table"], s["prefix"], s["cos"], s["sin"],
                       q_start=s["q_start"])
    k, v = ops.kv4_gather(s["pool"], s["table"], s["prefix"], s["q"].shape[0], q_start=s["q_start"],
                          dtype=s["q"].dtype)
    return {"q": q, "k": k, "v": v}


def _own_attend(s):
    from fitllm_b200 import ops
    return ops.kv4_attention(s["q"], s["pool"], s["table"], s["prefix"], s["max_len"], q_start=s["q_start"],
                             max_new=s["max_new"])


def _own_logprobs(s):
    from fitllm_b200.lm_head import token_logprobs
    r = token_logprobs(s["logits"], s["ids"], top=s["case"]["top"])
    out = {"logp": r.logp, "entropy": r.entropy}
    if s["case"]["top"]:
        out["top_logp"], out["top_ids"] = r.top_logp, r.top_ids
    if s["case"]["grad"]:
        wanted = [r.logp, r.entropy] + ([r.top_logp] if s["case"]["top"] else [])
        out["grad"] = torch.autograd.grad(wanted, s["logits"], s["ups"])[0]
    return out


def _tokens(s):
    """Sequence and position of each new token, and the sequences' starts."""
    n, b = s["q"].shape[0], s["prefix"].shape[0]
    at = torch.arange(n, device="cuda")
    start = s["q_start"].long() if s["q_start"] is not None else torch.arange(b + 1, device="cuda") * (n // b)
    seq = torch.searchsorted(start, at, right=True) - 1
    return start, seq, s["prefix"].long()[seq] + at - start[seq]


def _rotate(x, cos, sin):
    a, b = x.float().chunk(2, dim=-1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)


def _coded(x):
    """The values that x [n, heads, D] (fp32) stands for in the cache."""
    x = x.unflatten(-1, (-1, 64))
    low = x.amin(-1, keepdim=True).half().float()
    scale = ((x.amax(-1, keepdim=True) - low) / 15).half().float()
    code = torch.where(scale > 0, torch.round((x - low) * (1 / scale)), torch.zeros_like(x)).clamp(0, 15)
    return (scale * code + low).flatten(-2)


def _append(s):
    _, _, pos = _tokens(s)
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
    dt = s["q"].dtype
    return {"q": _rotate(s["q"], cos, sin).to(dt), "k": _coded(_rotate(s["k"], cos, sin)).to(dt),
            "v": _coded(s["v"].float()).to(dt)}


def _nibbles(b):
    return torch.stack([b & 15, b >> 4], dim=-1).flatten(-2)


def _cache(s):
    """Keys and values [B, kv_heads, positions, D] in fp32 behind the page table."""
    blocks = s["pool"][s["table"].clamp(min=0).long()]  # [B, pages, kv_heads, blocks, bytes]
    b, pages, kvh, per, nbytes = blocks.shape
    d = nbytes // 18
    g = d // 64
    lead = (b, pages, kvh, per)
    par = blocks[..., 16 * d:].contiguous().view(torch.float16).float().view(*lead, 16, 2, g, 1, 2)
    k = _nibbles(blocks[..., :8 * d]).view(*lead, 16, 4, g, 16).transpose(-2, -3).reshape(*lead, 16, g, 64)
    v = _nibbles(blocks[..., 8 * d:16 * d]).view(*lead, 2, 8, 4, 2, g, 8)
    v = v.permute(0, 1, 2, 3, 4, 6, 7, 8, 5, 9).reshape(*lead, 16, g, 64)
    k = k.float() * par[..., 0, :, :, 0] + par[..., 0, :, :, 1]
    v = v.float() * par[..., 1, :, :, 0] + par[..., 1, :, :, 1]
    return [x.view(b, pages, kvh, per * 16, d).transpose(1, 2).reshape(b, kvh, pages * per * 16, d) for x in (k, v)]


def _attend(s):
    c = s["case"]
    start, seq, pos = _tokens(s)
    b, h, d = c["batch"], c["heads"], c["dim"]
    t, kvh = s["max_new"], c["kv_heads"]
    k, v = _cache(s)
    at = start[:-1, None] + torch.arange(t, device="cuda")
    inside = at < start[1:, None]
    q = s["q"][at.clamp(max=s["q"].shape[0] - 1)].float()  # [B, t, H, D]
    q = q.view(b, t, kvh, h // kvh, d).permute(0, 2, 3, 1, 4).reshape(b, kvh, -1, d)
    score = (q @ k.transpose(-1, -2)).mul_(1 / math.sqrt(d)).view(b, kvh, h // kvh, t, -1)
    last = torch.where(inside, s["prefix"].long()[:, None] + torch.arange(t, device="cuda"), 0)
    hidden = torch.arange(k.shape[2], device="cuda") > last[:, :, None]
    score.masked_fill_(hidden[:, None, None], NEG)
    score.sub_(score.amax(-1, keepdim=True)).exp_()
    score.div_(score.sum(-1, keepdim=True))
    o = (score.view(b, kvh, -1, k.shape[2]) @ v).view(b, kvh, h // kvh, t, d).permute(0, 3, 1, 2, 4).reshape(b, t, h, d)
    return o[seq, torch.arange(seq.shape[0], device="cuda") - start[seq]].to(s["q"].dtype)


def _logprobs(s):
    c, ids = s["case"], s["ids"]
    z = s["logits"].detach().float()
    vocab, top = c["vocab"], c["top"]
    m = z.amax(-1, keepdim=True)
    x = z - m
    e = x.exp()
    total = e.sum(-1, keepdim=True)
    log_total = total.log()
    entropy = log_total - torch.where(e > 0, e * x, torch.zeros_like(x)).sum(-1, keepdim=True) / total
    valid = (ids >= 0) & (ids < vocab)
    safe = ids.clamp(0, vocab - 1)[:, None]
    logp = torch.where(valid, (x.gather(-1, safe) - log_total)[:, 0], torch.zeros_like(log_total[:, 0]))
    out = {"logp": logp, "entropy": entropy[:, 0]}
    if top:
        # unique keys: the logit's order first, then the lowest index
        bits = (z + 0.0).view(torch.int32)
        rank = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
        key = rank * (1 << 20) + ((1 << 20) - 1 - torch.arange(vocab, device="cuda"))
        out["top_ids"] = (1 << 20) - 1 - (torch.topk(key, top, dim=-1).values & ((1 << 20) - 1))
        out["top_logp"] = x.gather(-1, out["top_ids"]) - log_total
    if c["grad"]:
        p = e / total
        g_logp = torch.where(valid, s["ups"][0], torch.zeros_like(s["ups"][0]))[:, None]
        g_top = s["ups"][2] if top else torch.zeros(c["rows"], 1, device="cuda")
        slope = torch.where(p > 0, p * (x - log_total + entropy), torch.zeros_like(p))
        d = -p * (g_logp + g_top.sum(-1, keepdim=True)) - s["ups"][1][:, None] * slope
        d.scatter_add_(-1, safe, g_logp)
        if top:
            d.scatter_add_(-1, out["top_ids"], g_top)
        out["grad"] = d.to(s["logits"].dtype)
    return out


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(c, seed):
    s = prepare(c, seed)
    if c["kind"] == "logprobs":
        return _exact_logprobs(s)
    ctx, new = _lengths(c)
    if c["kind"] == "append":
        return _exact_append(s, ctx, new)
    d, ps, group = c["dim"], c["page"], c["heads"] // c["kv_heads"]
    # where each element of a block's keys and values lies: byte and shift
    p, e = torch.arange(16, device="cuda")[:, None], torch.arange(d, device="cuda")[None, :]
    g, f = e // 64, e % 64
    key_word = ((p * 4 + f // 16) * (d // 64) + g) * 2 + (f % 16) // 8
    val_word = 2 * d + ((((p // 8) * 8 + f // 8) * 4 + (p % 8) // 2) * 2 + p % 2) * (d // 64) + g
    par = 16 * d + ((p * 2) * (d // 64) + g) * 4
    low_half = torch.tensor([0, 1], device="cuda")
    out, at = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda"), 0
    for i, (n0, n1) in enumerate(zip(ctx, new)):
        length = n0 + n1
        pages = s["table"][i, : -(-length // ps)].long()
        b = s["pool"][pages].permute(1, 0, 2, 3).reshape(c["kv_heads"], -1, 18 * d)

        def side(word, which):
            code = (b[..., word * 4 + (e % 8) // 2] >> (4 * (e % 2)).to(torch.uint8)) & 15
            sc, lo = (b[..., (par + which * (d // 64) * 4 + o)[..., None] + low_half].contiguous()
                      .view(torch.float16)[..., 0].double() for o in (0, 2))
            return (code.double() * sc + lo).reshape(c["kv_heads"], -1, d)[:, :length]

        k, v = side(key_word, 0), side(val_word, 1)
        q = s["q"][at:at + n1].double()
        mask = torch.arange(length, device="cuda")[None, :] > torch.arange(n0, length, device="cuda")[:, None]
        for hd in range(c["heads"]):
            w = (q[:, hd] @ k[hd // group].T / math.sqrt(d)).masked_fill_(mask, NEG)
            out[at:at + n1, hd] = torch.softmax(w, dim=-1) @ v[hd // group]
        at += n1
    return out


def _exact_append(s, ctx, new):
    pos = torch.cat([torch.arange(p, p + n, device="cuda") for p, n in zip(ctx, new)])
    w = torch.complex(s["cos"][pos].double(), s["sin"][pos].double())[:, None]

    def turn(x):
        half = x.shape[-1] // 2
        z = torch.complex(x[..., :half].double(), x[..., half:].double()) * w
        return torch.cat([z.real, z.imag], dim=-1)

    def stand(x):
        y = torch.empty_like(x)
        for g in range(x.shape[-1] // 64):
            part = x[..., 64 * g:64 * g + 64]
            lo = part.min(-1, keepdim=True).values.half().double()
            step = ((part.max(-1, keepdim=True).values - lo) / 15).half().double()
            code = ((part - lo) / step.clamp(min=1e-30)).round().clamp(0, 15)
            y[..., 64 * g:64 * g + 64] = lo + step * code
        return y

    return {"q": turn(s["q"]), "k": stand(turn(s["k"])), "v": stand(s["v"].double())}


def _exact_logprobs(s):
    c, ids = s["case"], s["ids"]
    z = s["logits"].detach().double()
    logp = torch.log_softmax(z, dim=-1)
    p = logp.exp()
    ent = -torch.nansum(p * logp, dim=-1)
    rows = torch.arange(c["rows"], device="cuda")
    ok = ids >= 0
    out = {"logp": torch.where(ok, logp[rows, ids.clamp(min=0)], 0.0), "entropy": ent}
    if c["top"]:
        top_ids = torch.sort(z, dim=-1, descending=True, stable=True).indices[:, :c["top"]]
        out["top_logp"], out["top_ids"] = logp.gather(-1, top_ids), None
    if c["grad"]:
        g1, g2 = (u.double()[:, None] for u in s["ups"][:2])
        d = -g2 * torch.nan_to_num(p * (logp + ent[:, None]), nan=0.0)
        g1 = g1 * ok[:, None]
        d -= p * g1
        d[rows, ids.clamp(min=0)] += g1[:, 0]
        if c["top"]:
            g3 = s["ups"][2].double()
            d -= p * g3.sum(-1, keepdim=True)
            for j in range(c["top"]):
                d[rows, top_ids[:, j]] += g3[:, j]
        out["grad"] = d
    return out
