"""Operators of a serving step that drafts trees of tokens for many requests: what
they compute, in elementary torch operations, and the calls that run them on the
library.

* ``attend`` -- attention of a tree of drafted tokens over a key/value cache whose
                sequences have lengths of their own: every token sees the cached
                positions, its ancestors and itself.
* ``cache``  -- the tree's tokens enter the cache (queries and keys rotated at the
                position that their depth gives) and, once a path is accepted, its
                tokens move to the front in every layer.
* ``verify`` -- the drafted tokens against the model's probabilities, from given
                random numbers: accepted path and next token.
* ``lora``   -- low-rank adapters of many requests added to a shared projection.

A tree is ``parents`` int32 [batch, T]: the index of a token's parent (smaller than its
own), -1 for a token right behind the cached positions, -2 where there is no token.
Token i of a sequence stands in cache slot prefix + i and is rotated at position
prefix + depth.

Verification walks from token 0.  At a token the model's distribution is p =
softmax(logits / temperature); its children, in order, are accepted where u q(x) <
p(x), and where one is refused p becomes max(p - q, 0) (without a q: p with p(x) = 0),
normalised.  Behind the last child the next token is the first whose cumulated
probability exceeds the random number of token 0.
"""
import math

import torch

own = False

NEG = float("-inf")
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------ cases
def listed():
    a = dict(kind="attend", heads=40, kv_heads=8, dim=128, dtype="bf16", shape="tree", ragged=False)
    c = dict(kind="cache", heads=40, kv_heads=8, dim=128, dtype="bf16", shape="tree", ragged=False)
    v = dict(kind="verify", vocab=152064, dtype="bf16", shape="chain", ragged=False, probs=True, temp=0.8)
    m = dict(kind="lora", k=5120, n=5120, rank=16, dtype="bf16", ragged=False)
    return [
        # four drafts in a row for one short sequence: latency
        dict(a, name="attend_chain_1", batch=1, new=5, ctx_lo=1023, ctx_hi=1023, shape="chain"),
        # a tree of 32 tokens for each of eight sequences
        dict(a, name="attend_tree_8", batch=8, new=32, ctx_lo=3500, ctx_hi=4099),
        # a full ragged batch with small trees of different sizes: bandwidth
        dict(a, name="attend_ragged_64", batch=64, new=8, ctx_lo=100, ctx_hi=8191, ragged=True),
        # one long document, the largest tree, fp16
        dict(a, name="attend_long", batch=1, new=64, ctx_lo=131071, ctx_hi=131071, dtype="fp16"),
        # one sequence's chain enters the cache of one layer and is accepted in part: latency
        dict(c, name="cache_chain_1", batch=1, new=5, ctx_lo=200, ctx_hi=200, layers=1, shape="chain"),
        # trees of a full batch enter six layers, the accepted paths move in all of them
        dict(c, name="cache_tree_64", batch=64, new=16, ctx_lo=3, ctx_hi=250, layers=6, dtype="fp16", ragged=True),
        # one sequence's chain against the drafting model's probabilities: latency
        dict(v, name="verify_chain_1", batch=1, new=5),
        # a full batch of chains
        dict(v, name="verify_chain_64", batch=64, new=5),
        # trees of a model's most likely tokens (no drafting distribution), an odd vocabulary in fp16
        dict(v, name="verify_tree_16", batch=16, new=32, vocab=32001, dtype="fp16", shape="tree", probs=False, temp=1.0),
        # one sequence decodes one token through its adapter: latency
        dict(m, name="lora_decode_1", batch=1, new=1, adapters=4),
        # a decode step of 64 requests, an adapter each, on the widest projection
        dict(m, name="lora_decode_64", batch=64, new=1, adapters=64, n=27648),
        # prompts of different lengths, few adapters of a high rank, fp16
        dict(m, name="lora_prompts", batch=6, new=1001, adapters=5, k=27648, rank=64, dtype="fp16", ragged=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "cache", "verify", "lora"])
    shape = rng.choice(["chain", "tree"])
    ragged = rng.random() < 0.5
    if kind == "verify":
        vocab = _log_int(rng, 1000, 152064)
        new = rng.randint(1, 8) if shape == "chain" else rng.randint(2, 64)
        batch = _log_int(rng, 1, max(1, min(64, 40_000_000 // (vocab * new))))
        return dict(kind=kind, vocab=vocab, batch=batch, new=new, shape=shape, ragged=ragged,
                    dtype=rng.choice(["bf16", "fp16", "fp32"]), probs=rng.random() < 0.6,
                    temp=rng.choice([0.0, 0.3, 0.7, 1.0, 1.3]))
    if kind == "lora":
        k, n = rng.choice([(5120, 5120), (5120, 1024), (5120, 27648), (27648, 5120), (1024, 1536), (512, 1048)])
        batch = _log_int(rng, 1, 128)
        new = rng.choice([1, 1, rng.randint(2, 8), _log_int(rng, 9, 2048)])
        return dict(kind=kind, k=k, n=n, rank=rng.choice([16, 32, 48, 64]), batch=batch,
                    new=max(1, min(new, 4096 // batch)), adapters=_log_int(rng, 1, 64),
                    dtype=rng.choice(["bf16", "fp16"]), ragged=ragged)
    heads, kv_heads = rng.choice([(40, 8), (32, 8), (32, 4), (28, 4), (16, 16), (8, 1)])
    batch = _log_int(rng, 1, 64)
    new = rng.randint(1, 8) if shape == "chain" else rng.randint(2, 64)
    c = dict(kind=kind, heads=heads, kv_heads=kv_heads, dim=rng.choice([64, 128, 128]), batch=batch, new=new,
             dtype=rng.choice(["bf16", "fp16"]), shape=shape, ragged=ragged)
    if kind == "cache":
        ctx_hi = _log_int(rng, 1, 400)
        return dict(c, ctx_lo=rng.randint(0, ctx_hi), ctx_hi=ctx_hi, layers=rng.randint(1, 5))
    ctx_hi = _log_int(rng, 1, max(2, min(131072, 2_000_000 // (batch * kv_heads))))
    while batch * new * (ctx_hi + new) * heads > 300_000_000 and ctx_hi > 1:
        ctx_hi //= 2
    return dict(c, ctx_lo=rng.randint(0, ctx_hi), ctx_hi=ctx_hi)


def _spread(lo, hi, n):
    """n whole numbers spread over lo..hi in a fixed scrambled order, the last one hi."""
    return [lo + int((hi - lo) * ((0.6180339887 * (i + 1)) % 1.0)) for i in range(n - 1)] + [hi]


def _counts(c):
    """Tokens of each sequence."""
    return _spread(max(1, c["new"] // 3), c["new"], c["batch"]) if c["ragged"] else [c["new"]] * c["batch"]


def work(c):
    size = 4 if c["dtype"] == "fp32" else 2
    b, news = c["batch"], _counts(c)
    if c["kind"] == "lora":
        tokens, used = sum(news), min(c["adapters"], b)
        k, n, r = c["k"], c["n"], c["rank"]
        return {"bytes": size * (tokens * (k + 2 * n) + used * r * (k + n)), "flops": 2 * r * (k + n) * tokens}
    if c["kind"] == "verify":
        # rows that the walk reads: on a chain a token is accepted about two times in three; a tree goes
        # about as deep.  A drafting distribution is read where a token was refused.
        deep = min(sum(news) / b, 2.5)
        rows = b * deep
        return {"bytes": int(rows * c["vocab"] * size + (b * c["vocab"] * 4 if c["probs"] else 0)),
                "flops": int(4 * rows * c["vocab"])}
    h, kvh, d = c["heads"], c["kv_heads"], c["dim"]
    if c["kind"] == "cache":  # q, k, v in; q and the slots out; about a third of the slots moved in each layer
        moved = c["layers"] * sum(n * (2 * h + 4 * kvh) * d * size + (n // 3) * 4 * kvh * d * size for n in news)
        return {"bytes": moved, "flops": c["layers"] * 3 * d * (h + kvh) * sum(news)}
    ctx = _spread(c["ctx_lo"], c["ctx_hi"], b)
    read = sum(p + n for p, n in zip(ctx, news)) * kvh * d * 2 * size
    return {"bytes": read + 2 * sum(news) * h * d * size, "flops": 4 * h * d * sum(n * (p + 1) for p, n in zip(ctx, news))}


# ------------------------------------------------------------------ inputs
def _trees(c, g):
    """parents [batch, T] on the GPU: chains, or trees in which earlier tokens have more children."""
    b, t = c["batch"], c["new"]
    at = torch.arange(t, device="cuda")
    if c["shape"] == "chain":
        parents = (at - 1).expand(b, t).clone()
    else:
        parents = (torch.rand(b, t, generator=g, device="cuda") ** 1.5 * at).long().clamp(max=t - 1)
        parents = torch.minimum(parents, at - 1)
    counts = torch.tensor(_counts(c), device="cuda")
    return torch.where(at < counts[:, None], parents, -2).int()


def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[c["dtype"]]
    b, t = c["batch"], c["new"]

    def randn(*shape, dtype=dt):
        return torch.randn(*shape, generator=g, device="cuda", dtype=dtype)

    def rand(*shape):
        return torch.rand(*shape, generator=g, device="cuda")

    if c["kind"] == "lora":
        news, n_ad, r = _counts(c), c["adapters"], c["rank"]
        tokens = sum(news)
        adapter = torch.randint(0, n_ad, (b,), generator=g, device="cuda")
        if n_ad >= b > 1:  # an adapter each
            adapter = torch.randperm(n_ad, generator=g, device="cuda")[:b]
        if b > 2:
            adapter[1] = -1  # one request uses the model as it is
        starts = torch.tensor([0] + list(torch.tensor(news).cumsum(0)), dtype=torch.int32, device="cuda")
        return {"case": c, "x": randn(tokens, c["k"]), "y": randn(tokens, c["n"]), "adapter": adapter.int(),
                "a": (rand(n_ad, r, c["k"]) * 2 - 1).div_(math.sqrt(c["k"])).to(dt),
                "b": randn(n_ad, c["n"], r).mul_(0.3), "scale": 0.5 + 2 * rand(n_ad),
                "q_start": starts if c["ragged"] else None}
    parents = _trees(c, g)
    s = {"case": c, "parents": parents}
    if c["kind"] == "verify":
        vocab = c["vocab"]
        logits = randn(b, t, vocab).mul_(1.5)
        # a few tokens stand out, as in a trained model's rows
        heads = torch.randint(0, vocab, (b, t, 6), generator=g, device="cuda")
        lift = torch.tensor([13.0, 12.5, 12.0, 11.0, 10.0, 9.0], device="cuda").to(dt).expand(b, t, 6)
        logits.scatter_(-1, heads, lift)
        logits[..., vocab // 3] = NEG  # a token that is never allowed
        s["logits"], s["uniforms"], s["temp"] = logits, rand(b, t), c["temp"]
        s["temp32"] = torch.tensor(c["temp"], dtype=torch.float32, device="cuda").double()
        row = parents.long().clamp(min=0)
        if c["probs"]:
            # the drafting model's distributions: the target's, blurred; tokens drawn from them
            soft = logits.float().add_(torch.randn(b, t, vocab, generator=g, device="cuda"), alpha=0.7)
            q = torch.softmax(soft / max(c["temp"], 0.5), dim=-1)
            del soft
            cdf = q.cumsum(-1, dtype=torch.float64)
            at = rand(b, t).double() * cdf[..., -1].gather(1, row)
            s["tokens"] = torch.stack([torch.searchsorted(cdf[i, row[i]], at[i][:, None], right=True)[:, 0]
                                       for i in range(b)]).clamp(max=vocab - 1)
            s["probs"] = q[:, :max(1, t - 1)].contiguous()
        else:
            # children are the parent row's most likely tokens, in no order
            pick = torch.randint(0, 6, (b, t), generator=g, device="cuda")
            s["tokens"] = heads[torch.arange(b, device="cuda")[:, None], row, pick]
            s["probs"] = None
        return s
    ctx = _spread(c["ctx_lo"], c["ctx_hi"], b)
    h, kvh, d = c["heads"], c["kv_heads"], c["dim"]
    s["prefix"] = torch.tensor(ctx, dtype=torch.int32, device="cuda")
    cap = max(ctx) + t + 3
    if c["kind"] == "attend":
        s["q"], s["k_cache"], s["v_cache"] = randn(b, t, h, d), randn(b, kvh, cap, d), randn(b, kvh, cap, d)
        return s
    s["new"] = [(randn(b, t, h, d), randn(b, t, kvh, d), randn(b, t, kvh, d)) for _ in range(c["layers"])]
    s["k_caches"] = [randn(b, kvh, cap, d) for _ in range(c["layers"])]
    s["v_caches"] = [randn(b, kvh, cap, d) for _ in range(c["layers"])]
    inv = 1.0 / (1e6 ** (torch.arange(0, d, 2, device="cuda", dtype=torch.float64) / d))
    angle = torch.outer(torch.arange(cap, device="cuda", dtype=torch.float64), inv)
    s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
    # the accepted path: from token 0 to a child at a time, now and then no further
    path = torch.full((b, t), -1, dtype=torch.int32, device="cuda")
    path[:, 0] = 0
    accepted = torch.zeros(b, dtype=torch.int64, device="cuda")
    cur = torch.zeros(b, dtype=torch.int64, device="cuda")
    go = rand(b, t) < 0.6
    for i in range(1, t):
        step = (parents[:, i].long() == cur) & go[:, i]
        accepted += step
        cur = torch.where(step, i, cur)
        path.scatter_(1, torch.where(step, accepted, 0)[:, None], torch.where(step, i, 0).int()[:, None])
    s["path"], s["accepted"] = path, accepted
    return s


# ------------------------------------------------------------------ the operators
def run(s):
    kind = s["case"]["kind"]
    if own:
        return {"attend": _own_attend, "cache": _own_cache, "verify": _own_verify, "lora": _own_lora}[kind](s)
    return {"attend": _attend, "cache": _cache, "verify": _verify, "lora": _lora}[kind](s)


def _own_attend(s):
    from fitllm_b200 import ops
    return ops.tree_attention(s["q"], s["k_cache"], s["v_cache"], s["prefix"], s["parents"])


def _own_cache(s):
    from fitllm_b200 import ops
    turned = [ops.tree_append(q, k, v, kc, vc, s["prefix"], s["parents"], s["cos"], s["sin"])
              for (q, k, v), kc, vc in zip(s["new"], s["k_caches"], s["v_caches"])]
    lengths = ops.tree_keep(s["k_caches"], s["v_caches"], s["prefix"], s["path"], s["accepted"])
    return {"q": turned, "lengths": lengths, "k": s["k_caches"], "v": s["v_caches"]}


def _own_verify(s):
    from fitllm_b200.verify import verify_tree
    r = verify_tree(s["logits"], s["tokens"], s["parents"], s["uniforms"], draft_probs=s["probs"],
                    temperature=s["temp"])
    return {"path": r.path, "accepted": r.accepted, "next_token": r.next_token}


def _own_lora(s):
    from fitllm_b200 import ops
    return ops.multi_lora(s["x"], s["a"], s["b"], s["scale"], s["adapter"], s["y"], q_start=s["q_start"])


def _ancestors(parents):
    """seen [B, T, T] (token i sees token j) and depth [B, T]; absent tokens see nothing."""
    b, t = parents.shape
    up = parents.long()
    here = up >= -1
    seen = torch.zeros(b, t, t, dtype=torch.bool, device="cuda")
    cur = torch.where(here, torch.arange(t, device="cuda").expand(b, t), -1)
    depth = torch.full((b, t), -1, dtype=torch.int64, device="cuda")
    for _ in range(t):
        on = cur >= 0
        seen |= (torch.arange(t, device="cuda") == cur[:, :, None]) & on[:, :, None]
        depth += on
        cur = torch.where(on, up.gather(1, cur.clamp(min=0)), -1)
    return seen, depth, here


def _attend(s):
    c = s["case"]
    b, t, h, d, kvh = c["batch"], c["new"], c["heads"], c["dim"], c["kv_heads"]
    seen, _, here = _ancestors(s["parents"])
    cap = s["k_cache"].shape[2]
    pre = s["prefix"].long()
    rel = torch.arange(cap, device="cuda")[None, :] - pre[:, None]  # [B, cap]
    among = seen.gather(2, rel.clamp(0, t - 1)[:, None, :].expand(b, t, cap))
    visible = here[:, :, None] & ((rel < 0)[:, None, :] | ((rel < t)[:, None, :] & (rel >= 0)[:, None, :] & among))
    q = s["q"].float().view(b, t, kvh, h // kvh, d).permute(0, 2, 3, 1, 4).reshape(b, kvh, -1, d)
    score = (q @ s["k_cache"].float().transpose(-1, -2)).mul_(1 / math.sqrt(d)).view(b, kvh, h // kvh, t, cap)
    score.masked_fill_(~visible[:, None, None], NEG)
    score.sub_(score.amax(-1, keepdim=True).clamp(min=-3e38)).exp_()
    score.div_(score.sum(-1, keepdim=True).clamp(min=1e-30))
    o = (score.view(b, kvh, -1, cap) @ s["v_cache"].float()).view(b, kvh, h // kvh, t, d)
    return o.permute(0, 3, 1, 2, 4).reshape(b, t, h, d).to(s["q"].dtype)


def _rotate(x, cos, sin):
    a, b = x.float().chunk(2, dim=-1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)


def _cache(s):
    b, t = s["parents"].shape
    _, depth, here = _ancestors(s["parents"])
    here = here[..., None, None]
    pre = s["prefix"].long()
    pos = pre[:, None] + depth.clamp(min=0)
    cos, sin = s["cos"][pos][:, :, None], s["sin"][pos][:, :, None]
    i = torch.arange(t, device="cuda")
    slot = pre[:, None] + i
    src = pre[:, None] + torch.where(i <= s["accepted"][:, None], s["path"].long(), i)
    rows = torch.arange(b, device="cuda")[:, None].expand(b, t)
    turned = []
    for (q, k, v), k_cache, v_cache in zip(s["new"], s["k_caches"], s["v_caches"]):
        turned.append(torch.where(here, _rotate(q, cos, sin), 0.0).to(q.dtype))
        for cache, new in ((k_cache, _rotate(k, cos, sin).to(k.dtype)), (v_cache, v)):
            cache[rows, :, slot] = torch.where(here, new, cache[rows, :, slot])
            cache[rows, :, slot] = cache[rows, :, src]
    return {"q": turned, "lengths": (pre + s["accepted"] + 1).int(), "k": s["k_caches"], "v": s["v_caches"]}


def _verify(s):
    # 64 bits throughout: a random number that falls next to a border decides by the last digits
    c, parents, tokens = s["case"], s["parents"].long(), s["tokens"]
    b, t = parents.shape
    vocab = c["vocab"]
    rows = torch.arange(b, device="cuda")

    def target(at):
        z = s["logits"][rows, at].double()
        top = z.amax(-1, keepdim=True)
        if c["temp"] == 0:
            best = torch.where(z == top, torch.arange(vocab, device="cuda"), vocab).amin(-1)
            w = torch.zeros_like(z)
            w[rows, best] = 1.0
            return w
        w = ((z - top) / s["temp32"]).exp_()
        return w / w.sum(-1, keepdim=True)

    cur = torch.zeros(b, dtype=torch.int64, device="cuda")
    path = torch.full((b, t), -1, dtype=torch.int32, device="cuda")
    path[:, 0] = 0
    accepted = torch.zeros(b, dtype=torch.int64, device="cuda")
    p = target(cur)
    for i in range(1, t):
        child = parents[:, i] == cur
        x = tokens[:, i]
        u = s["uniforms"][:, i].double()
        px = p[rows, x]
        if s["probs"] is None or c["temp"] == 0:
            ok = child & (u < px)
            left = p.clone()
            left[rows, x] = 0.0
            if c["temp"] == 0:
                left = p
        else:
            q = s["probs"][rows, cur.clamp(max=s["probs"].shape[1] - 1)].double()
            ok = child & (u * q[rows, x] < px)
            left = (p - q).clamp_(min=0.0)
        left = left / left.sum(-1, keepdim=True)
        accepted += ok
        path.scatter_(1, torch.where(ok, accepted, 0)[:, None], torch.where(ok, i, 0).int()[:, None])
        cur = torch.where(ok, i, cur)
        p = torch.where(ok[:, None], target(cur), torch.where(child[:, None], left, p))
    cdf = p.cumsum(-1)
    above = cdf > s["uniforms"][:, :1].double() * cdf[:, -1:]
    nxt = torch.where(above & (p > 0), torch.arange(vocab, device="cuda"), vocab).amin(-1)
    return {"path": path, "accepted": accepted, "next_token": nxt}


def _lora(s):
    c = s["case"]
    tokens, n_ad, r = s["x"].shape[0], c["adapters"], c["rank"]
    if s["q_start"] is None:
        seq = torch.arange(tokens, device="cuda") // (tokens // c["batch"])
    else:
        seq = torch.searchsorted(s["q_start"].long(), torch.arange(tokens, device="cuda"), right=True) - 1
    own_one = s["adapter"].long()[seq][:, None] == torch.arange(n_ad, device="cuda")
    t = (s["x"].float() @ s["a"].float().view(n_ad * r, -1).T).view(tokens, n_ad, r)
    t = t * (own_one * s["scale"])[..., None]
    b_all = s["b"].float().permute(0, 2, 1).reshape(n_ad * r, -1)
    return (s["y"].float() + t.view(tokens, -1) @ b_all).to(s["y"].dtype)


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(c, seed):
    if c["kind"] == "verify":
        return None  # whole numbers
    s = prepare(c, seed)
    if c["kind"] == "lora":
        return _exact_lora(s)
    if c["kind"] == "cache":
        return _exact_cache(s)
    b, t, group, d = c["batch"], c["new"], c["heads"] // c["kv_heads"], c["dim"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    parents = s["parents"].tolist()
    for i, n0 in enumerate(s["prefix"].tolist()):
        mask = torch.zeros(t, n0 + t, dtype=torch.bool)
        for j in range(t):
            at = j if parents[i][j] != -2 else -1
            if at >= 0:
                mask[j, :n0] = True
            while at >= 0:
                mask[j, n0 + at] = True
                at = parents[i][at]
        real = [j for j in range(t) if parents[i][j] != -2]
        mask = mask[real].repeat_interleave(group, 0).cuda()
        for kv in range(c["kv_heads"]):
            k, v = s["k_cache"][i, kv, :n0 + t].double(), s["v_cache"][i, kv, :n0 + t].double()
            q = s["q"][i, real, kv * group:(kv + 1) * group].double().reshape(-1, d)
            w = (q @ k.T / math.sqrt(d)).masked_fill_(~mask, NEG)
            out[i, real, kv * group:(kv + 1) * group] = (torch.softmax(w, dim=-1) @ v).view(len(real), group, d)
    return out


def _exact_cache(s):
    parents, path = s["parents"].tolist(), s["path"].tolist()
    half = s["new"][0][0].shape[-1] // 2
    table = torch.complex(s["cos"].double(), s["sin"].double())
    q = [torch.zeros(n[0].shape, dtype=torch.float64, device="cuda") for n in s["new"]]
    k = [x.double() for x in s["k_caches"]]
    v = [x.double() for x in s["v_caches"]]

    def turn(x, pos):
        z = torch.complex(x[..., :half].double(), x[..., half:].double()) * table[pos]
        return torch.cat([z.real, z.imag], dim=-1)

    for i, n0 in enumerate(s["prefix"].tolist()):
        depth = {}
        for j, up in enumerate(parents[i]):
            if up == -2:
                continue
            depth[j] = depth[up] + 1 if up >= 0 else 0
            for layer, new in enumerate(s["new"]):
                q[layer][i, j] = turn(new[0][i, j], n0 + depth[j])
                k[layer][i, :, n0 + j] = turn(new[1][i, j], n0 + depth[j])
                v[layer][i, :, n0 + j] = new[2][i, j].double()
        n = int(s["accepted"][i]) + 1
        src = torch.tensor([n0 + j for j in path[i][:n]], device="cuda")
        for x in k + v:
            x[i, :, n0:n0 + n] = x[i, :, src].clone()
    return {"q": q, "lengths": None, "k": k, "v": v}


def _exact_lora(s):
    c = s["case"]
    news = _counts(c)
    out, at = s["y"].double(), 0
    for i, ad in enumerate(s["adapter"].tolist()):
        rows = slice(at, at + news[i])
        at += news[i]
        if ad >= 0:
            t = s["x"][rows].double() @ s["a"][ad].double().T
            out[rows] += s["scale"][ad].double() * (t @ s["b"][ad].double().T)
    return out
