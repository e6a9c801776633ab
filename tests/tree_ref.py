"""Plain restatements in 64 bits of the calls on trees of drafted tokens and of the
adapters of many requests, one sequence and one token at a time."""
import math

import torch

EPS = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def lineage(parents):
    """{token: (its ancestors and itself, its depth)} of the tokens that are there."""
    out = {}
    for i, up in enumerate(parents):
        if up == -1:
            out[i] = ([i], 0)
        elif 0 <= up < i and up in out:
            out[i] = (out[up][0] + [i], out[up][1] + 1)
    return out


def attention(q, k_cache, v_cache, prefix, parents):
    """[B, T, H, D] in 64 bits; visible slots only are looked at."""
    b, t, h, d = q.shape
    kvh = k_cache.shape[1]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    for s in range(b):
        n0 = int(prefix[s])
        for i, (line, _) in lineage(parents[s]).items():
            slots = torch.tensor(list(range(n0)) + [n0 + j for j in line], device=q.device)
            k, v = (c[s].double().index_select(1, slots).repeat_interleave(h // kvh, 0) for c in (k_cache, v_cache))
            w = torch.softmax(torch.einsum("hd,hnd->hn", q[s, i].double(), k) / math.sqrt(d), dim=-1)
            out[s, i] = torch.einsum("hn,hnd->hd", w, v)
    return out


def rotate(x, angle_cos, angle_sin):
    a, b = x.double().chunk(2, dim=-1)
    c, s = angle_cos.double(), angle_sin.double()
    return torch.cat([a * c - b * s, b * c + a * s], dim=-1)


def verify(logits, tokens, parents, uniforms, probs, temperature):
    """(path, accepted, next_token) of one sequence, lists and numbers of the host."""
    v = logits.shape[-1]

    def target(row):
        z = logits[row].double().cpu()
        if torch.isnan(z).any() or z.max() == -math.inf or (temperature != 0 and z.max() == math.inf):
            return None
        if temperature == 0:
            p = torch.zeros(v, dtype=torch.float64)
            p[int((z == z.max()).nonzero()[0])] = 1.0
            return p
        return torch.softmax(z / float(torch.tensor(temperature, dtype=torch.float32)), dim=-1)

    if parents[0] != -1:
        return [], -1, -1
    path, cur = [0], 0
    p = target(0)
    for i in range(1, len(parents)):
        if p is None or parents[i] != cur:
            continue
        x = int(tokens[i])
        known = 0 <= x < v
        if known and (p[x] > 0 if temperature == 0 else
                      float(uniforms[i]) * (float(probs[cur, x]) if probs is not None else 1.0) < p[x]):
            path.append(i)
            cur = i
            p = target(i)
        elif temperature != 0:
            if probs is not None:
                p = (p - probs[cur].double().cpu()).clamp(min=0)
            elif known:
                p = p.clone()
                p[x] = 0
            if p.sum() > 0:
                p = p / p.sum()
            else:
                break
    if p is None:
        return path, len(path) - 1, -1
    if not p.sum() > 0:
        z = logits[cur].double().cpu()
        return path, len(path) - 1, int((z == z.max()).nonzero()[0])
    c = p.cumsum(0)
    above = ((c > float(uniforms[0]) * c[-1]) & (p > 0)).nonzero()
    return path, len(path) - 1, int(above[0]) if len(above) else int((p > 0).nonzero()[-1])


def multi_lora(x, a, b, scale, adapter, y, starts):
    """[tokens, N] in 64 bits; rows of no sequence as in y."""
    out = y.double().clone()
    for s, l in enumerate(adapter.tolist()):
        r = slice(starts[s], starts[s + 1])
        if l >= 0:
            out[r] += scale[l].double() * ((x[r].double() @ a[l].double().T) @ b[l].double().T)
    return out


def multi_lora_bound(x, a, b, scale, adapter, y, starts, dtype):
    """How far a result may lie from the one in 64 bits: one rounding of the result; x.A^T as
    two numbers of dtype, eps^2 of it; fp32 sums of K and of 2 R products and the sum over at
    most 64 parts, each step 2^-24 of the sum of magnitudes."""
    k, r2 = x.shape[1], 2 * a.shape[1]
    eps, e32 = EPS[dtype], 2.0 ** -24
    out = torch.zeros(y.shape, dtype=torch.float64, device=y.device)
    for s, l in enumerate(adapter.tolist()):
        r = slice(starts[s], starts[s + 1])
        if l >= 0:
            mag = (x[r].double().abs() @ a[l].double().abs().T) @ b[l].double().abs().T * scale[l].double().abs()
            out[r] = mag * (eps * eps + e32 * (k + 64 + r2 + 4))
    exact = multi_lora(x, a, b, scale, adapter, y, starts)
    return out + exact.abs() * eps * 1.001 + 1e-7 * (dtype == torch.float16) + 1e-30
