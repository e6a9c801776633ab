"""The 4-bit paged cache in plain torch: coding, block layout, reading and
attention in 64 bits, written from the layout that include/fitq.h states, element
by element (no code shared with the library)."""
import math

import torch


def fp32(x):
    return torch.tensor(x, dtype=torch.float32)


def code_group(x):
    """(codes, scale, low) of x [..., 64] fp32, each step rounded to fp32."""
    low = x.amin(-1, keepdim=True).half()
    scale = ((x.amax(-1, keepdim=True) - low.float()) * (fp32(1.0) / fp32(15.0)).to(x.device)).half()
    inv = torch.ones_like(scale, dtype=torch.float32) / scale.float()
    code = torch.where(scale > 0, torch.round((x - low.float()) * inv), torch.zeros_like(x)).clamp(0, 15)
    return code.nan_to_num(0).to(torch.uint8), scale, low


def coded_values(x):
    """The fp32 values that x [..., D] (fp32) stands for once coded."""
    c, s, l = code_group(x.unflatten(-1, (-1, 64)))
    return (c.float() * s.float() + l.float()).flatten(-2)


def rotate(x, cos, sin):
    """Rotate-half of x [n, heads, D] in fp32, products and sums rounded one by one."""
    a, b = x.float().chunk(2, dim=-1)
    cos, sin = cos[:, None], sin[:, None]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)


def offsets(dim):
    """Byte and shift of every (block position, element) of keys and values, and the
    byte of its (scale, low) pair for each side."""
    G = dim // 64
    kb, vb, sh, pb = (torch.zeros(16, dim, dtype=torch.long) for _ in range(4))
    for p in range(16):
        for d in range(dim):
            g, f = d // 64, d % 64
            c, w, j = f // 16, (f % 16) // 8, f % 8
            kb[p, d] = ((((p * 4 + c) * G + g) * 2 + w) * 4) + j // 2
            h, q, o, e = p // 8, (p % 8) // 2, p % 2, f // 8
            vb[p, d] = 8 * dim + ((((h * 8 + e) * 4 + q) * 2 + o) * G + g) * 4 + j // 2
            sh[p, d] = 4 * (j % 2)
            pb[p, d] = 16 * dim + (p * 2 * G + g) * 4
    return kb, vb, sh, pb


def read_blocks(blocks):
    """(k, v) float64 [..., 16, D] of uint8 blocks [..., 18 D]."""
    dim = blocks.shape[-1] // 18
    kb, vb, sh, pb = (t.to(blocks.device) for t in offsets(dim))

    def pair(byte):
        raw = torch.stack([blocks[..., byte], blocks[..., byte + 1]], dim=-1).contiguous()
        return raw.view(torch.float16)[..., 0].double()

    out = []
    for side, at in ((0, kb), (1, vb)):
        code = (blocks[..., at].long() >> sh) & 15
        base = pb + side * (dim // 64) * 4
        out.append(code.double() * pair(base) + pair(base + 2))
    return out


def read_sequence(pool, table_row, length):
    """(k, v) float64 [KVH, length, D] behind one row of a page table (pages that do
    not exist read as NaN)."""
    pages, kvh, per, nbytes = pool.shape
    ps = per * 16
    n = -(-length // ps)
    rows = [int(x) for x in table_row[:n]]
    blocks = torch.stack([pool[p] if 0 <= p < pages else torch.full_like(pool[0], 255) for p in rows])
    k, v = read_blocks(blocks)  # [n, KVH, per, 16, D]
    return [x.permute(1, 0, 2, 3, 4).reshape(kvh, n * ps, -1)[:, :length] for x in (k, v)]


def attention(q, pool, table, prefix, starts, counts):
    """o float64 [tokens, H, D]; NaN rows for tokens of no sequence."""
    h, d = q.shape[1], q.shape[2]
    kvh = pool.shape[1]
    out = torch.full(q.shape, float("nan"), dtype=torch.float64, device=q.device)
    for b, (pre, a, n) in enumerate(zip(prefix, starts, counts)):
        if n == 0:
            continue
        k, v = read_sequence(pool, table[b], pre + n)
        qq = q[a:a + n].double()
        hidden = torch.arange(pre + n, device=q.device)[None] > torch.arange(pre, pre + n, device=q.device)[:, None]
        for i in range(h):
            s = (qq[:, i] @ k[i // (h // kvh)].T / math.sqrt(d)).masked_fill(hidden, float("-inf"))
            out[a:a + n, i] = torch.softmax(s, -1) @ v[i // (h // kvh)]
    return out


def random_pool(pages, kvh, ps, dim, g, dev):
    """A pool of random codes whose groups have scales in 0.1..0.3 and small means."""
    pool = torch.randint(0, 256, (pages, kvh, ps // 16, 18 * dim), generator=g, device=dev, dtype=torch.uint8)
    par = pool[..., 16 * dim:].view(torch.float16).view(pages, kvh, ps // 16, 16, 2, dim // 64, 2)
    scale = torch.rand(par.shape[:-1], generator=g, device=dev) * 0.2 + 0.1
    par[..., 0] = scale.half()
    par[..., 1] = (torch.randn(scale.shape, generator=g, device=dev) * 0.1 - 7.5 * scale).half()
    return pool


def page_table(lengths, ps, g, dev, spare=2):
    """(table, pages): distinct pages in random order, -1 behind each sequence."""
    need = [max(0, -(-n // ps)) for n in lengths]
    order = torch.randperm(sum(need) + spare, generator=g, device=dev).int()
    table = torch.full((len(lengths), max(1, max(need))), -1, dtype=torch.int32, device=dev)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, sum(need) + spare


def tables(length, dim, dev, theta=1e6):
    inv = 1.0 / (theta ** (torch.arange(0, dim, 2, device=dev, dtype=torch.float64) / dim))
    a = torch.outer(torch.arange(length, device=dev, dtype=torch.float64), inv)
    return a.cos().float().contiguous(), a.sin().float().contiguous()
