"""Plain 64-bit statements of the block-scaled cache (include/magicdec_hip.h: MD_KV_MXFP8, MD_KV_MXFP4) and of attention with a sliding window and
first tokens that stay visible, for the tests of both."""
import math

import torch

GRID = {"mxfp4": [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0],
        "mxfp8": [(m / 8 if e == 0 else 1 + m / 8) * 2.0 ** (max(e, 1) - 7) for e in range(16) for m in range(8)][:127]}
U_BF16, U_F32 = 2.0 ** -8, 2.0 ** -24


def element_bytes(kind, D):
    return {"bf16": 2 * D, "fp8": D, "mxfp8": D, "mxfp4": D // 2}[kind]


def quantize(x, kind):
    """Rows [..., D] of bf16 to (codes [..., D], scale bytes [..., D / 32]): by trying every scale from the smallest on."""
    grid = torch.tensor(GRID[kind], dtype=torch.float64)
    top, step = float(grid[-1]), float(grid[-1] - grid[-2])
    x = x.double().unflatten(-1, (-1, 32))
    amax = x.abs().amax(-1)
    binade = int(math.floor(math.log2(top)))
    e = torch.full(amax.shape, -100, dtype=torch.int64)
    while True:
        more = torch.isfinite(amax) & (amax > (top + step / 2) * 2.0 ** e.double()) & (e < 127 - binade)
        if not more.any():
            break
        e += more
    y = (x / 2.0 ** e.double().unsqueeze(-1)).abs().nan_to_num(0.0, 0.0).clamp(max=top)
    d = (y.unsqueeze(-1) - grid).abs()
    odd = torch.arange(grid.numel()) % 2
    near = d == d.amin(-1, keepdim=True)
    code = torch.where(near, torch.arange(grid.numel()) * 2 + odd * 10000, 10 ** 8).argmin(-1)           # ties: the even code
    code = code + (GRID_HALF[kind] * torch.signbit(x)).long()
    bad = ~torch.isfinite(amax)
    code = torch.where(bad.unsqueeze(-1), 0, code)
    return code.flatten(-2).to(torch.uint8), torch.where(bad, 255, e + 127).to(torch.uint8)


GRID_HALF = {"mxfp4": 8, "mxfp8": 128}


def dequantize(code, scale, kind):
    half = GRID_HALF[kind]
    grid = torch.tensor(GRID[kind] + [math.nan] * (half - len(GRID[kind])), dtype=torch.float64)
    code = code.long()
    v = grid[code % half] * torch.where(code >= half, -1.0, 1.0)
    s = torch.where(scale == 255, math.nan, 2.0 ** (scale.double() - 127))
    return (v.unflatten(-1, (-1, 32)) * s.unsqueeze(-1)).flatten(-2)


def pack(code, scale, kind):
    """Codes [pages, 2, KH, page, D] and scales [pages, 2, KH, page, D / 32] as a cache's bytes."""
    if kind == "mxfp4":
        code = code[..., 0::2] + 16 * code[..., 1::2]
    P, two, KH, page, eb = code.shape
    return torch.cat([code.flatten(3), scale.flatten(3)], -1).view(P, two, KH, page, -1).contiguous()


def unpack(cache, kind, D):
    P, two, KH, page, _ = cache.shape
    eb = element_bytes(kind, D)
    raw = cache.flatten(3)
    code, scale = raw[..., :page * eb].unflatten(3, (page, eb)), raw[..., page * eb:].unflatten(3, (page, D // 32))
    if kind == "mxfp4":
        code = torch.stack([code & 15, code >> 4], -1).flatten(4)
    return code, scale


def table(lens, page, seed=0, spare=2):
    """A page table in no order: (indices, indptr, last_page_len, pages of the cache, most pages of a request)."""
    pages = [-(-n // page) for n in lens]
    order = torch.randperm(sum(pages) + spare, generator=torch.Generator().manual_seed(seed))
    indptr = torch.tensor([0] + pages).cumsum(0)
    last = [(n - 1) % page + 1 if n else 0 for n in lens]
    return (order[:sum(pages)].to(torch.int32), indptr.to(torch.int32), torch.tensor(last, dtype=torch.int32), sum(pages) + spare, max(1, max(pages)))


def indptr_of(rows):
    return torch.tensor([0] + list(rows)).cumsum(0).to(torch.int32)


def request_rows(values, indices, indptr, b, n):
    """Values [pages, 2, KH, page, D] of request b's n tokens: (k, v) [n, KH, D]."""
    mine = values[indices[int(indptr[b]):int(indptr[b + 1])].long()]
    kv = mine.permute(1, 0, 3, 2, 4).flatten(1, 2)[:, :n]
    return kv[0], kv[1]


def window_attention(q, values, lens, rows, indices, indptr, window, sinks, scale=None):
    """(out, sum of weight * |value|) [rows, H, D] in 64 bits; hidden keys have no part in either, whatever they hold."""
    H, D = q.shape[1:]
    out, size = [], []
    at = 0
    for b, (n, m) in enumerate(zip(lens, rows)):
        qb = q[at:at + m].double()
        at += m
        k, v = (x.double() for x in request_rows(values, indices, indptr, b, n))
        g = H // values.shape[2]
        t = (n - m + torch.arange(m))[:, None]
        s = torch.arange(n)
        seen = s <= t
        if window:
            seen = seen & ((s > t - window) | (s < sinks))
        o, a = torch.zeros(m, H, D, dtype=torch.float64), torch.zeros(m, H, D, dtype=torch.float64)
        for h in range(H):
            x = (qb[:, h] @ k[:, h // g].T) * (1 / math.sqrt(D) if scale is None else scale)
            w = torch.softmax(torch.where(seen, x, -math.inf), -1) if n else x
            w = torch.where(seen.any(-1, keepdim=True), w, 0.0)
            vh = v[:, h // g]
            if torch.isfinite(vh).all():
                o[:, h], a[:, h] = w @ vh, w @ vh.abs()
            else:
                prod = torch.where(seen[..., None], w[..., None] * vh, 0.0)
                o[:, h], a[:, h] = prod.sum(1), prod.abs().sum(1)
        out.append(o)
        size.append(a)
    return torch.cat(out), torch.cat(size)


def attention_bound(size, q, values, scale=None):
    """How far a row may be off: the weights are rounded to bf16 in front of the product and the result behind it, half a step (2^-8 of the value)
    each.  Scores are 32-bit sums of D products, off by (D + 2) 2^-24 of |q| |k| at most, and the exponential of a score off by e is off by e of
    itself; the weights' 32-bit sum and the reference's changes add a few 2^-24, for which 16 stand."""
    D = q.shape[-1]
    finite = torch.where(torch.isfinite(values[:, 0]), values[:, 0], 0.0)
    most = q.double().norm(dim=-1).max() * finite.double().norm(dim=-1).max() * (1 / math.sqrt(D) if scale is None else scale)
    e = 2 * (D + 2) * U_F32 * float(most) + 16 * U_F32
    return (2 * U_BF16 + 2 * e) * (1 + U_BF16) * size + 1e-37
