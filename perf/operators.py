"""Block-scaled KV pages and the attention that reads them, as measurable cases: rows quantised as they are written, rows read back, and a
chunk of new tokens (one token, the rows of a verify step, a prompt's portion) attending over the pages, with or without a sliding window
whose first tokens stay visible.

A block-scaled cache is a uint8 tensor [pages, 2 (K, V), KH, page, row bytes].  The `page * row bytes` bytes of a (page, half, head) are the
rows' elements, [page, D] e4m3 bytes ("mxfp8") or [page, D / 2] pairs of e2m1 numbers, the even one in the low half ("mxfp4"), and behind
them one byte of scale per block of 32 elements, [page, D / 32].  An element's value is element * 2^(byte - 127); 255 is NaN.  The scale is
the smallest power of two at which no element is more than half a step of its binade off (the largest e4m3 number is 448, so up to 464; e2m1's
is 6, so up to 7), from 2^-100 up to 2^127 over the largest element's binade; elements round to nearest, ties to even.  A block that holds
an infinity or a NaN has scale 255 and elements 0.

Row i of the n_b new rows of a request of len_b tokens is at position t = len_b - n_b + i and sees the positions s <= t with s > t - window or
s < sinks.  Rows that see nothing are 0.
"""
import itertools
import math
from types import SimpleNamespace

import torch

own = False
PAGE = 128
DEV = "cuda:0"
LARGEST = {"mxfp8": (448.0, 8, 1.8125), "mxfp4": (6.0, 2, 1.75)}     # largest element, its binade, mantissa up to which it rounds to it


def listed():
    return [
        # the target's rows of a verify step of the headline benchmark's batch, rotated, quantised, and read back
        dict(name="append-verify-b64-mxfp8", op="append", kind="mxfp8", B=64, n=4, H=32, KH=8, D=128, past=16032, ragged=False, rope=True),
        # a portion of the prompts of the same model, 8192 rows
        dict(name="append-prompt-b64-mxfp4", op="append", kind="mxfp4", B=64, n=128, H=32, KH=8, D=128, past=3968, ragged=False, rope=True),
        # prompts of unequal lengths of a model with heads of 64, whose keys are not rotated here
        dict(name="append-ragged-b7-mxfp8-d64", op="append", kind="mxfp8", B=7, n=301, H=32, KH=4, D=64, past=777, ragged=True, rope=False),
        # what a compression of a few long requests has to read back
        dict(name="read-b8-16k-mxfp4", op="read", kind="mxfp4", B=8, L=16032, H=32, KH=8, D=128, ragged=False),
        dict(name="read-ragged-b5-mxfp8-d64", op="read", kind="mxfp8", B=5, L=2081, H=32, KH=2, D=64, ragged=True),
        # the verify step's attention of the headline benchmark over 8-bit and over 4-bit pages
        dict(name="verify-b64-16k-mxfp8", op="attend", kind="mxfp8", B=64, n=4, L=16036, H=32, KH=8, D=128, window=0, sinks=0, ragged=False),
        dict(name="verify-b64-16k-mxfp4", op="attend", kind="mxfp4", B=64, n=4, L=16036, H=32, KH=8, D=128, window=0, sinks=0, ragged=False),
        # one token of one request behind a long document
        dict(name="token-b1-32k-mxfp4", op="attend", kind="mxfp4", B=1, n=1, L=32065, H=32, KH=8, D=128, window=0, sinks=0, ragged=False),
        # a draft step of the small model that looks at 16 first tokens and a window of its full 16-bit cache
        dict(name="draft-window-b64-bf16-d64", op="attend", kind="bf16", B=64, n=1, L=16033, H=32, KH=8, D=64, window=241, sinks=16, ragged=False),
        # a portion of 128 tokens of sixteen prompts behind 16K
        dict(name="chunk-b16-16k-mxfp8", op="attend", kind="mxfp8", B=16, n=128, L=16160, H=32, KH=8, D=128, window=0, sinks=0, ragged=False),
        # whole prompts of a sliding-window model
        dict(name="prompt-window-b2-4k-bf16", op="attend", kind="bf16", B=2, n=4133, L=4133, H=32, KH=8, D=128, window=1024, sinks=4, ragged=False),
        # continuous batching: requests of unequal lengths with none to a few dozen new tokens, seven query heads on each of four kv heads
        dict(name="mixed-ragged-b9-mxfp4", op="attend", kind="mxfp4", B=9, n=33, L=3001, H=28, KH=4, D=128, window=500, sinks=1, ragged=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    op = rng.choice(["append", "append", "read", "attend", "attend", "attend", "attend"])
    KH, g = rng.choice([1, 2, 4, 8]), rng.choice([1, 4, 5, 7, 8])
    case = dict(op=op, kind=rng.choice(["mxfp8", "mxfp4"]), B=_log(rng, 1, 64), H=KH * g, KH=KH, D=rng.choice([64, 128]), ragged=rng.random() < 0.5)
    if op == "append":
        case.update(n=_log(rng, 1, 8192 // case["B"]), past=_log(rng, 1, 16032), rope=rng.random() < 0.6)
    elif op == "read":
        case.update(L=_log(rng, 1, min(32000, 128000 // case["B"])))
    else:
        n = rng.choice([1, 1, 2, 4, 4, 6, _log(rng, 7, 4096)])
        most = min(32000, 1000000 // case["B"], 900_000_000 // (case["B"] * case["H"] * n))        # keys, and scores in all
        case.update(kind=rng.choice(["mxfp8", "mxfp4", "bf16"]), L=max(n, _log(rng, min(64, most), most)), n=n, window=0, sinks=0)
        if n > most:
            case.update(n=1, L=_log(rng, 1, most))
        if rng.random() < 0.5:
            case.update(window=_log(rng, 1, 2048), sinks=rng.choice([0, 1, 4, 16, 100]))
    return case


def _rows(case):
    """Per request: tokens after the call, and new rows among them."""
    B = case["B"]
    if case["op"] == "read":
        lens = [case["L"] - (b * 7919 % (case["L"] // 2 + 1) if case["ragged"] else 0) for b in range(B)]
        return lens, lens
    new = [(case["n"] - b * 5 % (case["n"] + 1)) if case["ragged"] else case["n"] for b in range(B)]
    if case["op"] == "append":
        return [case["past"] - (b * 7919 % (case["past"] // 2 + 1) if case["ragged"] else 0) + m for b, m in enumerate(new)], new
    return [max(m, case["L"] - (b * 7919 % (case["L"] // 2 + 1) if case["ragged"] else 0)) for b, m in enumerate(new)], new


def _row_bytes(kind, D):
    return 2 * D if kind == "bf16" else (D if kind == "mxfp8" else D // 2) + D // 32


# ------------------------------------------------------------------------------------------------------------ the format, in elementary operations
def quantize(x, kind):
    """[..., D] to (element bytes [..., D] or [..., D / 2], scale bytes [..., D / 32])."""
    largest, binade, full = LARGEST[kind]
    x = x.float().unflatten(-1, (-1, 32))
    amax = x.abs().amax(-1)
    fraction, exponent = torch.frexp(amax)                               # amax = fraction * 2^exponent, fraction from 1/2 to 1
    scale = (exponent - 1 - binade + (2 * fraction > full)).clamp(-100, 127 - binade)
    scale = torch.where(amax == 0, -100, scale)
    finite = torch.isfinite(amax)
    y = torch.where(finite.unsqueeze(-1), torch.ldexp(x, -torch.where(finite, scale, 0).unsqueeze(-1)), 0.0).clamp(-largest, largest)
    scale = torch.where(finite, scale + 127, 255).to(torch.uint8)
    if kind == "mxfp8":
        return y.to(torch.float8_e4m3fn).view(torch.uint8).flatten(-2), scale
    a = y.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    a = torch.round(a / step) * step                                     # 0, 0.5, 1, 1.5, 2, 3, 4, 6
    code = torch.where(a < 2, 2 * a, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8) + 8 * torch.signbit(y).to(torch.uint8)
    code = code.flatten(-2)
    return code[..., 0::2] + 16 * code[..., 1::2], scale


def dequantize(elements, scales, kind):
    """The values, in 32 bits."""
    if kind == "mxfp8":
        v = elements.view(torch.float8_e4m3fn).float()
    else:
        code = torch.stack([elements & 15, elements >> 4], -1).flatten(-2)
        table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=elements.device)
        v = table[(code & 7).long()] * torch.where(code > 7, -1.0, 1.0)
    s = torch.where(scales == 255, math.nan, torch.exp2(scales.float() - 127))
    return (v.unflatten(-1, (-1, 32)) * s.unsqueeze(-1)).flatten(-2)


def _planes(cache, kind, D):
    """Views [pages, 2, KH, page, .] of the elements and of the scales of a block-scaled cache."""
    P, _, KH, page, _ = cache.shape
    flat, eb = cache.view(P, 2, KH, -1), D if kind == "mxfp8" else D // 2
    return flat[..., :page * eb].unflatten(-1, (page, eb)), flat[..., page * eb:].unflatten(-1, (page, D // 32))


# ------------------------------------------------------------------------------------------------------------ inputs
def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _table(lens, gen):
    """A page table whose requests' pages lie in no order: indices, indptr, tokens in the last page."""
    pages = [-(-n // PAGE) for n in lens]
    indptr = [0, *itertools.accumulate(pages)]
    order = torch.randperm(max(1, indptr[-1]), generator=gen, device=DEV)[:indptr[-1]].to(torch.int32)
    return order, _ints(indptr), _ints([(n - 1) % PAGE + 1 if n else 0 for n in lens])


def _keys(shape, gen):
    """Rows as a model's: channels of unequal sizes, a few of them large."""
    size = torch.exp(0.5 * torch.randn(shape[-2:], generator=gen, device=DEV))
    return (torch.randn(shape, generator=gen, device=DEV) * size).to(torch.bfloat16)


def _cache(case, pages, gen):
    KH, D, kind = case["KH"], case["D"], case["kind"]
    if kind == "bf16":
        cache = torch.empty((pages, 2, KH, PAGE, D), dtype=torch.bfloat16, device=DEV)
        for a in range(0, pages, 512):
            n = min(512, pages - a)
            cache[a:a + n] = _keys((n, 2, PAGE, KH, D), gen).transpose(2, 3)
        return cache
    cache = torch.empty((pages, 2, KH, PAGE, _row_bytes(kind, D)), dtype=torch.uint8, device=DEV)
    elements, scales = _planes(cache, kind, D)
    for a in range(0, pages, 512):
        n = min(512, pages - a)
        elements[a:a + n], scales[a:a + n] = quantize(_keys((n, 2, PAGE, KH, D), gen).transpose(2, 3), kind)
    return cache


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    lens, new = _rows(case)
    B, H, KH, D = case["B"], case["H"], case["KH"], case["D"]
    indices, indptr, last = _table(lens, gen)
    cache = _cache(case, max(1, indices.numel()), gen)
    rows, at = sum(new), [0, *itertools.accumulate(new)]
    state = dict(case=case, cache=cache, indices=indices, indptr=indptr, last=last, qo=_ints(at), rows=rows, n_max=max(1, max(new)),
                 longest=max(lens), max_pages=max(1, -(-max(lens) // PAGE)))
    if case["op"] == "append":
        qkv = _keys((rows, H + 2 * KH, D), gen)                                 # one product's output, as the engine slices it
        state.update(q=qkv[:, :H], k=qkv[:, H:H + KH], v=qkv[:, H + KH:], offsets=_ints([n - m for n, m in zip(lens, new)]))
        if case["rope"]:
            freq = 500000.0 ** (-2.0 * torch.arange(D // 2, dtype=torch.float64, device=DEV) / D)
            angle = torch.arange(max(lens) + 1, dtype=torch.float64, device=DEV)[:, None] * freq
            state["turns"] = torch.stack([angle.cos(), angle.sin()], -1).float().contiguous()
    if case["op"] == "attend":
        # scores of a spread that leaves some keys much heavier than others
        state["q"] = (torch.randn((rows, H, D), generator=gen, device=DEV) * (2.4 / 1.28)).to(torch.bfloat16)
    # what rope_append takes of an ops.RopeTable, so that both sides turn by the same 32-bit numbers
    state["rope_table"] = SimpleNamespace(table=state.get("turns"), max_pos=max(lens) + 1, head_dim=D)
    state["scratch"] = {}                                                # the attention's workspace, kept from call to call
    return state


# ------------------------------------------------------------------------------------------------------------ the plain form
def _places(st):
    """Of every new row: its request, its position, its page and its slot there."""
    qo, indptr = st["qo"].long(), st["indptr"].long()
    n = qo[1:] - qo[:-1]
    b = torch.repeat_interleave(torch.arange(n.numel(), device=DEV), n, output_size=st["rows"])
    pages = indptr[1:] - indptr[:-1]
    lens = torch.where(pages > 0, (pages - 1) * PAGE + st["last"].long(), 0)
    pos = lens[b] - n[b] + torch.arange(st["rows"], device=DEV) - qo[:-1][b]
    return b, pos, st["indices"].long()[indptr[b] + pos // PAGE], pos % PAGE


def _read(st, page, slot):
    elements, scales = _planes(st["cache"], st["case"]["kind"], st["case"]["D"])
    return [dequantize(elements[page, h, :, slot], scales[page, h, :, slot], st["case"]["kind"]).to(torch.bfloat16) for h in (0, 1)]


def _turn(x, cs):
    x = x.float().unflatten(-1, (-1, 2))
    c, s = cs[:, None, :, 0], cs[:, None, :, 1]
    return torch.stack([x[..., 0] * c - x[..., 1] * s, x[..., 1] * c + x[..., 0] * s], -1).flatten(-2).to(torch.bfloat16)


def _append_plain(st):
    case = st["case"]
    _, pos, page, slot = _places(st)
    q, k, v = st["q"], st["k"], st["v"]
    if case["rope"]:
        q, k = _turn(q, st["turns"][pos]), _turn(k, st["turns"][pos])
    elements, scales = _planes(st["cache"], case["kind"], case["D"])
    ke, ks = quantize(k, case["kind"])
    ve, vs = quantize(v, case["kind"])
    elements[page, 0, :, slot], scales[page, 0, :, slot] = ke, ks
    elements[page, 1, :, slot], scales[page, 1, :, slot] = ve, vs
    k, v = _read(st, page, slot)
    return (q, k, v) if case["rope"] else (k, v)


def _attend_plain(st):
    case = st["case"]
    B, H, KH, D, L, n_max = case["B"], case["H"], case["KH"], case["D"], st["longest"], st["n_max"]
    qo, indptr = st["qo"].long(), st["indptr"].long()
    n, pages = qo[1:] - qo[:-1], indptr[1:] - indptr[:-1]
    lens = torch.where(pages > 0, (pages - 1) * PAGE + st["last"].long(), 0)
    s = torch.arange(L, device=DEV)
    # [B, L]: every key's page and slot; what lies behind a request's end is not looked at
    held = s < lens[:, None]
    page = st["indices"].long()[torch.where(held, indptr[:-1, None] + s // PAGE, 0)]
    slot = (s % PAGE).expand(B, L)
    if case["kind"] == "bf16":
        k, v = (st["cache"][page, h, :, slot].float() for h in (0, 1))
    else:
        elements, scales = _planes(st["cache"], case["kind"], D)
        k, v = (dequantize(elements[page, h, :, slot], scales[page, h, :, slot], case["kind"]) for h in (0, 1))
    k, v = (torch.where(held[:, :, None, None], x, 0.0).permute(0, 2, 1, 3).contiguous() for x in (k, v))          # [B, KH, L, D]
    i = torch.arange(n_max, device=DEV)
    there = i < n[:, None]
    q = st["q"].float()[torch.where(there, qo[:-1, None] + i, 0)]                                                    # [B, n_max, H, D]
    q = q.unflatten(2, (KH, H // KH)).permute(0, 2, 3, 1, 4).flatten(2, 3).contiguous()                              # [B, KH, g * n_max, D]
    t = torch.where(there, lens[:, None] - n[:, None] + i, -1)[:, :, None]
    seen = (s <= t) & held[:, None, :]
    if case["window"]:
        seen &= (s > t - case["window"]) | (s < case["sinks"])
    seen = seen[:, None, None]                                                                                      # [B, 1, 1, n_max, L]
    p = torch.matmul(q, k.transpose(2, 3)).unflatten(2, (H // KH, n_max)) * (D ** -0.5)
    p = torch.where(seen, p, -math.inf)
    p = torch.exp(p - p.amax(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.flatten(2, 3), v).unflatten(2, (H // KH, n_max))
    out = torch.where(total > 0, out / total, 0.0)
    b = torch.repeat_interleave(torch.arange(B, device=DEV), n, output_size=st["rows"])
    return out.permute(0, 3, 1, 2, 4).flatten(2, 3)[b, torch.arange(st["rows"], device=DEV) - qo[:-1][b]].to(torch.bfloat16)


def run(st):
    case = st["case"]
    if not own:
        if case["op"] == "append":
            return _append_plain(st)
        if case["op"] == "read":
            _, _, page, slot = _places(st)
            return _read(st, page, slot)
        return _attend_plain(st)
    from magicdec_amd import ops
    table = (st["indices"], st["indptr"], st["last"])
    if case["op"] == "attend":
        if "ws" not in st["scratch"]:
            st["scratch"]["ws"] = ops.AttnWorkspace(DEV)
        return ops.paged_attention(st["q"], st["cache"], st["qo"], *table, st["n_max"], st["max_pages"], st["scratch"]["ws"], kv_layout="HND",
                                   window=case["window"] or None, sinks=case["sinks"])
    q = None
    if case["op"] == "append":
        if case["rope"]:
            q = ops.rope_append(st["q"], st["k"], st["v"], st["qo"], st["offsets"], st["rope_table"], st["cache"], *table, n_max=st["n_max"],
                                kv_layout="HND")
        else:
            ops.update_kv(st["k"], st["v"], st["qo"], st["cache"], *table, n_max=st["n_max"], kv_layout="HND")
    k, v = (torch.empty((st["rows"], case["KH"], case["D"]), dtype=torch.bfloat16, device=DEV) for _ in (0, 1))
    ops.read_kv(k, v, st["qo"], st["cache"], *table, n_max=st["n_max"], kv_layout="HND")
    return (k, v) if q is None else (q, k, v)


# ------------------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    lens, new = _rows(case)
    H, KH, D, rows = case["H"], case["KH"], case["D"], sum(new)
    row = 2 * KH * _row_bytes(case["kind"], D)
    if case["op"] == "append":
        moved = rows * (2 * KH * D * 2 + row + 2 * KH * D * 2)                                 # rows in, pages out, values out
        if case["rope"]:
            moved += rows * (2 * H * D * 2 + D * 4)
        return {"bytes": moved, "flops": rows * (H + KH) * D * 3 if case["rope"] else 0}
    if case["op"] == "read":
        return {"bytes": rows * (row + 2 * KH * D * 2), "flops": 0}
    keys = pairs = 0
    for n, m in zip(lens, new):
        if m == 0:
            continue
        w, sinks = case["window"], case["sinks"]
        for_all = 0
        if not w:
            for_all, keys = sum(range(n - m + 1, n + 1)), keys + n
        else:
            first = max(0, n - m + 1 - w)                                                      # of the window of the first row
            keys += n - first + min(first, sinks)
            for t in range(n - m, n):
                a = max(0, t + 1 - w)
                for_all += t + 1 - a + min(a, sinks)
        pairs += for_all
    return {"bytes": keys * row + 2 * rows * H * D * 2, "flops": 4 * pairs * H * D}


# ------------------------------------------------------------------------------------------------------------ from the definition, in 64 bits
def _grid(kind):
    """Every non-negative element, in the order of its code."""
    if kind == "mxfp4":
        return [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
    return [(m / 8 if e == 0 else 1 + m / 8) * 2.0 ** (max(e, 1) - 7) for e in range(16) for m in range(8)][:127]


def _stored64(x, kind):
    """What a block-scaled cache holds for rows x."""
    grid = torch.tensor(_grid(kind), dtype=torch.float64, device=x.device)
    x = x.double().unflatten(-1, (-1, 32))
    amax = x.abs().amax(-1, keepdim=True)
    top = float(grid[-1])
    half = (top - float(grid[-2])) / 2
    lowest, highest = -100, 127 - int(math.log2(top))
    # the smallest scale under which the largest element is at most half a step above the largest number
    e = torch.ceil(torch.log2(amax.clamp_min(1e-300) / (top + half)))
    e = e.clamp(lowest, highest)
    y = (x.abs() / torch.exp2(e)).clamp(max=top)
    above = torch.searchsorted(grid, y.contiguous()).clamp(max=grid.numel() - 1)
    below = (above - 1).clamp(min=0)
    up, down = grid[above] - y, y - grid[below]
    code = torch.where((up < down) | ((up == down) & (above % 2 == 0)), above, below)
    return (torch.sign(x) * grid[code] * torch.exp2(e)).flatten(-2)


def _of_pages64(st):
    """Values of the whole cache from its bytes, [pages, KH, page, D] of K and of V."""
    case = st["case"]
    KH, D, kind = case["KH"], case["D"], case["kind"]
    if kind == "bf16":
        return [st["cache"][:, h].double() for h in (0, 1)]
    raw = st["cache"].flatten(3)
    eb = PAGE * (D if kind == "mxfp8" else D // 2)
    codes, scale = raw[..., :eb].int(), raw[..., eb:].unflatten(-1, (PAGE, D // 32)).double()
    if kind == "mxfp4":
        codes = torch.stack([codes % 16, codes // 16], -1).flatten(3)
    codes = codes.unflatten(3, (PAGE, D))
    half = 128 if kind == "mxfp8" else 8
    grid = torch.tensor(_grid(kind), dtype=torch.float64, device=DEV)
    v = grid[codes % half] * (1 - 2 * (codes // half))
    v = (v.unflatten(-1, (-1, 32)) * torch.exp2(scale - 127).unsqueeze(-1)).flatten(-2)
    return v[:, 0], v[:, 1]


def exact(case, seed):
    st = prepare(case, seed)
    lens, new = _rows(case)
    H, KH, D = case["H"], case["KH"], case["D"]
    at, starts = st["qo"].tolist(), st["indptr"].tolist()
    if case["op"] == "append":
        if not case["rope"]:
            return _stored64(st["k"], case["kind"]), _stored64(st["v"], case["kind"])
        pos = torch.cat([torch.arange(n - m, n, device=DEV) for n, m in zip(lens, new)]).long()
        turn = torch.view_as_complex(st["turns"].double())[pos][:, None]
        q = torch.view_as_real(torch.view_as_complex(st["q"].double().unflatten(-1, (-1, 2)).contiguous()) * turn).flatten(-2)
        return q, None, _stored64(st["v"], case["kind"])          # (a rotated key next to a border of its rounding has two neighbours)
    # a request at a time, so that 64 bits of a large cache need not lie in memory at once
    out, ks, vs = [], [], []
    for b, (n, m) in enumerate(zip(lens, new)):
        mine = st["indices"][starts[b]:starts[b + 1]].long()
        k, v = (x.transpose(0, 1).flatten(1, 2)[:, :n] for x in _of_pages64(dict(case=case, cache=st["cache"][mine])))   # [KH, n, D]
        if case["op"] == "read":
            ks.append(k.transpose(0, 1))
            vs.append(v.transpose(0, 1))
            continue
        q = st["q"][at[b]:at[b + 1]].double().unflatten(1, (KH, -1))                                                # [m, KH, g, D]
        o = torch.zeros_like(q)
        t = torch.arange(n - m, n, device=DEV)[:, None]
        s = torch.arange(n, device=DEV)
        hidden = s > t
        if case["window"]:
            hidden = hidden | ((s <= t - case["window"]) & (s >= case["sinks"]))
        for h in range(KH if m else 0):
            w = (q[:, h].flatten(0, 1) @ k[h].T / math.sqrt(D)).unflatten(0, (m, -1)).masked_fill_(hidden[:, None], -math.inf)
            o[:, h] = torch.softmax(w, -1) @ v[h]
        out.append(o.flatten(1, 2))
    return torch.cat(out) if case["op"] == "attend" else (torch.cat(ks), torch.cat(vs))
