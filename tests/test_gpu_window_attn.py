"""Attention with a sliding window and first tokens that stay visible, and attention over block-scaled pages, against 64 bits."""
import math

import pytest
import torch

from tests import mx_util as mx
from tests.conftest import parity_report

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16
F8 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def ops():
    from magicdec_amd import ops as _ops
    _ops._lib.load()
    return _ops


def caches(kind, pages, KH, page, D, seed, ops, layout="HND", edit=None):
    """(the cache on the GPU, its kv_scales, the values it stands for [pages, 2, KH, page, D])."""
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(pages, 2, KH, page, D, generator=g) * torch.exp(0.5 * torch.randn(KH, 1, D, generator=g))).to(BF)
    if edit is not None:
        edit(x)
    if kind == "bf16":
        values, cache, scales = x, x, None
    elif kind == "fp8":
        ks, vs = 0.02 * (1 + torch.arange(KH, dtype=torch.float32)), 0.01 / (1 + torch.arange(KH, dtype=torch.float32))
        s = torch.stack([ks, vs])[None, :, :, None, None]
        cache = (x.float() / s).clamp(-448, 448).to(F8)
        values, scales = cache.float().double() * s.double(), (ks.to(DEV), vs.to(DEV))
    else:
        code, scale = mx.quantize(x, kind)
        return mx.pack(code, scale, kind).to(DEV), None, mx.dequantize(code, scale, kind)
    if layout == "NHD":
        cache = cache.transpose(2, 3).contiguous()
    return cache.to(DEV), scales, values


def attend(ops, q, cache, rows, lens, page, tab, window, sinks, scales=None, layout="HND", ws=None, n_max=None, most=None, **more):
    indices, indptr, last = tab[:3]
    return ops.paged_attention(q.to(DEV), cache, mx.indptr_of(rows).to(DEV), indices.to(DEV), indptr.to(DEV), last.to(DEV), n_max or max(1, max(rows)),
                               most or tab[4],
                               ws or ops.AttnWorkspace(DEV), kv_scales=scales, kv_layout=layout, window=window or None, sinks=sinks, **more)


def check(tag, out, want, size, bound):
    got = out.cpu().double()
    assert not got.isnan().any(), f"{tag}: NaN"
    ratio = (got - want).abs() / bound
    parity_report(f"[window attn] {tag:60s} max err/bound {ratio.max().item():.3f}  rms error {((got - want).norm() / want.norm().clamp_min(1e-30)).item():.2e}")
    assert bool((got[size == 0] == 0).all())
    assert ratio.max().item() <= 1.0, tag


# (name, D, H, KH, page, tokens of a request, new rows of it, window, sinks)
CASES = [
    ("token", 128, 8, 2, 128, [300, 1, 128, 33], [1, 1, 1, 1], 0, 0),
    ("token-d64-page32", 64, 6, 3, 32, [97, 32, 1], [1, 1, 1], 0, 0),
    ("token-long-split", 128, 8, 1, 128, [5003], [1], 0, 0),
    ("verify", 128, 32, 8, 128, [300, 257, 4], [4, 4, 4], 0, 0),
    ("verify-g5", 128, 10, 2, 128, [500, 129], [4, 4], 0, 0),
    ("verify-split-d64", 64, 8, 2, 128, [3001, 1700], [4, 4], 0, 0),
    ("seven-heads", 128, 14, 2, 128, [700, 90], [3, 5], 0, 0),
    ("no-rows-no-tokens", 64, 8, 2, 128, [0, 200, 7, 0], [0, 2, 0, 3], 0, 0),
    ("more-rows-than-tokens", 128, 4, 1, 128, [3, 130], [9, 2], 0, 0),
    ("chunk", 128, 8, 2, 128, [384, 130], [128, 130], 0, 0),
    ("chunk-d64-odd", 64, 12, 4, 64, [301, 77, 64], [45, 77, 1], 0, 0),
    ("chunk-behind-split", 128, 4, 1, 128, [2500], [40], 0, 0),
    ("prompt", 128, 4, 1, 128, [611], [611], 0, 0),
    ("prompt-d64", 64, 4, 2, 128, [700, 515], [700, 515], 0, 0),
    ("one-head", 64, 1, 1, 32, [1000], [7], 0, 0),
    ("window-1", 128, 8, 2, 128, [300, 1, 50], [1, 1, 2], 1, 0),
    ("window-1-sink-1", 64, 8, 2, 128, [300, 1, 50], [1, 1, 30], 1, 1),
    ("window-token", 128, 8, 2, 128, [1000, 40, 257], [1, 1, 1], 100, 4),
    ("window-verify-edge", 128, 8, 2, 128, [292, 291, 96], [4, 4, 4], 33, 32),
    ("window-sinks-meet", 64, 8, 2, 128, [200, 150], [4, 4], 64, 130),
    ("window-sinks-over-tiles", 128, 16, 4, 128, [2000, 1500], [5, 3], 200, 300),
    ("window-chunk", 128, 8, 2, 128, [900, 300], [130, 300], 100, 16),
    ("window-chunk-d64", 64, 8, 2, 32, [900, 65], [257, 65], 65, 3),
    ("window-prompt", 128, 4, 1, 128, [1300], [1300], 250, 0),
    ("window-longer-than-all", 128, 8, 2, 128, [300, 20], [3, 20], 5000, 2),
    ("window-split", 128, 4, 1, 128, [6000], [2], 3000, 700),
    ("window-ragged", 64, 7, 1, 128, [777, 0, 130, 2000], [33, 0, 1, 19], 127, 1),
]
KINDS = ["bf16", "fp8", "mxfp8", "mxfp4"]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("name,D,H,KH,page,lens,rows,window,sinks", CASES, ids=[c[0] for c in CASES])
def test_against_64_bits(ops, kind, name, D, H, KH, page, lens, rows, window, sinks):
    if kind in ("bf16", "fp8") and not window:
        window = 1 << 20                                       # (no window over these caches is md_paged_attn)
    tab = mx.table(lens, page, seed=len(name))
    layout = "NHD" if kind in ("bf16", "fp8") and len(name) % 2 else "HND"
    cache, scales, values = caches(kind, tab[3], KH, page, D, 5, ops, layout)
    q = (2 * torch.randn(sum(rows), H, D, generator=torch.Generator().manual_seed(1))).to(BF)
    want, size = mx.window_attention(q, values, lens, rows, tab[0], tab[1], window, sinks)
    out = attend(ops, q, cache, rows, lens, page, tab, window, sinks, scales, layout)
    check(f"{kind}/{name}", out, want, size, mx.attention_bound(size, q, values))


# Each way in which rows and keys are laid over workgroups: the bounds that a caller gives (rows and pages of a request, at most) choose it, whatever
# lies in them.  (name, D, H, KH, page, tokens, new rows, window, sinks, n_max, pages)
PLANS = [
    ("row-groups-of-32", 64, 8, 4, 128, [60 + 5 * b for b in range(25)], [b % 21 for b in range(25)], 0, 0, 20, 1),
    ("row-groups-of-32-d128", 128, 8, 4, 128, [60 + 5 * b for b in range(25)], [b % 21 for b in range(25)], 40, 3, 20, 2),
    ("64-splits", 128, 8, 1, 128, [700], [2], 0, 0, 2, 700),
    ("64-splits-tiles-of-64", 64, 8, 1, 128, [1500], [2], 0, 0, 2, 700),
    ("64-splits-window", 64, 8, 1, 64, [1500, 3], [2, 1], 1000, 100, 2, 1400),
    ("one-part-tiles-of-64", 64, 2, 2, 64, [800 + 3 * b for b in range(70)], [1] * 70, 0, 0, 1, 300),
    ("4-waves-32-splits", 128, 4, 1, 128, [900], [30], 0, 0, 30, 300),
    ("8-waves-32-splits", 128, 1, 1, 128, [700], [300], 0, 0, 300, 470),
    ("8-waves-32-splits-d64", 64, 1, 1, 128, [700], [300], 100, 4, 300, 470),
    ("8-waves-whole", 128, 2, 1, 128, [300, 150, 0, 260], [300, 131, 0, 257], 0, 0, 4000, 60),
    ("8-waves-page-64", 128, 1, 1, 64, [700], [300], 0, 0, 300, 940),
    ("8-waves-page-96", 128, 1, 1, 96, [700], [300], 130, 70, 300, 700),
    ("8-waves-page-32-d64", 64, 1, 1, 32, [700], [300], 130, 7, 300, 1900),
    ("4-waves-page-32", 128, 5, 1, 32, [300, 40], [13, 9], 0, 0, 13, 10),
    ("4-waves-page-160", 128, 5, 1, 160, [400, 40], [13, 9], 50, 20, 13, 3),
    ("4-waves-page-96-d64", 64, 5, 1, 96, [300, 40], [13, 9], 50, 20, 13, 4),
    ("few-of-8-waves", 128, 4, 1, 128, [600, 200], [30, 32], 0, 0, 32, 5),
    ("tokens-page-96", 128, 8, 2, 96, [300, 97, 5], [1, 2, 3], 0, 0, 3, 4),
    ("far-more-rows-allowed", 64, 8, 2, 128, [300, 97, 5], [1, 2, 3], 0, 0, 2000, 4),
]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("name,D,H,KH,page,lens,rows,window,sinks,n_max,most", PLANS, ids=[c[0] for c in PLANS])
def test_every_layout_of_the_work(ops, kind, name, D, H, KH, page, lens, rows, window, sinks, n_max, most):
    if kind in ("bf16", "fp8") and not window:
        window = 1 << 20
    tab = mx.table(lens, page, seed=len(name))
    cache, scales, values = caches(kind, tab[3], KH, page, D, 5, ops)
    # queries as a slice of a wider product's output
    wide = (2 * torch.randn(sum(rows), H + 3, D, generator=torch.Generator().manual_seed(1))).to(BF)
    q = wide[:, 1:H + 1]
    want, size = mx.window_attention(q, values, lens, rows, tab[0], tab[1], window, sinks)
    out = torch.full((sum(rows), H, D), 7.0, dtype=BF, device=DEV)
    dq = wide.to(DEV)[:, 1:H + 1]
    got = ops.paged_attention(dq, cache, mx.indptr_of(rows).to(DEV), *(t.to(DEV) for t in tab[:3]), n_max, most, ops.AttnWorkspace(DEV), out=out,
                              kv_scales=scales, kv_layout="HND", window=window or None, sinks=sinks)
    assert got.data_ptr() == out.data_ptr()
    check(f"{kind}/{name}", got, want, size, mx.attention_bound(size, q, values))


# Four and eight wavefronts that share tiles, of every length, whole and in parts, pairs of request and kv head in eights and not: as above, by the
# bounds.  (D, H, KH, page, requests, window, sinks, n_max, pages)
SHARED = [
    (64, 8, 8, 128, 3, 0, 0, 300, 40), (64, 4, 1, 128, 3, 0, 0, 300, 40), (64, 8, 2, 128, 3, 0, 0, 1100, 2), (64, 4, 1, 64, 5, 100, 3, 520, 2),
    (64, 4, 1, 96, 3, 0, 0, 130, 300), (64, 8, 8, 96, 3, 100, 3, 520, 2), (64, 4, 1, 96, 9, 0, 0, 520, 2), (64, 4, 1, 32, 9, 100, 3, 520, 2),
    (64, 4, 1, 128, 3, 0, 0, 100, 300), (64, 8, 8, 128, 5, 0, 0, 1100, 9), (64, 5, 5, 128, 3, 100, 3, 1100, 2), (64, 8, 8, 96, 3, 0, 0, 130, 300),
    (64, 4, 1, 96, 9, 0, 0, 1100, 9), (64, 6, 3, 96, 3, 100, 3, 1100, 2), (128, 8, 8, 64, 3, 0, 0, 100, 40), (128, 4, 1, 128, 3, 0, 0, 300, 40),
    (128, 8, 8, 128, 3, 0, 0, 1100, 2), (128, 4, 1, 64, 3, 100, 3, 40, 2), (128, 4, 1, 32, 3, 0, 0, 130, 300), (128, 8, 8, 96, 3, 100, 3, 520, 2),
    (128, 4, 1, 32, 5, 0, 0, 520, 2), (128, 8, 8, 128, 3, 0, 0, 130, 40), (128, 4, 1, 128, 3, 0, 0, 100, 300), (128, 8, 2, 128, 3, 0, 0, 1100, 9),
    (128, 5, 5, 128, 3, 100, 3, 1100, 2), (128, 4, 1, 64, 3, 0, 0, 100, 300), (128, 6, 3, 96, 5, 100, 3, 1100, 2), (128, 4, 1, 64, 9, 0, 0, 1100, 9),
]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D,H,KH,page,B,window,sinks,n_max,most", SHARED)
def test_tiles_shared_by_wavefronts(ops, kind, D, H, KH, page, B, window, sinks, n_max, most):
    if kind in ("bf16", "fp8") and not window:
        window = 1 << 20
    lens = [[min(most * page - 5, 700), min(most * page, 333), 0, 40][b] if b < 4 else 1 + 13 * b for b in range(B)]
    rows = [[min(n_max, lens[0], 290), min(n_max, 5), 0, 1][b] if b < 4 else b % 3 for b in range(B)]
    tab = mx.table(lens, page, seed=D + n_max)
    cache, scales, values = caches(kind, tab[3], KH, page, D, 5, ops)
    q = (2 * torch.randn(sum(rows), H, D, generator=torch.Generator().manual_seed(1))).to(BF)
    want, size = mx.window_attention(q, values, lens, rows, tab[0], tab[1], window, sinks)
    out = attend(ops, q, cache, rows, lens, page, tab, window, sinks, scales, n_max=n_max, most=most)
    check(f"{kind}/{D} {H}/{KH} pages of {page}, {B} x {n_max}", out, want, size, mx.attention_bound(size, q, values))


@pytest.mark.parametrize("kind", ["bf16", "mxfp8"])
@pytest.mark.parametrize("lens,rows", [([3, 130], [9, 2]), ([100, 0], [150, 60])])
def test_the_largest_window_and_more_rows_than_tokens(ops, kind, lens, rows):
    """A window and first tokens of 2^31 - 1 are all of them, for rows in front of a request's first token too, which see nothing."""
    D, H, KH, page = 64, 4, 2, 128
    tab = mx.table(lens, page)
    cache, _, values = caches(kind, tab[3], KH, page, D, 5, ops)
    q = torch.randn(sum(rows), H, D, generator=torch.Generator().manual_seed(1)).to(BF).to(DEV)
    want, size = mx.window_attention(q.cpu(), values, lens, rows, tab[0], tab[1], 1 << 20, 0)
    most, n = 2**31 - 1, max(rows)
    lib, kind_ = ops._lib.load(), {"bf16": ops.MD_KV_BF16, "mxfp8": ops.MD_KV_MXFP8}[kind] | ops.MD_KV_LAYOUT_HND
    indptr, table = mx.indptr_of(rows).to(DEV), [t.to(DEV) for t in tab[:3]]
    for window, sinks in ((most, 0), (most, most), (5, most)):
        ws = torch.zeros(lib.md_window_attn_workspace_bytes(len(lens), n, H, KH, D, tab[4], page, kind_, window, sinks), dtype=torch.uint8, device=DEV)
        out = torch.full_like(q, 7.0)
        assert lib.md_window_attn(q.data_ptr(), q.stride(0), cache.data_ptr(), out.data_ptr(), indptr.data_ptr(), *(t.data_ptr() for t in table),
                                  len(lens), n, H, KH, D, page, window, sinks, 1 / math.sqrt(D), tab[4], kind_, None, None, ws.data_ptr(), ws.numel(),
                                  torch.cuda.current_stream().cuda_stream) == 0
        check(f"{kind}/window {window}, {sinks} first", out, want, size, mx.attention_bound(size, q.cpu(), values))


@pytest.mark.parametrize("kind", ["bf16", "mxfp4"])
@pytest.mark.parametrize("n", [1, 60])
def test_rows_behind_the_last_request_stay(ops, kind, n):
    """A batch padded behind its last request: those rows of the result are not written.  Requests that share pages read the same ones."""
    D, H, KH, page = 64, 4, 2, 128
    lens, rows = [300, 300], [n, n]
    indices, indptr, last, pages, most = mx.table(lens, page)
    indices[3:5] = indices[0:2]                                  # the second request's first pages are the first one's
    cache, scales, values = caches(kind, pages, KH, page, D, 5, ops)
    q = torch.randn(2 * n + 5, H, D, generator=torch.Generator().manual_seed(1)).to(BF)
    out = torch.full((2 * n + 5, H, D), 7.0, dtype=BF, device=DEV)
    ops.paged_attention(q.to(DEV), cache, mx.indptr_of(rows).to(DEV), indices.to(DEV), indptr.to(DEV), last.to(DEV), n, most, ops.AttnWorkspace(DEV),
                        out=out, kv_layout="HND", window=290, sinks=2)
    assert bool((out[2 * n:] == 7.0).all())
    want, size = mx.window_attention(q[:2 * n], values, lens, rows, indices, indptr, 290, 2)
    check(f"{kind}/shared pages", out[:2 * n], want, size, mx.attention_bound(size, q[:2 * n], values))


def test_refusals_on_the_gpu(ops):
    """What the wrapper refuses before a launch."""
    D, H, KH, page = 128, 4, 2, 128
    tab = mx.table([200], page)
    cache, _, _ = caches("mxfp8", tab[3], KH, page, D, 5, ops)
    q = torch.zeros(1, H, D, dtype=BF)
    call = lambda q=q, cache=cache, tab=tab, **more: attend(ops, q, cache, [1], [200], page, tab, more.pop("window", 0), more.pop("sinks", 0), **more)  # noqa: E731
    call()
    for more in (dict(layout="NHD"), dict(causal=False), dict(sinks=-1), dict(window=-3), dict(scales=(q, q)), dict(q=torch.zeros(1, 3, D, dtype=BF)),
                 dict(q=torch.zeros(1, H, 64, dtype=BF)), dict(q=torch.zeros(1, H, D)), dict(q=torch.zeros(1, H, 2 * D, dtype=BF, device=DEV)[..., ::2]),
                 dict(out=torch.zeros(1, H, D, device=DEV)), dict(out=torch.zeros(2, H, D, dtype=BF, device=DEV))):
        with pytest.raises(ValueError):
            call(**more)
    with pytest.raises(TypeError):
        call(tab=(tab[0].long(), *tab[1:]))
    with pytest.raises(ops.MagicDecHipError, match="sm_scale"):
        call(sm_scale=-1.0)
    for op in (lambda: ops.snapkv_select(q.to(DEV), cache, *(t.to(DEV) for t in tab[:2]), 200, 32, 64, 5, cache, *(t.to(DEV) for t in tab[:3]),
                                         ops.AttnWorkspace(DEV), kv_layout="HND"),):
        with pytest.raises(ValueError, match="block-scaled"):
            op()


@pytest.mark.parametrize("n,H", [(1, 2), (3, 8), (200, 4)])
def test_scales_of_zero(ops, n, H):
    """A static scale of 0, of a head whose first rows were all 0: keys and values of 0, so that a row is the mean of what it sees, and 0."""
    D, KH, page, lens = 128, 2, 128, [300]
    tab = mx.table(lens, page)
    cache, (ks, vs), values = caches("fp8", tab[3], KH, page, D, 5, ops)
    ks, vs = ks.clone(), vs.clone()
    ks[0], vs[1] = 0.0, 0.0
    values[:, 0, 0], values[:, 1, 1] = 0.0, 0.0
    q = torch.randn(n, H, D, generator=torch.Generator().manual_seed(1)).to(BF)
    want, size = mx.window_attention(q, values, lens, [n], tab[0], tab[1], 77, 3)
    out = attend(ops, q, cache, [n], lens, page, tab, 77, 3, (ks, vs))
    check(f"scales of 0, {n} rows", out, want, size, mx.attention_bound(size, q, values))
    assert bool((out[:, H // 2:] == 0).all())


def hidden_garbage(lens, rows, tab, page, window, sinks):
    """An edit of a cache that puts infinities, NaN and the largest numbers into every place that no row of the request sees."""
    indices, indptr = tab[0], tab[1]

    def edit(x):
        junk = torch.tensor([math.nan, math.inf, -math.inf, 3.3895313892515355e38]).to(BF).repeat(x.shape[-1] // 4)
        used = set()
        for b, (n, m) in enumerate(zip(lens, rows)):
            seen = set()
            for t in range(n - m, n):
                seen |= {s for s in range(0, t + 1) if not window or s > t - window or s < sinks}
            for i in range(int(indptr[b]), int(indptr[b + 1])):
                pg = int(indices[i])
                used.add(pg)
                for slot in range(page):
                    if (i - int(indptr[b])) * page + slot not in seen:
                        x[pg, :, :, slot] = junk
        for pg in range(x.shape[0]):
            if pg not in used:
                x[pg] = junk
    return edit


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("lens,rows,window,sinks,D", [([300, 70], [1, 4], 40, 3, 128), ([600, 129], [130, 60], 90, 5, 128), ([333, 500], [65, 3], 33, 0, 64),
                                                      ([300, 200], [4, 130], 1 << 20, 0, 64)])
def test_what_no_row_sees_has_no_effect(ops, kind, lens, rows, window, sinks, D):
    H, KH, page = 8, 2, 128
    tab = mx.table(lens, page, seed=4)
    q = torch.randn(sum(rows), H, D, generator=torch.Generator().manual_seed(1)).to(BF)
    cache, scales, values = caches(kind, tab[3], KH, page, D, 5, ops, edit=hidden_garbage(lens, rows, tab, page, window, sinks))
    clean, _, clean_values = caches(kind, tab[3], KH, page, D, 5, ops)
    a = attend(ops, q, cache, rows, lens, page, tab, window, sinks, scales)
    c = attend(ops, q, clean, rows, lens, page, tab, window, sinks, scales)
    assert torch.equal(a, c)
    want, size = mx.window_attention(q, clean_values, lens, rows, tab[0], tab[1], window, sinks)
    check(f"{kind}/hidden garbage", a, want, size, mx.attention_bound(size, q, clean_values))


@pytest.mark.parametrize("kind", ["bf16", "mxfp8", "mxfp4"])
@pytest.mark.parametrize("n,D,window,most", [(4, 128, 150, None), (40, 64, 150, None), (130, 128, 150, None), (300, 128, 150, None),
                                             (4, 64, 1 << 20, None), (300, 128, 1 << 20, 470), (300, 64, 1 << 20, 470)])
def test_infinite_keys_and_values_reach_the_rows_that_see_them_alone(ops, kind, n, D, window, most):
    """The token at position p of a chunk has a NaN in its key, another an infinity in its value: rows before them are as without, rows behind
    the key's are NaN, rows that see the value are not finite in its place (block-scaled: its block)."""
    H, KH, page, past, sinks = 4, 1, 128, 200, 2
    lens, rows = [past + n], [n]
    tab = mx.table(lens, page)
    nan_at, inf_at = past + n - 1, past + n // 2

    def edit(x):
        pg, slot = int(tab[0][inf_at // page]), inf_at % page
        x[pg, 1, :, slot, 5] = math.inf
        pg, slot = int(tab[0][nan_at // page]), nan_at % page
        x[pg, 0, :, slot, 7] = math.nan
    q = torch.randn(n, H, D, generator=torch.Generator().manual_seed(1)).to(BF)
    cache, _, _ = caches(kind, tab[3], KH, page, D, 5, ops, edit=edit)
    clean, _, _ = caches(kind, tab[3], KH, page, D, 5, ops)
    a = attend(ops, q, cache, rows, lens, page, tab, window, sinks, most=most).cpu()
    c = attend(ops, q, clean, rows, lens, page, tab, window, sinks, most=most).cpu()
    first = n // 2                                              # rows from here on see the value
    assert torch.equal(a[:first], c[:first])
    assert bool(a[n - 1].isnan().all())
    where = torch.zeros(D, dtype=torch.bool)
    where[5 if kind == "bf16" else slice(0, 32)] = True
    behind = a[first:min(n - 1, first + window)]
    assert not torch.isfinite(behind[..., where]).any()
    if kind == "bf16":
        assert bool((behind[..., where] == math.inf).all())
    assert torch.equal(behind[..., ~where], c[first:first + behind.shape[0]][..., ~where])


def test_scores_of_the_largest_size_and_of_the_lowest(ops):
    """Scores near the largest 32-bit numbers of both signs: the one largest key takes all; where all are equal and very low, their mean."""
    D, H, KH, page, n = 64, 2, 1, 128, 100
    tab = mx.table([n], page)
    q = torch.zeros(1, H, D, dtype=BF)
    q[0, 0, 0], q[0, 1, 0] = 1e19, -1e18
    x = torch.zeros(tab[3], 2, KH, page, D, dtype=BF)
    x[:, 0, :, :, 0] = 1e18
    x[int(tab[0][0]), 0, 0, 37, 0] = 1.5e18
    x[:, 1] = torch.randn(tab[3], KH, page, D, generator=torch.Generator().manual_seed(2)).to(BF)
    out = attend(ops, q, x.to(DEV), [1], [n], page, tab, 1 << 20, 0).cpu()
    v = x[int(tab[0][0]), 1, 0, :n].double()
    assert torch.equal(out[0, 0].double(), v[37])
    rest = torch.cat([v[:37], v[38:]])
    assert bool(((out[0, 1].double() - rest.mean(0)).abs() <= 2 * mx.U_BF16 * rest.abs().mean(0) * 1.01).all())


@pytest.mark.parametrize("kind,n", [("mxfp4", 1), ("mxfp8", 4), ("bf16", 1), ("mxfp8", 150)])
def test_steps_of_a_captured_graph_follow_the_lengths(ops, kind, n):
    """Append and attention of a step captured once: replays read the rows, lengths and page tables as they are then, two graphs share a workspace
    and eager calls run between the replays."""
    B, H, KH, D, page, room = 3, 8, 2, 128, 128, 1024
    window, sinks = (64, 4) if kind == "bf16" else (300, 7)
    pages = B * room // page
    cache = (torch.zeros(pages, 2, KH, page, D, dtype=BF, device=DEV) if kind == "bf16" else ops.mx_kv_cache(pages, KH, D, kind))
    g = torch.Generator().manual_seed(3)
    rows_total = room - 200
    k, v = (torch.randn(B, room, KH, D, generator=g).to(BF).to(DEV) for _ in (0, 1))
    q = torch.randn(B * n, H, D, generator=g).to(BF).to(DEV)
    ix = torch.arange(pages, dtype=torch.int32, device=DEV)
    pi, la = (torch.zeros(m, dtype=torch.int32, device=DEV) for m in (B + 1, B))
    ip = mx.indptr_of([n] * B).to(DEV)
    kn, vn = (torch.zeros(B * n, KH, D, dtype=BF, device=DEV) for _ in (0, 1))
    ws = ops.AttnWorkspace(DEV)

    def place(length):
        """Page tables of `length` tokens a request, the requests' pages apart by `room`."""
        np_ = -(-length // page)
        ix[:B * np_].copy_((torch.arange(B)[:, None] * (room // page) + torch.arange(np_)).flatten().to(torch.int32))
        pi.copy_((torch.arange(B + 1) * np_).to(torch.int32))
        la.fill_((length - 1) % page + 1)

    def append():
        ops.update_kv(kn, vn, ip, cache, ix, pi, la, n_max=n, kv_layout="HND")

    def attention(out=None):
        return ops.paged_attention(q, cache, ip, ix, pi, la, n, room // page, ws, out=out, kv_layout="HND", window=window, sinks=sinks)

    # the past
    place(200)
    past = mx.indptr_of([200] * B).to(DEV)
    ops.update_kv(k[:, :200].reshape(-1, KH, D), v[:, :200].reshape(-1, KH, D), past, cache, ix, pi, la, n_max=200, kv_layout="HND")
    outs = [torch.zeros(B * n, H, D, dtype=BF, device=DEV) for _ in (0, 1)]
    attention()
    graphs = []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for i in (0, 1):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=side):
            append()
            attention(outs[i])
        graphs.append(gr)
    length = 200
    for step in range(6):
        length += n
        if length > rows_total:
            break
        kn.copy_(k[:, length - n:length].reshape(-1, KH, D))
        vn.copy_(v[:, length - n:length].reshape(-1, KH, D))
        place(length)
        out = outs[step % 2]
        graphs[step % 2].replay()
        torch.cuda.synchronize()
        got = out.clone()
        append()
        assert torch.equal(got, attention())
        if kind == "bf16":
            values = torch.stack([k, v], 1)[:, :, :length].transpose(2, 3).cpu()             # one long page a request
            one = (torch.arange(B), torch.arange(B + 1))
            want, size = mx.window_attention(q.cpu(), values, [length] * B, [n] * B, *one, window, sinks)
            check(f"graph step {step}", got, want, size, mx.attention_bound(size, q.cpu(), values))


def test_calls_on_two_streams_with_a_workspace_each(ops):
    """The same calls as one after another on the default stream."""
    kind, D, H, KH, page, lens, rows = "mxfp4", 128, 8, 1, 128, [9000], [1]
    tab = mx.table(lens, page)
    cache, _, _ = caches(kind, tab[3], KH, page, D, 5, ops)
    qs = [torch.randn(1, H, D, generator=torch.Generator().manual_seed(s)).to(BF) for s in (1, 2)]
    want = [attend(ops, q, cache, rows, lens, page, tab, 0, 0) for q in qs]
    torch.cuda.synchronize()
    streams, spaces, got = [torch.cuda.Stream() for _ in qs], [ops.AttnWorkspace(DEV) for _ in qs], [[], []]
    for _ in range(5):
        for i, q in enumerate(qs):
            with torch.cuda.stream(streams[i]):
                got[i].append(attend(ops, q, cache, rows, lens, page, tab, 0, 0, ws=spaces[i]))
    torch.cuda.synchronize()
    for i in (0, 1):
        assert all(torch.equal(o, want[i]) for o in got[i])


def test_one_request_alone_is_as_in_a_batch(ops):
    """Rows do not depend on what lies beside them, but for how their keys are split: a batch as large as to split none against its parts."""
    kind, D, H, KH, page = "mxfp8", 128, 8, 8, 128
    lens, rows = [100 + 7 * b for b in range(64)], [1 + b % 4 for b in range(64)]
    tab = mx.table(lens, page)
    cache, _, _ = caches(kind, tab[3], KH, page, D, 5, ops)
    q = torch.randn(sum(rows), H, D, generator=torch.Generator().manual_seed(1)).to(BF)
    a = attend(ops, q, cache, rows, lens, page, tab, 50, 3)
    again = attend(ops, q, cache, rows, lens, page, tab, 50, 3)
    assert torch.equal(a, again)
