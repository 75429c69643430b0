"""Calls of the windowed attention and of read_kv that the documentation allows, on the GPU, against 64 bits."""
import pytest
import torch

from tests import mx_util as mx
from tests.test_gpu_window_attn import attend, caches, check

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16


@pytest.fixture(scope="module")
def ops():
    from magicdec_amd import ops as _ops
    _ops._lib.load()
    return _ops


@pytest.mark.parametrize("D,n,H", [(128, 1, 2), (64, 3, 16), (128, 200, 4), (64, 500, 4)])
def test_negative_scales_of_heads(ops, D, n, H):
    """A static scale's sign is the sign of all that it scales: of one head's keys, of another's values.  Rows that see one key are its value, whose
    sign is the scale's."""
    KH, page, lens = 2, 128, [max(300, n)]
    tab = mx.table(lens, page)
    cache, (ks, vs), values = caches("fp8", tab[3], KH, page, D, 5, ops)
    ks, vs = ks.clone(), vs.clone()
    ks[0], vs[1] = -ks[0], -vs[1]
    values[:, 0, 0], values[:, 1, 1] = -values[:, 0, 0], -values[:, 1, 1]
    q = torch.randn(n, H, D, generator=torch.Generator().manual_seed(1)).to(BF)
    for window, sinks in ((77, 3), (1, 0)):
        want, size = mx.window_attention(q, values, lens, [n], tab[0], tab[1], window, sinks)
        out = attend(ops, q, cache, [n], lens, page, tab, window, sinks, (ks, vs))
        check(f"negative scales, {n} rows, window {window}", out, want, size, mx.attention_bound(size, q, values))


@pytest.mark.parametrize("kind", ["bf16", "mxfp8"])
def test_read_kv_refuses_one_place_for_keys_and_values(ops, kind):
    """k and v are written by many workgroups in no order; slices of one buffer whose rows lie between each other's are two places."""
    D, KH, page, n = 64, 2, 128, 5
    cache = ops.mx_kv_cache(1, KH, D, kind) if kind != "bf16" else torch.zeros(1, 2, KH, page, D, dtype=BF, device=DEV)
    table = [torch.tensor(t, dtype=torch.int32, device=DEV) for t in ([0, n], [0], [0, 1], [n])]
    x = (torch.arange(n * 2 * KH * D) % 13).to(BF).view(n, 2 * KH, D).to(DEV)
    ops.update_kv(x[:, :KH], x[:, KH:], table[0], cache, *table[1:], kv_layout="HND")
    both = torch.zeros(n + 1, 2 * KH, D, dtype=BF, device=DEV)
    out = both[:n, :KH]
    for v in (out, both[:n, 1:KH + 1], both[1:, :KH]):
        with pytest.raises(ValueError, match="share memory"):
            ops.read_kv(out, v, table[0], cache, *table[1:], kv_layout="HND")
    assert bool((both == 0).all())
    ops.read_kv(out, both[:n, KH:], table[0], cache, *table[1:], kv_layout="HND")
    assert torch.equal(both[:n], x) and bool((both[n] == 0).all())


@pytest.mark.parametrize("kind", ["bf16", "mxfp8", "mxfp4"])
@pytest.mark.parametrize("window,sinks", [(50, 3), (0, 0)])
def test_each_request_of_a_batch_by_itself(ops, kind, window, sinks):
    """A batch as large as to split no keys, and its requests one a call: the same bits where their keys are in one part there too (a window of few keys);
    otherwise, in up to five parts, both within the bound of 64 bits."""
    from tests import window_layouts as wl
    D, H, KH, page, most = 64, 2, 2, 64, 10
    lens, rows = [100 + 2 * b for b in range(130)], [1 + b % 4 for b in range(130)]
    indices, indptr, last, pages, _ = mx.table(lens, page)
    cache, _, values = caches(kind, pages, KH, page, D, 5, ops)
    q = torch.randn(sum(rows), H, D, generator=torch.Generator().manual_seed(1)).to(BF)
    window = wl.window_of(window, kind)
    want, size = mx.window_attention(q, values, lens, rows, indices, indptr, window, sinks)
    bound = mx.attention_bound(size, q, values)
    ws = ops.AttnWorkspace(DEV)
    at, parts = mx.indptr_of(rows).tolist(), set()
    with wl.reported(ops._lib.load()) as layout:
        whole = attend(ops, q, cache, rows, lens, page, (indices, indptr, last, pages, most), window, sinks, ws=ws)
        of_batch = layout()
        check(f"{kind}/130 requests", whole, want, size, bound)
        for b in range(130):
            mine = slice(at[b], at[b + 1])
            tab = (indices[int(indptr[b]):int(indptr[b + 1])], torch.tensor([0, int(indptr[b + 1] - indptr[b])], dtype=torch.int32), last[b:b + 1], 0, most)
            alone = attend(ops, q[mine], cache, rows[b:b + 1], lens[b:b + 1], page, tab, window, sinks, ws=ws)
            parts.add(layout())
            if window == 50:
                assert torch.equal(alone, whole[mine])
            else:
                assert bool(((alone.cpu().double() - want[mine]).abs() <= bound[mine]).all()), b
    if of_batch is not None:
        assert of_batch == (0, 16, 32, "whole") and parts == {(0, 16, 32, "whole" if window == 50 else "few")}


# (D, H, KH, requests, n_max, wavefronts that share tiles): pages of 32 rows, so that a part walks more of them than a wavefront holds numbers of
LONG = [(64, 1, 1, 520, 1, 0), (128, 1, 1, 520, 1, 0), (64, 4, 1, 520, 8, 0), (128, 4, 1, 520, 8, 0), (64, 2, 1, 160, 150, 4), (64, 4, 1, 80, 400, 8),
        (128, 2, 1, 160, 150, 4), (128, 4, 1, 80, 400, 8)]


@pytest.mark.parametrize("kind", ["bf16", "fp8", "mxfp8", "mxfp4"])
@pytest.mark.parametrize("window,sinks", [(0, 0), (2960, 70), (2300, 2100)])
@pytest.mark.parametrize("D,H,KH,B,n_max,nw", LONG, ids=[f"{c[0]}-{c[5]}-waves-{c[4]}-rows" for c in LONG])
def test_streams_of_more_pages_than_a_wavefront_holds_numbers_of(ops, kind, window, sinks, D, H, KH, B, n_max, nw):
    """A request of 157 pages among short ones, whole or in two parts, with infinities and NaN in front of its window: where they are hidden from some row of
    a tile, the wavefronts go back to that tile's page."""
    from tests import window_layouts as wl
    page, n = 32, 5000
    window = wl.window_of(window, kind)
    new = min(n_max, 70)
    lens, rows = [n, 1, 40, 7] + [0] * (B - 4), [new, 1, 0, 2] + [0] * (B - 4)
    tab = mx.table(lens, page, seed=3)
    first = n - new                                           # the first row's position
    seen = torch.arange(n) <= n - 1
    if window:
        seen &= (torch.arange(n) > first - window) | (torch.arange(n) < sinks)

    def edit(x):
        junk = torch.tensor([float("nan"), float("inf"), float("-inf"), 3.3895313892515355e38]).to(BF).repeat(D // 4)
        for pos in (~seen).nonzero().flatten().tolist():
            x[int(tab[0][pos // page]), :, :, pos % page] = junk
    cache, scales, _ = caches(kind, tab[3], KH, page, D, 5, ops, edit=edit)
    _, _, values = caches(kind, tab[3], KH, page, D, 5, ops)
    q = torch.randn(sum(rows), H, D, generator=torch.Generator().manual_seed(1)).to(BF)
    want, size = mx.window_attention(q, values, lens, rows, tab[0], tab[1], window, sinks)
    with wl.reported(ops._lib.load()) as layout:
        out = attend(ops, q, cache, rows, lens, page, tab, window, sinks, scales, n_max=n_max)
        took = layout()
    check(f"{kind}/157 pages, {nw} wavefronts, window {window}", out, want, size, mx.attention_bound(size, q, values))
    assert took is None or (took[0] == nw and took[3] in ("whole", "few")), took


def test_scales_in_one_tensor(ops):
    """kv_scales is two tensors: a tuple's, or the rows of one of [2, heads]."""
    D, H, KH, page, lens, n = 128, 4, 2, 128, [300], 3
    tab = mx.table(lens, page)
    cache, scales, _ = caches("fp8", tab[3], KH, page, D, 5, ops)
    q = torch.randn(n, H, D, generator=torch.Generator().manual_seed(1)).to(BF)
    table = [t.to(DEV) for t in (mx.indptr_of([n]), *tab[:3])]
    outs, rows = [], []
    for s in (scales, torch.stack(scales)):
        outs.append(attend(ops, q, cache, [n], lens, page, tab, 77, 3, s))
        k, v = (torch.zeros(n, KH, D, dtype=BF, device=DEV) for _ in (0, 1))
        rows.append(torch.cat(ops.read_kv(k, v, table[0], cache, *table[1:], n_max=n, kv_scales=s, kv_layout="HND")))
    assert torch.equal(*outs) and torch.equal(*rows) and bool(rows[0].any())
