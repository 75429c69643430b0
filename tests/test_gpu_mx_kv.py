"""Block-scaled KV pages on the GPU: rows quantised as they are written (update_kv, rope_append) and read back (read_kv), byte for byte against a
plain statement of the format."""
import pytest
import torch

from tests import mx_util as mx

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16
KINDS = ["mxfp8", "mxfp4"]


@pytest.fixture(scope="module")
def ops():
    from magicdec_amd import ops as _ops
    _ops._lib.load()
    return _ops


def dev(*ts):
    return [t.to(DEV) for t in ts]


def rows_of(n, KH, D, seed, special=False):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(n, KH, D, generator=g) * torch.exp(2 * torch.randn(n, KH, 1, generator=g))).to(BF)
    if special:
        flat = x.view(-1, 32)
        flat[0] = 0.0
        flat[1] = -0.0
        flat[2, 3] = float("inf")
        flat[3, 31] = float("-inf")
        flat[4, 0] = float("nan")
        flat[5] = 2.0 ** -130                                                # bf16 subnormal numbers
        flat[6, :4] = torch.tensor([3.3895313892515355e38, -3.3895313892515355e38, 1.0, 2.0 ** 120])          # the largest
        flat[7] = torch.tensor([2.0 ** -110, 2.0 ** -101, 1.5 * 2.0 ** -101, 2.0 ** -99] * 8).to(BF)             # next to the smallest scale
        # ties of both grids, and largest elements on both sides of the scale's border
        flat[8] = torch.arange(32).to(BF) * 0.25
        flat[9] = torch.cat([torch.tensor([7.0]), torch.arange(31) * 0.25]).to(BF)
        flat[10] = torch.cat([torch.tensor([7.0625]), torch.arange(31) * 0.25]).to(BF)
        flat[11] = torch.cat([torch.tensor([464.0]), torch.arange(31) * 4.5]).to(BF)
        flat[12] = torch.cat([torch.tensor([466.0]), torch.arange(31) * 4.5]).to(BF)
        flat[13] = torch.cat([torch.tensor([-448.0]), (torch.arange(31) + 0.5) * 2.0 ** -9]).to(BF)                # e4m3 subnormals and ties
    return x


def expected(cache, k, v, rows, lens, indices, indptr, page, kind):
    """The cache's bytes behind update_kv."""
    D = k.shape[-1]
    code, scale = mx.unpack(cache.clone(), kind, D)
    code, scale = code.clone(), scale.clone()
    at = 0
    for b, (m, n) in enumerate(zip(rows, lens)):
        room = int(indptr[b + 1] - indptr[b]) * page
        for j in range(m):
            pos = n - m + j
            if 0 <= pos < room:
                pg = int(indices[int(indptr[b]) + pos // page])
                for half, x in ((0, k), (1, v)):
                    code[pg, half, :, pos % page], scale[pg, half, :, pos % page] = mx.quantize(x[at + j], kind)
        at += m
    return mx.pack(code, scale, kind)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D,KH,page,lens,rows,special", [
    (128, 8, 128, [5, 129, 300], [1, 1, 1], False),             # single tokens, one in a new page
    (128, 2, 128, [260, 4, 131, 4], [4, 4, 4, 4], True),        # a verify step's rows over a page's end
    (64, 3, 32, [70, 33, 0, 64], [37, 33, 0, 1], True),         # pages of 32 rows, a request without rows
    (64, 1, 128, [500], [301], True),                           # a prompt's portion, an odd number of rows
    (128, 5, 64, [1, 77], [1, 60], True),
], ids=["tokens", "verify", "pages32-d64", "prompt-d64", "odd"])
def test_update_kv_writes_the_format_and_read_kv_its_values(ops, kind, D, KH, page, lens, rows, special):
    indices, indptr, last, pages, _ = mx.table(lens, page, seed=3)
    total = sum(rows)
    k, v = rows_of(total, KH, D, 1, special and total * KH * D >= 14 * 32), rows_of(total, KH, D, 2)
    g = torch.Generator().manual_seed(9)
    before = torch.randint(0, 256, (pages, 2, KH, page, ops.mx_row_bytes(D, kind)), dtype=torch.uint8, generator=g)
    want = expected(before, k, v, rows, lens, indices, indptr, page, kind)
    # rows as slices of one product's output
    wide = torch.zeros(total, 2 * KH + 1, D, dtype=BF)
    wide[:, 1:KH + 1], wide[:, KH + 1:] = k, v
    wide = wide.to(DEV)
    cache = before.to(DEV)
    ip, ix, pi, la = dev(mx.indptr_of(rows), indices, indptr, last)
    ops.update_kv(wide[:, 1:KH + 1], wide[:, KH + 1:], ip, cache, ix, pi, la, n_max=max(rows), kv_layout="HND")
    assert torch.equal(cache.cpu(), want)                       # every byte, those of rows that were not written too
    ko, vo = (torch.full((total + 3, KH, D), 7.0, dtype=BF, device=DEV) for _ in (0, 1))
    back = ops.read_kv(ko[:total], vo[:total], ip, cache, ix, pi, la, n_max=max(rows), kv_layout="HND")
    assert back[0].data_ptr() == ko.data_ptr()
    for got, x in ((ko, k), (vo, v)):
        values = mx.dequantize(*mx.quantize(x, kind), kind)
        assert torch.equal(values.nan_to_num(1e30), values.to(BF).double().nan_to_num(1e30))      # bf16 holds them
        assert torch.equal(got[:total].cpu().view(torch.int16)[~values.isnan()], values.to(BF).view(torch.int16)[~values.isnan()])
        assert torch.equal(got[:total].cpu().isnan(), values.isnan())
        assert bool((got[total:] == 7.0).all())


def test_elements_are_off_by_half_a_step_at_most():
    """The format itself, on the CPU's statement of it: for e4m3 half a step is 2^-4 of a number from 2^-6 of the scale on and 2^-10 of the
    scale below, for e2m1 a quarter of the scale, or of the binade's step above 2 (half of it)."""
    x = rows_of(400, 4, 64, 5)
    for kind, rel, floor in (("mxfp8", 2.0 ** -4, 2.0 ** -10), ("mxfp4", 0.25, 0.25)):
        code, scale = mx.quantize(x, kind)
        err = (mx.dequantize(code, scale, kind) - x.double()).abs()
        s = 2.0 ** (scale.double() - 127).unsqueeze(-1).expand(*scale.shape, 32).flatten(-2)
        assert bool((err <= torch.maximum(rel * x.double().abs(), floor * s)).all())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D,n,second", [(128, 4, False), (64, 130, True), (128, 33, True)])
def test_rope_append_is_rope_and_update_kv(ops, kind, D, n, second):
    B, H, KH, page = 3, 12, 4, 128
    lens = [n, 200 + n, 127 + n]
    indices, indptr, last, pages, _ = mx.table(lens, page, seed=1)
    qkv = rows_of(B * n, H + 2 * KH, D, 3).to(DEV)
    q, k, v = qkv[:, :H], qkv[:, H:H + KH], qkv[:, H + KH:]
    tab = ops.RopeTable(512, D, 10000.0, 1.0, device=DEV)
    off = torch.tensor([0, 300, 511 - n // 2], dtype=torch.int32)            # (the last one's positions end behind the table)
    ip, off, ix, pi, la = dev(mx.indptr_of([n] * B), off, indices, indptr, last)
    a, c = (ops.mx_kv_cache(pages, KH, D, kind) for _ in (0, 1))
    bf, bf_want = (torch.zeros(pages, 2, page, KH, D, dtype=BF, device=DEV) for _ in (0, 1))
    more = (bf, ix, pi, la) if second else ()
    got = ops.rope_append(q, k, v, ip, off, tab, a, ix, pi, la, *more, n_max=n, kv_layout="HND")
    rq, rk = ops.rope(q, k, ip, off, tab, n_max=n)
    ops.update_kv(rk, v, ip, c, ix, pi, la, n_max=n, kv_layout="HND")
    assert torch.equal(got.view(torch.int16), rq.view(torch.int16))
    assert torch.equal(a, c)
    if second:
        ops.update_kv(rk, v, ip, bf_want, ix, pi, la, n_max=n)
        assert torch.equal(bf.view(torch.int16), bf_want.view(torch.int16))


def test_rows_outside_the_pages_are_dropped_counted_and_not_read(ops):
    D, KH, page = 64, 2, 128
    indices, indptr, last, pages, _ = mx.table([128, 40], page)
    last = torch.tensor([130, 3], dtype=torch.int32)             # request 0: two rows behind its page; request 1: five rows of three tokens
    k = rows_of(10, KH, D, 1).to(DEV)
    ip, ix, pi, la = dev(mx.indptr_of([5, 5]), indices, indptr, last)
    cache = ops.mx_kv_cache(pages, KH, D, "mxfp8")
    ops.page_overflow_count(reset=True)
    ops.update_kv(k, k, ip, cache, ix, pi, la, n_max=5, kv_layout="HND")
    assert ops.page_overflow_count(reset=True) == 2
    ko, vo = (torch.full((10, KH, D), 7.0, dtype=BF, device=DEV) for _ in (0, 1))
    ops.read_kv(ko, vo, ip, cache, ix, pi, la, n_max=5, kv_layout="HND")
    left = [3, 4, 5, 6]
    assert bool((ko[left] == 7.0).all()) and bool((vo[left] == 7.0).all())
    want = mx.dequantize(*mx.quantize(k.cpu(), "mxfp8"), "mxfp8")
    there = [0, 1, 2, 7, 8, 9]
    assert torch.equal(ko[there].cpu().double(), want[there])


@pytest.mark.parametrize("layout", ["NHD", "HND"])
@pytest.mark.parametrize("D", [64, 128])
def test_read_kv_of_other_caches(ops, layout, D):
    KH, page, lens, rows = 3, 64, [200, 64, 9], [200, 10, 9]
    indices, indptr, last, pages, _ = mx.table(lens, page, seed=2)
    k, v = rows_of(sum(rows), KH, D, 1).clamp(-100, 100).to(DEV), rows_of(sum(rows), KH, D, 2).clamp(-100, 100).to(DEV)
    ip, ix, pi, la = dev(mx.indptr_of(rows), indices, indptr, last)
    shape = (pages, 2, page, KH, D) if layout == "NHD" else (pages, 2, KH, page, D)
    for dtype, scales in ((BF, None), (torch.float8_e4m3fn, tuple(dev(torch.tensor([0.3, 0.02, 1.7]), torch.tensor([0.011, 0.25, 0.6]))))):
        cache = torch.zeros(shape, device=DEV).to(dtype)
        ops.update_kv(k, v, ip, cache, ix, pi, la, n_max=200, kv_scales=scales, kv_layout=layout)
        ko, vo = torch.empty_like(k), torch.empty_like(v)
        ops.read_kv(ko, vo, ip, cache, ix, pi, la, kv_scales=scales, kv_layout=layout)
        for got, x, sc in ((ko, k, 0), (vo, v, 1)):
            if scales is None:
                assert torch.equal(got.view(torch.int16), x.view(torch.int16))
            else:                                             # the stored byte times its head's scale, rounded once
                s = scales[sc][None, :, None]
                stored = (x.float() * (1.0 / s)).clamp(-448, 448).to(torch.float8_e4m3fn).float()
                assert torch.equal(got, (stored * s).to(BF))


def test_pages_behind_four_gib(ops):
    """A cache of over 2^32 bytes: rows in its last pages are where their page numbers say."""
    D, KH, page, kind = 128, 8, 128, "mxfp8"
    pages = 2 ** 32 // (2 * KH * page * ops.mx_row_bytes(D, kind)) + 40
    cache = torch.zeros((pages, 2, KH, page, ops.mx_row_bytes(D, kind)), dtype=torch.uint8, device=DEV)
    n = 300
    k, v = rows_of(n, KH, D, 1).to(DEV), rows_of(n, KH, D, 2).to(DEV)
    ip, pi, la = dev(mx.indptr_of([n]), torch.tensor([0, 3], dtype=torch.int32), torch.tensor([n - 256], dtype=torch.int32))
    ix = torch.tensor([pages - 1, 5, pages - 7], dtype=torch.int32, device=DEV)
    ops.update_kv(k, v, ip, cache, ix, pi, la, n_max=n, kv_layout="HND")
    small = ops.mx_kv_cache(3, KH, D, kind)
    low = torch.tensor([0, 1, 2], dtype=torch.int32, device=DEV)
    ops.update_kv(k, v, ip, small, low, pi, la, n_max=n, kv_layout="HND")
    assert torch.equal(cache[ix.long()], small)
    ko, vo = torch.empty_like(k), torch.empty_like(v)
    ops.read_kv(ko, vo, ip, cache, ix, pi, la, kv_layout="HND")
    assert torch.equal(ko.double().cpu(), mx.dequantize(*mx.quantize(k.cpu(), kind), kind))
    q = rows_of(4, 32, D, 7).to(DEV)
    qo, ws = mx.indptr_of([4]).to(DEV), ops.AttnWorkspace(DEV)
    a = ops.paged_attention(q, cache, qo, ix, pi, la, 4, 3, ws, kv_layout="HND")
    c = ops.paged_attention(q, small, qo, low, pi, la, 4, 3, ws, kv_layout="HND")
    assert torch.equal(a, c)


def test_read_kv_refuses_rows_that_share_memory(ops):
    """An expanded row can be appended many times, but not be written as many."""
    D, KH, page = 64, 2, 128
    cache = ops.mx_kv_cache(1, KH, D, "mxfp8")
    table = [torch.tensor(t, dtype=torch.int32, device=DEV) for t in ([0, 3], [0], [0, 1], [3])]
    one = torch.randn(1, KH, D, generator=torch.Generator().manual_seed(1)).to(BF).to(DEV)
    many, out = one.expand(3, KH, D), torch.zeros(3, KH, D, dtype=BF, device=DEV)
    ops.update_kv(many, many, table[0], cache, *table[1:], kv_layout="HND")
    for k, v in ((many, out), (out, many)):
        with pytest.raises(ValueError, match="share memory"):
            ops.read_kv(k, v, table[0], cache, *table[1:], kv_layout="HND")
    k, v = ops.read_kv(out, torch.zeros_like(out), table[0], cache, *table[1:], kv_layout="HND")
    assert torch.equal(k[0], k[2]) and torch.equal(v, k)
    assert bool(((k[0] - one[0]).abs() <= one.abs().amax() / 16).all())
