"""The windowed attention on every way of laying rows and keys over workgroups, each with what it is taken for asserted: against 64 bits with infinities,
NaN and the largest numbers in all places that no row sees, and with infinities and NaN in places that some rows see."""
import math

import pytest
import torch

from tests import mx_util as mx
from tests import window_layouts as wl
from tests.test_gpu_window_attn import caches, check

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16
IDS = ["-".join(map(str, b)) for b, _ in wl.LAYOUTS]


@pytest.fixture(scope="module")
def ops():
    from magicdec_amd import ops as _ops
    _ops._lib.load()
    return _ops


class Call:
    """A call within the bounds, over caches that an edit of the 16-bit rows changes."""

    def __init__(self, ops, bounds, layout, kind):
        self.ops, self.bounds, self.kind, self.layout = ops, bounds, kind, wl.of_kind(layout, kind, bounds[0])
        self.D, self.H, self.KH, self.page, _, window, self.sinks, self.n_max, self.most = bounds
        self.window = wl.window_of(window, kind)
        self.lens, self.rows = wl.lengths(bounds)
        self.tab = mx.table(self.lens, self.page, seed=self.n_max)
        self.q = torch.randn(sum(self.rows), self.H, self.D, generator=torch.Generator().manual_seed(1)).to(BF)

    def cache(self, edit=None):
        return caches(self.kind, self.tab[3], self.KH, self.page, self.D, 5, self.ops, edit=edit)

    def __call__(self, cache, scales):
        with wl.reported(self.ops._lib.load()) as layout:
            out = self.ops.paged_attention(self.q.to(DEV), cache, mx.indptr_of(self.rows).to(DEV), *(t.to(DEV) for t in self.tab[:3]), self.n_max,
                                           self.most, self.ops.AttnWorkspace(DEV), kv_scales=scales, kv_layout="HND", window=self.window or None,
                                           sinks=self.sinks)
            assert layout() in (None, self.layout)
        return out.cpu()

    def place(self, b, pos):
        """Page and slot of a request's position."""
        return int(self.tab[0][int(self.tab[1][b]) + pos // self.page]), pos % self.page

    def sees(self, b):
        """[rows, tokens] of a request."""
        t, s = (self.lens[b] - self.rows[b] + torch.arange(self.rows[b]))[:, None], torch.arange(self.lens[b])
        return (s <= t) & ((s > t - self.window) | (s < self.sinks) if self.window else True)


@pytest.mark.parametrize("kind", wl.KINDS)
@pytest.mark.parametrize("bounds,layout", wl.LAYOUTS, ids=IDS)
def test_hidden_places_hold_anything(ops, bounds, layout, kind):
    call = Call(ops, bounds, layout, kind)
    junk = torch.tensor([math.nan, math.inf, -math.inf, 3.3895313892515355e38]).to(BF).repeat(call.D // 4)

    def edit(x):
        seen = torch.zeros(x.shape[0], call.page, dtype=torch.bool)
        for b, n in enumerate(call.lens):
            if call.rows[b]:
                for pos in call.sees(b).any(0).nonzero().flatten().tolist():
                    seen[call.place(b, pos)] = True
        x.copy_(torch.where(seen[:, None, None, :, None], x, junk))
    cache, scales, _ = call.cache(edit)
    clean, _, values = call.cache()
    got, want_bits = call(cache, scales), call(clean, scales)
    assert torch.equal(got, want_bits)
    want, size = mx.window_attention(call.q, values, call.lens, call.rows, call.tab[0], call.tab[1], call.window, call.sinks)
    check(f"{kind}/{call.layout}", got, want, size, mx.attention_bound(size, call.q, values))


@pytest.mark.parametrize("kind", wl.KINDS)
@pytest.mark.parametrize("bounds,layout", wl.LAYOUTS, ids=IDS)
def test_infinities_reach_the_rows_that_see_them_alone(ops, bounds, layout, kind):
    """The first request's first token has -infinity in its value, one in the middle of its new rows +infinity, the last one (of three rows and more) NaN in
    its key.  Each counts, in its element (block-scaled: its block; of static-scale fp8, which has none, a NaN), for the rows that see it, and nothing else
    changes by a bit."""
    call = Call(ops, bounds, layout, kind)
    new = call.rows[0]
    past = call.lens[0] - new
    middle, block = past + new // 2, kind in ("mxfp8", "mxfp4")
    put = {0: (40, -math.inf), middle: (5, math.inf)}

    def edit(x):
        for pos, (d, value) in put.items():
            page, slot = call.place(0, pos)
            x[page, 1, :, slot, d] = value if kind != "fp8" else math.nan
        if new > 2:
            page, slot = call.place(0, call.lens[0] - 1)
            x[page, 0, :, slot, 7] = math.nan
    cache, scales, _ = call.cache(edit)
    got, clean = call(cache, scales), call(call.cache()[0], scales)
    assert torch.equal(got[new:], clean[new:])
    if new > 2:
        assert bool(got[new - 1].isnan().all())
    rows = new - (new > 2)
    reached = torch.zeros(rows, call.D, dtype=torch.bool)
    sees = call.sees(0)
    for pos, (d, value) in put.items():
        at = slice(d // 32 * 32, d // 32 * 32 + 32) if block else d
        mark = torch.zeros(call.D, dtype=torch.bool)
        mark[at] = True
        mine = sees[:rows, pos][:, None] & mark
        reached |= mine
        if kind == "bf16":
            assert bool((got[:rows][mine[:, None].expand(-1, call.H, -1)] == value).all())
    wide = reached[:, None].expand(-1, call.H, -1)
    assert not torch.isfinite(got[:rows][wide]).any()
    assert torch.equal(got[:rows][~wide], clean[:rows][~wide])
