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
