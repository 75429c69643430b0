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
