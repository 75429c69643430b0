"""Block-scaled pages that hold any bytes at all, as a cache that was loaded or that another program wrote may, read back."""
import pytest
import torch

from tests import mx_util as mx

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16


@pytest.fixture(scope="module")
def ops():
    from magicdec_amd import ops as _ops
    _ops._lib.load()
    return _ops


def every_byte(kind, D, page):
    """A cache of one kv head whose rows hold every element under every scale, and how many rows those are."""
    codes = 256 if kind == "mxfp8" else 16
    code = torch.arange(codes).repeat(-(-D // codes)) if codes < D else torch.arange(codes)
    code = code.view(-1, D).repeat(256, 1)
    scale = torch.arange(256).repeat_interleave(code.shape[0] // 256)[:, None].expand(-1, D // 32)
    n, pages = code.shape[0], -(-code.shape[0] // page)
    full = [torch.zeros(pages * page, x.shape[1], dtype=torch.uint8) for x in (code, scale)]
    for f, x in zip(full, (code, scale)):
        f[:n] = x.to(torch.uint8)
    code, scale = (torch.stack([f, f.flip(-1)]).view(2, pages, 1, page, -1).transpose(0, 1).contiguous() for f in full)
    return code, scale, n


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("kind", ["mxfp8", "mxfp4"])
def test_every_element_under_every_scale(ops, kind, D):
    """element * 2^(byte - 127), rounded to bf16 where that has fewer bits left; NaN under 255, and of e4m3's NaN."""
    page = 128
    code, scale, n = every_byte(kind, D, page)
    cache = mx.pack(code, scale, kind).to(DEV)
    pages = cache.shape[0]
    i = lambda *t: torch.tensor(t, dtype=torch.int32, device=DEV)  # noqa: E731
    k, v = (torch.empty(n, 1, D, dtype=BF, device=DEV) for _ in (0, 1))
    ops.read_kv(k, v, i(0, n), cache, i(*range(pages)), i(0, pages), i((n - 1) % page + 1), n_max=n, kv_layout="HND")
    values = mx.dequantize(code, scale, kind)
    for half, got in ((0, k), (1, v)):
        want = values[:, half].reshape(-1, D)[:n].to(BF)
        got = got[:, 0].cpu()
        assert torch.equal(got.isnan(), want.isnan())
        wrong = (got.view(torch.int16) != want.view(torch.int16)) & ~want.isnan()
        at = wrong.nonzero()[:5].tolist()
        assert not at, [(a, int(code[a[0] // page, half, 0, a[0] % page, a[1]]), int(scale[a[0] // page, half, 0, a[0] % page, 0]),
                         got[tuple(a)].item(), want[tuple(a)].item()) for a in at]
