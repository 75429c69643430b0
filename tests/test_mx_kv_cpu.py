"""Block-scaled caches and windowed attention: what is refused, without a GPU (the library's checks come before any launch)."""
import ctypes

import pytest
import torch

from magicdec_amd import _lib, ops

BF = torch.bfloat16
HND, BF16, FP8, MX8, MX4 = 0x100, 0, 1, 2, 3
OK, INVALID, UNSUPPORTED, WORKSPACE = 0, -1, -2, -4
P = ctypes.c_void_p(4096)                 # an aligned address that no check reads


def test_row_bytes():
    lib = _lib.load()
    for kind, name in ((MX8, "mxfp8"), (MX4, "mxfp4")):
        for D in (64, 128):
            assert lib.md_kv_row_bytes(kind | HND, D) == ops.mx_row_bytes(D, name)
    assert lib.md_kv_row_bytes(BF16, 128) == 256 and lib.md_kv_row_bytes(FP8, 64) == 64
    assert lib.md_kv_row_bytes(MX8, 96) == 0 and lib.md_kv_row_bytes(4, 128) == 0
    for bad in (("fp8", 128), ("mxfp8", 96), ("mxfp4", 32)):
        with pytest.raises(ValueError):
            ops.mx_row_bytes(bad[1], bad[0])
    assert ops.mx_kv_cache(3, 2, 64, "mxfp4", page_size=32, device="cpu").shape == (3, 2, 2, 32, 34)


def append(kind=MX8 | HND, D=128, page=128, k=P, B=2, n=4, KH=2, ks=256):
    return _lib.load().md_append_paged_kv(k, P, ks, ks, P, P, P, P, P, B, n, KH, D, page, kind, None, None, None)


def read(kind=MX8 | HND, D=128, page=128, out=P, B=2, n=4, KH=2, ks=256):
    return _lib.load().md_read_paged_kv(out, P, ks, ks, P, P, P, P, P, B, n, KH, D, page, kind, None, None, None)


def attend(kind=MX8 | HND, D=128, page=128, q=P, B=2, n=4, H=8, KH=2, stride=1024, window=0, sinks=0, scale=0.1, pages=4, ws=P, ws_bytes=1 << 40):
    return _lib.load().md_window_attn(q, stride, P, P, P, P, P, P, B, n, H, KH, D, page, window, sinks, scale, pages, kind, None, None, ws, ws_bytes, None)


@pytest.mark.parametrize("call,args,code,words", [
    (append, dict(kind=MX8), INVALID, "HND"), (append, dict(D=96), UNSUPPORTED, "head_dim"), (append, dict(page=48), INVALID, "32 rows"),
    (append, dict(k=ctypes.c_void_p(4098)), INVALID, "aligned"), (append, dict(ks=257), INVALID, "aligned"), (append, dict(kind=4 | HND), INVALID, "MD_KV_MXFP8"),
    (append, dict(B=70000), INVALID, "B=70000"), (append, dict(k=None), INVALID, "null"), (append, dict(n=0), INVALID, "n_max=0"),
    (read, dict(kind=MX4), INVALID, "HND"), (read, dict(D=32), UNSUPPORTED, "head_dim"), (read, dict(page=100), INVALID, "32 rows"),
    (read, dict(kind=FP8), INVALID, "scales"), (read, dict(kind=0x200), INVALID, "flags"), (read, dict(out=ctypes.c_void_p(4104)), INVALID, "aligned"),
    (read, dict(out=None), INVALID, "null"), (read, dict(n=0), INVALID, "n_max=0"),
    (attend, dict(kind=MX4), INVALID, "HND"), (attend, dict(D=256), UNSUPPORTED, "head_dim"), (attend, dict(page=16), INVALID, "32 rows"),
    (attend, dict(H=9), INVALID, "H=9"), (attend, dict(window=-1), INVALID, "window"), (attend, dict(sinks=-2), INVALID, "sinks"),
    (attend, dict(scale=0.0), INVALID, "sm_scale"), (attend, dict(scale=float("nan")), INVALID, "sm_scale"), (attend, dict(kind=FP8), INVALID, "scales"),
    (attend, dict(kind=0x400), INVALID, "flags"), (attend, dict(stride=1025), INVALID, "aligned"), (attend, dict(q=None), INVALID, "null"),
    (attend, dict(n=0), INVALID, "n_max=0"), (attend, dict(pages=0), INVALID, "pages=0"),
    (append, dict(page=131072), INVALID, "65 536"), (read, dict(page=131072), INVALID, "65 536"), (attend, dict(page=131072), INVALID, "65 536"),
    (append, dict(n=2147483647), INVALID, "n_max=2147483647"), (read, dict(n=2147483647), INVALID, "n_max=2147483647"),
    (attend, dict(B=1, KH=1, pages=200, ws=None), WORKSPACE, "workspace"), (attend, dict(B=1, KH=1, pages=200, ws_bytes=100), WORKSPACE, "workspace"),
])
def test_the_library_refuses(call, args, code, words):
    assert call(**args) == code
    assert words in _lib.load().md_last_error_string().decode()


def test_other_entry_points_refuse_block_scaled_caches():
    lib = _lib.load()
    assert lib.md_paged_attn(P, 1024, P, P, P, P, P, P, 2, 4, 8, 2, 128, 128, 1, 0.1, 4, MX8 | HND, None, None, P, 1 << 40, None) == INVALID
    assert lib.md_snapkv_select(P, P, P, P, 2, 8, 2, 128, 128, 512, 32, 129, 5, P, P, P, P, P, MX4 | HND, None, None, P, 1 << 40, None) == INVALID


def test_workspace_is_for_splits_alone():
    lib = _lib.load()
    need = lambda **a: lib.md_window_attn_workspace_bytes(*[a.get(n, d) for n, d in (  # noqa: E731
        ("B", 1), ("n", 1), ("H", 8), ("KH", 1), ("D", 128), ("pages", 256), ("page", 128), ("kind", MX8 | HND), ("window", 0), ("sinks", 0))])
    assert need() > 512 * 16 and need(B=512, KH=8, H=8) == 256 and need(pages=1) == 256
    assert need(window=64) == 256                               # few keys are seen, however many there are
    assert need(n=0) == 0 and need(page=33) == 0 and need(window=-1) == 0


def test_python_refuses_on_the_cpu():
    """No CPU path, and a block-scaled cache is HND and without scales."""
    cache = ops.mx_kv_cache(2, 2, 64, "mxfp8", device="cpu")
    k = torch.zeros(1, 2, 64, dtype=BF)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU"):
        ops.update_kv(k, k, i, cache, i, i, i, kv_layout="HND")
    with pytest.raises(ValueError, match="GPU"):
        ops.read_kv(k, k, i, cache, i, i, i, kv_layout="HND")
    with pytest.raises(ValueError, match="GPU"):
        ops.paged_attention(k, cache, i, i, i, i, 1, 1, None, kv_layout="HND")
    with pytest.raises(ValueError, match="HND"):
        ops._kv_args(cache, None, "NHD", 64)
    with pytest.raises(ValueError, match="kv_scales"):
        ops._kv_args(cache, (i, i), "HND", 64)
    with pytest.raises(ValueError, match="no block-scaled"):
        ops._kv_args(cache, None, "HND")
    with pytest.raises(ValueError, match="66 bytes"):
        ops._kv_args(cache, None, "HND", 128)
    assert ops._kv_args(cache, None, "HND", 64) == (MX8 | HND, None, None)
