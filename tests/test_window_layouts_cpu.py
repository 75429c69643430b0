"""Which kernel of the windowed attention a call takes, and in how many parts: the workspace query lays a call out as the call itself, without a GPU."""
import pytest

from magicdec_amd import _lib
from tests import window_layouts as wl


@pytest.fixture(scope="module")
def lib():
    library = _lib.load()
    if not hasattr(library, "md_debug_set_window_report"):
        pytest.skip("a library without the development knobs")
    return library


def layout_of(lib, bounds, kind):
    D, H, KH, page, B, window, sinks, n_max, most = bounds
    with wl.reported(lib) as layout:
        lib.md_window_attn_workspace_bytes(B, n_max, H, KH, D, most, page, wl.KIND[kind] | wl.HND, wl.window_of(window, kind), sinks)
        return layout()


@pytest.mark.parametrize("kind", wl.KINDS)
@pytest.mark.parametrize("bounds,layout", wl.LAYOUTS, ids=["-".join(map(str, b)) for b, _ in wl.LAYOUTS])
def test_bounds_take_the_layout_that_they_are_listed_for(lib, bounds, layout, kind):
    assert layout_of(lib, bounds, kind) == wl.of_kind(layout, kind, bounds[0])


@pytest.mark.parametrize("kind", wl.KINDS)
def test_the_list_reaches_every_kernel_whole_and_in_parts(lib, kind):
    kernels = {(D, 0, rows, 32) for D in (64, 128) for rows in (16, 32)}
    kernels |= {(64, nw, 32 * nw, keys) for nw in (4, 8) for keys in (32, 64)}
    kernels |= {(128, nw, 32 * nw, keys) for nw, keys in ((4, 32), (4, 64), (8, 32), (8, 128))}
    if kind == "mxfp4":
        kernels.add((64, 0, 16, 64))
    reached = {(b[0], *layout_of(lib, b, kind)) for b, _ in wl.LAYOUTS}
    assert reached == {(*k, parts) for k in kernels for parts in ("whole", "few", "many")}


@pytest.mark.parametrize("kind", wl.KINDS)
def test_windows_that_hide_keys_are_among_them(lib, kind):
    """Of every kernel whole, and of every kernel in parts, but for the joins of more than 8 parts."""
    hiding = {(b[0], *layout_of(lib, b, kind)) for b, _ in wl.LAYOUTS if 0 < b[5] < wl.lengths(b)[0][0]}
    assert hiding >= {(b[0], *layout_of(lib, b, kind)) for b, layout in wl.LAYOUTS if layout[3] != "many" and not (layout[0] == 0 and layout[2] == 64)}


def test_no_report_without_asking(lib):
    with wl.reported(lib) as layout:
        pass
    lib.md_window_attn_workspace_bytes(1, 1, 8, 1, 128, 256, 128, 2 | wl.HND, 0, 0)
    assert layout()[:3] == (0, 0, 0)
