"""Bounds of calls of the windowed attention that between them take every way of laying rows and keys over workgroups, and what a library with
development knobs says of a call's."""
import contextlib
import ctypes

KINDS = ["bf16", "fp8", "mxfp8", "mxfp4"]
KIND = {"bf16": 0, "fp8": 1, "mxfp8": 2, "mxfp4": 3}
HND = 0x100

# (D, H, KH, page, requests, window, sinks, n_max, pages of a request at most), and the layout that they take whatever the cache's kind:
# (wavefronts that share tiles, or 0; rows of a workgroup; keys of a tile; parts of the keys: "whole", "few", to 8, or "many", which are joined another way).
# Tiles of 64 keys of the kernel of few rows are those of 4-bit heads of 64, others have 32 there.
LAYOUTS = [
    ((64, 4, 1, 64, 2, 0, 0, 1, 2), (0, 16, 32, "whole")), ((64, 4, 1, 64, 2, 20, 3, 1, 2), (0, 16, 32, "whole")),
    ((64, 4, 1, 64, 2, 0, 0, 1, 9), (0, 16, 32, "few")), ((64, 4, 1, 32, 2, 600, 70, 1, 40), (0, 16, 32, "few")),
    ((64, 4, 1, 128, 2, 0, 0, 1, 9), (0, 16, 32, "many")), ((64, 8, 8, 128, 17, 0, 0, 1, 9), (0, 16, 64, "whole")),
    ((64, 8, 2, 128, 17, 0, 0, 1, 100), (0, 16, 64, "few")), ((64, 4, 1, 128, 9, 0, 0, 1, 300), (0, 16, 64, "many")),
    ((64, 7, 1, 64, 2, 0, 0, 4, 2), (0, 32, 32, "whole")), ((64, 7, 1, 64, 2, 20, 3, 4, 2), (0, 32, 32, "whole")),
    ((64, 7, 1, 64, 2, 0, 0, 4, 9), (0, 32, 32, "few")), ((64, 7, 1, 32, 2, 600, 70, 4, 40), (0, 32, 32, "few")),
    ((64, 7, 1, 128, 2, 0, 0, 4, 9), (0, 32, 32, "many")),
    ((64, 1, 1, 96, 9, 0, 0, 2500, 2), (4, 128, 32, "whole")), ((64, 4, 1, 32, 2, 20, 3, 1100, 4), (4, 128, 32, "whole")),
    ((64, 7, 1, 96, 17, 0, 0, 40, 100), (4, 128, 32, "few")), ((64, 4, 1, 32, 17, 900, 5, 130, 40), (4, 128, 32, "few")),
    ((64, 7, 1, 96, 9, 0, 0, 16, 300), (4, 128, 32, "many")),
    ((64, 1, 1, 64, 9, 0, 0, 2500, 3), (4, 128, 64, "whole")), ((64, 4, 1, 64, 2, 20, 3, 1100, 2), (4, 128, 64, "whole")),
    ((64, 1, 1, 64, 3, 0, 0, 2500, 40), (4, 128, 64, "few")), ((64, 4, 1, 128, 17, 900, 5, 130, 40), (4, 128, 64, "few")),
    ((64, 7, 1, 128, 9, 0, 0, 16, 300), (4, 128, 64, "many")),
    ((64, 1, 1, 160, 17, 0, 0, 2500, 3), (8, 256, 32, "whole")), ((64, 6, 3, 32, 3, 20, 3, 1100, 4), (8, 256, 32, "whole")),
    ((64, 1, 1, 96, 3, 0, 0, 2500, 40), (8, 256, 32, "few")), ((64, 1, 1, 32, 17, 900, 5, 1100, 40), (8, 256, 32, "few")),
    ((64, 1, 1, 160, 2, 0, 0, 520, 300), (8, 256, 32, "many")),
    ((64, 1, 1, 128, 17, 0, 0, 2500, 4), (8, 256, 64, "whole")), ((64, 6, 3, 64, 3, 20, 3, 1100, 2), (8, 256, 64, "whole")),
    ((64, 1, 1, 128, 3, 0, 0, 2500, 40), (8, 256, 64, "few")), ((64, 1, 1, 128, 17, 900, 5, 1100, 40), (8, 256, 64, "few")),
    ((64, 1, 1, 128, 2, 0, 0, 520, 300), (8, 256, 64, "many")),
    ((128, 4, 1, 64, 2, 0, 0, 1, 2), (0, 16, 32, "whole")), ((128, 4, 1, 64, 2, 20, 3, 1, 2), (0, 16, 32, "whole")),
    ((128, 4, 1, 64, 2, 0, 0, 1, 9), (0, 16, 32, "few")), ((128, 4, 1, 32, 2, 600, 70, 1, 40), (0, 16, 32, "few")),
    ((128, 4, 1, 128, 2, 0, 0, 1, 9), (0, 16, 32, "many")),
    ((128, 7, 1, 64, 2, 0, 0, 4, 2), (0, 32, 32, "whole")), ((128, 7, 1, 64, 2, 20, 3, 4, 2), (0, 32, 32, "whole")),
    ((128, 7, 1, 64, 2, 0, 0, 4, 9), (0, 32, 32, "few")), ((128, 7, 1, 32, 2, 600, 70, 4, 40), (0, 32, 32, "few")),
    ((128, 7, 1, 128, 2, 0, 0, 4, 9), (0, 32, 32, "many")),
    ((128, 4, 1, 32, 9, 0, 0, 520, 4), (4, 128, 32, "whole")), ((128, 4, 1, 32, 2, 100, 4, 40, 4), (4, 128, 32, "whole")),
    ((128, 1, 1, 96, 2, 0, 0, 2500, 40), (4, 128, 32, "few")), ((128, 1, 1, 32, 9, 900, 5, 1100, 40), (4, 128, 32, "few")),
    ((128, 7, 1, 96, 9, 0, 0, 16, 300), (4, 128, 32, "many")),
    ((128, 4, 1, 64, 9, 0, 0, 520, 2), (4, 128, 64, "whole")), ((128, 4, 1, 64, 2, 100, 4, 40, 2), (4, 128, 64, "whole")),
    ((128, 1, 1, 128, 3, 0, 0, 1100, 40), (4, 128, 64, "few")), ((128, 1, 1, 128, 9, 900, 5, 1100, 40), (4, 128, 64, "few")),
    ((128, 7, 1, 128, 9, 0, 0, 16, 100), (4, 128, 64, "many")),
    ((128, 1, 1, 64, 17, 0, 0, 2500, 4), (8, 256, 32, "whole")), ((128, 6, 3, 64, 2, 20, 3, 1100, 2), (8, 256, 32, "whole")),
    ((128, 1, 1, 64, 3, 0, 0, 2500, 100), (8, 256, 32, "few")), ((128, 1, 1, 32, 17, 900, 5, 1100, 40), (8, 256, 32, "few")),
    ((128, 7, 1, 96, 3, 0, 0, 40, 300), (8, 256, 32, "many")),
    ((128, 1, 1, 128, 17, 0, 0, 2500, 2), (8, 256, 128, "whole")), ((128, 1, 1, 128, 9, 100, 4, 2500, 2), (8, 256, 128, "whole")),
    ((128, 1, 1, 128, 2, 0, 0, 2500, 40), (8, 256, 128, "few")), ((128, 1, 1, 128, 17, 900, 5, 1100, 40), (8, 256, 128, "few")),
    ((128, 7, 1, 128, 3, 0, 0, 40, 300), (8, 256, 128, "many")),
]


def of_kind(layout, kind, D):
    """The layout of a call over a cache of this kind."""
    nw, rows, keys, parts = layout
    return nw, rows, keys if nw or (kind == "mxfp4" and D == 64) else 32, parts


def window_of(window, kind):
    """No window over the caches that md_paged_attn is for is one longer than all."""
    return window or (1 << 20 if kind in ("bf16", "fp8") else 0)


@contextlib.contextmanager
def reported(lib):
    """What the library's last call inside took: () -> (wavefronts, rows, keys, parts in words), or None of a library without the knobs."""
    if not hasattr(lib, "md_debug_set_window_report"):
        yield lambda: None
        return
    report = (ctypes.c_int * 5)()
    lib.md_debug_set_window_report(ctypes.cast(report, ctypes.c_void_p))
    try:
        yield lambda: (report[0], report[1], report[4], "whole" if report[3] == 1 else "few" if report[3] <= 8 else "many")
    finally:
        lib.md_debug_set_window_report(None)


def lengths(bounds):
    """Tokens and new rows of the requests, within the bounds: one long, one with few rows, an empty one, short ones."""
    D, H, KH, page, B, window, sinks, n_max, most = bounds
    long = min(most * page - 5, 1300 if window >= 600 else 700)
    new = max(1, min(n_max, long - 40, 290))
    lens = [long, min(most * page, 333), 0, 40] + [1 + 13 * (b % 8) for b in range(4, B)]
    rows = [new, min(n_max, 5), 0, 1] + [b % 2 for b in range(4, B)]
    return lens[:B], rows[:B]
