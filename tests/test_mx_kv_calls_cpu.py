"""Calls of read_kv and paged_attention that the wrappers refuse before they reach the library, without a GPU."""
import pytest
import torch

from magicdec_amd import ops

BF = torch.bfloat16


@pytest.mark.parametrize("kind", ["bf16", "mxfp8"])
@pytest.mark.parametrize("window,sinks", [(None, -1), (5, -1), (0, 0), (-3, 2)])
def test_windows_and_first_tokens_out_of_range(kind, window, sinks):
    """Over every cache, with a window and without one."""
    cache = ops.mx_kv_cache(2, 2, 64, "mxfp8", device="cpu") if kind == "mxfp8" else torch.zeros(2, 2, 2, 128, 64, dtype=BF)
    q, i = torch.zeros(1, 2, 64, dtype=BF), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="window must be at least 1 and sinks at least 0"):
        ops.paged_attention(q, cache, i, i, i, i, 1, 1, None, kv_layout="HND", window=window, sinks=sinks)


def test_rows_that_are_written_twice_are_found():
    """Two tensors of rows in one buffer, against the sets of their elements; rows of unequal distance whose ranges meet count as shared."""
    heads, D, at = 2, 8, torch.arange(2000)
    buffer = torch.zeros(2000, dtype=BF)
    seen = set()
    for n in (1, 2, 3):
        for stride in (16, 24, 32, 40):
            for other in {stride, 24}:
                for d in range(0, 160, 8):
                    k, v = (torch.as_strided(buffer, (n, heads, D), (s, D, 1), o) for s, o in ((stride, 0), (other, d)))
                    places = [set(torch.as_strided(at, (n, heads, D), (s, D, 1), o).flatten().tolist()) for s, o in ((stride, 0), (other, d))]
                    common = bool(places[0] & places[1])
                    for a, b in ((k, v), (v, k)):
                        got = ops._share_memory(a, b)
                        assert got == common or (got and n > 1 and stride != other), (n, stride, other, d)
                    seen.add((common, n))
    assert len(seen) == 6
