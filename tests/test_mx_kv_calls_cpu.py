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
