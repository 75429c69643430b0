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


class OnDevice:
    """A CPU tensor that says it is on a GPU."""

    def __init__(self, t, index):
        self.t, self.index, self.is_cuda, self.device = t, index, True, f"cuda:{index}"

    def __getattr__(self, name):
        return getattr(self.t, name)

    def get_device(self):
        return self.index


@pytest.mark.parametrize("call", ["read_kv", "paged_attention"])
def test_scales_of_another_device_are_refused(call, monkeypatch):
    """The kernels read a static-scale cache's scales on the current device, as all else."""
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    monkeypatch.setattr(ops._lib, "load", lambda: pytest.fail("the library was called"))
    KH, D = 2, 64
    here = lambda t: OnDevice(t, 0)  # noqa: E731
    cache = here(torch.zeros(1, 2, KH, 128, D).to(ops.FP8_DTYPE))
    rows = [here(torch.zeros(1, KH, D, dtype=BF)) for _ in (0, 1)]
    i = here(torch.tensor([0, 1], dtype=torch.int32))
    for other in (0, 1):
        scales = [here(torch.ones(KH)) for _ in (0, 1)]
        scales[other] = OnDevice(torch.ones(KH), 1)
        with pytest.raises(ValueError, match="cuda:1"):
            if call == "read_kv":
                ops.read_kv(*rows, i, cache, i, i, i, kv_scales=tuple(scales), kv_layout="HND")
            else:
                ops.paged_attention(rows[0], cache, i, i, i, i, 1, 1, None, kv_scales=tuple(scales), kv_layout="HND", window=5)
