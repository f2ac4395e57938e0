"""Sizes, ranges and host-side state of the training losses, without a GPU."""

import ctypes

import pytest
import torch

from fuselse_amd import _lib, ext


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("alone", [0, 1])
def test_a_forwards_workspace_does_not_grow_with_the_logits(dtype, alone):
    """Packed hidden states, some words a row, and a piece of at most 256 MB each
    of the packed projection and of the rows' (max, sum) pairs."""
    lib = _lib.load()
    for n in (100, 4096, 65536, 1 << 20):
        for v in (32000, 128256, 1 << 21, 1 << 24):
            for d in (64, 130):
                nbytes = lib.fl_linear_ce_workspace_bytes(n, v, d, dtype, alone, 0, d)
                rows = n * (2 * (2 if dtype == 0 else 1) * (-(-d // 64) * 64) + 32)
                # a piece is 2048 vocabulary entries at least: 17 pairs a row
                assert nbytes <= rows + (1 << 28) * 2 + 17 * 8 * n + (1 << 16), (n, v, d, nbytes)


def test_distillation_pairs_refusals():
    lib = _lib.load()
    vp = ctypes.c_void_p(4096)

    def fwd(pairs):
        return lib.fl_distill_fwd_pairs(vp, 2, 2, 8, 8, 8, 0, vp, 0, vp, 2, 1.0, 0, vp, vp, vp, pairs, None, vp, 1 << 30,
                                        None)

    def bwd(pairs, rows=2):
        return lib.fl_distill_bwd_pairs(vp, 1, None, vp, rows, 2, 8, 8, 8, 0, vp, 0, vp, 2, 1.0, pairs, vp, None)

    for call in (fwd, bwd):
        assert call(None) == 1 and "NULL" in lib.fl_last_error().decode()
        assert call(ctypes.c_void_p(4104)) == 1 and "16-byte" in lib.fl_last_error().decode()
    assert bwd(None, rows=0) == 0


def test_remembered_workspace_sizes_stay_few(monkeypatch):
    """Calls of ever new numbers of rows do not make the host's table grow
    without end, whichever operator they call."""
    monkeypatch.setattr(ext._lib, "call", lambda *a: None)
    monkeypatch.setattr(ext, "_stream", lambda t: 0)
    monkeypatch.setattr(ext, "_ws_cache", {})
    x, i = torch.zeros(5000, 2), torch.zeros(5000, 1, dtype=torch.int64)
    for n in range(1, 5000):
        ext._distill_fwd(x[:n], x[:n, :1].contiguous(), i[:n], 1.0, 0, False)
    assert len(ext._ws_cache) <= 4096
    ext._ws_cache.clear()
    for n in range(1, 5000):
        ext._router_fwd(x[:n], i[:n], None)
    assert len(ext._ws_cache) <= 4096
    ext._ws_cache.clear()
    for n in range(1, 5000):
        ext._linear_fwd(x[:n], x[:3], i[:n, 0], -100, 0, 0.0, False)
    assert len(ext._ws_cache) <= 4096


@pytest.mark.parametrize("call", ["fl_distill_fwd", "fl_distill_bwd"])
def test_distillation_temperatures_whose_square_leaves_the_type(call):
    """The loss carries T^2: where that or its inverse is no normal fp32 number
    the call is refused rather than answered with 0, infinity or NaN."""
    lib = _lib.load()
    vp = ctypes.c_void_p(4096)

    def code(temp):
        if call == "fl_distill_fwd":
            return lib.fl_distill_fwd(vp, 0, 2, 8, 8, 8, 0, vp, 0, vp, 2, temp, 0, vp, vp, vp, None, vp, 1 << 30, None)
        return lib.fl_distill_bwd(vp, 1, None, vp, 0, 2, 8, 8, 8, 0, vp, 0, vp, 2, temp, vp, vp, vp, None)

    for temp in (1e-25, 1e-20, 2e19, 1e30, -1.0):
        assert code(temp) == 1 and "temperature" in lib.fl_last_error().decode(), temp
    for temp in (2e-19, 1e-6, 1.0, 1e6, 5e18):
        assert code(temp) == 0, temp
