"""Sizes, ranges and host-side state of the training losses, without a GPU."""

import pytest

from fuselse_amd import _lib


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
