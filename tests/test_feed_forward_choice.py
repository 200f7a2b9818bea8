"""Which kernel and tile a 16-bit product takes (host code): the shapes that the GPU tests run reach every one."""

import pytest

from ffn_shapes import FEW_ROWS, PAIRS
from triton_metal import _core, cuda


@pytest.mark.parametrize("case", PAIRS, ids=str)
def test_shapes_of_the_pairs(case):
    mode, M, N, K, epilogue, columns, tiles = case
    extra = dict(activation="gelu", pre=True, residual=mode == "linear") if epilogue else {}
    assert cuda.linear_choice(mode, M, N, K, x_by_k=mode != "pair", **extra) == ("pairs", columns, tiles)
    assert tiles > 74 and M % 256 and N % 128 and K % 64


@pytest.mark.parametrize("case", FEW_ROWS, ids=str)
def test_shapes_of_the_few_row_kernel(case):
    mode, M, N, K, rows, split = case
    assert cuda.linear_choice(mode, M, N, K) == ("few rows", rows, split)


def test_every_tile_is_reached():
    widths = {(mode, columns) for mode, _, _, _, _, columns, _ in PAIRS}
    assert widths == {(mode, columns) for mode in cuda.LINEAR_MODES for columns in (128, 256, 512)}
    tiles = {(mode, rows, split) for mode, _, _, _, rows, split in FEW_ROWS}
    for mode in ("linear", "gated", "sum"):
        assert {(rows, split) for m, rows, split in tiles if m == mode} >= (
            {(rows, split) for rows in (16, 32, 64) for split in (2, 4, 8)} | {(128, 1), (128, 2), (128, 4)})


def test_refusals():
    for bad in (("linear", 0, 8, 8), ("linear", 8, 1 << 31, 8), ("linear", 8, 8, -1)):
        with pytest.raises(RuntimeError, match="positive 32-bit extents"):
            cuda.linear_choice(*bad)
    assert cuda._lib.tmx_debug_linear_choice(4, 0, 0, 0, 1, 1, 1, 1, 148, None) == -1
    assert "mode 0...3" in _core.last_error()


def test_a_grid_whose_extent_passes_64_bits_covers_everything():
    """2^60 programs of 128 rows are not 0 rows: the operands are looked at, and found too short."""
    import ctypes

    from triton_metal import kernels
    for cls, scalars in ((kernels.Linear, (8, 16, 32, 32, 1, 16, 1, 16, 16, 16)),
                         (kernels.ResidualNorm, (8, 16, _core.float_bits(1.0), _core.float_bits(1e-6), 16))):
        kern = cls("bf16")
        try:
            n = len(kern.names)
            values = (ctypes.c_int64 * n)(0x10000000, 0x20000000, 0x30000000, *scalars)
            lengths = (ctypes.c_int64 * n)(64, 64, 64)
            for gx, gy in ((1 << 60, 1), (1 << 57, 1), (1, 1 << 57)):
                assert cuda._lib.tmx_launch_on(kern.handle, 0, gx, gy, 1, 128, kern._kinds, values, lengths, n) == -1
                assert "beyond its" in _core.last_error()
        finally:
            kern.release()
