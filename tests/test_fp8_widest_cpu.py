"""The widest rows that 8-bit tiles take: a tile's rows of codes lie within what one descriptor of its loads can hold, 2^32 - 1 bytes."""
import pytest

from sharpinference_amd.ops import fp8, lib

MOST = (1 << 32) - 1
WIDEST = [fp8.FP8_MOST_K, fp8.FP8_MOST_K - 126, fp8.FP8_MOST_K - 127, 1 << 23, 5120, 128, 1]


@pytest.mark.parametrize("K", WIDEST)
def test_tiles_are_no_higher_than_their_loads_reach(K):
    row = -(-K // 128) * 128
    assert fp8.grouped_tile_fp8(K) * row <= MOST
    for M in (65, 193, 256, 1024, 8192):
        for N in (1, 128, 2048, 16384):
            for gated in (False, True):
                assert fp8.tile_fp8(M, N, K, gated, 256)[0] * row <= MOST, (M, N, gated)


def test_heights_of_rows_that_are_not_so_wide_stay():
    assert fp8.tile_fp8(8192, 16384, 5120, False, 256)[0] == 256 and fp8.grouped_tile_fp8(5120) == 256 and fp8.grouped_tile_fp8(2048) == 128
    assert fp8.grouped_tile_fp8(fp8.FP8_MOST_K - 127) == 256 and fp8.grouped_tile_fp8(fp8.FP8_MOST_K) == 192


def test_the_entries_refuse_a_tile_beyond_it():
    """(1001: the argument error; nothing is launched)"""
    K, x = fp8.FP8_MOST_K, 1 << 20
    assert lib.load().sharpi_fp8_tiles(x, x, 300, x, x, 64, x, 1, 300, 40, K, 0, 0, 1, 0, 256, 2, 1, None) == 1001
    assert lib.load().sharpi_fp8_tiles_gated(x, x, 300, x, x, 128, x, x, 300, 40, K, 0, 0, 1, 0, 0, 1, 0.0, 256, None) == 1001
