"""Which launch a product with a 4-bit matrix takes, by its sizes alone (CPU)."""
import pytest

from pdscope_amd import _lib

REGISTERS, SPLIT, TILES_64, HALVES_128, TILES_128, TILES_256 = range(1, 7)


def launch(T, N, K, G):
    return _lib.load().pdscope_linear_int4_launch(T, N, K, G)


@pytest.mark.parametrize("T,N,K,G,want", [
    # x in registers: from 131072 units on with two whole units a wave, from 98304 on with more than 12 rows
    (1, 151936, 2048, 64, REGISTERS), (8, 131088, 2048, 128, REGISTERS), (16, 131088, 2016, 32, REGISTERS),
    (16, 98320, 2048, 64, REGISTERS), (13, 121024, 1664, 64, REGISTERS), (16, 112352, 1792, 128, REGISTERS),
    # not where the other launch takes less time
    (1, 98304, 2048, 128, SPLIT), (8, 98304, 2048, 128, SPLIT), (12, 98304, 2048, 128, SPLIT), (8, 151936, 1664, 64, SPLIT),
    (1, 131072, 2048, 64, SPLIT), (16, 98304, 1664, 64, SPLIT), (14, 80000, 1664, 64, SPLIT), (16, 200064, 1536, 64, SPLIT),
    (16, 151936, 2176, 64, SPLIT), (16, 1000, 2048, 64, SPLIT), (17, 151936, 2048, 64, TILES_128),
    # more rows
    (17, 4096, 2048, 128, SPLIT), (64, 4096, 2048, 128, SPLIT), (128, 4096, 2048, 128, TILES_64),
    (512, 4096, 2048, 128, HALVES_128), (1100, 4096, 2048, 128, TILES_128), (2048, 4096, 2048, 128, TILES_256),
    (2048, 4097, 2048, 128, TILES_128), (16384, 4096, 4096, 32, TILES_256), (200, 77, 160, 32, SPLIT)])
def test_launches(T, N, K, G, want):
    assert launch(T, N, K, G) == want


@pytest.mark.parametrize("T,N,K,G", [(0, 64, 128, 32), (-1, 64, 128, 32), (1 << 25, 64, 128, 32), (4, 0, 128, 32),
                                     (4, 64, 96, 64), (4, 64, 128, 16), (4, 1 << 24, 1 << 20, 32)])
def test_sizes_outside_the_limits(T, N, K, G):
    assert launch(T, N, K, G) == 0
