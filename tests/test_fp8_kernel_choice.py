"""Which kernel the 8-bit product takes (no GPU here): a size for each of them, for the tests that have to reach
every one, and none besides."""
import math
import random

import pytest

from tierlm_amd import fp8

# name: (T, rows, n), part tiles of rows and tokens and a part block each
SIZES = {"rows_16x16_w8": (3, 301, 311), "rows_16x16_w16": (1, 308, 8486), "rows_32x16_w8": (195, 314, 314),
         "rows_32x16_w16": (9, 8500, 1982), "rows_32x32_w4": (290, 429, 302), "rows_32x32_w8": (306, 414, 525),
         "rows_64x32_w4": (65, 8424, 330), "rows_64x32_w8": (687, 356, 520), "rows_64x64_w4": (1098, 684, 1700),
         "tile_64x64_s2": (33, 12574, 306), "tile_128x64_s2": (68, 24975, 318), "tile_128x64_s4": (33, 16651, 2164),
         "tile_128x128_s2": (193, 26448, 314)}


@pytest.mark.parametrize("name", SIZES)
def test_a_size_for_each_kernel(name):
    T, rows, n = SIZES[name]
    assert fp8.matmul_kernel(rows, n, T) == name


def test_no_other_kernel():
    rng, seen = random.Random(1), set()

    def log(lo, hi):
        return int(math.exp(rng.uniform(math.log(lo), math.log(hi))))

    for _ in range(100000):
        T, rows, n = log(1, 1 << 20), log(1, 1 << 18), log(1, 1 << 14)
        if T * rows <= 1 << 35:
            seen.add(fp8.matmul_kernel(rows, n, T))
    assert seen == set(SIZES)


def test_no_launch_no_name():
    for args in ((0, 128, 1), (16, 0, 1), (16, 128, 0), (16, 128, (1 << 20) + 1), (1 << 20, 128, (1 << 15) + 1)):
        assert fp8.matmul_kernel(*args) is None
