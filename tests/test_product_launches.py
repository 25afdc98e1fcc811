"""Which tiles the products of the feed-forward section run on: the sizes that the GPU tests hold against formulas reach every kernel.

The GPU tests of test_gpu_tiles.py tell the library of eight CUs, so that sizes of a few thousand rows are as many rounds of tiles as
large calls are on a whole GPU."""
import ctypes

import pytest

from physicsnemo_amd import _lib

BF16, F32, INT8 = 2, 4, 1
PLAIN, GATED, BACK, PEAK, CODES = range(5)
LARGE, MEDIUM, SMALL, FEW = range(4)

# rows, channels, hidden units, with eight CUs
GATED_SIZES = [(300, 264, 300), (700, 272, 520), (1100, 512, 700), (2100, 512, 700), (3000, 512, 700), (3001, 519, 701), (2060, 264, 520)]
INT8_SIZES = [(300, 264, 300), (300, 512, 700), (700, 272, 520), (3000, 512, 700), (3001, 519, 701), (4200, 512, 700), (2100, 700, 512)]


@pytest.fixture
def lib():
    yield _lib.load()
    _lib.load().pa_set_compute_units(0)


def launches(lib, bytes_, kind, rows, columns, K, K2=0):
    out = (ctypes.c_int64 * 4)()
    assert lib.pa_product_launches(bytes_, kind, rows, columns, K, K2, out) == 0
    return [(out[0], out[1])] + ([(out[2], out[3])] if out[2] else [])


def padded(n, to):
    return (n + to - 1) // to * to


def products_of_gated(lib, bytes_, rows, C, F):
    """(kind, launches) of a forward and backward pass on the tile kernels."""
    Fp, Cp = padded(max(F, 16 if bytes_ == 4 else 8), 32 // bytes_), padded(max(C, 16 if bytes_ == 4 else 8), 16 // bytes_)
    return [(GATED, launches(lib, bytes_, GATED, rows, F, C)), (PLAIN, launches(lib, bytes_, PLAIN, rows, C, F)),
            (BACK, launches(lib, bytes_, BACK, rows, F, Cp, Cp)), (PLAIN, launches(lib, bytes_, PLAIN, rows, C, 2 * Fp))]


def products_of_int8(lib, rows, C, F):
    return [(PLAIN, launches(lib, INT8, PLAIN, rows, F, C)), (PEAK, launches(lib, INT8, PEAK, rows, F, C)),
            (CODES, launches(lib, INT8, CODES, rows, F, C)), (PLAIN, launches(lib, INT8, PLAIN, rows, C, F))]


def reached(found):
    return {(kind, size) for kind, parts in found for _, size in parts}, {kind for kind, parts in found if len(parts) == 2}


@pytest.mark.parametrize("bytes_", [BF16, F32])
def test_tested_sizes_of_the_gated_block_reach_every_tile(lib, bytes_):
    lib.pa_set_compute_units(8)
    sizes, split = reached([p for s in GATED_SIZES for p in products_of_gated(lib, bytes_, *s)])
    assert sizes >= {(kind, size) for kind in (PLAIN, GATED, BACK) for size in (LARGE, MEDIUM, SMALL)}
    assert split >= {PLAIN, GATED, BACK}


def test_tested_sizes_in_8_bits_reach_every_tile(lib):
    lib.pa_set_compute_units(8)
    sizes, split = reached([p for s in INT8_SIZES for p in products_of_int8(lib, *s)])
    assert sizes >= {(kind, size) for kind in (PLAIN, PEAK, CODES) for size in (LARGE, MEDIUM, SMALL)}
    assert split >= {PLAIN, PEAK, CODES}


def test_large_calls_run_on_large_tiles(lib):
    lib.pa_set_compute_units(256)
    assert launches(lib, BF16, GATED, 100_003, 1365, 512) == [(100_003, LARGE)]
    assert [size for _, size in launches(lib, BF16, PLAIN, 100_003, 512, 1365)] == [LARGE, SMALL]
    assert launches(lib, INT8, PLAIN, 200_003, 2048, 512) == [(200_003, LARGE)]
    for kind in (PEAK, CODES):
        assert launches(lib, INT8, kind, 131_072, 2048, 512) == [(131_072, LARGE)]
    assert launches(lib, F32, BACK, 28_900, 512, 128, 128) == [(28_900, LARGE)]
    assert launches(lib, BF16, PLAIN, 64, 512, 2048) == launches(lib, F32, PLAIN, 64, 512, 2048) == [(64, FEW)]
    assert launches(lib, INT8, PEAK, 1, 2048, 512) == [(1, SMALL)]


def test_every_row_has_a_launch(lib):
    for cus in (1, 8, 256, 304):
        lib.pa_set_compute_units(cus)
        for rows in (1, 63, 64, 65, 2047, 2048, 65_537, 1_000_003):
            for columns in (1, 65, 256, 1365, 4097):
                for bytes_, kinds in ((BF16, (PLAIN, GATED, BACK)), (F32, (PLAIN, GATED, BACK)), (INT8, (PLAIN, PEAK, CODES))):
                    for kind in kinds:
                        parts = launches(lib, bytes_, kind, rows, columns, 100, 100)
                        assert sum(n for n, _ in parts) == rows and all(n > 0 for n, _ in parts)
                        if len(parts) == 2:
                            assert parts[0][0] % 32 == 0  # results in blocks of 32 rows go on where the first launch ends


def test_rows_on_chip(lib):
    lib.pa_set_compute_units(256)
    on_chip = lib.pa_gated_mlp_rows_on_chip
    assert on_chip(1, 262_144, 256, 1024) == 262_144 and on_chip(1, 40, 64, 96) == 40 and on_chip(1, 100, 128, 512) == 0
    assert on_chip(1, 32_768 + 1000, 256, 1024) == 32_768  # less than half a round more
    assert on_chip(0, 262_144, 256, 1024) == on_chip(1, 262_144, 264, 1024) == on_chip(1, 262_144, 250, 1024) == 0
    assert on_chip(1, 0, 256, 1024) == -2 and on_chip(2, 8, 8, 8) == -3


def test_refusals(lib):
    out = (ctypes.c_int64 * 4)()
    ask = lambda b=2, kind=0, rows=8, columns=8, K=8, K2=0, to=out: lib.pa_product_launches(b, kind, rows, columns, K, K2, to)
    assert ask() == 0 and ask(to=None) == -1
    assert ask(rows=0) == ask(columns=0) == ask(K=0) == ask(K2=-1) == -2
    assert ask(b=3) == ask(kind=-1) == ask(kind=5) == ask(kind=PEAK) == ask(b=1, kind=GATED) == ask(b=1, kind=BACK) == -3
    assert ask(rows=1 << 41) == ask(columns=1 << 20) == ask(K=1 << 20) == ask(K2=1 << 20) == -3
