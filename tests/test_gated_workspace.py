"""What the gated block asks of its caller's memory."""
import pytest

from physicsnemo_amd import _lib

F32, BF16 = 0, 1
MB = 1 << 20


@pytest.fixture
def lib():
    lib = _lib.load()
    lib.pa_set_compute_units(256)
    yield lib
    lib.pa_set_compute_units(0)


@pytest.mark.parametrize("C,F", [(64, 256), (128, 512), (160, 640), (192, 768), (200, 533), (256, 1024)])
def test_rows_whose_hidden_layer_stays_on_chip_have_no_room_for_it(lib, C, F):
    """Whatever the number of rows: the weights, pieces of rows off a boundary, and less than a round of rows left over."""
    sizes = [lib.pa_gated_mlp_workspace_bytes(BF16, rows, C, F) for rows in (1 << 16, 1 << 18, 1 << 20, (1 << 20) + 7, 1 << 24)]
    weights = 2 * 2 * 3 * (C + 32) * (F + 64) + MB
    assert 0 < min(sizes) and max(sizes) <= 32768 * (C + F + 16) * 2 + weights
    assert sizes[1] == sizes[2] == sizes[4]


@pytest.mark.parametrize("dtype,C,F", [(BF16, 512, 1365), (BF16, 1024, 4096), (F32, 128, 512)])
def test_rows_of_whole_units_have_no_room_for_copies(lib, dtype, C, F):
    rows, e = 1 << 18, 2 if dtype == BF16 else 4
    hidden = rows * ((F + 15) // 16 * 16) * e
    assert hidden <= lib.pa_gated_mlp_workspace_bytes(dtype, rows, C, F) <= hidden + 2 * 3 * (C + 16) * (F + 16) * e + MB


def test_rows_that_are_not_do(lib):
    rows, C, F = 1 << 18, 257, 1028
    assert lib.pa_gated_mlp_workspace_bytes(BF16, rows, C, F) >= rows * (1028 + 264) * 2


def test_few_rows(lib):
    """The room of a small call holds either way: rows as they lie, and copied."""
    for rows in (1, 31, 300, 4096):
        for C, F in ((64, 96), (256, 1024), (512, 1365), (257, 100)):
            for dtype, e in ((BF16, 2), (F32, 4)):
                assert lib.pa_gated_mlp_workspace_bytes(dtype, rows, C, F) >= rows * (C + F) * e


@pytest.mark.parametrize("dtype,C,F", [(BF16, 256, 1024), (BF16, 512, 1365), (BF16, 64, 64), (F32, 128, 512), (F32, 64, 40)])
def test_the_backward_of_rows_of_whole_units_has_no_room_for_copies(lib, dtype, C, F):
    """dg, du and h, a 32nd of two of them in float32 for the bias gradients (bf16), and partial weight gradients: at most two per CU
    of 3 F C float32 values, in float32 for each of the pieces that rows off a boundary run in."""
    e = 2 if dtype == BF16 else 4
    group = 32 // e  # the hidden layer's columns come in 32 bytes
    Fp = (F + group - 1) // group * group
    for rows in (1 << 18, 1 << 20, 1 << 22):
        hidden = rows * 3 * Fp * e + (rows // 32 * 2 * Fp * 4 if dtype == BF16 else 0)
        need = lib.pa_gated_mlp_backward_workspace_bytes(dtype, rows, C, F)
        assert hidden <= need
        weights = 6 * (C + 32) * (Fp + 64) * e + (Fp * 2 * 4 * 64) + MB
        pieces = 1 if dtype == BF16 else (3 * Fp + 2 * C) // (3 * Fp) + 2
        assert need - hidden <= weights + pieces * 512 * (3 * Fp * C + 2 * Fp + C) * 4
    grows = [lib.pa_gated_mlp_backward_workspace_bytes(dtype, rows, C, F) for rows in (1 << 24, 1 << 25)]
    per_row = (grows[1] - grows[0]) / (1 << 24)
    assert per_row <= 1.001 * (3 * Fp * e + (2 * Fp * 4 / 32 if dtype == BF16 else 0)) + 1
