"""Every width in tiles of 32 channels of the kernels that keep the gated block's hidden layer on chip, bf16, several blocks of rows a
workgroup: the library is told of eight CUs, so that a round is 2 048 rows (up to 128 channels) or 1 024.  Against the formulas in
64 bits, tolerances of test_gpu_gated.py."""
import pytest
import torch

from gpu_util import announce
from physicsnemo_amd import _lib
from physicsnemo_amd import functional as PF
from test_gpu_gated import NAMES, check, derived, make, on_gpu

pytestmark = pytest.mark.gpu
CUS = 8


@pytest.fixture
def eight_cus():
    lib = _lib.load()
    lib.pa_set_compute_units(CUS)
    yield
    lib.pa_set_compute_units(0)


# F: an even and an odd number of chunks of 32 hidden units, part of one, several slots of a wave's stream
@pytest.mark.parametrize("F", [96, 130, 256])
@pytest.mark.parametrize("C", [24, 64, 96, 128, 152, 160, 184, 192, 200, 224, 256])
def test_several_blocks_a_workgroup(eight_cus, C, F):
    block = 256 if C <= 128 else 128
    rows = 3 * CUS * block + (CUS - 1) * block + 45  # three whole rounds and most of a fourth, its last block part of one
    act = ("silu", "gelu", "tanh")[(C // 8 + F) % 3]
    announce("gated widths", C, F, act)
    st = make(rows, C, F, torch.bfloat16, bias=F % 2 == 0 and C != 64, seed=C + F)
    values, tols = derived(st, act, torch.bfloat16)
    gpu = on_gpu(st)
    params = [gpu[n] for n in NAMES]
    check(PF.gated_mlp_forward(gpu["x"], *params, act=act, residual=gpu["residual"]), values[0], tols[0], "y")
    for what, g, v, t in zip(("dx",) + NAMES, PF.gated_mlp_backward(gpu["x"], gpu["dy"], *params[:5], act=act), values[1:], tols[1:]):
        check(g, v, t, what)


@pytest.mark.parametrize("C", [128, 160, 256])
def test_whole_rounds_and_rows_left_over(eight_cus, C):
    """Two rounds here, less than half a round on the tile kernels."""
    block, F = 256 if C <= 128 else 128, 100
    rows = 2 * CUS * block + 3 * block - 7
    announce("gated rounds and rest", C)
    st = make(rows, C, F, torch.bfloat16, seed=C)
    values, tols = derived(st, "silu", torch.bfloat16)
    gpu = on_gpu(st)
    params = [gpu[n] for n in NAMES]
    check(PF.gated_mlp_forward(gpu["x"], *params, residual=gpu["residual"]), values[0], tols[0], "y")
    for what, g, v, t in zip(("dx",) + NAMES, PF.gated_mlp_backward(gpu["x"], gpu["dy"], *params[:5]), values[1:], tols[1:]):
        check(g, v, t, what)
