"""GELU and its derivative inside the feed-forward kernels, point by point: a gated block on rows of zeros has the gate g = b_gate and
the factor u = b_up = 1, W_down is the identity, so that y is the hidden layer itself and d b_gate the derivative.

Tolerances.  bf16: one rounding (2^-8 of the value) and the fit, which is good to 3.6e-4 of GELU down to -9 and, with float32's
roundings of an exponent up to 65 in magnitude (2^-24 65 ln 2 each, three of them), to 4e-4; its derivative is good to 7.3e-7 and
four roundings of 2^-24.  float32: the exponent -a^2 / 2 is rounded three times, 1.5 a^2 2^-24 of the value, and everything else
(reciprocal, exponential, nine multiply-adds, a product, a sum, the fit's own 5.8e-8) stays within 16 2^-24; the derivative, which
is at most 1.13, within 8 2^-24."""
import math

import pytest
import torch

from gpu_util import announce
from physicsnemo_amd import functional as PF

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float32]
# channels, rows: on chip (up to 64 channels always), few rows, tiles
PLACES = [(64, 3), (512, 1), (512, 2000)]


def points(n):
    """Gate values from -9 to 9, closest around 0, a whole number of n."""
    x = torch.cat([torch.linspace(-9, 9, 2500, dtype=torch.float64), torch.logspace(-6, 0, 200, dtype=torch.float64)])
    x = torch.cat([x, -x[-200:]])
    return x[:x.numel() // n * n].float()


def gelu64(x):
    x = x.double()
    tail = 0.5 * torch.erfc(x.abs() / math.sqrt(2))
    phi = torch.where(x > 0, 1 - tail, tail)
    return x * phi, phi + x * torch.exp(-0.5 * x * x) / math.sqrt(2 * math.pi)


def weights(C, dtype):
    return torch.zeros(C, C, device="cuda", dtype=dtype), torch.eye(C, device="cuda", dtype=dtype), torch.ones(C, device="cuda")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("C,rows", PLACES)
def test_values(C, rows, dtype):
    announce("gelu values", C, rows, dtype)
    zero, eye, one = weights(C, dtype)
    x, p = torch.zeros(rows, C, device="cuda", dtype=dtype), points(C)
    got = torch.cat([PF.gated_mlp_forward(x, zero, b, zero, one, eye, None, act="gelu")[-1] for b in p.cuda().split(C)])
    want = gelu64(p)[0]
    if dtype == torch.bfloat16:
        tol = (2.0 ** -8 + 4e-4) * want.abs()
    else:
        tol = (16 + 1.5 * p.double() ** 2) * 2.0 ** -24 * want.abs()
    over = ((got.double().cpu() - want).abs() / tol.clamp_min(1e-30)).max()
    assert over <= 1, f"{float(over):.3f} of the tolerance"


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("C,rows", [(64, 1), (512, 1)])
def test_derivatives(C, rows, dtype):
    announce("gelu derivatives", C, rows, dtype)
    zero, eye, one = weights(C, dtype)
    x, dy, p = torch.zeros(rows, C, device="cuda", dtype=dtype), torch.ones(rows, C, device="cuda", dtype=dtype), points(C)
    wanted = (False, False, True, False, False, False, False)
    got = torch.cat([PF.gated_mlp_backward(x, dy, zero, b, zero, one, eye, act="gelu", wanted=wanted)[2] for b in p.cuda().split(C)])
    want = rows * gelu64(p)[1]
    tol = 7.3e-7 + 4 * 2.0 ** -24 if dtype == torch.bfloat16 else 8 * 2.0 ** -24
    over = float((got.double().cpu() - want).abs().max() / tol)
    assert over <= 1, f"{over:.3f} of the tolerance"


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("C,rows", [(64, 2), (512, 1)])
def test_far_gates(C, rows, dtype):
    """Where GELU is x or 0 and its derivative 1 or 0, also where a float32 square overflows."""
    announce("gelu far", C, rows, dtype)
    zero, eye, one = weights(C, dtype)
    big = torch.tensor([20.0, 1e3, 2.0 ** 60, 1e18, 1e22, 2.0 ** 64, 2.0 ** 70, 3e30, 3e38], dtype=torch.float32)
    far = torch.cat([big, -big])
    b = torch.nn.functional.pad(far, (0, C - far.numel())).cuda()
    x, dy = torch.zeros(rows, C, device="cuda", dtype=dtype), torch.ones(rows, C, device="cuda", dtype=dtype)
    y = PF.gated_mlp_forward(x, zero, b, zero, one, eye, None, act="gelu")
    # float32 products are sums of three parts' products, exact for an identity
    assert torch.equal(y[0, :far.numel()].cpu(), far.clamp_min(0).to(dtype))
    slope = PF.gated_mlp_backward(x, dy, zero, b, zero, one, eye, act="gelu", wanted=(False, False, True) + (False,) * 4)[2]
    assert torch.equal(slope[:far.numel()].cpu(), rows * (far > 0).float())


@pytest.mark.parametrize("C,rows", PLACES)
def test_an_infinite_gate(C, rows):
    announce("gelu infinite", C, rows)
    gen = torch.Generator().manual_seed(C)
    draw = lambda *s: (torch.rand(*s, generator=gen) + 0.25).bfloat16().cuda()
    x, wg, wu, wd = draw(rows, C), draw(C, C), draw(C, C), draw(C, C)
    b = torch.zeros(C, device="cuda")
    b[C // 2] = float("inf")
    y = PF.gated_mlp_forward(x, wg, b, wu, None, wd, None, act="gelu")
    assert torch.equal(y, torch.full_like(y, float("inf")))
    b[C // 2] = -float("inf")  # that unit's h is 0
    y = PF.gated_mlp_forward(x, wg, b, wu, None, wd, None, act="gelu")
    wd[:, C // 2] = 0
    assert torch.equal(y, PF.gated_mlp_forward(x, wg, torch.zeros_like(b), wu, None, wd, None, act="gelu"))
    b[C // 2] = float("nan")
    assert torch.isnan(PF.gated_mlp_forward(x, wg, b, wu, None, wd + 0.25, None, act="gelu")).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [1, 5000])
def test_behind_an_8_bit_product(rows, dtype):
    """Rows of zeros have scale 0: what the activation takes is the bias."""
    announce("gelu int8", rows, dtype)
    p = points(1)
    bias = torch.cat([p, torch.tensor([float("inf"), -float("inf"), float("nan"), 1e30, -1e30])]).cuda()
    q, s = PF.quantize_int8(torch.ones(bias.numel(), 32, device="cuda"))
    y = PF.linear_int8(torch.zeros(rows, 32, device="cuda", dtype=dtype), q, s, bias, act="gelu")
    assert torch.equal(y[0].nan_to_num(), y[-1].nan_to_num())
    want = gelu64(p)[0]
    tol = (2.0 ** -8 + 4e-4 if dtype == torch.bfloat16 else (16 + 1.5 * p.double() ** 2) * 2.0 ** -24) * want.abs()
    over = ((y[0, :p.numel()].double().cpu() - want).abs() / tol.clamp_min(1e-30)).max()
    assert over <= 1, f"{float(over):.3f} of the tolerance"
    last = y[0, p.numel():].tolist()
    assert last[0] == float("inf") and last[1] == 0 and math.isnan(last[2]) and last[3] == float(torch.tensor(1e30).to(dtype)) and last[4] == 0
