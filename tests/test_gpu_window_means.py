"""Gradients of attention over long windows whose inputs have means far from zero: what cancels in the definition has to cancel in the kernels.

Compared in the 2-norm with the definition in 64 bits and with its plain float32 form.  float32: twice the plain form's error, and 16 u (u = 2^-24)
for running sums over some sixty tiles, each a truncation of the matrix unit's of up to u of the partial sum (a third of sixty u, on both sums that a
weight goes through).  bfloat16: one r = 2^-8 for the three roundings of weights, ds and result (each r / sqrt(3) at most in the 2-norm, independent)."""
import pytest
import torch

from gpu_util import announce
from physicsnemo_amd import autograd as PA
from test_gpu_window import BF, F32

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
MEANS = [(0, 0, 0, 0), (0, 8, 0, 0), (0, 0, 8, 0), (8, 0, 0, 0), (0, 0, 0, 8), (0, 8, 8, 0), (1, 8, 8, 8), (0, 64, 64, 0)]  # of q, k, v, dy


def gradients(q, k, v, dy, reach, dtype):
    """The definition in `dtype`, a thousand queries at a time."""
    q, k, v, dy = (t[0].to(dtype) for t in (q, k, v, dy))
    N, H, D = q.shape
    y, dq, dk, dv = (torch.zeros_like(q) for _ in range(4))
    j = torch.arange(N, device="cuda")
    for h in range(H):
        for a in range(0, N, 1000):
            b = min(N, a + 1000)
            lo, hi = max(0, a - reach), min(N, b + reach)
            far = (j[None, lo:hi] - j[a:b, None]).abs() > reach
            K, V = k[lo:hi, h].contiguous(), v[lo:hi, h].contiguous()
            p = torch.softmax((torch.mm(q[a:b, h], K.t()) * D ** -0.5).masked_fill(far, -torch.inf), -1)
            dp = torch.mm(dy[a:b, h], V.t())
            ds = p * (dp - (p * dp).sum(-1, keepdim=True))
            y[a:b, h] = torch.mm(p, V)
            dq[a:b, h] = D ** -0.5 * torch.mm(ds, K)
            dk[lo:hi, h] += D ** -0.5 * torch.mm(ds.t(), q[a:b, h])
            dv[lo:hi, h] += torch.mm(p.t(), dy[a:b, h])
    return y, dq, dk, dv


def errors(means, D, dtype, bias):
    N, reach = 3000, 1000
    gen = torch.Generator("cuda").manual_seed(D)
    q, k, v, dy = ((torch.randn(1, N, 2, D, generator=gen, device="cuda") + m).to(dtype) for m in means)
    want, plain = (gradients(q, k, v, dy, reach, t) for t in (torch.float64, torch.float32))
    leaves = [t.requires_grad_(True) for t in (q, k, v)] + ([torch.zeros(8, 2, device="cuda", requires_grad=True)] if bias else [])
    out = PA.window_attention(*leaves[:3], window=(reach, reach), bias=leaves[3] if bias else None, max_distance=20)
    got = (out.detach(), *torch.autograd.grad(out, leaves, dy)[:3])
    off = lambda t, w: float((t.reshape(w.shape).double() - w).norm() / w.norm())
    return {n: (off(g, w), off(p, w)) for n, g, w, p in zip(("y", "dq", "dk", "dv"), got, want, plain)}


@pytest.mark.parametrize("D", [16, 64, 128])
@pytest.mark.parametrize("means", [m for m in MEANS if m[2] == 0])
def test_sums_that_a_start_would_bias(means, D):
    """float32: dk and dv, whose products started from the denominators and from delta."""
    announce("starts", means, D)
    for name, (own, plain) in errors(means, D, F32, False).items():
        print(f"{name} {own:.2e} {plain:.2e}", flush=True)
        if name in ("dk", "dv"):
            assert own <= 2 * plain + 16 * U, (name, own, plain)


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [16, 32, 40, 64, 128])
@pytest.mark.parametrize("means", MEANS)
def test_means_far_from_zero(means, D, dtype, bias):
    """delta from a rounded result, and score gradients that are rounded before they meet the keys, leave multiples of the means behind."""
    announce("means", means, D, dtype, bias)
    for name, (own, plain) in errors(means, D, dtype, bias).items():
        print(f"{name} {own:.2e} {plain:.2e}", flush=True)
        assert own <= 2 * plain + (16 * U if dtype == F32 else 2.0 ** -8), (name, own, plain)
