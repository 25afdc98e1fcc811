"""The same tensor in two places of a feed-forward operator: gradients add up.  Against autograd in float64; tolerances as for
independent tensors, of both places together."""
import pytest
import torch

from gpu_util import announce
from oracle import numpy_oracle as no
from physicsnemo_amd import autograd as PA

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float32]


def close(got, want, r, terms, what):
    """Within roundings r of the results and of every term's size."""
    err = (got.detach().double().cpu() - want).abs()
    tol = r * (want.abs() + terms)
    assert float((err - tol).max()) <= 0, f"{what}: {float((err / tol.clamp_min(1e-30)).max()):.2f} of the tolerance"


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,C,F", [(50, 64, 96), (300, 264, 130)])
def test_gated(rows, C, F, dtype):
    """The input is the residual, gate and up have one weight and one bias."""
    announce("shared, gated", rows, C, F, dtype)
    gen = torch.Generator().manual_seed(rows)
    x = torch.randn(rows, C, generator=gen).to(dtype)
    w, wd = ((torch.rand(*s, generator=gen) - 0.5).mul_(2 / s[1] ** 0.5).to(dtype) for s in ((F, C), (C, F)))
    b, dy = torch.randn(F, generator=gen) * 0.1, torch.randn(rows, C, generator=gen).to(dtype)
    d = [t.double().requires_grad_() for t in (x, w, wd, b)]
    g = d[0] @ d[1].t() + d[3]
    y = torch.nn.functional.silu(g) * g @ d[2].t() + d[0]
    want = torch.autograd.grad(y, d, dy.double())
    gpu = [t.cuda().requires_grad_() for t in (x, w, wd, b)]
    out = PA.gated_mlp(gpu[0], gpu[1], gpu[3], gpu[1], gpu[3], gpu[2], None, act="silu", residual=gpu[0])
    got = torch.autograd.grad(out, gpu, dy.cuda())
    # sums of roundings of terms: bounded by the sums of the terms' sizes
    r = 4 * (torch.finfo(dtype).eps / 2 + (C + F + rows) * 2.0 ** -23)
    with torch.no_grad():
        h = torch.nn.functional.silu(g) * g
        dh = dy.double() @ d[2]
        dg, du = (dh * g * 1.1).abs(), (dh * torch.nn.functional.silu(g)).abs()
        sizes = [(dg + du) @ d[1].abs() + dy.double().abs(), (dg + du).t() @ d[0].abs(), dy.double().abs().t() @ h.abs(), (dg + du).sum(0)]
        close(out, y, r, h.abs() @ d[2].abs().t() + d[0].abs(), "y")
    for what, a, v, s in zip(("x", "w", "w_down", "b"), got, want, sizes):
        close(a, v, r, s, what)


@pytest.mark.parametrize("dtype", TYPES)
def test_dropout(dtype):
    """The rows are their own residual; one vector is the LayerNorm's weight and bias."""
    announce("shared, dropout", dtype)
    gen = torch.Generator().manual_seed(3)
    x, v = torch.randn(40, 72, generator=gen).to(dtype), torch.rand(72, generator=gen) + 0.5
    dy, dn = torch.randn(40, 72, generator=gen).to(dtype), torch.randn(40, 72, generator=gen).to(dtype)
    keep = torch.from_numpy(no.dropout_keep(7, 9, range(40), 72, 0.25)).double() / 0.75
    d = [t.double().requires_grad_() for t in (x, v)]
    s = d[0] + d[0] * keep
    n = torch.nn.functional.layer_norm(s, (72,), d[1], d[1], 1e-5)
    want = torch.autograd.grad([s, n], d, [dy.double(), dn.double()])
    gpu = [t.cuda().requires_grad_() for t in (x, v)]
    out = PA.dropout_add_norm(gpu[0], gpu[0], 0.25, torch.tensor([7, 9], device="cuda"), gpu[1], gpu[1], 1e-5)
    got = torch.autograd.grad(out, gpu, [dy.cuda(), dn.cuda()])
    r = 4 * (torch.finfo(dtype).eps / 2 + 80 * 2.0 ** -23)
    with torch.no_grad():
        xh = torch.nn.functional.layer_norm(s, (72,), eps=1e-5)
        rstd = 1 / (s.var(-1, unbiased=False, keepdim=True) + 1e-5).sqrt()
        t = (dn.double() * d[1]).abs()
        ds = dy.double().abs() + rstd * (t + t.mean(-1, keepdim=True) + xh.abs() * (t * xh.abs()).mean(-1, keepdim=True))
        close(out[0], s, r, s.abs(), "y")
        close(out[1], n, r, (xh * d[1]).abs() + d[1], "n")
        close(got[0], want[0], r, ds * (1 + keep), "dx")
        close(got[1], want[1], r, (dn.double().abs() * (1 + xh.abs())).sum(0), "d gamma + d beta")
