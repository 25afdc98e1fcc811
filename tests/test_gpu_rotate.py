"""Norms of queries and keys with the rotation by their positions on the GPU against the formulas in 64 bits.

r = eps / 2 of the type, u = 2^-24: the norm's factor is off by (D + 8) u of itself, an angle's cos and sin by 4 u, a channel by that of its pair's
magnitude; gradients carry the same factors through their formula; weight gradients are float32 sums of n terms, (n + 8) u of their magnitudes."""
import pytest
import torch

from gpu_util import announce
from physicsnemo_amd import autograd as PA
from physicsnemo_amd import functional as PF

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def turned(x, angle, interleaved):
    """Pairs of x's channels turned by `angle` (.., pairs), in x's type."""
    R = 2 * angle.shape[-1]
    a, b = (x[..., 0:R:2], x[..., 1:R:2]) if interleaved else (x[..., :R // 2], x[..., R // 2:R])
    c, s = torch.cos(angle), torch.sin(angle)
    c, s = a * c - b * s, a * s + b * c
    return torch.cat([torch.stack([c, s], -1).flatten(-2) if interleaved else torch.cat([c, s], -1), x[..., R:]], -1)


def pair_size(x, pairs, interleaved):
    """Magnitude of every channel's pair, at the channel."""
    R = 2 * pairs
    a, b = (x[..., 0:R:2], x[..., 1:R:2]) if interleaved else (x[..., :R // 2], x[..., R // 2:R])
    m = a.abs() + b.abs()
    return torch.cat([torch.stack([m, m], -1).flatten(-2) if interleaved else torch.cat([m, m], -1), x[..., R:].abs()], -1)


def derived(x, w, angle, dy, eps, norm, interleaved):
    """(y, dx, dw) with tolerances; angle (B or 1, N, 1, pairs) float64."""
    r, D, pairs = torch.finfo(x.dtype).eps / 2, x.shape[-1], angle.shape[-1]
    x, dy, e = x.double(), dy.double(), (D + 24) * U
    w = torch.ones(D, dtype=torch.float64, device=x.device) if w is None else w.double()
    rs = (x.square().mean(-1, keepdim=True) + eps).rsqrt() if norm else torch.ones_like(x[..., :1])
    xh = x * rs
    y = turned(xh * w, angle, interleaved)
    tol_y = r * y.abs() + e * pair_size(xh * w, pairs, interleaved)
    g = turned(dy, -angle, interleaved)
    e_g = 8 * U * pair_size(dy, pairs, interleaved)
    t = g * w
    dot = (t * xh).mean(-1, keepdim=True) if norm else torch.zeros_like(rs)
    dx = rs * (t - xh * dot)
    e_t = e_g * w.abs() + 2 * U * t.abs()
    e_dot = ((e_t + 2 * e * t.abs()) * xh.abs()).mean(-1, keepdim=True) if norm else 0 * rs
    tol_dx = r * dx.abs() + rs * (e_t + xh.abs() * e_dot + 2 * e * (t.abs() + (xh * dot).abs()))
    n = x.shape[0] * x.shape[1] * x.shape[2]
    dw, tol_dw = (g * xh).sum((0, 1, 2)), ((e_g + (e + (n + 8) * U) * g.abs()) * xh.abs()).sum((0, 1, 2))
    return (y, tol_y), (dx, tol_dx), (dw, tol_dw)


def check(got, want, what):
    value, tol = want
    got = got.detach().double()
    assert torch.isfinite(got).all(), f"{what}: not finite"
    worst = float(((got - value).abs() / tol.clamp_min(1e-30)).max())
    assert bool(((got - value).abs() <= tol + 1e-30).all()), f"{what}: {worst:.3f} of the tolerance"
    return worst


def angles(positions, frequencies):
    pos = positions.double()
    f = frequencies.double()
    a = pos[..., None] * f if f.ndim == 1 else (pos[..., None] * f).sum(-2)
    return (a if a.ndim == 3 else a[None])[:, :, None]


def compare(q, k, wq, wk, positions, frequencies, dyq, dyk, eps=1e-6, norm=True, interleaved=False):
    angle = angles(positions, frequencies) if positions is not None else torch.zeros(1, q.shape[1], 1, 0, dtype=torch.float64, device="cuda")
    sides = [derived(x, w, angle, dy, eps, norm, interleaved) for x, w, dy in ((q, wq, dyq), (k, wk, dyk))]
    call = dict(eps=eps, norm=norm, interleaved=interleaved)
    out = PF.norm_rotate(q, k, wq, wk, positions, frequencies, **call)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, wq, wk) if t is not None]
    with_w = leaves[2:] if wq is not None else [None, None]
    got = PA.norm_rotate(*leaves[:2], *with_w, positions, frequencies, **call)
    grads = torch.autograd.grad(got, leaves, [dyq, dyk])
    worst = []
    for s, name in enumerate("qk"):
        assert torch.equal(out[s], got[s])
        worst += [check(out[s], sides[s][0], name), check(grads[s], sides[s][1], "d" + name)]
        if wq is not None:
            worst.append(check(grads[2 + s], sides[s][2], "dw" + name))
    print("worst", [f"{w:.2f}" for w in worst], flush=True)


def make(B, N, Hq, Hk, D, dtype, seed=0):
    gen = torch.Generator("cuda").manual_seed(seed)
    draw = lambda h: (torch.randn(B, N, h, D, generator=gen, device="cuda") * 1.5).to(dtype)
    w = lambda: torch.rand(D, generator=gen, device="cuda") + 0.5
    return draw(Hq), draw(Hk), w(), w(), draw(Hq), draw(Hk)


def speeds(pairs, axes=1):
    f = 10_000.0 ** (-torch.arange(pairs, device="cuda").float() / max(pairs, 1))
    return f if axes == 1 else torch.stack([f * (a + 1) / axes for a in range(axes)])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,N,Hq,Hk,D,R", [(1, 1, 1, 1, 8, 8), (2, 3, 2, 1, 1, 0), (1, 7, 3, 2, 5, 4), (2, 65, 4, 4, 32, 32), (1, 130, 8, 2, 32, 30), (1, 33, 2, 2, 64, 32),
                                           (1, 40, 3, 3, 33, 32), (1, 17, 2, 1, 128, 128), (2, 50, 1, 1, 100, 50), (1, 9, 2, 2, 127, 64), (1, 5000, 2, 2, 16, 16)])
def test_values_and_gradients(B, N, Hq, Hk, D, R, interleaved, dtype):
    announce("rotate", B, N, Hq, Hk, D, R, interleaved, dtype)
    q, k, wq, wk, dyq, dyk = make(B, N, Hq, Hk, D, dtype, seed=N)
    positions = torch.arange(N, device="cuda") if R else None
    compare(q, k, wq, wk, positions, speeds(R // 2) if R else None, dyq, dyk, interleaved=interleaved)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("kind", [torch.int32, torch.int64, torch.float32])
@pytest.mark.parametrize("axes,batched", [(1, False), (1, True), (2, False), (3, True), (8, True)])
def test_positions(axes, batched, kind, dtype):
    """Several numbers a position, shared or one set for each sequence, far ones and negative ones among them."""
    announce("positions", axes, batched, kind, dtype)
    B, N, D = 2, 60, 32
    q, k, wq, wk, dyq, dyk = make(B, N, 3, 2, D, dtype, seed=1)
    shape = ((B,) if batched else ()) + (N,) + ((axes,) if axes > 1 else ())
    gen = torch.Generator("cuda").manual_seed(axes)
    most = 10 if kind == torch.float32 else 1 << 20
    positions = ((torch.rand(shape, generator=gen, device="cuda") * 2 - 1) * most).to(kind)
    compare(q, k, wq, wk, positions, speeds(D // 2, axes), dyq, dyk)


@pytest.mark.parametrize("far", [10 ** 5, 2 ** 24 + 1, 2 ** 31 - 1, -(2 ** 31), 10 ** 15])
def test_far_positions(far):
    """Against angles reduced with 100 digits: a product of a whole number and a float32 has more bits than a double."""
    from decimal import Decimal, getcontext
    import math
    getcontext().prec = 100
    two_pi = 2 * Decimal("3.14159265358979323846264338327950288419716939937510582097494459230781640628620899862803482534211706798214808651")
    announce("far", far)
    f = speeds(8)
    positions = torch.tensor([far, far + 1, far + 12345], device="cuda")
    angle = [[float((Decimal(int(p)) * Decimal(float(w))) % two_pi) for w in f.tolist()] for p in positions.tolist()]
    want_c, want_s = (torch.tensor([[fn(a) for a in row] for row in angle], dtype=torch.float64) for fn in (math.cos, math.sin))
    one = torch.zeros(1, 3, 1, 16, device="cuda")
    one[..., :8] = 1
    q, _ = PF.norm_rotate(one, one, positions=positions, frequencies=f, norm=False)
    got = q[0, :, 0].double().cpu()
    assert (got[:, :8] - want_c).abs().max() <= 4 * U and (got[:, 8:] - want_s).abs().max() <= 4 * U


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_parts_of_it(dtype):
    """Without weights, without the norm, without the turn; large eps; rows of zeros."""
    announce("parts", dtype)
    q, k, wq, wk, dyq, dyk = make(2, 37, 3, 1, 24, dtype, seed=2)
    positions, f = torch.arange(37, device="cuda"), speeds(12)
    compare(q, k, None, None, positions, f, dyq, dyk)
    compare(q, k, wq, wk, None, None, dyq, dyk, eps=10.0)
    compare(q, k, None, None, positions, f, dyq, dyk, norm=False)
    out = PF.norm_rotate(torch.zeros_like(q), k, wq, wk, positions, f)
    assert not out[0].any()
    same = PF.norm_rotate(q, k, norm=False)
    assert torch.equal(same[0], q) and torch.equal(same[1], k)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_views(dtype):
    announce("views", dtype)
    gen = torch.Generator("cuda").manual_seed(3)
    draw = lambda *s: torch.randn(*s, generator=gen, device="cuda").to(dtype)
    B, N, H, D = 2, 50, 4, 32
    w, positions, f = torch.rand(D, device="cuda"), torch.arange(N, device="cuda"), speeds(D // 2)
    for t in (draw(B, N, 3 * H, D), draw(B * N * 3 * H * D + 1)[1:].view(B, N, 3 * H, D), draw(B, 3 * H, N, D).transpose(1, 2), draw(B, N, 3 * H, D + 3)[..., 2:D + 2],
              draw(B, N, 1, D).expand(B, N, 3 * H, D)):
        q, k, dy = t[:, :, :H], t[:, :, H:2 * H], t[:, :, 2 * H:]
        got, want = (PF.norm_rotate(*(x.contiguous() if c else x for x in (q, k)), w, None, positions, f) for c in (False, True))
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        got, want = (PF.norm_rotate_backward(*(x.contiguous() if c else x for x in (dy, dy, q, k)), w, None, positions, f, wanted=(True, True, True, False))
                     for c in (False, True))
        assert got[3] is None and all(torch.allclose(a.float(), b.float(), rtol=0, atol=1e-3) if n == 2 else torch.equal(a, b)
                                      for n, (a, b) in enumerate(zip(got[:3], want[:3])))


def test_gradients_against_differences():
    announce("differences")
    q, k, wq, wk, dyq, dyk = make(1, 20, 2, 1, 12, torch.float32, seed=4)
    positions, f = torch.arange(20, device="cuda"), speeds(5)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, wq, wk)]
    grads = torch.autograd.grad(PA.norm_rotate(*leaves, positions, f), leaves, [dyq, dyk])
    h, size = 2.0 ** -7, 4 * float(dyq.norm() + dyk.norm())
    for n, (leaf, g) in enumerate(zip(leaves, grads)):
        way = torch.randn(leaf.shape, generator=torch.Generator("cuda").manual_seed(n), device="cuda")
        way /= way.norm()
        def value(s):
            a, b = PF.norm_rotate(*[t.detach() + (s * way if m == n else 0) for m, t in enumerate(leaves)], positions, f)
            return (a.double() * dyq).sum() + (b.double() * dyk).sum()
        assert abs(float((value(h) - value(-h)) / (2 * h)) - float((g.double() * way).sum())) <= size * (h * h + 2.0 ** -22 / h), n


def test_far_rows():
    """Elements past 2^31 and more rows than a launch has workgroups."""
    announce("far rows")
    N, H, D = (1 << 22) + 5, 4, 128
    q = torch.randn(1, N, H, D, device="cuda", dtype=torch.bfloat16)
    positions, f, w = torch.arange(N, device="cuda"), speeds(64), torch.rand(D, device="cuda") + 0.5
    assert q.numel() > 1 << 31
    out, _ = PF.norm_rotate(q, q[:, :, :1], w, w, positions, f)
    tail, _ = PF.norm_rotate(q[:, -500:].contiguous(), q[:, -500:, :1], w, w, positions[-500:], f)
    assert torch.equal(out[:, -500:], tail)
