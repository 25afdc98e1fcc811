"""Dropout + residual add + LayerNorm on the GPU: the mask bit for bit against the generator's definition, values and
gradients against the formulas in 64 bits.

Tolerances follow the roundings: r = eps / 2 of the type for each result; float32 arithmetic of a row of C elements
(C + 8) 2^-23 of its magnitudes, carried through the formulas."""
import numpy as np
import pytest
import torch

from gpu_util import announce
from oracle import numpy_oracle as no
from physicsnemo_amd import autograd as PA
from physicsnemo_amd import functional as PF

pytestmark = pytest.mark.gpu


def rng_of(seed, offset):
    return torch.tensor([seed, offset], dtype=torch.int64, device="cuda")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,C", [(1, 1), (5, 3), (7, 8), (130, 33), (64, 64), (9, 256), (33, 260), (17, 512), (6, 1000), (3, 2048),
                                    (4, 4096), (3, 4100), (2, 10007)])
def test_mask(rows, C, dtype):
    announce("mask", rows, C, dtype)
    one = torch.ones(rows, C, dtype=dtype, device="cuda")
    for seed, offset, p in ((0, 0, 0.5), (2 ** 63 - 1, 2 ** 32 - 1, 0.1), (-12345, 7, 0.9), (81985529216486895, 2 ** 32 + 3, 0.25)):
        got = PF.dropout_add_norm(one, None, p, rng_of(seed, offset)) != 0
        assert np.array_equal(got.cpu().numpy(), no.dropout_keep(seed, offset, np.arange(rows), C, p)), (seed, offset, p)


def test_mask_of_far_rows():
    """Row numbers past 2^16 with a narrow width; the mask does not depend on how many rows the call has."""
    announce("far rows")
    rows = 3_000_001
    one = torch.ones(rows, 2, dtype=torch.bfloat16, device="cuda")
    got = PF.dropout_add_norm(one, None, 0.3, rng_of(5, 6)) != 0
    pick = np.array([0, 65_535, 65_536, 1_000_003, rows - 1])
    assert np.array_equal(got.cpu().numpy()[pick], no.dropout_keep(5, 6, pick, 2, 0.3))
    assert torch.equal(PF.dropout_add_norm(one[:1000], None, 0.3, rng_of(5, 6)) != 0, got[:1000])


def test_share_kept():
    """0.9 of 2^24 elements: the count's standard deviation is sqrt(0.09 2^24) = 1229; six of them."""
    announce("share")
    one = torch.ones(1 << 16, 256, dtype=torch.bfloat16, device="cuda")
    kept = int((PF.dropout_add_norm(one, None, 0.1, rng_of(11, 0)) != 0).sum())
    assert abs(kept - 0.9 * 2 ** 24) < 6 * 1229


def derived(x, res, keep, p, gamma, beta, eps, dy, dn, dtype):
    r, C = torch.finfo(dtype).eps / 2, x.shape[-1]
    u = (C + 8) * 2.0 ** -23
    x, res, dy, dn, gamma, beta = (t.double() for t in (x, res, dy, dn, gamma, beta))
    scale = 1 / (1 - p) if p < 1 else 0.0
    s = res + torch.where(keep, x * scale, torch.zeros_like(x))
    mean, var = s.mean(-1, keepdim=True), s.var(-1, unbiased=False, keepdim=True)
    rstd = (var + eps).rsqrt()
    xh = (s - mean) * rstd
    n = xh * gamma + beta
    most = s.abs().amax(-1, keepdim=True)
    e_s = 2.0 ** -22 * (res.abs() + x.abs() * scale)
    e_xh = u * (most * rstd + xh.abs()) + e_s * rstd
    t = dn * gamma
    m1, m2 = t.mean(-1, keepdim=True), (t * xh).mean(-1, keepdim=True)
    ds = dy + rstd * (t - m1 - xh * m2)
    dx = torch.where(keep, ds * scale, torch.zeros_like(ds))
    e_back = e_xh  # the backward pass forms the same sums again
    e_ds = 2.0 ** -22 * ds.abs() + rstd * (u * (t.abs().mean(-1, keepdim=True) + t.abs() + xh.abs() * (t * xh).abs().mean(-1, keepdim=True)) +
                                           e_back * m2.abs() + xh.abs() * (t.abs() * e_back).mean(-1, keepdim=True) +
                                           u * (t - m1 - xh * m2).abs())
    rows = (x.shape[0] + 8) * 2.0 ** -23
    values = [s, n, dx, ds, (dn * xh).sum(0), dn.sum(0)]
    tols = [r * s.abs() + e_s, r * n.abs() + e_xh * gamma.abs() + 2.0 ** -22 * (xh * gamma).abs() + 2.0 ** -23 * beta.abs(),
            r * dx.abs() + scale * e_ds, r * ds.abs() + e_ds,
            (dn.abs() * e_back).sum(0) + rows * (dn * xh).abs().sum(0), rows * dn.abs().sum(0)]
    return values, tols


def check(got, want, tol, what):
    got = got.detach().double().cpu().reshape(want.shape)
    assert torch.isfinite(got).all(), f"{what}: not finite"
    over = ((got - want).abs() / tol.clamp_min(1e-30)).max()
    assert over <= 1, f"{what}: {float(over):.3f} of the tolerance"


def make(rows, C, dtype, seed=0, shift=0.0):
    gen = torch.Generator().manual_seed(seed)
    draw = lambda: torch.randn(rows, C, generator=gen).to(dtype)
    return dict(x=draw(), residual=(draw() + shift).to(dtype), dy=draw(), dn=draw(), gamma=torch.rand(C, generator=gen) + 0.5,
                beta=torch.randn(C, generator=gen))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,C", [(1, 8), (3, 2), (7, 5), (100, 33), (130, 64), (257, 128), (1000, 256), (77, 333), (65, 512), (40, 1000),
                                    (31, 2048), (19, 4096), (5, 4104), (6, 9001)])
def test_values_and_gradients(rows, C, dtype):
    announce("dropout_add_norm", rows, C, dtype)
    st = make(rows, C, dtype, seed=rows)
    p, seed, offset = 0.2, 77, 3
    keep = torch.from_numpy(no.dropout_keep(seed, offset, np.arange(rows), C, p))
    values, tols = derived(st["x"], st["residual"], keep, p, st["gamma"], st["beta"], 1e-5, st["dy"], st["dn"], dtype)
    g = {k: v.cuda() for k, v in st.items()}
    leaves = [g[k].requires_grad_(True) for k in ("x", "residual", "gamma", "beta")]
    y, n = PA.dropout_add_norm(leaves[0], leaves[1], p, rng_of(seed, offset), leaves[2], leaves[3])
    grads = torch.autograd.grad([y, n], leaves, [g["dy"], g["dn"]])
    for what, got, v, t in zip(("y", "n", "dx", "dr", "dgamma", "dbeta"), (y, n, *grads), values, tols):
        check(got, v, t, what)


@pytest.mark.parametrize("p", [0.0, 1e-12, 0.5, 1 - 1e-12, 1.0])
def test_probabilities_to_the_ends(p):
    announce("p", p)
    st = make(50, 72, torch.float32)
    keep = torch.from_numpy(no.dropout_keep(4, 4, np.arange(50), 72, p))
    assert (p > 0.9) <= bool((~keep).all()) and (p < 0.1) <= bool(keep.all())
    values, tols = derived(st["x"], st["residual"], keep, p if p < 0.9 else 1.0, st["gamma"], st["beta"], 1e-5, st["dy"], st["dn"], torch.float32)
    g = {k: v.cuda() for k, v in st.items()}
    y, n, stats = PF.dropout_add_norm(g["x"], g["residual"], p, rng_of(4, 4), g["gamma"], g["beta"], return_stats=True)
    grads = PF.dropout_add_norm_backward(g["dy"], g["dn"], g["x"], g["residual"], stats, g["gamma"], p, rng_of(4, 4))
    for what, got, v, t in zip(("y", "n", "dx", "dr", "dgamma", "dbeta"), (y, n, *grads), values, tols):
        check(got, v, t, what)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("C", [40, 37])
def test_forms(C, dtype):
    """Without a residual, without a LayerNorm, with one of the two gradients missing."""
    announce("forms", C, dtype)
    st = make(90, C, dtype)
    p = 0.3
    keep = torch.from_numpy(no.dropout_keep(1, 2, np.arange(90), C, p))
    g = {k: v.cuda() for k, v in st.items()}
    rng, zero = rng_of(1, 2), torch.zeros(90, C, dtype=dtype)
    val = lambda res, dy, dn: derived(st["x"], res, keep, p, st["gamma"], st["beta"], 1e-5, dy, dn, dtype)
    v, t = val(zero, st["dy"], zero)
    check(PF.dropout_add_norm(g["x"], None, p, rng), v[0], t[0], "y alone")
    x = g["x"].clone().requires_grad_(True)
    check(torch.autograd.grad(PA.dropout_add_norm(x, None, p, rng), x, g["dy"])[0], v[2], t[2], "dx of y alone")
    for dy, dn in ((None, "dn"), ("dy", None)):
        v, t = val(st["residual"], st[dy] if dy else zero, st[dn] if dn else zero)
        leaves = [g[k].clone().requires_grad_(True) for k in ("x", "residual", "gamma", "beta")]
        y, n = PA.dropout_add_norm(leaves[0], leaves[1], p, rng, leaves[2], leaves[3])
        got = torch.autograd.grad([y if dy else n], leaves, [g[dy or dn]], allow_unused=True)
        for what, a, b, c in zip(("dx", "dr", "dgamma", "dbeta"), got, v[2:], t[2:]):
            if a is None:
                assert not dn and what in ("dgamma", "dbeta")
            else:
                check(a, b, c, (what, dy, dn))


def test_rows_far_from_zero():
    """Rows of mean 300 and spread 1 in float32: the statistics are taken about the mean."""
    announce("shifted rows")
    st = make(64, 256, torch.float32, shift=300.0)
    keep = torch.from_numpy(no.dropout_keep(1, 1, np.arange(64), 256, 0.1))
    values, tols = derived(st["x"], st["residual"], keep, 0.1, st["gamma"], st["beta"], 1e-5, st["dy"], st["dn"], torch.float32)
    g = {k: v.cuda() for k, v in st.items()}
    y, n = PF.dropout_add_norm(g["x"], g["residual"], 0.1, rng_of(1, 1), g["gamma"], g["beta"])
    check(y, values[0], tols[0], "y")
    check(n, values[1], tols[1], "n")


def test_dropped_infinities_and_nan_do_not_pass():
    announce("dropped nan")
    keep = torch.from_numpy(no.dropout_keep(9, 9, np.arange(20), 64, 0.5)).cuda()
    x = torch.randn(20, 64, device="cuda")
    bad = torch.where(keep, x, torch.tensor([float("nan"), float("inf")], device="cuda").repeat(32))
    res = torch.randn(20, 64, device="cuda")
    assert torch.equal(PF.dropout_add_norm(bad, res, 0.5, rng_of(9, 9)), PF.dropout_add_norm(x, res, 0.5, rng_of(9, 9)))


def test_views_off_a_boundary():
    announce("dropout views")
    st = make(33, 64, torch.bfloat16)
    g = {k: v.cuda() for k, v in st.items()}
    odd = lambda t: torch.cat([torch.full((3,), float("nan"), dtype=t.dtype, device="cuda"), t.reshape(-1)])[3:].view(t.shape)
    args = (0.25, rng_of(3, 3), g["gamma"], g["beta"])
    want = PF.dropout_add_norm(g["x"], g["residual"], *args)
    got = PF.dropout_add_norm(odd(g["x"]), odd(g["residual"]), 0.25, rng_of(3, 3), odd(g["gamma"]), odd(g["beta"]))
    r = torch.finfo(torch.bfloat16).eps  # the sums run in another order: at most a step apart
    for a, b in zip(got, want):
        assert ((a.float() - b.float()).abs() <= r * b.float().abs() + 1e-5).all()


def test_graph_draws_a_new_mask_on_every_replay():
    announce("dropout graph")
    st = {k: v.cuda() for k, v in make(200, 128, torch.bfloat16).items()}
    state = rng_of(21, 100)

    def step(state):
        x = st["x"].detach().requires_grad_(True)
        y, n = PA.dropout_add_norm(x, st["residual"], 0.5, PF.dropout_advance(state), st["gamma"], st["beta"])
        return [y, n, *torch.autograd.grad([y, n], x, [st["dy"], st["dn"]])]

    eager_state = rng_of(21, 100)
    warm = torch.cuda.Stream()
    warm.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(warm):
        step(rng_of(0, 0))
    torch.cuda.current_stream().wait_stream(warm)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(state)
    seen = []
    for k in range(3):
        graph.replay()
        torch.cuda.synchronize()
        want = step(eager_state)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want)), k
        seen.append(held[0].clone())
    assert state.tolist() == eager_state.tolist() == [21, 103]
    assert not torch.equal(seen[0], seen[1]) and not torch.equal(seen[1], seen[2])


def test_changing_the_counter_before_the_backward_pass_is_refused():
    announce("dropout state changed")
    x = torch.randn(4, 16, device="cuda", requires_grad=True)
    state = rng_of(1, 0)
    y = PA.dropout_add_norm(x, None, 0.5, state)
    state.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_no_rows():
    announce("dropout empty")
    x = torch.zeros(0, 16, device="cuda", requires_grad=True)
    w, b = (torch.ones(16, device="cuda", requires_grad=True) for _ in range(2))
    y, n = PA.dropout_add_norm(x, x, 0.5, rng_of(1, 1), w, b)
    assert y.shape == n.shape == (0, 16)
    gx, gw, gb = torch.autograd.grad([y, n], [x, w, b], [torch.zeros_like(y), torch.zeros_like(n)])
    assert gx.shape == (0, 16) and not gw.any() and not gb.any()
