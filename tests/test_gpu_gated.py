"""The gated feed-forward block on the GPU against its formulas in 64 bits, values and gradients.

Tolerances are element by element and follow the roundings of the kernels: r = eps / 2 of the type wherever a value is
rounded to it (h, dg, du, the results; the bias gradients are summed before that), n 2^-23 of the sum of magnitudes for a float32 sum of n terms, 1e-6 (1 + |g|) for the
activation and 2e-6 (1 + |g|) for its derivative (their fits are good to 4e-7 and 1e-6), each carried through the products."""
import pytest
import torch

from gpu_util import announce
from physicsnemo_amd import autograd as PA
from physicsnemo_amd import functional as PF

pytestmark = pytest.mark.gpu

ACTS = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu, "relu": torch.relu, "sigmoid": torch.sigmoid,
        "tanh": torch.tanh, None: lambda v: v}
NAMES = ("w_gate", "b_gate", "w_up", "b_up", "w_down", "b_down")


def make(rows, C, F, dtype, bias=True, seed=0, shape=None):
    gen = torch.Generator().manual_seed(seed)
    draw = lambda *s: torch.rand(*s, generator=gen) * 2 - 1
    st = {"x": torch.randn(*(shape or (rows,)), C, generator=gen).to(dtype), "dy": torch.randn(*(shape or (rows,)), C, generator=gen).to(dtype),
          "residual": torch.randn(*(shape or (rows,)), C, generator=gen).to(dtype)}
    for name, o, i in (("gate", F, C), ("up", F, C), ("down", C, F)):
        st["w_" + name] = (draw(o, i) / i ** 0.5).to(dtype)
        st["b_" + name] = draw(o) / i ** 0.5 if bias else None
    return st


def on_gpu(st):
    return {k: None if v is None else v.cuda() for k, v in st.items()}


def derived(st, act, dtype):
    """(values, tolerances) of y and the seven gradients."""
    r, u23 = torch.finfo(dtype).eps / 2, 2.0 ** -23
    d = {k: None if v is None else v.double().reshape(-1, v.shape[-1]) if v.ndim != 1 else v.double() for k, v in st.items()}
    x, dy, wg, wu, wd = (d[k] for k in ("x", "dy", "w_gate", "w_up", "w_down"))
    zero = torch.zeros((), dtype=torch.float64)
    bg, bu, bd = (zero if d[k] is None else d[k] for k in ("b_gate", "b_up", "b_down"))
    M, C, F = x.shape[0], x.shape[1], wg.shape[0]
    g = (x @ wg.t() + bg).requires_grad_(True)
    a = ACTS[act](g)
    slope = torch.autograd.grad(a.sum(), g)[0]
    g, a, u = g.detach(), a.detach(), x @ wu.t() + bu
    h = a * u
    y = h @ wd.t() + bd + d["residual"]
    e_g = (C + 4) * u23 * (x.abs() @ wg.abs().t() + bg.abs())
    e_u = (C + 4) * u23 * (x.abs() @ wu.abs().t() + bu.abs())
    e_a = 1.13 * e_g + 1e-6 * (1 + g.abs())
    e_h = r * h.abs() + u.abs() * e_a + a.abs() * e_u
    tol_y = r * y.abs() + e_h @ wd.abs().t() + (F + 6) * u23 * (h.abs() @ wd.abs().t() + bd.abs() + d["residual"].abs())
    dh = dy @ wd
    e_dh = (C + 4) * u23 * (dy.abs() @ wd.abs())
    e_s = e_g + 2e-6 * (1 + g.abs()) + (g.abs() <= e_g).double() * (act == "relu")
    dg, du = dh * u * slope, dh * a
    s_dg = (u * slope).abs() * e_dh + (dh * slope).abs() * e_u + (dh * u).abs() * e_s
    s_du = a.abs() * e_dh + dh.abs() * e_a
    e_dg, e_du = r * dg.abs() + s_dg, r * du.abs() + s_du
    dx = dg @ wg + du @ wu
    sums = lambda A, B: A.t() @ B
    many = (M + 6) * u23
    values = [y, dx, sums(dg, x), dg.sum(0), sums(du, x), du.sum(0), sums(dy, h), dy.sum(0)]
    tols = [tol_y, r * dx.abs() + e_dg @ wg.abs() + e_du @ wu.abs() + (2 * F + 6) * u23 * (dg.abs() @ wg.abs() + du.abs() @ wu.abs())]
    tols += [r * values[2].abs() + sums(e_dg, x.abs()) + many * sums(dg.abs(), x.abs()), s_dg.sum(0) + many * dg.abs().sum(0)]
    tols += [r * values[4].abs() + sums(e_du, x.abs()) + many * sums(du.abs(), x.abs()), s_du.sum(0) + many * du.abs().sum(0)]
    tols += [r * values[6].abs() + sums(dy.abs(), e_h) + many * sums(dy.abs(), h.abs()), many * dy.abs().sum(0)]
    return values, tols


def check(got, want, tol, what):
    got = got.detach().double().cpu().reshape(want.shape)
    assert torch.isfinite(got).all(), f"{what}: not finite"
    over = ((got - want).abs() / tol.clamp_min(1e-30)).max()
    assert over <= 1, f"{what}: {float(over):.3f} of the tolerance"


SIZES = [(1, 1, 1), (1, 8, 8), (3, 7, 5), (2, 33, 65), (31, 64, 128), (33, 32, 96), (64, 96, 130), (127, 128, 512), (129, 200, 533),
         (300, 256, 1024), (257, 257, 100), (65, 512, 1365), (1000, 64, 170), (5, 1024, 40), (700, 24, 2050),
         (2500, 200, 533), (4000, 96, 260), (3001, 257, 130), (9000, 40, 72)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,C,F", SIZES)
def test_values_and_gradients(rows, C, F, dtype):
    announce("gated", rows, C, F, dtype)
    st = make(rows, C, F, dtype, bias=C % 2 == 0, seed=rows + C)
    values, tols = derived(st, "silu", dtype)
    gpu = on_gpu(st)
    params = [gpu[n] for n in NAMES]
    check(PF.gated_mlp_forward(gpu["x"], *params, residual=gpu["residual"]), values[0], tols[0], "y")
    got = PF.gated_mlp_backward(gpu["x"], gpu["dy"], *params[:5])
    for what, g, v, t in zip(("dx",) + NAMES, got, values[1:], tols[1:]):
        check(g, v, t, what)


@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("rows,C,F", [(39_400, 32, 33), (65_539, 64, 96), (66_000, 96, 200), (40_001, 128, 64), (32_700, 200, 70),
                                      (33_000, 256, 130)])
def test_many_rows(rows, C, F, act):
    """Enough rows for the kernel that keeps the hidden layer on chip, with and without rows left over for the tile kernels."""
    announce("gated many rows", rows, C, F, act)
    st = make(rows, C, F, torch.bfloat16, bias=F % 2 == 0, seed=C)
    values, tols = derived(st, act, torch.bfloat16)
    gpu = on_gpu(st)
    params = [gpu[n] for n in NAMES]
    check(PF.gated_mlp_forward(gpu["x"], *params, act=act, residual=gpu["residual"]), values[0], tols[0], "y")
    y = PF.gated_mlp_forward(gpu["x"], *params, act=act)
    bare = values[0] - st["residual"].double()  # rounded relative to itself, not to its sum with the residual
    check(y, bare, tols[0] + torch.finfo(torch.bfloat16).eps / 2 * bare.abs(), "y without a residual")
    for what, g, v, t in zip(("dx",) + NAMES, PF.gated_mlp_backward(gpu["x"], gpu["dy"], *params[:5], act=act), values[1:], tols[1:]):
        check(g, v, t, what)
    x = gpu["x"].clone()
    x[17, 3], x[rows - 1, 0] = float("nan"), float("inf")
    hit = PF.gated_mlp_forward(x, *params, act=act)
    clean = torch.ones(rows, dtype=torch.bool, device="cuda")
    clean[17] = clean[rows - 1] = False
    assert torch.equal(hit[clean], y[clean]) and torch.isnan(hit[17]).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("act", list(ACTS))
def test_activations(act, dtype):
    announce("gated act", act, dtype)
    st = make(200, 64, 192, dtype, seed=3)
    st["w_gate"] = st["w_gate"] * 8  # tails of the activations
    values, tols = derived(st, act, dtype)
    gpu = on_gpu(st)
    params = [gpu[n] for n in NAMES]
    check(PF.gated_mlp_forward(gpu["x"], *params, act=act, residual=gpu["residual"]), values[0], tols[0], "y")
    for what, g, v, t in zip(("dx",) + NAMES, PF.gated_mlp_backward(gpu["x"], gpu["dy"], *params[:5], act=act), values[1:], tols[1:]):
        check(g, v, t, what)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_autograd_of_strided_inputs_and_float32_parameters(dtype):
    """Batched rows, a transposed input, a sliced weight, a residual, parameters in float32."""
    announce("gated autograd", dtype)
    st = make(0, 72, 136, dtype, shape=(3, 41))
    values, tols = derived(st, "gelu", dtype)
    gpu = on_gpu(st)
    x = gpu["x"].transpose(0, 1).contiguous().transpose(0, 1).requires_grad_(True)
    res = gpu["residual"].requires_grad_(True)
    wide = torch.zeros(136, 80, device="cuda")
    wide[:, 5:77] = gpu["w_gate"].float()
    leaves = [wide.requires_grad_(True)] + [gpu[n].float().requires_grad_(True) for n in NAMES[1:]]
    y = PA.gated_mlp(x, leaves[0][:, 5:77], *leaves[1:], act="gelu", residual=res)
    check(y, values[0], tols[0], "y")
    grads = torch.autograd.grad(y, [x, res, *leaves], gpu["dy"])
    assert torch.equal(grads[1], gpu["dy"])
    assert not grads[2][:, :5].any() and not grads[2][:, 77:].any()
    got = [grads[0], grads[2][:, 5:77], *grads[3:]]
    for what, g, v, t in zip(("dx",) + NAMES, got, values[1:], tols[1:]):
        check(g, v, t, what)


def test_gradient_against_differences():
    """float32 gradients against central differences of the float64 formula along random directions."""
    announce("gated differences")
    st = make(40, 24, 56, torch.float32, seed=9)
    gpu = on_gpu(st)
    dx, *grads = PF.gated_mlp_backward(gpu["x"], gpu["dy"], *[gpu[n] for n in NAMES[:5]], act="silu")
    d = {k: v.double() for k, v in st.items()}

    def loss(d):
        h = torch.nn.functional.silu(d["x"] @ d["w_gate"].t() + d["b_gate"]) * (d["x"] @ d["w_up"].t() + d["b_up"])
        return float(((h @ d["w_down"].t() + d["b_down"]) * d["dy"]).sum())

    gen, eps = torch.Generator().manual_seed(1), 1e-5
    for name, grad in zip(("x",) + NAMES, [dx] + grads):
        v = torch.randn(d[name].shape, generator=gen, dtype=torch.float64)
        slope = (loss({**d, name: d[name] + eps * v}) - loss({**d, name: d[name] - eps * v})) / (2 * eps)
        got = float((grad.double().cpu() * v).sum())
        # the difference is good to eps^2 of a third derivative, about 1e-8 here; the float32 gradient to 1e-5 of its terms
        bound = 1e-5 * float((grad.double().cpu() * v).abs().sum()) + 1e-6
        assert abs(got - slope) <= bound, (name, got, slope)


def test_views_off_a_boundary_and_a_larger_buffer():
    """Inputs and outputs that start off a 16-byte boundary; what lies around them is neither read into results nor written."""
    announce("gated views")
    dtype = torch.bfloat16
    st = make(50, 64, 96, dtype)
    values, tols = derived(st, "silu", dtype)
    gpu = on_gpu(st)
    odd = lambda t: torch.cat([torch.full((3,), float("nan"), dtype=t.dtype, device="cuda"), t.reshape(-1),
                               torch.full((5,), float("nan"), dtype=t.dtype, device="cuda")])[3:-5].view(t.shape)
    params = [odd(gpu[n]) for n in NAMES]
    check(PF.gated_mlp_forward(odd(gpu["x"]), *params, residual=odd(gpu["residual"])), values[0], tols[0], "y")
    got = PF.gated_mlp_backward(odd(gpu["x"]), odd(gpu["dy"]), *params[:5])
    for what, g, v, t in zip(("dx",) + NAMES, got, values[1:], tols[1:]):
        check(g, v, t, what)


@pytest.mark.parametrize("where", [0, 63])
def test_infinities_and_nan_stay_in_their_rows(where):
    announce("gated nan", where)
    st = make(70, 64, 80, torch.bfloat16)
    gpu = on_gpu(st)
    params = [gpu[n] for n in NAMES]
    clean = PF.gated_mlp_forward(gpu["x"], *params)
    x = gpu["x"].clone()
    x[11, where], x[69, where] = float("nan"), float("inf")
    y = PF.gated_mlp_forward(x, *params)
    hit = torch.zeros(70, dtype=torch.bool, device="cuda")
    hit[11] = hit[69] = True
    assert torch.equal(y[~hit], clean[~hit]) and not torch.isfinite(y[hit]).any()


@pytest.mark.parametrize("rows,C,F", [(33, 24, 40), (40_001, 128, 64)])
def test_bias_gradients_with_an_infinite_last_row(rows, C, F):
    """Rows are worked off in blocks; what fills the last one takes no part: inf x 0 of it would be NaN."""
    announce("gated, infinite last row", rows, C, F)
    st = make(rows, C, F, torch.bfloat16, seed=21)
    st["x"][-1, 0] = float("inf")
    st["w_gate"][:, 0] = st["w_gate"][:, 0].abs() + 0.25
    st["w_up"][:, 0] = st["w_up"][:, 0].abs() + 0.25
    gpu = on_gpu(st)
    grads = PF.gated_mlp_backward(gpu["x"], gpu["dy"], *[gpu[n] for n in NAMES[:5]], act=None, wanted=(False, False, True, False, True, False, False))
    sign = torch.sign(st["dy"][-1].double() @ st["w_down"].double())  # of d h in the last row, whose g and u are + infinity
    assert bool((sign != 0).all())
    for got in (grads[2], grads[4]):
        assert torch.equal(got.double().cpu(), sign * float("inf"))


def test_no_rows_and_wanted_gradients():
    announce("gated empty")
    st = on_gpu(make(6, 16, 24, torch.float32))
    params = [st[n] for n in NAMES]
    assert PF.gated_mlp_forward(st["x"][:0], *params).shape == (0, 16)
    for g in PF.gated_mlp_backward(st["x"][:0], st["dy"][:0], *params[:5])[1:]:
        assert not g.any()
    every = PF.gated_mlp_backward(st["x"], st["dy"], *params[:5])
    for k in range(7):
        some = PF.gated_mlp_backward(st["x"], st["dy"], *params[:5], wanted=[j == k for j in range(7)])
        assert torch.equal(some[k], every[k]) and all(s is None for j, s in enumerate(some) if j != k)


def test_repeats_exactly_on_two_streams_and_in_a_graph():
    announce("gated streams and graph")
    st = on_gpu(make(5000, 128, 344, torch.bfloat16))
    params = [st[n] for n in NAMES]
    run = lambda x: [PF.gated_mlp_forward(x, *params, residual=st["residual"]), *PF.gated_mlp_backward(x, st["dy"], *params[:5])]
    other = st["x"].flip(0).contiguous()
    want, want_other = run(st["x"]), run(other)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    outs = []
    for s, x in zip(streams, (st["x"], other)):
        with torch.cuda.stream(s):
            outs.append(run(x))
    torch.cuda.synchronize()
    for got, ref in zip(outs, (want, want_other)):
        assert all(torch.equal(a, b) for a, b in zip(got, ref))
    x = st["x"].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run(x)
    for source, ref in ((other, want_other), (st["x"], want), (other, want_other)):
        x.copy_(source)
        graph.replay()
        torch.cuda.synchronize()
        run(source)  # eager work between the replays
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, ref))
