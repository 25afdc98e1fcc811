"""8-bit integer Linears on the GPU: codes and scales bit for bit, products against 64 bits.

A product of codes is exact, so y is off by its rounding r = eps / 2 of the type, a few float32 roundings (8 2^-23 of the
scaled sum and the bias) and the activation's 1e-6 (1 + |v|)."""
import pytest
import torch

from gpu_util import announce
from physicsnemo_amd import functional as PF

pytestmark = pytest.mark.gpu

ACTS = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu, "relu": torch.relu, "sigmoid": torch.sigmoid,
        "tanh": torch.tanh, None: lambda v: v}


def codes(x):
    """The definition in float32, row by row.  127 as a tensor: torch forms the quotient of a number and a tensor from a
    reciprocal, which is one rounding more than a quotient has."""
    most = x.float().abs().amax(-1, keepdim=True)
    top = torch.full_like(most, 127)
    inv = torch.where(most > 0, top / most, torch.zeros_like(most))
    return (x.float() * inv).round().to(torch.int8), (most / top).squeeze(-1)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", [(1, 1), (3, 5), (7, 16), (65, 100), (2, 9, 256), (33, 511), (10, 512), (5, 513), (4, 2048), (3, 2051),
                                   (2, 70000)])
def test_codes_and_scales(shape, dtype):
    announce("int8 codes", shape, dtype)
    x = (torch.randn(*shape) * 3).to(dtype)
    x.view(-1, shape[-1])[0] = 0
    q, s = PF.quantize_int8(x.cuda())
    want_q, want_s = codes(x)
    assert q.shape == x.shape and s.shape == x.shape[:-1]
    assert torch.equal(q.cpu(), want_q) and torch.equal(s.cpu(), want_s)


def test_halves_go_to_even_and_extremes():
    announce("int8 halves")
    x = torch.tensor([[127.0, 0.5, 1.5, 2.5, -0.5, -1.5, -127.0, 126.5], [1e-40, -1e-40, 0, 0, 0, 5e-41, 0, 0],
                      [3e38, -3e38, 1.0, 0, 0, 0, 0, 1e38], [-0.0, 0, 0, 0, 0, 0, 0, 0]], device="cuda")
    q, s = PF.quantize_int8(x)
    assert q[0].tolist() == [127, 0, 2, 2, 0, -2, -127, 126]
    assert q[1, 0] == 127 and q[1, 1] == -127 and 63 <= q[1, 5] <= 64 and not q[1, 2:5].any()
    assert q[2].tolist() == [127, -127, 0, 0, 0, 0, 0, 42] and not q[3].any()
    assert s[0] == 1 and s[3] == 0 and 0 < s[1] < 1e-41 and torch.isfinite(s).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_rows_that_are_not_finite(bad):
    announce("int8 not finite", bad)
    x = torch.randn(9, 40, device="cuda")
    w, sw = PF.quantize_int8(torch.randn(24, 40, device="cuda"))
    clean = PF.linear_int8(x, w, sw)
    x[4, 39] = bad
    q, s = PF.quantize_int8(x)
    assert torch.isnan(s[4]) and not q[4].any() and torch.isfinite(s[:4]).all() and torch.isfinite(s[5:]).all()
    y = PF.linear_int8(x, w, sw)
    assert torch.isnan(y[4]).all() and torch.equal(y[:4], clean[:4]) and torch.equal(y[5:], clean[5:])


def linear64(x, w, sw, b, act, res):
    q, s = codes(x)
    acc = q.double() @ w.double().t()
    scaled = acc * (s.double()[..., None] * sw.double())
    v = scaled + (0 if b is None else b.double())
    y = ACTS[act](v) + (0 if res is None else res.double())
    err = 8 * 2.0 ** -23 * (scaled.abs() + (0 if b is None else b.double().abs())) * 1.13 + (1e-6 * (1 + v.abs()) if act else 0)
    err = err + (0 if res is None else 2.0 ** -23 * (y.abs() + res.double().abs()))
    return y, torch.finfo(x.dtype).eps / 2 * y.abs() + err


def check(got, want, tol, what):
    got = got.double().cpu()
    assert torch.isfinite(got).all(), f"{what}: not finite"
    over = ((got - want).abs() / tol.clamp_min(1e-30)).max()
    assert over <= 1, f"{what}: {float(over):.3f} of the tolerance"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,K,N", [(1, 1, 1), (1, 16, 8), (2, 17, 3), (31, 64, 33), (33, 100, 130), (64, 256, 1024), (130, 512, 512),
                                      (257, 130, 96), (70, 2048, 64), (5, 33000, 20), (1000, 32, 250), (3001, 100, 700), (9000, 40, 33),
                                      (2500, 320, 257)])
def test_linear(rows, K, N, dtype):
    announce("linear_int8", rows, K, N, dtype)
    gen = torch.Generator().manual_seed(rows)
    x = torch.randn(rows, K, generator=gen).to(dtype)
    w, sw = codes(torch.randn(N, K, generator=gen))
    b, res = torch.randn(N, generator=gen), torch.randn(rows, N, generator=gen).to(dtype)
    dev = lambda t: t.cuda()
    for act, bias, r in ((None, None, None), ("gelu", b, None), ("silu", b, res)):
        y = PF.linear_int8(dev(x), dev(w), dev(sw), None if bias is None else dev(bias), act, None if r is None else dev(r))
        want, tol = linear64(x, w, sw, bias, act, r)
        check(y, want, tol, (act, bias is not None, r is not None))


@pytest.mark.parametrize("act", list(ACTS))
def test_activations(act):
    announce("int8 act", act)
    x, (w, sw) = torch.randn(100, 48), codes(torch.randn(72, 48))
    want, tol = linear64(x, w, sw, None, act, None)
    check(PF.linear_int8(x.cuda(), w.cuda(), sw.cuda(), act=act), want, tol, act)


def test_largest_sums_are_exact():
    """131 072 products of 127 by 127: 2 114 060 288, below 2^31; one term more is refused."""
    announce("int8 largest")
    x = torch.ones(2, 131072, device="cuda")
    w = torch.full((3, 131072), 127, dtype=torch.int8, device="cuda")
    w[1] = -127
    y = PF.linear_int8(x, w, torch.ones(3, device="cuda"))
    want = torch.tensor([1.0, -1.0, 1.0], dtype=torch.float64) * 127 * 131072
    assert ((y.double().cpu() - want).abs() <= 4 * 2.0 ** -23 * want.abs()).all()
    with pytest.raises(RuntimeError, match="pa_int8_linear_workspace_bytes"):
        PF.linear_int8(torch.ones(1, 131073, device="cuda"), torch.ones(1, 131073, dtype=torch.int8, device="cuda"), torch.ones(1, device="cuda"))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,C,F", [(1, 1, 1), (3, 9, 5), (33, 32, 96), (100, 200, 533), (130, 256, 1024), (65, 512, 1365)])
def test_gated(rows, C, F, dtype):
    """Against the hidden layer without its rounding to 8 bits: half a step of its row's scale per hidden unit at most, and
    as independent errors of variance scale^2 / 12 on the whole (three times that allowed)."""
    announce("gated_mlp_int8", rows, C, F, dtype)
    gen = torch.Generator().manual_seed(C)
    x, res = torch.randn(rows, C, generator=gen).to(dtype), torch.randn(rows, C, generator=gen).to(dtype)
    ws = {n: codes(torch.randn(o, i, generator=gen) / i ** 0.5) for n, o, i in (("gate", F, C), ("up", F, C), ("down", C, F))}
    bs = {n: torch.randn(o, generator=gen) * 0.1 for n, o in (("gate", F), ("up", F), ("down", C))}
    args = [t.cuda() for n in ("gate", "up", "down") for t in (*ws[n], bs[n])]
    y = PF.gated_mlp_int8(x.cuda(), *args, act="silu", residual=res.cuda())
    g, e_g = linear64(x.float(), *ws["gate"], bs["gate"], None, None)
    u, e_u = linear64(x.float(), *ws["up"], bs["up"], None, None)
    a = ACTS["silu"](g)
    h = a * u
    r = torch.finfo(dtype).eps / 2
    e_h = r * h.abs() + u.abs() * (1.1 * e_g + 1e-6 * (1 + g.abs())) + a.abs() * e_u
    step = h.abs().amax(-1, keepdim=True) / 127
    wd = ws["down"][0].double() * ws["down"][1].double()[:, None]
    want = h @ wd.t() + bs["down"].double() + res.double()
    sums = (F + 8) * 2.0 ** -23 * (h.abs() @ wd.abs().t() + bs["down"].double().abs() + res.double().abs())
    tol = r * want.abs() + (e_h + 0.5 * (1 + 2 * r) * step) @ wd.abs().t() + sums
    check(y, want, tol, "y")
    if F >= 64:
        noise = (step.pow(2) / 12 * wd.pow(2).sum(1) + (r * h.abs()).pow(2) @ wd.pow(2).t() / 3 + (r * want).pow(2) / 3).sum().sqrt()
        assert (y.double().cpu() - want).norm() <= 3 * noise


def test_views_off_a_boundary_and_no_rows():
    announce("int8 views")
    x, (w, sw) = torch.randn(20, 64).bfloat16(), codes(torch.randn(32, 64))
    odd = lambda t: torch.cat([t.reshape(-1)[:3], t.reshape(-1)]).cuda()[3:].view(t.shape)
    want = PF.linear_int8(x.cuda(), w.cuda(), sw.cuda())
    assert torch.equal(PF.linear_int8(odd(x), odd(w), odd(sw)), want)
    assert PF.linear_int8(x[:0].cuda(), w.cuda(), sw.cuda()).shape == (0, 32)
    assert PF.quantize_int8(x[:0].cuda())[0].shape == (0, 64)


def test_repeats_exactly_in_a_graph():
    announce("int8 graph")
    x, other = torch.randn(3000, 128, device="cuda").bfloat16(), torch.randn(3000, 128, device="cuda").bfloat16()
    ws = [t for o, i in ((344, 128), (344, 128), (128, 344)) for t in (*PF.quantize_int8(torch.randn(o, i, device="cuda")), None)]
    run = lambda x: PF.gated_mlp_int8(x, *ws)
    want = [run(x), run(other)]
    held_in = x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run(held_in)
    for k in (1, 0, 1):
        held_in.copy_((x, other)[k])
        graph.replay()
        torch.cuda.synchronize()
        run(other)
        assert torch.equal(held, want[k])
