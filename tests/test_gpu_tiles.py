"""The tile kernels at every tile size, with rows on two launches and several tiles a workgroup, against the formulas in 64 bits.  The
library is told of eight CUs; test_product_launches.py says which tiles the sizes reach.  Tolerances are those of test_gpu_gated.py
and test_gpu_int8.py."""
import pytest
import torch

from gpu_util import announce
from physicsnemo_amd import _lib
from physicsnemo_amd import functional as PF
from test_gpu_gated import NAMES, check, derived, make, on_gpu
from test_gpu_int8 import ACTS, codes, linear64
from test_product_launches import GATED_SIZES, INT8_SIZES

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float32]


@pytest.fixture
def eight_cus():
    _lib.load().pa_set_compute_units(8)
    yield
    _lib.load().pa_set_compute_units(0)


def forward_and_backward(st, act, dtype, values, tols):
    gpu = on_gpu(st)
    params = [gpu[n] for n in NAMES]
    check(PF.gated_mlp_forward(gpu["x"], *params, act=act, residual=gpu["residual"]), values[0], tols[0], "y")
    for what, g, v, t in zip(("dx",) + NAMES, PF.gated_mlp_backward(gpu["x"], gpu["dy"], *params[:5], act=act), values[1:], tols[1:]):
        check(g, v, t, what)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,C,F", GATED_SIZES)
def test_gated_block(eight_cus, rows, C, F, dtype):
    act = ("silu", "gelu", "sigmoid")[rows % 3]
    announce("tiles, gated", rows, C, F, act, dtype)
    st = make(rows, C, F, dtype, bias=C % 3 != 0, seed=rows)
    forward_and_backward(st, act, dtype, *derived(st, act, dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,C,F", INT8_SIZES)
def test_int8_linear(eight_cus, rows, C, F, dtype):
    announce("tiles, linear_int8", rows, C, F, dtype)
    gen = torch.Generator().manual_seed(rows)
    for K, N, act in ((C, F, "gelu"), (F, C, "silu")):
        x, res = torch.randn(rows, K, generator=gen).to(dtype), torch.randn(rows, N, generator=gen).to(dtype)
        w, sw = codes(torch.randn(N, K, generator=gen))
        b = torch.randn(N, generator=gen)
        for bias, r in ((None, None), (b, res)):
            dev = lambda t: None if t is None else t.cuda()
            y = PF.linear_int8(dev(x), dev(w), dev(sw), dev(bias), act, dev(r))
            check(y, *linear64(x, w, sw, bias, act, r), (K, N, bias is not None))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,C,F", INT8_SIZES)
def test_int8_gated(eight_cus, rows, C, F, dtype):
    """As test_gpu_int8.py: half a step of the row's scale per hidden unit at most, and as independent errors on the whole."""
    announce("tiles, gated_mlp_int8", rows, C, F, dtype)
    gen = torch.Generator().manual_seed(rows + C)
    x, res = torch.randn(rows, C, generator=gen).to(dtype), torch.randn(rows, C, generator=gen).to(dtype)
    ws = {n: codes(torch.randn(o, i, generator=gen) / i ** 0.5) for n, o, i in (("gate", F, C), ("up", F, C), ("down", C, F))}
    bs = {n: torch.randn(o, generator=gen) * 0.1 for n, o in (("gate", F), ("up", F), ("down", C))}
    args = [t.cuda() for n in ("gate", "up", "down") for t in (*ws[n], bs[n])]
    y = PF.gated_mlp_int8(x.cuda(), *args, act="silu", residual=res.cuda())
    g, e_g = linear64(x.float(), *ws["gate"], bs["gate"], None, None)
    u, e_u = linear64(x.float(), *ws["up"], bs["up"], None, None)
    a = ACTS["silu"](g)
    h, r = a * u, torch.finfo(dtype).eps / 2
    e_h = u.abs() * (1.1 * e_g + 1e-6 * (1 + g.abs())) + a.abs() * e_u  # from float32 straight to codes
    step = h.abs().amax(-1, keepdim=True) / 127
    wd = ws["down"][0].double() * ws["down"][1].double()[:, None]
    want = h @ wd.t() + bs["down"].double() + res.double()
    sums = (F + 8) * 2.0 ** -23 * (h.abs() @ wd.abs().t() + bs["down"].double().abs() + res.double().abs())
    check(y, want, r * want.abs() + (e_h + 0.5 * (1 + 2 * r) * step) @ wd.abs().t() + sums, "y")
    # the codes are what 64 bits give but for those whose value lies within its error of a half, one step each: per output the
    # distance from the formula on those codes
    q = (h / step).round()
    near = ((h / step - q).abs() >= 0.5 - (e_h + 4 * 2.0 ** -24 * h.abs()) / step).double()
    assert near.mean() < 1e-3
    exact = (q * step) @ wd.t() + bs["down"].double() + res.double()
    e_s = 2.0 ** -22 * (h.abs() + step) + q.abs() * e_h.amax(-1, keepdim=True) / 127
    check(y, exact, r * exact.abs() + (near * step + e_s) @ wd.abs().t() + sums, "y of the codes")


@pytest.mark.parametrize("rows,C,F,dtype,act", [(100_003, 512, 1365, torch.bfloat16, "silu"), (28_900, 128, 512, torch.float32, "silu"),
                                                (140_000, 256, 1024, torch.bfloat16, "gelu")])
def test_large_gated_blocks(rows, C, F, dtype, act):
    """Whole calls on all CUs, the formulas in float64 on the GPU."""
    announce("tiles, large", rows, C, F, dtype, act)
    st = make(rows, C, F, dtype, bias=F % 2 == 0, seed=C)
    values, tols = derived(on_gpu(st), act, dtype)
    forward_and_backward(st, act, dtype, [v.cpu() for v in values], [t.cpu() for t in tols])


@pytest.mark.parametrize("rows,K,N", [(100_003, 512, 700), (131_072, 700, 512)])
def test_large_int8_linears(rows, K, N):
    announce("tiles, large int8", rows, K, N)
    gen = torch.Generator("cuda").manual_seed(K)
    draw = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    x, (w, sw), b, res = draw(rows, K).bfloat16(), codes(draw(N, K)), draw(N), draw(rows, N).bfloat16()
    want, tol = linear64(x, w, sw, b, "gelu", res)
    check(PF.linear_int8(x, w, sw, b, "gelu", res), want.cpu(), tol.cpu(), "y")


@pytest.mark.parametrize("rows,C,F", [(70, 64, 80), (1, 64, 80), (3000, 512, 700)])
def test_float32_rows_that_are_not_finite(eight_cus, rows, C, F):
    """They give rows that are not finite and change no other."""
    announce("tiles, float32 not finite", rows, C, F)
    gpu = on_gpu(make(rows, C, F, torch.float32, seed=5))
    params = [gpu[n] for n in NAMES]
    clean = PF.gated_mlp_forward(gpu["x"], *params, act="gelu")
    for k, bad in enumerate((float("nan"), float("inf"), -float("inf"))):
        x, row = gpu["x"].clone(), (rows - 1, 0, rows // 2)[k]
        x[row, (0, C - 1, C // 2)[k]] = bad
        y = PF.gated_mlp_forward(x, *params, act="gelu")
        others = torch.arange(rows, device="cuda") != row
        assert torch.equal(y[others], clean[others]) and not bool(torch.isfinite(y[row]).any())
