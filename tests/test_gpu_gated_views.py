"""Gated blocks over many rows that start off a 16-byte boundary: they run in pieces, each on the tile kernels.  Tolerances are those
of test_gpu_gated.py."""
import ctypes

import pytest
import torch

from gpu_util import announce
from physicsnemo_amd import _lib
from physicsnemo_amd import functional as PF
from test_gpu_gated import NAMES, check, derived, make, on_gpu

pytestmark = pytest.mark.gpu


def shifted(t):
    """The same values one element behind a boundary, NaN around them."""
    fill = torch.full((1,), float("nan"), dtype=t.dtype, device=t.device)
    return torch.cat([fill, t.reshape(-1), fill])[1:-1].view(t.shape)


def call(x, params, residual, y):
    """The C entry, which writes where it is told."""
    lib, (rows, C), F = _lib.load(), x.shape, params[0].shape[0]
    code = _lib.dtype_code(x.dtype)
    nbytes = lib.pa_gated_mlp_workspace_bytes(code, rows, C, F)
    guard = 4096
    ws = torch.full((nbytes + guard,), 77, dtype=torch.uint8, device=x.device)
    p = _lib.PaGatedParams(*map(_lib.ptr, params))
    _lib.check(lib.pa_gated_mlp_forward(code, rows, C, F, ctypes.byref(p), _lib.ACTS["silu"], x.data_ptr(), _lib.ptr(residual), y.data_ptr(),
                                        ws.data_ptr(), nbytes, _lib.current_stream_ptr(x.device)), "pa_gated_mlp_forward")
    torch.cuda.synchronize()
    assert bool((ws[nbytes:] == 77).all())


@pytest.mark.parametrize("rows,C,F,dtype", [(70_001, 64, 96, torch.bfloat16), (32_768, 72, 40, torch.bfloat16), (65_537, 32, 33, torch.bfloat16),
                                            (33_000, 264, 72, torch.bfloat16), (40_000, 36, 50, torch.float32), (500, 256, 64, torch.bfloat16),
                                            (140_000, 64, 16, torch.bfloat16)])
def test_rows_off_a_boundary(rows, C, F, dtype):
    announce("gated views", rows, C, F, dtype)
    st = make(rows, C, F, dtype, seed=rows)
    values, tols = derived(st, "silu", dtype)
    gpu = on_gpu(st)
    params = [gpu[n] for n in NAMES]
    x, residual = gpu["x"], gpu["residual"]
    check(PF.gated_mlp_forward(shifted(x), *params, residual=shifted(residual)), values[0], tols[0], "x, residual")
    check(PF.gated_mlp_forward(x, *params, residual=shifted(residual)), values[0], tols[0], "residual")
    for what, source, add in (("y", x, residual), ("x, y", shifted(x), residual)):
        out = shifted(torch.zeros_like(x))
        call(source, params, add, out)
        check(out, values[0], tols[0], what)
    both = shifted(residual)  # y over the residual
    call(x, params, both, both)
    check(both, values[0], tols[0], "y over the residual")
    out = torch.zeros_like(x)
    call(x, params, residual, out)
    check(out, values[0], tols[0], "on boundaries")


@pytest.mark.parametrize("rows,C,F,dtype", [(70_001, 64, 96, torch.bfloat16), (65_537, 32, 33, torch.bfloat16), (33_000, 264, 72, torch.bfloat16),
                                            (40_000, 36, 50, torch.float32), (500, 256, 64, torch.bfloat16), (140_000, 64, 16, torch.bfloat16),
                                            (90_000, 256, 256, torch.bfloat16)])
def test_gradients_of_rows_off_a_boundary(rows, C, F, dtype):
    """x, dy or both; the result's place as well; every gradient, and the biases' alone."""
    announce("gated views, gradients", rows, C, F, dtype)
    st = make(rows, C, F, dtype, seed=rows)
    values, tols = derived(st, "silu", dtype)
    gpu = on_gpu(st)
    params = [gpu[n] for n in NAMES]
    for xs, ys in ((shifted(gpu["x"]), gpu["dy"]), (gpu["x"], shifted(gpu["dy"])), (shifted(gpu["x"]), shifted(gpu["dy"]))):
        got = PF.gated_mlp_backward(xs, ys, *params[:5])
        for what, g, v, t in zip(("dx",) + NAMES, got, values[1:], tols[1:]):
            check(g, v, t, what)
    some = PF.gated_mlp_backward(xs, ys, *params[:5], wanted=(False, False, True, False, True, False, True))
    assert all(torch.equal(some[k], got[k]) for k in (2, 4, 6)) and [g is None for g in some] == [True, True, False, True, False, True, False]
    lib, code, guard = _lib.load(), _lib.dtype_code(dtype), 4096
    nbytes = lib.pa_gated_mlp_backward_workspace_bytes(code, rows, C, F)
    ws = torch.full((nbytes + guard,), 77, dtype=torch.uint8, device="cuda")
    dx = shifted(torch.zeros_like(gpu["x"]))
    p, grads = _lib.PaGatedParams(*map(_lib.ptr, params)), _lib.PaGatedGrads()
    _lib.check(lib.pa_gated_mlp_backward(code, rows, C, F, ctypes.byref(p), _lib.ACTS["silu"], xs.data_ptr(), ys.data_ptr(), dx.data_ptr(),
                                         ctypes.byref(grads), ws.data_ptr(), nbytes, _lib.current_stream_ptr(dx.device)), "pa_gated_mlp_backward")
    check(dx, values[1], tols[1], "dx alone, off a boundary")
    torch.cuda.synchronize()
    assert bool((ws[nbytes:] == 77).all())


def test_an_on_chip_call_takes_little_memory():
    announce("gated memory")
    rows, C, F = 1 << 18, 256, 1024
    st = {k: torch.randn(*s, device="cuda").bfloat16() for k, s in (("x", (rows, C)), ("g", (F, C)), ("u", (F, C)), ("d", (C, F)))}
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    y = PF.gated_mlp_forward(st["x"], st["g"], None, st["u"], None, st["d"], None)
    torch.cuda.synchronize()
    extra = torch.cuda.max_memory_allocated() - before - y.numel() * 2
    assert extra <= 32768 * (C + F + 16) * 2 + 2 * 2 * 3 * (C + 32) * (F + 64) + (1 << 20)
