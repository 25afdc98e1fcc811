"""What the gated block, counter-based dropout and the 8-bit Linears refuse, without a GPU: argument checks of the C ABI (no
kernel is launched) and of the tensor-level functions; the generator's published test vectors."""
import ctypes

import numpy as np
import pytest
import torch

import physicsnemo_amd as pn
from oracle import numpy_oracle as no
from physicsnemo_amd import _lib
from physicsnemo_amd import functional as PF

P = ctypes.c_void_p(1 << 20)  # never read: every call below ends in its checks
BIG = 1 << 50


def test_philox_known_answers():
    """Known answers published with the generator (ten rounds)."""
    hexes = lambda words: [f"{int(w):08x}" for w in words]
    assert hexes(no.philox4x32((0, 0, 0, 0), (0, 0))) == ["6627e8d5", "e169c58d", "bc57ac4c", "9b00dbd8"]
    ones = 0xFFFFFFFF
    assert hexes(no.philox4x32((ones,) * 4, (ones,) * 2)) == ["408f276d", "41c83b0e", "a20bc7c6", "6d5451fd"]


@pytest.mark.parametrize("rows,C,F,dtype,code", [
    (0, 8, 8, 1, -2), (-1, 8, 8, 1, -2), (8, 0, 8, 1, -2), (8, 8, 0, 0, -2), (8, 8, 8, 2, -3), (8, 8, 8, -1, -3),
    (1 << 41, 8, 8, 1, -3), (8, (1 << 18) + 1, 8, 1, -3), (8, 8, (1 << 18) + 1, 1, -3), (8, 2 ** 62, 2 ** 62, 1, -3)])
def test_sizes_of_the_gated_block(rows, C, F, dtype, code):
    lib = _lib.load()
    p, g = _lib.PaGatedParams(P, None, P, None, P, None), _lib.PaGatedGrads()
    assert lib.pa_gated_mlp_workspace_bytes(dtype, rows, C, F) == code
    assert lib.pa_gated_mlp_backward_workspace_bytes(dtype, rows, C, F) == code
    assert lib.pa_gated_mlp_forward(dtype, rows, C, F, ctypes.byref(p), 1, P, None, P, P, BIG, None) == code
    assert lib.pa_gated_mlp_backward(dtype, rows, C, F, ctypes.byref(p), 1, P, P, P, ctypes.byref(g), P, BIG, None) == code


def test_arguments_of_the_gated_block():
    lib = _lib.load()
    p, g = _lib.PaGatedParams(P, None, P, None, P, None), _lib.PaGatedGrads()
    ref = ctypes.byref(p)
    need = lib.pa_gated_mlp_workspace_bytes(1, 100, 64, 96)
    assert need > 0
    forward = lambda p=ref, act=3, x=P, y=P, ws=P, n=need: lib.pa_gated_mlp_forward(1, 100, 64, 96, p, act, x, None, y, ws, n, None)
    assert forward(p=None) == forward(x=None) == forward(y=None) == forward(ws=None) == -1
    assert forward(act=-1) == forward(act=6) == -3
    assert forward(ws=ctypes.c_void_p(8)) == -4 and forward(n=need - 1) == -5
    for missing in ("w_gate", "w_up", "w_down"):
        q = _lib.PaGatedParams(P, None, P, None, P, None)
        setattr(q, missing, None)
        assert forward(p=ctypes.byref(q)) == -1
    need = lib.pa_gated_mlp_backward_workspace_bytes(1, 100, 64, 96)
    back = lambda p=ref, dy=P, g=ctypes.byref(g), ws=P, n=need: lib.pa_gated_mlp_backward(1, 100, 64, 96, p, 3, P, dy, P, g, ws, n, None)
    assert back(p=None) == back(dy=None) == back(g=None) == back(ws=None) == -1
    assert back(ws=ctypes.c_void_p(8)) == -4 and back(n=need - 1) == -5


def test_arguments_of_dropout():
    lib = _lib.load()
    nan = float("nan")
    call = lambda dtype=1, rows=8, C=8, x=P, p=0.5, rng=P, y=P, gamma=None, beta=None, n=None: lib.pa_dropout_add_norm(
        dtype, rows, C, x, None, p, rng, y, gamma, beta, 1e-5, n, None, None)
    assert call(rows=0) == call(C=0) == call(rows=-1) == -2
    assert call(p=-0.01) == call(p=1.01) == call(p=nan) == -2
    assert call(dtype=2) == call(rows=1 << 41) == call(C=(1 << 23) + 1) == -3
    assert call(x=None) == call(rng=None) == call(y=None) == call(n=P) == call(n=P, gamma=P) == call(n=P, beta=P) == -1
    need = lib.pa_dropout_add_norm_backward_workspace_bytes(1, 1000, 64)
    assert need > 0 and lib.pa_dropout_add_norm_backward_workspace_bytes(1, 0, 64) == -2
    back = lambda dy=P, dn=P, x=P, stats=P, gamma=P, p=0.5, rng=P, grads=P, ws=P, n=need: lib.pa_dropout_add_norm_backward(
        1, 1000, 64, dy, dn, x, None, stats, gamma, p, rng, P, P, grads, ws, n, None)
    assert back(dy=None, dn=None) == back(rng=None) == back(x=None) == back(stats=None) == back(gamma=None) == back(ws=None) == -1
    assert back(p=2.0) == -2 and back(ws=ctypes.c_void_p(4)) == -4 and back(n=need - 1) == -5
    assert lib.pa_dropout_advance(None, P, None) == lib.pa_dropout_advance(P, None, None) == -1


def test_arguments_of_the_8_bit_linears():
    lib = _lib.load()
    quantize = lambda dtype=1, rows=4, K=32, x=P, q=P, ld=32, s=P: lib.pa_int8_quantize_rows(dtype, rows, K, x, q, ld, s, None)
    assert quantize(rows=0) == quantize(K=0) == quantize(ld=31) == quantize(ld=36) == -2
    assert quantize(dtype=3) == quantize(K=131073) == quantize(ld=1 << 40) == -3
    assert quantize(x=None) == quantize(q=None) == quantize(s=None) == -1 and quantize(q=ctypes.c_void_p(4)) == -4
    need = lib.pa_int8_linear_workspace_bytes(1, 4, 32, 16)
    linear = lambda K=32, N=16, w=P, s=P, act=0, x=P, y=P, ws=P, n=need: lib.pa_int8_linear(1, 4, K, N, w, s, None, act, x, None, y, ws, n, None)
    assert need > 0 and linear(K=0) == linear(N=0) == -2 and linear(K=131073) == linear(N=(1 << 18) + 1) == linear(act=9) == -3
    assert linear(w=None) == linear(s=None) == linear(x=None) == linear(y=None) == linear(ws=None) == -1
    assert linear(ws=ctypes.c_void_p(8)) == -4 and linear(n=need - 1) == -5
    p = _lib.PaInt8GatedParams(P, P, None, P, P, None, P, P, None)
    need = lib.pa_int8_gated_workspace_bytes(1, 4, 32, 48)
    gated = lambda C=32, F=48, p=ctypes.byref(p), act=3, x=P, ws=P, n=need: lib.pa_int8_gated(1, 4, C, F, p, act, x, None, P, ws, n, None)
    assert need > 0 and gated(C=0) == gated(F=0) == -2 and gated(C=131073) == gated(F=131073) == gated(act=7) == -3
    assert gated(p=None) == gated(x=None) == gated(ws=None) == -1 and gated(ws=ctypes.c_void_p(8)) == -4 and gated(n=need - 1) == -5
    for name, _ in _lib.PaInt8GatedParams._fields_:
        q = _lib.PaInt8GatedParams(P, P, None, P, P, None, P, P, None)
        setattr(q, name, None)
        if not name.startswith("b_"):
            assert gated(p=ctypes.byref(q)) == -1, name


def test_tensors_on_the_cpu_are_refused():
    x, w, v = torch.zeros(4, 8), torch.zeros(8, 8), torch.zeros(8)
    state, codes = torch.zeros(2, dtype=torch.int64), torch.zeros(8, 8, dtype=torch.int8)
    for call in (lambda: PF.gated_mlp_forward(x, w, v, w, v, w, v), lambda: PF.gated_mlp_backward(x, x, w, v, w, v, w),
                 lambda: PF.dropout_add_norm(x, x, 0.1, state), lambda: PF.dropout_add_norm_backward(x, None, None, None, None, None, 0.1, state),
                 lambda: PF.dropout_advance(state), lambda: PF.quantize_int8(x), lambda: PF.linear_int8(x, codes, v),
                 lambda: PF.gated_mlp_int8(x, codes, v, v, codes, v, v, codes, v, v)):
        with pytest.raises(RuntimeError, match="GPU tensors only"):
            call()


def test_unknown_activations_are_refused():
    for name in ("swish", "GELU", 3, ["silu"]):
        with pytest.raises(ValueError, match="not found"):
            PF._act_code(name)
    assert [PF._act_code(a) for a in (None, "gelu", "relu", "silu", "sigmoid", "tanh")] == list(range(6))


def test_mask_is_a_function_of_the_place():
    """Neither the number of rows nor the width changes an element's bit; seeds, offsets and rows do."""
    full = no.dropout_keep(3, 4, np.arange(64), 64, 0.5)
    assert np.array_equal(no.dropout_keep(3, 4, np.arange(10), 33, 0.5), full[:10, :33])
    for other in (no.dropout_keep(4, 4, np.arange(64), 64, 0.5), no.dropout_keep(3, 5, np.arange(64), 64, 0.5),
                  no.dropout_keep(3, 4, np.arange(64) + 2 ** 32, 64, 0.5)):
        assert 0.4 < (other == full).mean() < 0.6


def test_gated_module_on_the_cpu_is_the_formula():
    for act, f in (("silu", torch.nn.functional.silu), ("gelu", torch.nn.functional.gelu), ("relu", torch.relu),
                   ("sigmoid", torch.sigmoid), ("tanh", torch.tanh), (None, lambda t: t)):
        mlp = pn.GatedMlp(6, 10, act, bias=act != "relu")
        x, r = torch.randn(3, 6), torch.randn(3, 6)
        lin = torch.nn.functional.linear
        h = f(lin(x, mlp.gate.weight, mlp.gate.bias)) * lin(x, mlp.up.weight, mlp.up.bias)
        assert torch.equal(mlp(x, r), lin(h, mlp.down.weight, mlp.down.bias) + r)
    with pytest.raises(KeyError, match="not found"):
        pn.GatedMlp(6, 10, "swish")


@pytest.mark.parametrize("cls", [pn.Transolver, pn.FLAREModel])
def test_models_of_gated_blocks(cls, tmp_path):
    make = lambda act: cls(functional_dim=3, out_dim=2, embedding_dim=2, n_layers=2, n_hidden=32, dropout=0.1, n_head=4, act=act, use_te=False)
    for act, gate, module in (("swiglu", "silu", torch.nn.SiLU), ("geglu", "gelu", torch.nn.GELU), ("reglu", "relu", torch.nn.ReLU),
                              ("GLU", "sigmoid", torch.nn.Sigmoid)):
        model = make(act)
        assert all(type(b.ln_mlp1[1]) is pn.GatedMlp and b.ln_mlp1[1].act == gate for b in model.blocks)
        assert type(model.preprocess.layers[1]) is module
    model.save(str(tmp_path / "gated.mdlus"))
    again = cls.from_checkpoint(str(tmp_path / "gated.mdlus"))
    assert all(torch.equal(a, b) for a, b in zip(model.state_dict().values(), again.state_dict().values()))
    assert type(make("gelu").blocks[0].ln_mlp1[1]) is pn.Mlp
    with pytest.raises(KeyError, match="not found"):
        make("swish")
    keys = list(model.state_dict())
    assert list(model.use_counter_dropout(5).state_dict()) == keys
    assert [b.Attn.out_dropout.state.tolist() for b in model.blocks] == [[5, 0], [5 + (1 << 32), 0]]
    assert model.use_counter_dropout(2 ** 63 - 1).blocks[1].Attn.out_dropout.state.tolist() == [-(2 ** 63) + 2 ** 32 - 1, 0]
    assert [b.Attn.out_dropout.p for b in model.blocks] == [0.1, 0.1]


def test_blocks_refuse_what_does_not_go_together():
    plain, gated = (pn.TransolverBlock(4, 32, 0.1, act=act, use_te=False) for act in ("gelu", "swiglu"))
    with pytest.raises(ValueError, match="fp8 weights"):
        gated.use_fp8_weights()
    with pytest.raises(ValueError, match="fp8 weights"):
        plain.use_int8_mlp().use_fp8_weights()
    plain.use_int8_mlp(False).use_fp8_weights()
    with pytest.raises(ValueError, match="fp8 weights"):
        plain.use_int8_mlp()
    plain.use_fp8_weights(False)
    plain.ln_mlp1[1].layers[0].register_forward_hook(lambda *a: None)
    with pytest.raises(ValueError, match="without hooks"):
        plain.use_int8_mlp()
    gated.ln_mlp1[1].up = torch.nn.Identity()
    with pytest.raises(ValueError, match="without hooks"):
        gated.use_int8_mlp()


def test_counter_dropout_off_the_gpu():
    drop = pn.CounterDropout(0.5)
    with pytest.raises(RuntimeError, match="GPU tensors only"):
        drop(torch.zeros(4))
    x = torch.zeros(4)
    assert drop.eval()(x) is x and pn.CounterDropout(0.0)(x) is x
    with pytest.raises(ValueError):
        pn.CounterDropout(1.5)
