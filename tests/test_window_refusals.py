"""What window attention, the query-key norm with rotation and their layer refuse, without a GPU; buckets against their definition."""
import ctypes
from fractions import Fraction

import pytest
import torch

import physicsnemo_amd as pn
from physicsnemo_amd import _lib
from physicsnemo_amd import autograd as PA
from physicsnemo_amd import functional as PF

P = 1 << 20  # never read: every call below ends in its checks
BIG = 1 << 50


def heads(data=P, batch=64, row=64, head=8):
    return _lib.PaHeads(data, batch, row, head)


def window(**kw):
    base = dict(B=2, N=100, Hq=4, Hk=2, D=32, left=8, right=8, sinks=0, buckets=0, distance=0, scale=0.2, lengths=None, bias=None)
    base.update(kw)
    return _lib.PaWindowParams(*base.values())


WINDOWS = [(dict(B=0), -2), (dict(N=0), -2), (dict(Hq=0), -2), (dict(Hk=0), -2), (dict(D=0), -2), (dict(Hq=5), -2), (dict(left=-2), -2), (dict(right=-2), -2),
           (dict(sinks=-1), -2), (dict(scale=0.0), -2), (dict(scale=-1.0), -2), (dict(scale=float("nan")), -2), (dict(scale=float("inf")), -2),
           (dict(D=129), -3), (dict(sinks=129), -3), (dict(N=(1 << 29) + 1), -3), (dict(Hq=8192, Hk=8192), -3), (dict(B=1 << 25), -3),
           (dict(B=1 << 20, N=1 << 20), -3), (dict(B=1 << 21), -3), (dict(N=1 << 28, Hq=8, Hk=8, B=1), -3), (dict(buckets=-1), -2), (dict(buckets=2, distance=9, bias=P), -2), (dict(buckets=7, distance=9, bias=P), -2),
           (dict(buckets=32, distance=8, bias=P), -2), (dict(buckets=32, distance=16, right=0, bias=P), -2), (dict(buckets=258, distance=500, bias=P), -3),
           (dict(buckets=32, distance=2049, bias=P), -3), (dict(buckets=32, distance=64), -1)]


@pytest.mark.parametrize("change,code", WINDOWS)
def test_sizes_of_the_window(change, code):
    lib, h = _lib.load(), heads()
    p, ref = window(**change), ctypes.byref(h)
    assert lib.pa_window_attention(1, ctypes.byref(p), ref, ref, ref, P, None, None) == code
    assert lib.pa_window_attention_backward_workspace_bytes(1, ctypes.byref(p), 0) == code
    assert lib.pa_window_attention_backward(1, ctypes.byref(p), ref, ref, ref, P, P, ref, P, P, P, None, P, BIG, None) == code
    if change.get("right", 0) == 0 and "buckets" not in change:
        p = window(**{**change, "right": 0, "lengths": P})
        assert lib.pa_window_attention_step_workspace_bytes(1, ctypes.byref(p), 1) == code


def test_arguments_of_the_window():
    lib = _lib.load()
    h, p = heads(), window()
    ref = ctypes.byref(h)
    forward = lambda dtype=1, p=p, q=ref, k=ref, v=ref, y=P: lib.pa_window_attention(dtype, None if p is None else ctypes.byref(p), q, k, v, y, None, None)
    assert forward(p=None) == forward(q=None) == forward(k=None) == forward(v=None) == forward(y=None) == -1
    assert forward(dtype=2) == forward(dtype=-1) == -3
    for bad, code in ((heads(data=None), -1), (heads(batch=-1), -2), (heads(row=-1), -2), (heads(head=-1), -2), (heads(data=P + 1), -4)):
        assert forward(q=ctypes.byref(bad)) == forward(k=ctypes.byref(bad)) == forward(v=ctypes.byref(bad)) == code
    assert forward(dtype=0, q=ctypes.byref(heads(data=P + 2))) == -4
    need = lib.pa_window_attention_backward_workspace_bytes(1, ctypes.byref(p), 0)
    assert need > 0 and lib.pa_window_attention_backward_workspace_bytes(1, ctypes.byref(p), 1) == -2
    back = lambda y=P, stats=P, dy=ref, dq=P, dk=P, dv=P, ws=P, n=need: lib.pa_window_attention_backward(1, ctypes.byref(p), ref, ref, ref, y, stats, dy, dq, dk, dv,
                                                                                                        None, ws, n, None)
    assert back(y=None) == back(stats=None) == back(dy=None) == back(dq=None) == back(dk=None) == back(dv=None) == back(ws=None) == -1
    assert back(ws=P + 8) == -4 and back(n=need - 1) == -5
    p = window(right=0, N=4000, left=-1, lengths=P)
    need = lib.pa_window_attention_step_workspace_bytes(1, ctypes.byref(p), 1)
    step = lambda p=p, T=1, q=ref, y=P, ws=P, n=need: lib.pa_window_attention_step(1, ctypes.byref(p), T, q, ref, ref, y, ws, n, None)
    assert need > 0 and step(T=0) == step(T=4001) == step(p=window(right=1, lengths=P)) == -2
    assert step(p=window(right=0)) == step(q=None) == step(y=None) == step(ws=None) == -1 and step(ws=P + 4) == -4 and step(n=need - 1) == -5


def rotate(**kw):
    base = dict(B=2, N=10, Hq=4, Hk=2, D=32, rotated=32, axes=1, position_batch=0, position_type=1, interleaved=0, norm=1, eps=1e-6, positions=P, frequencies=P,
                q_weight=None, k_weight=None)
    base.update(kw)
    return _lib.PaRotateParams(*base.values())


def test_arguments_of_the_rotation():
    lib = _lib.load()
    h = heads()
    ref = ctypes.byref(h)
    forward = lambda dtype=1, q=ref, k=ref, a=P, b=P, **kw: lib.pa_norm_rotate(dtype, ctypes.byref(rotate(**kw)), q, k, a, b, None)
    for kw in (dict(B=0), dict(N=0), dict(Hq=0), dict(Hk=0), dict(D=0), dict(rotated=-2), dict(rotated=34), dict(rotated=31), dict(axes=0), dict(position_batch=5),
               dict(eps=-1.0), dict(eps=float("nan"))):
        assert forward(**kw) == -2, kw
        assert lib.pa_norm_rotate_backward_workspace_bytes(1, ctypes.byref(rotate(**kw))) == -2
    for kw in (dict(D=130), dict(Hq=5000), dict(axes=9), dict(position_type=3), dict(position_type=-1), dict(B=1 << 41), dict(N=1 << 41), dict(dtype=2)):
        assert forward(**kw) == -3, kw
    assert forward(positions=None) == forward(frequencies=None) == forward(q=None) == forward(k=None) == forward(a=None) == forward(b=None) == -1
    assert forward(q=ctypes.byref(heads(data=P + 1))) == -4 and forward(k=ctypes.byref(heads(row=-3))) == -2
    need = lib.pa_norm_rotate_backward_workspace_bytes(1, ctypes.byref(rotate()))
    back = lambda p=rotate(), dq=ref, w=P, ws=P, n=need: lib.pa_norm_rotate_backward(1, ctypes.byref(p), ref, ref, dq, ref, P, P, w, w, ws, n, None)
    assert back(dq=None) == back(ws=None) == -1 and back(ws=P + 8) == -4 and back(n=need - 1) == -5 and back(p=rotate(norm=0)) == -3


def test_tensors_that_do_not_go_together():
    x = torch.zeros(1, 4, 2, 8)
    for call in (lambda: PF.window_attention(x, x, x), lambda: PF.norm_rotate(x, x), lambda: PF.window_attention_step(x, x, x, torch.zeros(1, dtype=torch.int32)),
                 lambda: PA.window_attention(x, x, x), lambda: PA.norm_rotate(x, x)):
        with pytest.raises(RuntimeError, match="GPU tensors only"):
            call()
    with pytest.raises(ValueError, match="multiple"):
        PF.window_attention(x[:, :, :1].expand(-1, -1, 3, -1), x, x)
    for bad in (x[0], torch.zeros(1, 5, 2, 8)):
        with pytest.raises(ValueError):
            PF.window_attention(x, bad, bad)
    with pytest.raises(ValueError, match="lengths"):
        PF.window_attention_step(x, x, x, None)
    with pytest.raises(ValueError, match="no gradient"):
        PA.norm_rotate(x, x, positions=torch.zeros(4, requires_grad=True), frequencies=torch.ones(2))
    for value in (-1, 1.5):
        with pytest.raises(ValueError):
            PF._bound(value, "window")


@pytest.mark.parametrize("buckets,distance,both", [(32, 128, True), (32, 128, False), (4, 2, True), (2, 2, False), (3, 100, False), (8, 64, True), (64, 500, False),
                                                   (256, 2048, True), (256, 2048, False)])
def test_buckets(buckets, distance, both):
    """Every distance's bucket from the definition in whole numbers, at exact powers as well (32 buckets to 128: 16, 32, 64)."""
    n = buckets // 2 if both else buckets
    E, L = n // 2, n - n // 2
    got = PF.relative_buckets(range(-distance - 5, distance + 6), buckets, distance, both)
    for off, b in zip(range(-distance - 5, distance + 6), got):
        d = min(abs(off), distance)
        want = d if d < E else E + max(k for k in range(L) if Fraction(d, E) ** L >= Fraction(distance, E) ** k)
        assert b == want + (n if off > 0 and both else 0), off


def test_buckets_that_are_refused():
    for buckets, distance, both in ((1, 9, False), (2, 9, True), (5, 9, True), (32, 8, True), (32, 16, False), (258, 600, True), (32, 2049, True), (32, 0, True)):
        with pytest.raises(ValueError):
            PF.relative_buckets((1,), buckets, distance, both)


def test_the_layer_refuses():
    with pytest.raises(ValueError, match="multiple"):
        pn.WindowAttention(32, heads=4, dim_head=8, kv_heads=3)
    with pytest.raises(ValueError):
        pn.WindowAttention(32, heads=4, dim_head=8, window=(-1, 4))
    with pytest.raises(ValueError):
        pn.WindowAttention(32, heads=4, dim_head=8, window=(4,))
    with pytest.raises(ValueError):
        pn.WindowAttention(32, heads=4, dim_head=8, bias_buckets=5)
    with pytest.raises(ValueError, match="pairs"):
        pn.WindowAttention(32, heads=4, dim_head=4, axes=3)
    layer = pn.WindowAttention(32, heads=4, dim_head=8)
    with pytest.raises(RuntimeError, match="GPU tensors only"):
        layer(torch.zeros(1, 4, 32))
    with pytest.raises(ValueError, match="Expected 3D"):
        layer(torch.zeros(4, 32))
    with pytest.raises(ValueError, match="reach ahead"):
        layer.step(torch.zeros(1, 1, 32), layer.cache(1, 4))
    with pytest.raises(ValueError, match="fp8"):
        layer.use_fp8_weights()
    cache = layer.cache(2, 3)
    k = torch.ones(2, 2, 4, 8)
    cache.append(k, 2 * k)
    with pytest.raises(ValueError, match="no room"):
        cache.append(k, k)
    assert cache.lengths.tolist() == [2, 2] and bool(cache.k[:, :2].eq(1).all()) and not cache.k[:, 2:].any() and bool(cache.v[:, :2].eq(2).all())
    cache.reset(torch.tensor([1, 0], dtype=torch.int32))
    cache.append(3 * k, k)
    assert cache.k[0, 1:, 0, 0].tolist() == [3, 3] and cache.k[1, :2, 0, 0].tolist() == [3, 3]
    for lengths in ([0, -1], [4, 0], [1]):
        with pytest.raises(ValueError, match="lengths have to be"):
            cache.reset(torch.tensor(lengths, dtype=torch.int32))
    assert cache.lengths.tolist() == [3, 2] and cache.used == 3
    cache.reset()
    assert cache.used == 0 and not cache.lengths.any()


def test_frequencies_of_a_cast_layer():
    """The type of the weights does not round the angles."""
    layer = pn.WindowAttention(32, heads=4, dim_head=16, axes=2)
    own = layer.frequencies.clone()
    for cast in (layer.to(torch.bfloat16), layer.half(), layer.double(), layer.to("meta"), layer.to_empty(device="cpu")):
        assert layer.frequencies.dtype == torch.float32
        assert layer.frequencies.is_meta or torch.equal(layer.frequencies, own)


def test_models_with_window_blocks(tmp_path):
    options = dict(functional_dim=3, out_dim=2, embedding_dim=2, n_layers=3, n_hidden=32, n_head=4, use_te=False)
    plain = pn.Transolver(**options)
    assert "window_blocks" not in plain._args and all(isinstance(b.Attn, pn.PhysicsAttentionBase) for b in plain.blocks)
    model = pn.Transolver(**options, window_blocks=(1,), window_options=dict(window=(7, 7), sinks=1, bias_buckets=8, max_distance=9))
    assert [type(b.Attn) is pn.WindowAttention for b in model.blocks] == [False, True, False]
    model.save(str(tmp_path / "m.mdlus"))
    again = pn.Transolver.from_checkpoint(str(tmp_path / "m.mdlus"))
    assert again.blocks[1].Attn.window == (7, 7) and all(torch.equal(a, b) for a, b in zip(model.state_dict().values(), again.state_dict().values()))
    with pytest.raises(ValueError, match="window_blocks"):
        pn.Transolver(**options, window_blocks=(3,))
    with pytest.raises(ValueError, match="window_options"):
        pn.Transolver(**options, window_options={})
    with pytest.raises(ValueError, match="fp8"):
        model.use_fp8_weights()
