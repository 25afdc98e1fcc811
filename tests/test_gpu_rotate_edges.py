"""Norm and rotation of queries and keys where values are infinite or NaN, where eps is zero, and at positions far out."""
import pytest
import torch

from gpu_util import announce
from physicsnemo_amd import autograd as PA
from physicsnemo_amd import functional as PF
from test_gpu_rotate import compare, make, speeds

pytestmark = pytest.mark.gpu
WILD = [float("inf"), float("-inf"), float("nan")]
# D, channels turned, interleaved: whole fours of either half, odd halves, neighbours; one and several lanes a row
PAIRINGS = [(32, 16, False), (8, 0, False), (32, 30, False), (33, 20, False), (128, 62, False), (5, 2, False), (32, 16, True), (24, 6, True), (7, 4, True), (128, 96, True)]


def same(a, b):
    return torch.equal(torch.nan_to_num(a, 3e38, 1e38, 2e38), torch.nan_to_num(b, 3e38, 1e38, 2e38)) and torch.equal(a.isnan(), b.isnan())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("value", WILD)
@pytest.mark.parametrize("D,R,interleaved", PAIRINGS)
def test_wild_channels_that_are_not_turned(D, R, interleaved, value, dtype):
    """Without the norm they are left as they are and touch no other, in results and in gradients."""
    announce("not turned", D, R, interleaved, value, dtype)
    N = 37
    q, k, _, _, dyq, dyk = make(1, N, 2, 2, D, dtype, seed=D)
    turn = (torch.arange(N, device="cuda"), speeds(R // 2)) if R else (None, None)
    call = dict(norm=False, interleaved=interleaved)
    clean = PF.norm_rotate(q, k, None, None, *turn, **call)
    back = lambda dq, dk: PF.norm_rotate_backward(dq, dk, q, k, None, None, *turn, **call)[:2]
    clean_d = back(dyq, dyk)
    for at in {R, (R + D) // 2, D - 1}:
        q2, k2, gq2, gk2 = (t.clone() for t in (q, k, dyq, dyk))
        for t in (q2, k2, gq2, gk2):
            t[0, 3::5, :, at] = value
        for got, want, given in zip((*PF.norm_rotate(q2, k2, None, None, *turn, **call), *back(gq2, gk2)), (*clean, *clean_d), (q2, k2, gq2, gk2)):
            want = want.clone()
            want[0, 3::5, :, at] = value
            assert same(got, want), at
            assert same(got[..., R:], given[..., R:]), at


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D,R,interleaved", PAIRINGS)
def test_infinite_channels_under_the_norm(D, R, interleaved, dtype):
    """x / infinity: NaN for the channel that is infinite itself, zero for the others of its head, nothing for other heads."""
    announce("infinite", D, R, interleaved, dtype)
    N = 21
    q, k, wq, wk, _, _ = make(1, N, 3, 2, D, dtype, seed=D + 1)
    turn = (torch.arange(N, device="cuda"), speeds(R // 2)) if R else (None, None)
    clean = PF.norm_rotate(q, k, wq, wk, *turn, interleaved=interleaved)
    for at in {R, D - 1}:
        q2 = q.clone()
        q2[0, 4, 1, at] = float("inf")
        got = PF.norm_rotate(q2, k, wq, wk, *turn, interleaved=interleaved)
        want = clean[0].clone()
        want[0, 4, 1] = 0
        want[0, 4, 1, at] = float("nan")
        assert same(got[0], want) and torch.equal(got[1], clean[1]), at


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("value", WILD)
@pytest.mark.parametrize("D,R,interleaved", PAIRINGS)
def test_gradients_without_the_norm_do_not_read_the_inputs(D, R, interleaved, value, dtype):
    """dx is dy turned back, whatever x holds."""
    announce("without the norm", D, R, interleaved, value, dtype)
    N = 19
    q, k, _, _, dyq, dyk = make(2, N, 2, 1, D, dtype, seed=D + 2)
    turn = (torch.arange(N, device="cuda"), speeds(R // 2)) if R else (None, None)
    call = dict(norm=False, interleaved=interleaved)
    wild = [torch.full_like(t, value) for t in (q, k)]
    clean = PF.norm_rotate_backward(dyq, dyk, q, k, None, None, *turn, **call)
    got = PF.norm_rotate_backward(dyq, dyk, *wild, None, None, *turn, **call)
    assert all(torch.equal(a, b) for a, b in zip(got[:2], clean[:2]))
    leaves = [t.requires_grad_(True) for t in wild]
    own = torch.autograd.grad(PA.norm_rotate(*leaves, None, None, *turn, **call), leaves, [dyq, dyk])
    assert all(torch.equal(a, b) for a, b in zip(own, clean[:2]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,N,Hq,Hk,D", [(1, 1, 1, 1, 8), (1, 5, 3, 1, 32), (2, 7, 2, 2, 33), (1, 1031, 3, 2, 64), (3, 2, 1, 1, 128)])
def test_no_eps(B, N, Hq, Hk, D, dtype):
    """eps = 0: rows that are not zero have their norm, and weight gradients sum them alone, also where rows do not fill a workgroup."""
    announce("no eps", B, N, Hq, Hk, D, dtype)
    q, k, wq, wk, dyq, dyk = make(B, N, Hq, Hk, D, dtype, seed=N)
    compare(q, k, wq, wk, torch.arange(N, device="cuda"), speeds(D // 2), dyq, dyk, eps=0.0)


TWO_PI = "6.283185307179586476925286766559005768394338798750211641949889184615632812572417997256069650684234135964296173026564613294187689219"


@pytest.mark.parametrize("kind,far", [(torch.float32, 2.0 ** 40), (torch.float32, -(2.0 ** 62)), (torch.float32, 2.0 ** 77), (torch.float32, -(2.0 ** 77)),
                                      (torch.int64, 2 ** 53 - 4), (torch.int64, -(2 ** 53))])
@pytest.mark.parametrize("axes", [1, 3])
def test_angles_far_out(axes, kind, far):
    """To the last product that is served, against angles reduced with 120 digits: the turn's own error is below 2^-25 there, sincos and its argument's
    rounding leave less than the rest of 4 u (u = 2^-24)."""
    import math
    from decimal import Decimal, getcontext
    getcontext().prec = 120
    announce("far out", axes, kind, far)
    f = torch.stack([speeds(8) / 2 ** a for a in range(axes)])
    steps = torch.arange(3 * axes, device="cuda").view(3, axes)
    positions = far * (1 + steps.float() * 2.0 ** -5) if kind == torch.float32 else far + steps % 4
    positions = positions.to(kind)
    assert positions.double().abs().max() <= (2.0 ** 78 if kind == torch.float32 else 2.0 ** 53)
    angle = [[float(sum(Decimal(p) * Decimal(w[c]) for p, w in zip(row, f.tolist())) % Decimal(TWO_PI)) for c in range(8)]
             for row in ([[Decimal(v) for v in row] for row in positions.tolist()])]
    want_c, want_s = (torch.tensor([[fn(a) for a in row] for row in angle], dtype=torch.float64) for fn in (math.cos, math.sin))
    one = torch.zeros(1, 3, 1, 16, device="cuda")
    one[..., :8] = 1
    q, _ = PF.norm_rotate(one, one, positions=positions, frequencies=f, norm=False)
    got = q[0, :, 0].double().cpu()
    assert (got[:, :8] - want_c).abs().max() <= 4 * 2.0 ** -24 and (got[:, 8:] - want_s).abs().max() <= 4 * 2.0 ** -24


@pytest.mark.parametrize("kind,far", [(torch.float32, 2.0 ** 79), (torch.float32, -3e38), (torch.float32, float("inf")), (torch.float32, float("nan")),
                                      (torch.int64, 2 ** 53 + 1), (torch.int64, -(2 ** 63)), (torch.int64, 2 ** 63 - 1)])
def test_angles_too_far_out(kind, far):
    """NaN, not a wrong turn, in the pairs that it concerns; other points and channels behind the pairs as ever."""
    announce("too far out", kind, far)
    q, k, _, _, _, _ = make(1, 5, 1, 1, 12, torch.float32, seed=1)
    f = torch.tensor([1.0, 0.5, 0.5, 0.0], device="cuda")
    positions = torch.tensor([3, 1, 4, 1, 5], device="cuda").to(kind)
    clean = PF.norm_rotate(q, k, None, None, positions, f)[0]
    positions[2] = far
    got = PF.norm_rotate(q, k, None, None, positions, f)[0]
    keep = [0, 1, 3, 4]
    assert torch.equal(got[:, keep], clean[:, keep]) and torch.equal(got[..., 8:], clean[..., 8:])
    touched = got[0, 2, 0, :8].isnan().view(2, 4)
    all_of_it = kind == torch.int64 or not abs(far) < float("inf")
    assert touched[:, 0].all() and bool(touched[:, 3].all()) == all_of_it and torch.equal(touched[0], touched[1])
