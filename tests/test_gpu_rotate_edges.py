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
