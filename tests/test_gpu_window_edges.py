"""Attention over a window at its edges: rows behind sequences, scores out of the ordinary, means far from zero, scales of the caller's."""
import pytest
import torch

import window_oracle as wo
from gpu_util import announce
from physicsnemo_amd import autograd as PA
from physicsnemo_amd import functional as PF
from test_gpu_window import BF, F32, compare, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("buckets", [0, 8])
@pytest.mark.parametrize("D", [32, 40, 64, 128])
def test_rows_behind_sequences_are_not_read(D, buckets, dtype):
    """NaN or zeros behind sequences whose last tiles are not whole: the same bits.  A NaN that came in would be multiplied by a weight of zero, and the sums
    it spoils formed again row by row, in other roundings."""
    announce("behind", D, buckets, dtype)
    N = 330
    q, k, v, dy, bias = make(4, N, 4, 2, D, dtype, buckets, seed=D)
    lengths = (1, 70, 201, 323)  # behind a tile's first row, behind its first rows, in the middle, short of the buffer's end
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    call = dict(window=(90, 0), sinks=3, lengths=n, bias=bias, max_distance=20)

    def all_of_it(behind):
        ts = [t.clone() for t in (q, k, v, dy)]
        for t in ts:
            for b, m in enumerate(lengths):
                t[b, m:] = behind
        y, stats = PF.window_attention(*ts[:3], return_stats=True, **call)
        grads = PF.window_attention_backward(ts[3], *ts[:3], y, stats, **call)
        first = [max(0, m - 5) for m in lengths]
        newest = torch.stack([q[b, f:f + 5] for b, f in enumerate(first)])
        step = PF.window_attention_step(newest, *ts[1:3], n, left=90, sinks=3, bias=bias, max_distance=20)
        return [t for t in (y, stats, *grads, step) if t is not None]

    for a, b in zip(all_of_it(0.0), all_of_it(float("nan"))):
        assert torch.isfinite(a[a != float("inf")]).all() and torch.equal(a, b)


def one_hot(size, N, D, dtype, falling, twice):
    """Scores of up to about `size` in steps of its 128th at the scale D^-0.5, formed without rounding: q, k, v and, for a window of everything up to a point
    (first points of it included), what a softmax of such scores leaves: the value of the largest, or the mean of the two that are largest."""
    gen = torch.Generator("cuda").manual_seed(5)
    draw = lambda: torch.randn(1, N, 2, D, generator=gen, device="cuda").to(dtype)
    q, k, v, dy = torch.zeros_like(draw()), torch.zeros_like(draw()), draw(), draw()
    step = torch.arange(N, device="cuda") % 64
    if falling:
        step = step.flip(0)
    if twice:
        step = step // 2 * 2
    root = 2.0 ** round(torch.tensor(size * D ** 0.5).double().log2().item() / 2)
    q[..., 0], k[..., 0] = root, (root * (1 + step / 128))[None, :, None].to(dtype)
    return q, k, v, dy, step


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("twice", [False, True])
@pytest.mark.parametrize("falling", [False, True])
@pytest.mark.parametrize("size", [1e5, 1e8, 3e9, 3e10, 1e11, 1e20, 2e37])
def test_scores_of_any_size(size, falling, twice, D, dtype):
    """Scores that are finite in float32 have their softmax: gaps of a 128th of the size, 780 and more, leave the largest alone.  A value is weighed and
    divided by its weight: r of itself and 8 u; the mean of two as well."""
    announce("size", size, falling, twice, D, dtype)
    N, back = 200, 50
    q, k, v, _, step = one_hot(size, N, D, dtype, falling, twice)
    i = torch.arange(N, device="cuda")
    ok = (i[None] <= i[:, None]) & (i[None] >= i[:, None] - back)
    best = torch.where(ok, step[None], -1).amax(1, keepdim=True)
    w = (ok & (step[None] == best)).double()
    w /= w.sum(1, keepdim=True)
    V = v[0].double()
    want, size_of = torch.einsum("ij,jhd->ihd", w, V), torch.einsum("ij,jhd->ihd", w, V.abs())
    r = torch.finfo(dtype).eps / 2
    tol = r * want.abs() + 8 * wo.U * size_of
    y = PF.window_attention(q, k, v, window=(back, 0))
    if float(q[..., 0].max()) * float(k[..., 0].min()) >= 2.0 ** 128:  # 2e37 at 128 channels: q . k is past float32, every score infinite
        assert y.isnan().all()
    else:
        assert ((y[0].double() - want).abs() <= tol).all()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("twice", [False, True])
@pytest.mark.parametrize("falling", [False, True])
@pytest.mark.parametrize("size", [1e5, 1e8, 3e9, 3e10, 1e11, 1e20, 2e37])
def test_steps_over_scores_of_any_size(size, falling, twice, D, dtype):
    """The same over a cache, in one part and in several, whose references differ."""
    announce("step of size", size, falling, twice, D, dtype)
    for N, back in ((200, 50), (3000, None)):
        q, k, v, _, step = one_hot(size, N, D, dtype, falling, twice)
        if back is None:  # every part has a largest of its own, all of them another
            step = torch.arange(N, device="cuda") * 64 // N
            step = step.flip(0) if falling else step
            k[..., 0] = (float(q[0, 0, 0, 0]) * (1 + step / 128))[None, :, None].to(dtype)
        n = torch.tensor([N], dtype=torch.int32, device="cuda")
        ok = torch.ones(N, dtype=torch.bool, device="cuda") if back is None else torch.arange(N, device="cuda") >= N - 1 - back
        w = (ok & (step == step[ok].max())).double()
        w /= w.sum()
        V = v[0].double()
        want, size_of = torch.einsum("j,jhd->hd", w, V), torch.einsum("j,jhd->hd", w, V.abs())
        tol = torch.finfo(dtype).eps / 2 * want.abs() + (16 + int(w.gt(0).sum())) * wo.U * size_of
        y = PF.window_attention_step(q[:, -1:], k, v, n, left=back)
        if float(q[..., 0].max()) * float(k[..., 0].min()) >= 2.0 ** 128:
            assert y.isnan().all()
        else:
            assert ((y[0, 0].double() - want).abs() <= tol).all(), N


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("buckets", [0, 8])
def test_gradients_of_scores_past_the_denominators(buckets, D, dtype):
    """A point whose scores are past what the kept denominator holds: NaN in its gradient and in those of the keys that it sees, not wrong ones; all others
    as they were."""
    announce("past the denominators", buckets, D, dtype)
    N, at = 200, 120
    q, k, v, dy, bias = make(1, N, 2, 2, D, dtype, buckets, seed=D)
    k[..., 0] = k[..., 0].abs() + 0.5  # its scores are all of one sign
    call = dict(window=(30, 10), sinks=2, bias=bias, max_distance=12)

    def all_of_it(q):
        y, stats = PF.window_attention(q, k, v, return_stats=True, **call)
        return y, stats, PF.window_attention_backward(dy, q, k, v, y, stats, **call)

    clean, q2 = all_of_it(q), q.clone()
    i = torch.arange(N, device="cuda")
    seen = ((i >= at - 30) & (i <= at + 10)) | (i < 2)
    for size in (1e8, -1e8, 1e12, 1e30):
        q2[0, at, 1] = 0
        q2[0, at, 1, 0] = size
        y, stats, (dq, dk, dv, db) = all_of_it(q2)
        assert torch.isfinite(y).all() and stats[0, 1, at].isnan() and int(stats.isnan().sum()) == 1
        assert dq[0, at, 1].isnan().all() and torch.equal(dq[0, i != at], clean[2][0][0, i != at])
        for got, was in ((dk, clean[2][1]), (dv, clean[2][2])):
            assert got[0, seen, 1].isnan().all() and torch.equal(got[0, ~seen], was[0, ~seen]) and torch.equal(got[:, :, 0], was[:, :, 0])
        if buckets:
            assert torch.equal(db[:, 0], clean[2][3][:, 0]) and db[0, 1].isnan()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("falling", [False, True])
@pytest.mark.parametrize("size", [1e3, 1e4, 1e5])
def test_gradients_of_large_scores(size, falling, dtype):
    announce("gradients of size", size, falling, dtype)
    q, k, v, dy, _ = one_hot(size, 200, 32, dtype, falling, True)
    compare(q, k, v, dy, None, window=(50, 0))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("buckets", [0, 12])
@pytest.mark.parametrize("D", [24, 64, 128])
@pytest.mark.parametrize("scale", [0.03, 1.0, 3.0])
def test_scales(scale, D, buckets, dtype):
    """The caller's scale, in values, all gradients, and steps."""
    announce("scale", scale, D, buckets, dtype)
    q, k, v, dy, bias = make(2, 210, 4, 2, D, dtype, buckets, seed=D)
    call = dict(sinks=3, scale=scale, max_distance=30)
    q = q * min(1.0, D ** -0.5 / scale * 2)  # scores of a softmax that is not one-hot
    lengths = torch.tensor([210, 133], dtype=torch.int32, device="cuda")
    for right in (0, 25):
        compare(q, k, v, dy, bias, window=(60, right), lengths=lengths, **call)
    want = wo.attention(q[:, -7:], k, v, window=(60, 0), lengths=lengths, bias=bias, first=lengths.long() - 7, **call)["y"]
    wo.check(PF.window_attention_step(q[:, -7:], k, v, lengths, left=60, bias=bias, **call), want, "step")
    other = PF.window_attention(q, k, v, window=(60, 0), bias=bias, **{**call, "scale": 2 * scale})
    assert not torch.equal(other, PF.window_attention(q, k, v, window=(60, 0), bias=bias, **call))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("scale", [1e-29, 1e-12, 1e12, 1e29])
def test_scales_at_their_limits(scale, dtype):
    """Inputs that make up for it: the results of ordinary ones, exactly so for scales and inputs that differ by powers of two."""
    announce("far scale", scale, dtype)
    q, k, v, dy, _ = make(1, 150, 2, 1, 32, dtype, 0, seed=3)
    power = 2.0 ** round(torch.tensor(scale).double().log2().item())
    call = dict(window=(40, 20), sinks=2)
    def all_of_it(q, scale):
        y, stats = PF.window_attention(q, k, v, scale=scale, return_stats=True, **call)
        return y, *PF.window_attention_backward(dy, q, k, v, y, stats, scale=scale, **call)[:3]
    want, got = all_of_it(q, 0.25), all_of_it(q / power, 0.25 * power)
    assert torch.equal(got[0], want[0]) and torch.equal(got[2], want[2]) and torch.equal(got[3], want[3])
    wo.check(got[1].double() / power, (want[1].double(), torch.finfo(dtype).eps * want[1].double().abs()), "dq")
