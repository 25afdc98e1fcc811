"""Attention over a window of neighbours on the GPU against the formulas in 64 bits (tests/window_oracle.py, with the tolerances)."""
import pytest
import torch

import window_oracle as wo
from gpu_util import announce
from physicsnemo_amd import autograd as PA
from physicsnemo_amd import functional as PF

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def make(B, N, Hq, Hk, D, dtype, buckets=0, seed=0, Nk=None):
    gen = torch.Generator("cuda").manual_seed(seed)
    draw = lambda n, h: torch.randn(B, n, h, D, generator=gen, device="cuda").to(dtype)
    Nk = N if Nk is None else Nk
    q, k, v, dy = draw(N, Hq), draw(Nk, Hk), draw(Nk, Hk), draw(N, Hq)
    bias = torch.randn(buckets, Hq, generator=gen, device="cuda") if buckets else None
    return q, k, v, dy, bias


def compare(q, k, v, dy, bias, grads=True, **call):
    want = wo.attention(q, k, v, bias=bias, dy=dy if grads else None, **call)
    y = PF.window_attention(q, k, v, bias=bias, **call)
    worst = [wo.check(y, want["y"], "y")]
    if grads:
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)] + ([] if bias is None else [bias.detach().requires_grad_(True)])
        out = PA.window_attention(*leaves[:3], bias=leaves[3] if bias is not None else None, **call)
        assert torch.equal(out, y)
        for name, g in zip(("dq", "dk", "dv", "dbias"), torch.autograd.grad(out, leaves, dy)):
            worst.append(wo.check(g, want[name], name))
    print("worst", [f"{w:.2f}" for w in worst], flush=True)


SIZES = [  # B, N, Hq, Hk, D, left, right, sinks
    (1, 1, 1, 1, 32, 4, 4, 0), (2, 5, 2, 2, 16, 2, 0, 1), (1, 33, 3, 1, 33, 40, 7, 0), (1, 64, 2, 1, 64, 0, 0, 0), (2, 129, 4, 2, 32, 31, 32, 3),
    (1, 300, 2, 2, 32, 32, 32, 0), (1, 257, 2, 1, 128, 100, 0, 33), (3, 200, 6, 3, 24, 17, 65, 8), (1, 515, 2, 2, 7, 64, 64, 40), (1, 131, 1, 1, 1, 5, 5, 2),
    (1, 700, 4, 1, 48, 127, 128, 128), (1, 385, 2, 2, 80, None, 0, 5), (1, 260, 2, 2, 100, None, None, 0), (2, 150, 2, 2, 64, 20, None, 4),
    (1, 1300, 2, 1, 32, 50, 0, 20)]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("B,N,Hq,Hk,D,left,right,sinks", SIZES)
def test_values_and_gradients(B, N, Hq, Hk, D, left, right, sinks, dtype):
    announce("window", B, N, Hq, Hk, D, left, right, sinks, dtype)
    q, k, v, dy, _ = make(B, N, Hq, Hk, D, dtype, seed=N)
    compare(q, k, v, dy, None, window=(left, right), sinks=sinks)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("buckets,distance", [(4, 2), (8, 100), (32, 128), (64, 500), (256, 2048)])
@pytest.mark.parametrize("B,N,Hq,Hk,D,left,right,sinks", [SIZES[k] for k in (0, 1, 4, 6, 11, 12, 14)])
def test_bias_and_its_gradient(B, N, Hq, Hk, D, left, right, sinks, buckets, distance, dtype):
    announce("bias", B, N, Hq, Hk, D, left, right, sinks, buckets, distance, dtype)
    if right == 0 and distance <= buckets // 2:
        distance = buckets // 2 + 1
    q, k, v, dy, bias = make(B, N, Hq, Hk, D, dtype, buckets, seed=N + 1)
    compare(q, k, v, dy, bias, window=(left, right), sinks=sinks, max_distance=distance)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("buckets", [0, 16])
@pytest.mark.parametrize("lengths", [[0, 1, 200], [129, 0, 0], [64, 200, 37], [-5, 500, 128]])
def test_padded_sequences(lengths, buckets, dtype):
    """Rows behind a sequence hold NaN: they are not read, and zero in results and gradients."""
    announce("padded", lengths, buckets, dtype)
    q, k, v, dy, bias = make(3, 200, 4, 2, 40, dtype, buckets, seed=5)
    for b, n in enumerate(lengths):
        for t in (q, k, v, dy):
            t[b, max(0, min(n, 200)):] = float("nan")
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    call = dict(window=(70, 0 if buckets else 33), sinks=6, lengths=n, max_distance=60)
    compare(q, k, v, dy, bias, **call)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    y = PA.window_attention(*leaves, bias=bias, **call)
    for t in (y, *torch.autograd.grad(y, leaves, dy)):
        for b, m in enumerate(lengths):
            assert not t[b, max(0, min(m, 200)):].any()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("value", [float("-inf"), torch.finfo(torch.float32).min, -1e9, -65536.0])
@pytest.mark.parametrize("all_of_it", [False, True])
def test_masking_biases(value, all_of_it, dtype):
    """Biases of -inf and down to the lowest float hide their distances, also all that a point sees: zeros, no gradients, no NaN."""
    announce("masking", value, all_of_it, dtype)
    q, k, v, dy, bias = make(2, 150, 2, 2, 32, dtype, 8, seed=9)
    bias[:, 0] = value  # head 0: everything, or all but the point itself
    if not all_of_it:
        bias[0, 0] = 0.5
    bias[3:5, 1] = value
    compare(q, k, v, dy, bias, window=(40, 40), max_distance=30)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v, bias)]
    y = PA.window_attention(*leaves[:3], bias=leaves[3], window=(40, 40), max_distance=30)
    grads = torch.autograd.grad(y, leaves, dy)
    assert not grads[3][3:5, 1].any()
    if all_of_it:
        assert not any(t[:, :, 0].any() for t in (y, *grads[:3])) and not grads[3][:, 0].any()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("value", [70000.0, 9000.0, -9000.0])
def test_large_biases(value, dtype):
    """One distance far above or below the others, by more than exp2 holds: what is above takes all, what is below nothing."""
    announce("large", value, dtype)
    q, k, v, dy, bias = make(1, 100, 2, 1, 16, dtype, 8, seed=3)
    bias[1] = value
    compare(q, k, v, dy, bias, window=(30, 30), max_distance=20)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
def test_wild_values_where_they_are_not_seen(value, dtype):
    """Infinities and NaN in points of the sequence itself reach the points that see them and no others, forward and backward."""
    announce("wild", value, dtype)
    q, k, v, dy, bias = make(1, 300, 4, 2, 32, dtype, 8, seed=12)
    call = dict(window=(37, 21), sinks=2, bias=bias, max_distance=25)
    def all_of_it(q, k, v, dy):
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        y = PA.window_attention(*leaves, **call)
        n = torch.full((1,), 300, dtype=torch.int32, device="cuda")
        step = PF.window_attention_step(q[:, -40:], k, v, n, left=37, sinks=2, bias=bias, max_distance=25)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy), step]
    clean, at, want = all_of_it(q, k, v, dy), 150, wo.attention(q, k, v, dy=dy, **call)
    i = torch.arange(300, device="cuda")
    sees = (i >= at - 21) & (i <= at + 37)  # the queries that see the point; the keys it sees: at - 37 .. at + 21 and the sinks
    seen = ((i >= at - 37) & (i <= at + 21)) | (i < 2)
    near = sees[:, None] & torch.stack([((i >= a - 37) & (i <= a + 21)) | (i < 2) for a in range(300)])
    through = near.any(0)  # keys of the queries that see the point
    for which, touched in (("q", (i == at, i == at, seen, seen)), ("k", (sees, sees, through, through)), ("v", (sees, sees, through, i == at)),
                           ("dy", (i < 0, i == at, seen, seen))):
        t = {n: x.clone() for n, x in zip(("q", "k", "v", "dy"), (q, k, v, dy))}
        t[which][0, at] = value
        got = all_of_it(**t)
        for n, (name, may) in enumerate(zip(("y", "dq", "dk", "dv"), touched)):
            wo.check(got[n][0][~may], [t[0][~may] for t in want[name]], (which, name))
            if may.any() and not (which == "v" and name == "dv"):
                assert not torch.isfinite(got[n][0][may]).all(), (which, name)
        assert torch.equal(got[4], clean[4])  # the step's windows lie behind the point


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [16, 64, 128])
def test_infinite_keys_in_sight(D, dtype):
    """A key whose scores are all -inf weighs nothing; one whose scores are +inf leaves NaN to the points that see it, as a softmax does."""
    announce("infinite", D, dtype)
    q, k, v, _, bias = make(1, 150, 2, 2, D, dtype, 8, seed=4)
    q = q.abs() + 1
    call = dict(window=(20, 9), sinks=3, bias=bias, max_distance=12)
    for at in (1, 70):  # a first point, which all see; a point in the middle
        k2 = k.clone()
        k2[0, at, :, 0] = float("-inf")
        low = k.clone()
        low[0, at, :, 0] = -2000.0  # weights below exp(-170)
        y = PF.window_attention(q, k2, v, **call)
        wo.check(y, wo.attention(q, low, v, **call)["y"], ("-inf", at))
        k2[0, at, :, 0] = float("inf")
        y = PF.window_attention(q, k2, v, **call)[0]
        i = torch.arange(150, device="cuda")
        sees = (i >= at - 9) if at < 3 else (i >= at - 9) & (i <= at + 20)
        assert torch.isnan(y[sees]).all() and torch.isfinite(y[~sees]).all()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("bias", [False, True])
def test_scores_that_outgrow_the_first(bias, dtype):
    """Scores that rise by hundreds along the window, beyond what exp2 holds: the weights of the largest, as a softmax has them."""
    announce("outgrow", bias, dtype)
    q, k, v, dy, table = make(2, 700, 2, 1, 32, dtype, 8, seed=6)
    q[..., 0], k[..., 0] = 8.0, torch.linspace(-160, 160, 700, device="cuda").to(dtype)[None, :, None]  # 226 a hundred points
    compare(q, k, v, dy, table if bias else None, window=(300, 150), sinks=2, **(dict(max_distance=20) if bias else {}))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_nan_and_the_bias_gradient(dtype):
    """A gradient that is NaN at one point reaches the buckets of the distances that the point sees; the others stay as they were."""
    announce("nan in d bias", dtype)
    q, k, v, dy, bias = make(1, 90, 2, 1, 32, dtype, 16, seed=2)
    def grad(dy):
        leaf = bias.detach().requires_grad_(True)
        return torch.autograd.grad(PA.window_attention(q, k, v, bias=leaf, window=(60, 0), max_distance=40), leaf, dy)[0]
    clean, bad = grad(dy), dy.clone()
    bad[0, 3, 0] = float("nan")  # sees distances 0 .. 3, of a bucket each
    got = grad(bad)
    assert torch.isnan(got[:4, 0]).all() and torch.equal(got[4:], clean[4:]) and torch.equal(got[:, 1], clean[:, 1])


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("which", ["all", "k", "v"])
def test_inputs_full_of_nan(which, dtype):
    """NaN everywhere is NaN everywhere; with NaN in the values alone the weights, and so dv, are those of the scores."""
    announce("full of nan", which, dtype)
    q, k, v, dy, _ = make(1, 3000, 2, 1, 40, dtype, seed=8)
    want = wo.attention(q, k, v, sinks=0, dy=dy)
    for name, t in (("q", q), ("k", k), ("v", v)):
        if which in ("all", name):
            t.fill_(float("nan"))
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    y = PA.window_attention(*leaves)
    dq, dk, dv = torch.autograd.grad(y, leaves, dy)
    assert all(torch.isnan(t).all() for t in (y, dq, dk))
    if which == "v":
        wo.check(dv, want["dv"], "dv")
    else:
        assert torch.isnan(dv).all()


@pytest.mark.parametrize("dtype", [BF, F32])
def test_first_points_of_many_sequences(dtype):
    """More sums of first points' gradients than one round of their workgroups holds."""
    announce("many", dtype)
    q, k, v, dy, _ = make(40, 130, 4, 4, 64, dtype, seed=1)
    compare(q, k, v, dy, None, window=(5, 0), sinks=128)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_views(dtype):
    """Slices of one projection, shared keys (stride 0), rows off 16-byte boundaries, heads in front of rows: the results of copies."""
    announce("views", dtype)
    gen = torch.Generator("cuda").manual_seed(3)
    B, N, H, D = 2, 170, 4, 32
    draw = lambda *s: torch.randn(*s, generator=gen, device="cuda").to(dtype)
    packed, odd, turned = draw(B, N, 3 * H, D), draw(B * N * 3 * H * D + 1)[1:].view(B, N, 3 * H, D), draw(B, 3 * H, N, D).transpose(1, 2)
    wide, one = draw(B, N, 3 * H, D + 3)[..., 2:D + 2], draw(B, N, 1, D).expand(B, N, 3 * H, D)
    dy = draw(B, N, H, D + 1)[..., 1:]
    call = dict(window=(50, 20), sinks=2)
    for t in (packed, odd, turned, wide, one):
        views = [t[:, :, :H], t[:, :, H:2 * H], t[:, :, 2 * H:]]
        y = [PA.window_attention(*(x.detach().contiguous() if copy else x.detach() for x in views), **call) for copy in (False, True)]
        assert torch.equal(*y)
        both = []
        for copy in (False, True):
            leaves = [(x.detach().contiguous() if copy else x.detach()).requires_grad_(True) for x in views]
            both.append(torch.autograd.grad(PA.window_attention(*leaves, **call), leaves, dy.contiguous() if copy else dy))
        assert all(torch.equal(a, b) for a, b in zip(*both))
    turned_channels = packed.transpose(-1, -2).contiguous().transpose(-1, -2)
    with pytest.raises(ValueError, match="last axis"):
        PF.window_attention(turned_channels, packed, packed)
    assert torch.equal(PA.window_attention(turned_channels, packed, packed, **call), PF.window_attention(packed, packed, packed, **call))


def test_gradients_of_broadcast_inputs():
    """One key and value row for all sequences: autograd adds their gradients up."""
    announce("broadcast")
    q, k, v, dy, _ = make(3, 90, 4, 2, 16, F32, seed=2)
    k1, v1 = (t[:1].detach().requires_grad_(True) for t in (k, v))
    call = dict(window=(20, 20), sinks=1)
    got = torch.autograd.grad(PA.window_attention(q, k1.expand(3, -1, -1, -1), v1.expand(3, -1, -1, -1), **call), (k1, v1), dy)
    want = wo.attention(q, k1.detach().expand(3, -1, -1, -1), v1.detach().expand(3, -1, -1, -1), dy=dy, **call)
    for g, name in zip(got, ("dk", "dv")):
        value, tol = want[name]
        wo.check(g, (value.sum(0, keepdim=True), tol.sum(0, keepdim=True) + 4 * wo.U * value.abs().sum(0, keepdim=True)), name)


def test_gradients_against_differences():
    """Central differences of the float32 result in one direction per input: h = 2^-7 leaves h^2 / 6 of the third derivative and 2^-24 / h of rounding."""
    announce("differences")
    q, k, v, dy, bias = make(1, 70, 2, 1, 8, F32, 6, seed=4)
    q, k = q * 0.5, k * 0.5
    call = dict(window=(25, 25), sinks=2, max_distance=20)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v, bias)]
    grads = torch.autograd.grad(PA.window_attention(*leaves[:3], bias=leaves[3], **call), leaves, dy)
    h = 2.0 ** -7
    for n, (leaf, g) in enumerate(zip(leaves, grads)):
        way = torch.randn(leaf.shape, generator=torch.Generator("cuda").manual_seed(n), device="cuda")
        way /= way.norm()
        f = lambda s: (PF.window_attention(*[(t.detach() + (s * way if m == n else 0)) for m, t in enumerate(leaves[:3])],
                                           bias=bias + (s * way if n == 3 else 0), **call).double() * dy).sum()
        difference, slope = float((f(h) - f(-h)) / (2 * h)), float((g.double() * way).sum())
        size = float(dy.double().norm()) * 4  # |d3 f| <= about |dy| |y| |way|^3; rounding: 2^-24 |dy| |y| / h
        assert abs(difference - slope) <= size * (h * h + 2.0 ** -22 / h), (n, difference, slope)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_results_repeat(dtype):
    announce("repeat", dtype)
    q, k, v, dy, bias = make(2, 1500, 4, 2, 32, dtype, 32, seed=6)
    def once():
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v, bias)]
        y = PA.window_attention(*leaves[:3], window=(300, 40), sinks=5, bias=leaves[3])
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]
    first = once()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, once()))


STEPS = [  # B, capacity, T, Hq, Hk, D, left, sinks
    (1, 1, 1, 1, 1, 32, None, 0), (3, 40, 1, 4, 4, 16, 10, 2), (2, 333, 1, 8, 2, 64, None, 0), (4, 1000, 1, 8, 1, 128, 255, 4), (2, 100, 5, 6, 3, 24, 31, 1),
    (1, 5000, 1, 2, 2, 33, None, 0), (1, 700, 40, 4, 1, 32, 100, 33), (5, 64, 64, 2, 2, 8, None, 0), (2, 3000, 3, 16, 1, 80, 2000, 0)]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("buckets,distance", [(0, 0), (9, 50), (64, 2048)])
@pytest.mark.parametrize("B,cap,T,Hq,Hk,D,left,sinks", STEPS)
def test_steps(B, cap, T, Hq, Hk, D, left, sinks, buckets, distance, dtype):
    """The newest points over caches whose rows behind the sequences hold NaN; sequences of no, one, few and all points."""
    announce("step", B, cap, T, Hq, Hk, D, left, sinks, buckets, distance, dtype)
    q, k, v, _, bias = make(B, T, Hq, Hk, D, dtype, buckets, seed=cap, Nk=cap)
    for lengths in ([cap] * B, [(0, 1, T, T - 1, cap // 2)[b % 5] for b in range(B)], [max(1, cap - 3 * b) for b in range(B)]):
        n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        kk, vv = k.clone(), v.clone()
        for b, m in enumerate(lengths):
            kk[b, m:], vv[b, m:] = float("nan"), float("nan")
        want = wo.attention(q, kk, vv, window=(left, 0), sinks=sinks, lengths=n, bias=bias, max_distance=distance, first=n.long() - T)
        got = PF.window_attention_step(q, kk, vv, n, left=left, sinks=sinks, bias=bias, max_distance=distance)
        wo.check(got, want["y"], f"lengths {lengths}")
        for b, m in enumerate(lengths):
            assert not got[b, :max(0, T - m)].any()


def test_step_by_step_is_the_whole():
    """A sequence point by point over its cache: the rows of the whole call, within both sides' tolerances."""
    announce("step by step")
    q, k, v, _, bias = make(2, 90, 4, 2, 32, F32, 12, seed=8)
    call = dict(sinks=2, bias=bias, max_distance=40)
    whole, want = PF.window_attention(q, k, v, window=(20, 0), **call), wo.attention(q, k, v, window=(20, 0), **call)["y"]
    for t in range(90):
        n = torch.full((2,), t + 1, dtype=torch.int32, device="cuda")
        y = PF.window_attention_step(q[:, t:t + 1], k, v, n, left=20, **call)
        assert ((y[:, 0] - whole[:, t]).abs() <= 2 * want[1][:, t]).all(), t


def test_far_rows():
    """Elements past 2^31: the last rows of a long sequence and of a long cache are those of the same rows alone."""
    announce("far rows")
    N, H, D, W = (1 << 22) + 77, 8, 64, 16
    gen = torch.Generator("cuda").manual_seed(1)
    q, k, v, dy = (torch.randn(1, N, H, D, generator=gen, device="cuda", dtype=BF) for _ in range(4))
    assert q.numel() > 1 << 31
    y, stats = PF.window_attention(q, k, v, window=(W, W), return_stats=True)
    d = PF.window_attention_backward(dy, q, k, v, y, stats, window=(W, W))
    cut, own = N - 1000, 1000 - 2 * W  # rows whose neighbours' neighbours are inside the cut
    tail = [t[:, cut:].contiguous() for t in (q, k, v, dy)]
    want = wo.attention(*tail[:3], window=(W, W), dy=tail[3])
    for got, name in zip((y, *d[:3]), ("y", "dq", "dk", "dv")):
        wo.check(got[:, -own:], [t[:, -own:] for t in want[name]], name)
    n = torch.tensor([N], dtype=torch.int32, device="cuda")
    wo.check(PF.window_attention_step(q[:, -1:], k, v, n, left=W), [t[:, -1:] for t in wo.attention(*tail[:3], window=(W, 0))["y"]], "step")


def test_other_stream_and_graph():
    """Captured with its workspaces and replayed among eager calls: every replay is the eager result."""
    announce("graph")
    q, k, v, dy, bias = make(2, 400, 4, 2, 32, BF, 16, seed=11)
    n = torch.tensor([400, 123], dtype=torch.int32, device="cuda")
    call = dict(window=(60, 60), sinks=3, bias=bias, lengths=n, max_distance=64)
    def all_of_it():
        y, stats = PF.window_attention(q, k, v, return_stats=True, **call)
        step = PF.window_attention_step(q[:, :1], k, v, n, left=60, sinks=3, bias=bias, max_distance=64)
        return [y, step, *PF.window_attention_backward(dy, q, k, v, y, stats, **call), *PF.norm_rotate(q, k, positions=torch.arange(400, device="cuda"),
                                                                                                       frequencies=torch.ones(8, device="cuda"))]
    eager = all_of_it()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert all(torch.equal(a, b) for a, b in zip(eager, all_of_it()))
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = all_of_it()
    for round_ in range(4):
        with torch.no_grad():
            q.copy_(torch.randn(q.shape, generator=torch.Generator("cuda").manual_seed(round_), device="cuda").to(BF))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(kept, all_of_it())), round_
