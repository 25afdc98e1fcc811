"""Attention over a window of neighbours and its gradients in 64 bits, with the errors that the kernels' roundings may leave.

r = eps / 2 of the results' type, u = 2^-24.  Scores are float32 sums of D products: |e_s| <= (D + 8) u scale sum |q| |k| + 4 u (|s| + |bias|), a
weight is off by e_p = 2 e_s + 8 u of itself (its exponent, exp2 and the division), bf16 weights and score gradients by r more in
the products they go into, sums of n terms by (n + 8) u of their magnitudes."""
import torch

from physicsnemo_amd import functional as PF

U = 2.0 ** -24


def visible(N, Nk, first, left, right, sinks, n):
    """(B, N, Nk): query t is position first_b + t."""
    i = first[:, None, None] + torch.arange(N, device=n.device)[None, :, None]
    j = torch.arange(Nk, device=n.device)[None, None]
    n = n[:, None, None]
    ok = (i >= 0) & (i < n) & (j < n)
    if left is not None:
        ok = ok & ((j >= i - left) | (j < sinks))
    if right is not None:
        ok = ok & (j <= i + right)
    return ok


def bias_of(bias, N, Nk, first, right, max_distance):
    """(B, Hq, N, Nk)"""
    both = right != 0
    off = torch.arange(Nk, device=bias.device)[None, None] - first[:, None, None] - torch.arange(N, device=bias.device)[None, :, None]
    table = torch.tensor(PF.relative_buckets(range(-max_distance, max_distance + 1), bias.shape[0], max_distance, both), device=bias.device)
    return bias[table[off.clamp(-max_distance, max_distance) + max_distance]].permute(0, 3, 1, 2)


def attention(q, k, v, window=(None, None), sinks=0, scale=None, lengths=None, bias=None, max_distance=128, first=None, dy=None):
    """Values and tolerances: dict with y (and dq, dk, dv, dbias) -> (value, tolerance), all float64 on the inputs' device."""
    dtype, dev = q.dtype, q.device
    B, N, Hq, D = q.shape
    Nk, Hk = k.shape[1], k.shape[2]
    G, r, low = Hq // Hk, torch.finfo(dtype).eps / 2, dtype == torch.bfloat16
    scale = D ** -0.5 if scale is None else scale
    n = torch.full((B,), Nk, device=dev) if lengths is None else lengths.long().clamp(0, Nk)
    first = torch.zeros(B, dtype=torch.long, device=dev) if first is None else first
    ok = visible(N, Nk, first, *window, sinks, n)[:, None]
    live = (torch.arange(Nk, device=dev)[None] < n[:, None])[:, :, None, None]
    qlive = ((first[:, None] + torch.arange(N, device=dev)[None] < n[:, None]) & (first[:, None] + torch.arange(N, device=dev)[None] >= 0))[:, :, None, None]
    heads = lambda t, m: torch.where(m, t.double(), torch.zeros((), dtype=torch.float64, device=dev)).transpose(1, 2)
    Q = heads(q, qlive)
    K, V = (heads(t, live).repeat_interleave(G, 1) for t in (k, v))
    s = torch.matmul(Q, K.mT) * scale
    e_s = (D + 8) * U * scale * torch.matmul(Q.abs(), K.abs().mT) + 4 * U * s.abs()
    if bias is not None:
        add = bias_of(bias.double(), N, Nk, first, window[1], max_distance)
        ok = ok & (add > -65536)  # hidden
        add = add.clamp(-65536, 65536)
        s, e_s = s + add, e_s + 4 * U * add.abs()
    s = torch.where(ok, s, torch.full_like(s, -torch.inf))
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top > -torch.inf, top, torch.zeros_like(top)))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, torch.ones_like(total))
    e_p = 2 * torch.where(ok, e_s, torch.zeros_like(e_s)).amax(-1, keepdim=True) + (Nk + 8) * U  # of a row's weights, relative
    w = r if low else 0.0
    y = torch.matmul(p, V)
    e_y = r * y.abs() + (w + 2 * e_p) * torch.matmul(p, V.abs())
    back = lambda t: t.transpose(1, 2)
    out = {"y": (back(y), back(e_y))}
    if dy is None:
        return out
    dY = heads(dy, qlive)
    dp = torch.matmul(dY, V.mT)
    e_dp = (D + 8) * U * torch.matmul(dY.abs(), V.abs().mT)
    delta = (p * dp).sum(-1, keepdim=True)
    e_delta = (dY.abs() * e_y).sum(-1, keepdim=True) + (D + 8) * U * (dY.abs() * y.abs()).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    e_ds = p * (e_dp + e_delta) + 2 * e_p * p * (dp - delta).abs()
    merged = lambda t: t.unflatten(1, (Hk, G)).sum(2)
    grad = lambda value, tol: (back(value), back(tol))
    out["dq"] = grad(scale * torch.matmul(ds, K), scale * torch.matmul(e_ds + (w + (Nk + 8) * U) * ds.abs(), K.abs()))
    out["dk"] = grad(scale * merged(torch.matmul(ds.mT, Q)), scale * merged(torch.matmul((e_ds + (w + (N * G + 8) * U) * ds.abs()).mT, Q.abs())))
    out["dv"] = grad(merged(torch.matmul(p.mT, dY)), merged(torch.matmul(((w + 2 * e_p + (N * G + 8) * U) * p).mT, dY.abs())))
    out = {name: (val, tol + (r * val.abs() if name != "y" else 0)) for name, (val, tol) in out.items()}
    if bias is not None:
        both = window[1] != 0
        off = torch.arange(Nk, device=dev)[None, :] - torch.arange(N, device=dev)[:, None]
        table = torch.tensor(PF.relative_buckets(range(-max_distance, max_distance + 1), bias.shape[0], max_distance, both), device=dev)
        bucket = table[off.clamp(-max_distance, max_distance) + max_distance].flatten()
        e_d = (Nk + D + 16) * U * (p * (dp.abs() + torch.matmul(dY.abs(), V.abs().mT))).sum(-1, keepdim=True) + 2 * e_p * (p * dp.abs()).sum(-1, keepdim=True)
        e = p * (e_dp + e_d) + 2 * e_p * p * (dp - delta).abs() + (N + 64) * U * ds.abs()
        sums = lambda t: torch.zeros(bias.shape[0], Hq, dtype=torch.float64, device=dev).index_add_(0, bucket, t.sum(0).flatten(1).t())
        out["dbias"] = (sums(ds), sums(e))
    return out


def check(got, want, what):
    value, tol = want
    got = got.detach().double().reshape(value.shape)
    assert torch.isfinite(got).all(), f"{what}: not finite"
    over = (got - value).abs() - tol
    worst = float(((got - value).abs() / tol.clamp_min(1e-30)).max()) if got.numel() else 0.0
    assert bool((over <= 1e-30).all()), f"{what}: {worst:.3f} of the tolerance"
    return worst
