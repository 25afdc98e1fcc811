"""The feed-forward half of a transformer block beyond Linear, GELU, Linear, as calls that can be timed and checked:

  gated    y = residual + W_down (act(W_gate x + b_gate) * (W_up x + b_up)) + b_down, served and trained
  dropout  y = residual + dropout(x), n = LayerNorm(y), the mask from a counter-based generator and never stored
  int8     a Linear and the gated feed-forward block on 8-bit integers, one scale per token and per output channel

A case is a plain dict; `listed` holds what in use is quoted or costs most, `draw` more of the same ranges.  With `own`
false `run` computes the definitions with elementary tensor operations, with `own` true it calls the library.
"""
import math

import torch

own = False

# ------------------------------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------------------------------


def listed():
    return [
        # one block's feed-forward half on a few hundred points: launches and host time count
        dict(name="gated_small", op="gated", train=False, rows=300, C=128, F=512, act="silu", bias=True, residual=True, dtype="bf16"),
        # a surface of 262 144 points through the usual width, with the block's residual add
        dict(name="gated_serve", op="gated", train=False, rows=262_144, C=256, F=1024, act="gelu", bias=True, residual=True, dtype="bf16"),
        # the wide model's block, hidden width 8/3 C (an odd number) as gated blocks are given to keep their parameter count
        dict(name="gated_wide", op="gated", train=False, rows=100_003, C=512, F=1365, act="silu", bias=False, residual=True, dtype="bf16"),
        # training step of the block's half: all gradients
        dict(name="gated_train", op="gated", train=True, rows=131_072, C=256, F=1024, act="silu", bias=True, residual=False, dtype="bf16"),
        # the same with widths that fill no tile and rows that do not either
        dict(name="gated_train_odd", op="gated", train=True, rows=30_001, C=200, F=533, act="gelu", bias=False, residual=True, dtype="bf16"),
        # float32 training on a regular grid's batch (4 x 85 x 85 points)
        dict(name="gated_train_f32", op="gated", train=True, rows=28_900, C=128, F=512, act="silu", bias=True, residual=False, dtype="f32"),
        # attention output dropped out, added and normalised, trained on a small batch
        dict(name="dropout_small", op="dropout", train=True, rows=2_000, C=256, p=0.1, norm=True, dtype="bf16"),
        # the same on a million points
        dict(name="dropout_million", op="dropout", train=True, rows=1 << 20, C=256, p=0.1, norm=True, dtype="bf16"),
        # float32 rows of an odd width
        dict(name="dropout_odd", op="dropout", train=True, rows=50_003, C=333, p=0.25, norm=True, dtype="f32"),
        # an 8-bit Linear for a handful of points
        dict(name="int8_small", op="int8", gated=False, rows=64, C=256, F=1024, act="gelu", bias=True, dtype="bf16"),
        # the first Linear of the wide model's Mlp in 8 bits, a ragged number of points
        dict(name="int8_linear", op="int8", gated=False, rows=200_003, C=512, F=2048, act="gelu", bias=True, dtype="bf16"),
        # the wide model's gated block served in 8 bits
        dict(name="int8_gated", op="int8", gated=True, rows=131_072, C=512, F=2048, act="silu", bias=True, dtype="bf16"),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_WIDTHS = [32, 64, 96, 128, 200, 256, 257, 384, 512]


def draw(rng):
    op = rng.choice(["gated", "gated", "gated", "dropout", "dropout", "int8"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if op == "gated":
        C, train = rng.choice(_WIDTHS), rng.random() < 0.6
        F = rng.choice([2 * C, 4 * C, 8 * C // 3, _log_uniform(rng, C, 4 * C)])
        most = (3e10 if train else 9e10) / (C * F) / (8 if dtype == "f32" else 1)
        return dict(op=op, train=train, rows=_log_uniform(rng, 100 if train else 1, max(1_000, min(most, 300_000))), C=C, F=F,
                    act=rng.choice(["silu", "silu", "gelu", "relu", "sigmoid", "tanh"]), bias=rng.random() < 0.6,
                    residual=rng.random() < 0.5, dtype=dtype)
    if op == "dropout":
        C = rng.choice(_WIDTHS + [1, 7, 1000, 1024, 2048, _log_uniform(rng, 16, 4096)])
        return dict(op=op, train=rng.random() < 0.6, rows=_log_uniform(rng, 1, max(2, min(1 << 20, (1 << 27) // C))), C=C,
                    p=rng.choice([0.0, 0.05, 0.1, 0.25, 0.5]), norm=rng.random() < 0.7, dtype=dtype)
    gated, C = rng.random() < 0.5, rng.choice(_WIDTHS)
    F = rng.choice([2 * C, 4 * C, 8 * C // 3])
    return dict(op=op, gated=gated, rows=_log_uniform(rng, 1, min(200_000, 1.2e11 / (C * F))), C=C, F=F,
                act=rng.choice(["silu", "gelu", "relu"]), bias=rng.random() < 0.6, dtype="bf16")


def work(case):
    e, M, C = (2 if case["dtype"] == "bf16" else 4), case["rows"], case["C"]
    if case["op"] == "dropout":
        tensors = 2 + 1 + case["norm"]  # x, residual; y and the normalised rows
        if case["train"]:
            tensors += 1 + case["norm"] + 2  # gradients of the outputs; of x and the residual
        return {"bytes": tensors * M * C * e + (4 * C * 4 if case["norm"] else 0), "flops": (4 + 10 * case["norm"]) * M * C}
    F = case["F"]
    if case["op"] == "int8":
        if case["gated"]:
            return {"bytes": 2 * M * C * e + 3 * C * F, "flops": 6 * M * C * F}
        return {"bytes": M * (C + F) * e + C * F, "flops": 2 * M * C * F}
    rows, weights = 2 + case["residual"], 1
    if case["train"]:
        rows, weights = rows + 2 + case["residual"], 2
    return {"bytes": rows * M * C * e + weights * 3 * C * F * e, "flops": (18 if case["train"] else 6) * M * C * F}


# ------------------------------------------------------------------------------------------------------------------
# what a program has in hand
# ------------------------------------------------------------------------------------------------------------------


def _dtype(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float32


def _linear(gen, out_features, in_features, bias, dtype):
    """A Linear's parameters as torch draws them."""
    bound = 1 / math.sqrt(in_features)
    w = (torch.rand(out_features, in_features, generator=gen, device="cuda") * 2 - 1) * bound
    b = (torch.rand(out_features, generator=gen, device="cuda") * 2 - 1) * bound if bias else None
    return w.to(dtype), b


def _codes(w):
    """(8-bit codes, one scale per output channel) of a weight: what a program keeps of it."""
    scale = w.float().abs().amax(1) / 127
    return (w.float() / scale[:, None]).round().clamp(-127, 127).to(torch.int8), scale


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    dtype, M, C = _dtype(case), case["rows"], case["C"]
    rows = lambda n, s=1.0: (torch.randn(M, n, generator=gen, device="cuda") * s).to(dtype)
    st = {"case": case}
    if case["op"] == "dropout":
        st.update(x=rows(C, 0.5), residual=rows(C), rng=torch.tensor([(1_000_003 * seed + 17) % 2 ** 62, 5], device="cuda"),
                  gamma=torch.rand(C, generator=gen, device="cuda") + 0.5,
                  beta=torch.randn(C, generator=gen, device="cuda") * 0.1, dy=rows(C, 0.1), dn=rows(C, 0.1))
        leaves = ["x", "residual"] + (["gamma", "beta"] if case["norm"] else [])
    else:
        F, int8 = case["F"], case["op"] == "int8"
        outs = [("gate", F, C), ("up", F, C), ("down", C, F)] if not int8 or case["gated"] else [("w", F, C)]
        st["x"] = rows(C)  # rows of a LayerNorm
        for name, o, i in outs:
            w, st["b_" + name] = _linear(gen, o, i, case["bias"], torch.float32 if int8 else dtype)
            if int8:
                st["w_" + name], st["s_" + name] = _codes(w)
            else:
                st["w_" + name] = w
        if not int8:
            st["residual"], st["dy"] = rows(C, 2.0) if case["residual"] else None, rows(C, 0.1)
        leaves = ["x"] + (["residual"] if not int8 and case["residual"] else []) + \
                 [k for n, _, _ in outs for k in ("w_" + n, "b_" + n) if st[k] is not None]
    if case.get("train"):
        for k in leaves:
            st[k].requires_grad_(True)
        st["leaves"] = leaves
    return st


# ------------------------------------------------------------------------------------------------------------------
# the definitions in 32 bits
# ------------------------------------------------------------------------------------------------------------------


def _act(name, v):
    """act(v) and its derivative."""
    if name == "relu":
        return v.clamp(min=0), (v > 0).to(v.dtype)
    if name == "gelu":
        phi = 0.5 * (1 + torch.erf(v * math.sqrt(0.5)))
        return v * phi, phi + v * torch.exp(-0.5 * v * v) * (1 / math.sqrt(2 * math.pi))
    if name == "tanh":
        t = torch.tanh(v)
        return t, 1 - t * t
    s = 1 / (1 + torch.exp(-v))
    if name == "sigmoid":
        return s, s * (1 - s)
    return v * s, s * (1 + v * (1 - s))


def _product(x, w, b):
    y = x @ w.t()
    return y if b is None else y + b


def _gated_plain(st):
    case, f = st["case"], (lambda k: None if st[k] is None else st[k].detach().float())
    x, wg, bg, wu, bu, wd, bd = (f(k) for k in ("x", "w_gate", "b_gate", "w_up", "b_up", "w_down", "b_down"))
    g, u = _product(x, wg, bg), _product(x, wu, bu)
    a, slope = _act(case["act"], g)
    h = a * u
    y = _product(h, wd, bd)
    if case["residual"]:
        y = y + f("residual")
    y = y.to(_dtype(case))
    if not case["train"]:
        return y
    dy = st["dy"].float()
    dh = dy @ wd
    dg, du = dh * u * slope, dh * a
    grads = {"x": dg @ wg + du @ wu, "residual": dy, "w_gate": dg.t() @ x, "b_gate": dg.sum(0), "w_up": du.t() @ x,
             "b_up": du.sum(0), "w_down": dy.t() @ h, "b_down": dy.sum(0)}
    return [y] + [grads[k].to(st[k].dtype) for k in st["leaves"]]


_M0, _M1, _W0, _W1, _LOW = 0xD2511F53, 0xCD9E8D57, 0x9E3779B9, 0xBB67AE85, 0xFFFFFFFF


def _philox(c, key):
    """Philox4x32-10 (Salmon et al., 2011) of four counter words, elementwise, in 64-bit arithmetic that wraps."""
    c0, c1, c2, c3 = c
    k0, k1 = key & _LOW, (key >> 32) & _LOW
    for _ in range(10):
        a, b = c0 * _M0, c2 * _M1
        c0, c1, c2, c3 = ((b >> 32) & _LOW) ^ c1 ^ k0, b & _LOW, ((a >> 32) & _LOW) ^ c3 ^ k1, a & _LOW
        k0, k1 = (k0 + _W0) & _LOW, (k1 + _W1) & _LOW
    return c0, c1, c2, c3


def _keep(rng, M, C, p):
    """The mask: element (r, c) is kept where word c % 4 of the block (c // 4, r, r >> 32, offset) under the seed is at least p 2^32."""
    quads = (C + 3) // 4
    r = torch.arange(M, device="cuda")[:, None].expand(M, quads)
    q = torch.arange(quads, device="cuda")[None, :].expand(M, quads)
    words = _philox((q, r & _LOW, r >> 32, (rng[1] & _LOW).expand(M, quads)), rng[0])
    return torch.stack(words, -1).view(M, 4 * quads)[:, :C] >= round(p * 2 ** 32)


_EPS = 1e-5


def _dropout_plain(st):
    case, dtype = st["case"], _dtype(st["case"])
    M, C, p = case["rows"], case["C"], case["p"]
    keep = _keep(st["rng"], M, C, p).float() * (1 / (1 - p))
    s = st["residual"].detach().float() + st["x"].detach().float() * keep
    out = [s.to(dtype)]
    if case["norm"]:
        gamma, beta = st["gamma"].detach(), st["beta"].detach()
        centred = s - s.mean(-1, keepdim=True)
        rstd = torch.rsqrt(centred.square().mean(-1, keepdim=True) + _EPS)
        xh = centred * rstd
        out.append((xh * gamma + beta).to(dtype))
    if case["train"]:
        ds = st["dy"].float()
        if case["norm"]:
            dn = st["dn"].float()
            t = dn * gamma
            ds = ds + rstd * (t - t.mean(-1, keepdim=True) - xh * (t * xh).mean(-1, keepdim=True))
        out += [(ds * keep).to(dtype), ds.to(dtype)]
        if case["norm"]:
            out += [(dn * xh).sum(0), dn.sum(0)]
    return out


def _tokens(x):
    """(whole numbers -127 .. 127, one scale per row) of float32 rows."""
    most = x.abs().amax(1, keepdim=True)
    top = torch.full_like(most, 127)  # a tensor: a number's quotient is formed from its reciprocal, one rounding more
    return (x * torch.where(most > 0, top / most, torch.zeros_like(most))).round(), most / top


def _int8_product(x, codes, scale, bias):
    # sums of whole numbers: exact below 2^24, above it off by 2^-24 of them
    q, s = _tokens(x)
    y = (q @ codes.float().t()) * (s * scale)
    return y if bias is None else y + bias


def _int8_plain(st):
    case, x = st["case"], st["x"].float()
    prod = lambda v, n: _int8_product(v, st["w_" + n], st["s_" + n], st["b_" + n])
    if not case["gated"]:
        return _act(case["act"], prod(x, "w"))[0].to(_dtype(case))
    return prod(_act(case["act"], prod(x, "gate"))[0] * prod(x, "up"), "down").to(_dtype(case))


# ------------------------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------------------------


def _run_own(st):
    from physicsnemo_amd import autograd as PA, functional as PF

    case = st["case"]
    if case["op"] == "int8":
        if not case["gated"]:
            return PF.linear_int8(st["x"], st["w_w"], st["s_w"], st["b_w"], act=case["act"])
        return PF.gated_mlp_int8(st["x"], st["w_gate"], st["s_gate"], st["b_gate"], st["w_up"], st["s_up"], st["b_up"],
                                 st["w_down"], st["s_down"], st["b_down"], act=case["act"])
    if case["op"] == "gated":
        args = [st[k] for k in ("x", "w_gate", "b_gate", "w_up", "b_up", "w_down", "b_down")]
        if not case["train"]:
            return PF.gated_mlp_forward(*args, act=case["act"], residual=st["residual"])
        y = PA.gated_mlp(*args, act=case["act"], residual=st["residual"])
        return [y.detach(), *torch.autograd.grad(y, [st[k] for k in st["leaves"]], st["dy"])]
    norm = (st["gamma"], st["beta"]) if case["norm"] else (None, None)
    if not case["train"]:
        out = PF.dropout_add_norm(st["x"], st["residual"], case["p"], st["rng"], *norm, ln_eps=_EPS)
        return list(out) if case["norm"] else [out]
    out = PA.dropout_add_norm(st["x"], st["residual"], case["p"], st["rng"], *norm, ln_eps=_EPS)
    out, upstream = (list(out), [st["dy"], st["dn"]]) if case["norm"] else ([out], [st["dy"]])
    return [o.detach() for o in out] + list(torch.autograd.grad(out, [st[k] for k in st["leaves"]], upstream))


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return {"gated": _gated_plain, "dropout": _dropout_plain, "int8": _int8_plain}[state["case"]["op"]](state)


# ------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ------------------------------------------------------------------------------------------------------------------


_TORCH_ACT = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu, "relu": torch.relu, "sigmoid": torch.sigmoid,
              "tanh": torch.tanh}


def _mulhilo(a, m):
    """(high, low) 32 bits of a * m for words held in 64-bit integers, from 16-bit halves so that nothing wraps."""
    al, ah, ml, mh = a & 0xFFFF, a >> 16, m & 0xFFFF, m >> 16
    low, mid = al * ml, ah * ml + al * mh  # mid < 2^33
    total = low + ((mid & 0xFFFF) << 16)
    return (ah * mh + (mid >> 16) + (total >> 32)) & _LOW, total & _LOW


def _exact_mask(rng, M, C, p):
    seed, offset = (int(v) & (2 ** 64 - 1) for v in rng.tolist())
    blocks, index = (C + 3) // 4, torch.arange(M * ((C + 3) // 4), device="cuda")
    row = index // blocks
    word = [index % blocks, row & _LOW, row >> 32, torch.full_like(index, offset & _LOW)]
    key = [seed & _LOW, seed >> 32]
    for _ in range(10):
        h0, l0 = _mulhilo(word[0], _M0)
        h1, l1 = _mulhilo(word[2], _M1)
        word = [h1 ^ word[1] ^ key[0], l1, h0 ^ word[3] ^ key[1], l0]
        key = [(key[0] + _W0) & _LOW, (key[1] + _W1) & _LOW]
    kept = torch.empty(M * blocks, 4, dtype=torch.bool, device="cuda")
    for k in range(4):
        kept[:, k] = word[k] >= round(p * 2 ** 32)
    return kept.view(M, -1)[:, :C]


def _exact_int8(x, codes, scale, bias):
    most = x.abs().amax(1, keepdim=True)
    q = torch.where(most > 0, x / (most / 127), torch.zeros_like(x)).round()
    return torch.nn.functional.linear(q * (most / 127), codes.double() * scale.double()[:, None],
                                      None if bias is None else bias.double())


def exact(case, seed):
    st, linear = prepare(case, seed), torch.nn.functional.linear
    d = {k: v.detach().double() for k, v in st.items() if torch.is_tensor(v) and v.is_floating_point()}
    act = _TORCH_ACT.get(case.get("act"))
    train = bool(case.get("train"))
    for k in st.get("leaves", ()):
        d[k].requires_grad_(True)
    with torch.set_grad_enabled(train):
        if case["op"] == "int8":
            prod = lambda v, n: _exact_int8(v, st["w_" + n], st["s_" + n], st["b_" + n])
            if not case["gated"]:
                return act(prod(d["x"], "w"))
            return prod(act(prod(d["x"], "gate")) * prod(d["x"], "up"), "down")
        if case["op"] == "gated":
            hidden = act(linear(d["x"], d["w_gate"], d.get("b_gate"))) * linear(d["x"], d["w_up"], d.get("b_up"))
            y = linear(hidden, d["w_down"], d.get("b_down"))
            outs, upstream = [y + d["residual"] if case["residual"] else y], [d["dy"]]
            if not train:
                return outs[0]
        else:
            kept = _exact_mask(st["rng"], case["rows"], case["C"], case["p"])
            s = d["residual"] + torch.where(kept, d["x"] / (1 - case["p"]), torch.zeros((), dtype=torch.float64, device="cuda"))
            outs, upstream = [s], [d["dy"]]
            if case["norm"]:
                outs.append(torch.nn.functional.layer_norm(s, (case["C"],), d["gamma"], d["beta"], _EPS))
                upstream.append(d["dn"])
            if not train:
                return outs
        return [o.detach() for o in outs] + list(torch.autograd.grad(outs, [d[k] for k in st["leaves"]], upstream))
