"""The gated MLP, counter-based dropout and the 8-bit block MLP where blocks and models use them.

The operators themselves are held against plain formulas in 64 bits in test_gpu_gated.py, test_gpu_dropout.py and
test_gpu_int8.py; here a block or a model has to be exactly the composition of them and of the attention layer (the kernels give
the same bits on every call), and its gradient the slope of what it computes."""
import copy

import pytest
import torch
import torch.utils.checkpoint

import physicsnemo_amd as pn
from physicsnemo_amd import autograd as PA
from physicsnemo_amd import functional as PF
from gpu_util import announce

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.bfloat16, torch.float32]


def gated_params(mlp, dtype):
    return [p.detach().to(dtype if p.ndim == 2 else torch.float32) for p in mlp.parameters_in_order()]


def randomized(module, seed):
    gen = torch.Generator().manual_seed(seed)
    with torch.no_grad():
        for p in module.parameters():
            if p.ndim == 1:
                p.add_((torch.randn(p.shape, generator=gen) * 0.1).to(p))
    return module


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bias", [True, False])
def test_gated_module(dtype, bias):
    announce("gated module", dtype, bias)
    torch.manual_seed(0)
    mlp = pn.GatedMlp(40, 100, "gelu", bias).to(DEV, dtype)
    x, r = torch.randn(2, 7, 40, device=DEV, dtype=dtype), torch.randn(2, 7, 40, device=DEV, dtype=dtype)
    params = [None if p is None else p.detach().to(dtype if p.ndim == 2 else torch.float32) for p in mlp.parameters_in_order()]
    want = PF.gated_mlp_forward(x, *params, act="gelu", residual=r)
    with torch.no_grad():
        assert torch.equal(mlp(x, r), want)
    got = mlp(x, r)
    assert got.grad_fn is not None and torch.equal(got, want)
    strided = torch.randn(40, 7, device=DEV, dtype=dtype).t()
    assert torch.equal(mlp(strided).detach(), PF.gated_mlp_forward(strided.contiguous(), *params, act="gelu"))
    other = torch.float32 if dtype == torch.bfloat16 else torch.bfloat16  # a residual of another type is added afterwards
    want2 = PF.gated_mlp_forward(x, *params, act="gelu") + r.to(other)
    got2 = mlp(x, r.to(other))
    assert got2.dtype == torch.float32 and torch.equal(got2, want2)
    with torch.no_grad():  # cached weights follow an update
        mlp(x)
        mlp.up.weight.mul_(2)
        params[2] = mlp.up.weight.detach().clone()
        assert torch.equal(mlp(x), PF.gated_mlp_forward(x, *params, act="gelu"))
    assert mlp(x[:0]).shape == (0, 7, 40)
    seen = []
    handle = mlp.up.register_forward_hook(lambda *a: seen.append(1))
    mlp(x)
    handle.remove()
    assert seen


def test_gated_module_under_autocast():
    announce("gated module, autocast")
    torch.manual_seed(1)
    mlp = pn.GatedMlp(64, 96).to(DEV)
    x = torch.randn(33, 64, device=DEV, requires_grad=True)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = mlp(x)
    assert y.dtype == torch.bfloat16
    assert torch.equal(y, PF.gated_mlp_forward(x.detach().bfloat16(), *gated_params(mlp, torch.bfloat16)))
    y.sum().backward()
    dx, *grads = PF.gated_mlp_backward(x.detach().bfloat16(), torch.ones_like(y), *gated_params(mlp, torch.bfloat16)[:5])
    assert torch.equal(x.grad, dx.float())
    for p, g in zip(mlp.parameters_in_order(), grads):
        assert torch.equal(p.grad, g.float())
    with torch.autocast("cuda", dtype=torch.float16):  # not a type of the kernels: the Linears themselves
        assert mlp(x).dtype == torch.float16


@pytest.mark.parametrize("dtype", TYPES)
def test_dropout_module(dtype):
    announce("dropout module", dtype)
    torch.manual_seed(2)
    drop, ln = pn.CounterDropout(0.3, seed=11, offset=5), randomized(torch.nn.LayerNorm(48), 3).to(DEV)
    x, r = torch.randn(2, 9, 48, device=DEV, dtype=dtype), torch.randn(2, 9, 48, device=DEV, dtype=dtype)
    rng = lambda offset: torch.tensor([11, offset], device=DEV)
    assert torch.equal(drop(x), PF.dropout_add_norm(x, None, 0.3, rng(5)))
    y, normed = drop.add_norm(x, r, ln)
    want, want_n = PF.dropout_add_norm(x, r, 0.3, rng(6), ln.weight.detach(), ln.bias.detach(), ln.eps)
    assert torch.equal(y, want) and torch.equal(normed, want_n)
    assert drop.state.tolist() == [11, 7]
    # a residual of another type: one after the other
    other = torch.float32 if dtype == torch.bfloat16 else torch.bfloat16
    y, _ = drop.add_norm(x, r.to(other), ln)
    assert torch.equal(y, PF.dropout_add_norm(x, None, 0.3, rng(7)) + r.to(other))
    half = drop(x.half())
    assert half.dtype == torch.float16 and torch.equal(half, PF.dropout_add_norm(x.half().float(), None, 0.3, rng(8)).half())
    assert drop.eval()(x) is x and pn.CounterDropout(0.0)(x) is x and drop.state.tolist() == [11, 9]


def make_block(kind, dtype, p=0.25, act="swiglu"):
    torch.manual_seed(4)
    if kind == "transolver":
        block = pn.TransolverBlock(4, 64, p, act=act, mlp_ratio=2, slice_num=32, use_te=False)
    elif kind == "structured":
        block = pn.TransolverBlock(4, 64, p, act=act, mlp_ratio=2, slice_num=32, spatial_shape=(8, 9), use_te=False)
    elif kind == "flare":
        block = pn.FLAREBlock(4, 64, p, act=act, mlp_ratio=2, n_global_queries=32)
    else:
        block = pn.GALEBlock(4, 64, p, act=act, mlp_ratio=2, slice_num=32)
    return randomized(block, 5).to(DEV, dtype)


def run(block, x):
    return block((x,), None)[0] if isinstance(block, pn.GALEBlock) else block(x)


def attention(block, x):
    """The attention layer of the block without its dropout."""
    keep, block.Attn.out_dropout = block.Attn.out_dropout, torch.nn.Dropout(0.0)
    y = block.Attn((x,), None)[0] if isinstance(block, pn.GALEBlock) else block.Attn(x)
    block.Attn.out_dropout = keep
    return y


def grads_of(y, dy, block, x):
    params = [p for p in block.parameters()]
    return torch.autograd.grad(y, [x] + params, dy, allow_unused=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["transolver", "structured", "flare", "gale"])
def test_block_trains_as_the_composition(kind, dtype):
    announce("block, training", kind, dtype)
    block = make_block(kind, dtype).train()
    assert type(block.Attn.out_dropout) is torch.nn.Dropout
    assert block.use_counter_dropout(9, 100) is block
    gen = torch.Generator().manual_seed(6)
    x = torch.randn(2, 72, 64, generator=gen).to(DEV, dtype).requires_grad_()
    dy = torch.randn(2, 72, 64, generator=gen).to(DEV, dtype)
    y = run(block, x)
    got = grads_of(y, dy, block, x)
    assert block.Attn.out_dropout.state.tolist() == [9, 101]

    normed_in, fx = (PA.layer_norm(x, block.ln_1), x) if kind == "gale" else PA.layer_norm_residual(x, block.ln_1)
    ln, mlp = block.ln_mlp1
    fx1, normed = PA.dropout_add_norm(attention(block, normed_in), fx, 0.25, torch.tensor([9, 100], device=DEV), ln.weight, ln.bias,
                                      ln.eps)
    want = PA.gated_mlp(normed, *mlp.parameters_in_order(), act="silu", residual=fx1)
    assert torch.equal(y, want)
    wanted = grads_of(want, dy, block, x)
    for name, g, w in zip(["x"] + [n for n, _ in block.named_parameters()], got, wanted):
        assert (g is None) == (w is None), name
        assert g is None or torch.equal(g, w), name


@pytest.mark.parametrize("kind", ["transolver", "flare", "gale"])
def test_block_gradient_against_differences(kind):
    """The slope along the gradient from values alone, with the same masks: the float32 block at x +- h d."""
    announce("block, differences", kind)
    block = make_block(kind, torch.float32).train().use_counter_dropout(3)
    gen = torch.Generator().manual_seed(7)
    x, dy = (torch.randn(1, 50, 64, generator=gen).to(DEV) for _ in range(2))

    def values(x):
        block.Attn.out_dropout.state = torch.tensor([3, 0])
        return run(block, x)

    x.requires_grad_()
    grad, = torch.autograd.grad(values(x), x, dy)
    d = grad / grad.abs().mean()
    slope = float((grad.double() * d.double()).sum())
    with torch.no_grad():
        size = float((values(x).double() * dy.double()).abs().sum())
        diff = {h: float(((values(x + h * d).double() - values(x - h * d).double()) * dy.double()).sum()) / (2 * h) for h in (2 ** -8, 2 ** -9)}
    # halving h takes three quarters off a difference's error of second order, so the change between the two bounds what is left;
    # values are good to 64 roundings of 2^-24 of their size, the gradient to as many of its terms
    bound = abs(diff[2 ** -8] - diff[2 ** -9]) + 64 * 2.0 ** -24 * (size * 2 ** 9 + float((grad * d).abs().sum()))
    assert bound < 0.1 * slope
    assert abs(diff[2 ** -9] - slope) <= bound, (diff, slope, bound)


def test_dropout_without_a_gradient_and_in_evaluation():
    announce("block, dropout without gradient")
    block = make_block("transolver", torch.bfloat16).train().use_counter_dropout(1)
    x = torch.randn(2, 60, 64, device=DEV, dtype=torch.bfloat16)
    with torch.no_grad():
        y = block(x)
        ln, mlp = block.ln_mlp1
        fx1, normed = PF.dropout_add_norm(attention(block, block.ln_1(x)), x, 0.25, torch.tensor([1, 0], device=DEV),
                                          ln.weight.detach().float(), ln.bias.detach().float(), ln.eps)
        assert torch.equal(y, PF.gated_mlp_forward(normed, *gated_params(mlp, torch.bfloat16), residual=fx1))
        assert not torch.equal(y, block(x))  # the next mask
        block.eval()
        plain = copy.deepcopy(block)
        plain.Attn.out_dropout = torch.nn.Dropout(0.25).eval()
        assert torch.equal(block(x), plain(x))
    x.requires_grad_()
    assert torch.equal(block(x), plain(x))  # evaluation with gradients: the fused tail either way
    assert block.Attn.out_dropout.state.tolist() == [1, 2]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ["gelu", "relu", "swiglu", "geglu"])
def test_block_serves_in_8_bits(act, dtype):
    announce("block, 8 bits", act, dtype)
    block = make_block("transolver", dtype, act=act).eval().use_int8_mlp()
    x = torch.randn(2, 60, 64, device=DEV, dtype=dtype)
    with torch.no_grad():
        y = block(x)
        ln, mlp = block.ln_mlp1
        fx1, normed = block.Attn.forward_block(block.ln_1(x), x, ln)
        lins = mlp.linears() if act.endswith("glu") else (mlp.layers[0], mlp.layers[2])
        q = [(*PF.quantize_int8(lin.weight.detach().float()), lin.bias.detach().float()) for lin in lins]

        def served(residual):
            if act.endswith("glu"):
                return PF.gated_mlp_int8(normed, *q[0], *q[1], *q[2], act={"swiglu": "silu", "geglu": "gelu"}[act], residual=residual)
            return PF.linear_int8(PF.linear_int8(normed, *q[0], act=act), *q[1], residual=residual)
        assert torch.equal(y, served(fx1))
        out, nxt = block.forward_chain(x, None, block.ln_1)
        want, want_n = PF.residual_layernorm(served(None), residual=fx1, ln_weight=block.ln_1.weight.detach().float(),
                                             ln_bias=block.ln_1.bias.detach().float(), ln_eps=block.ln_1.eps)
        assert torch.equal(out, want) and torch.equal(nxt, want_n)
        lins[-1].weight.mul_(0.5)  # the codes follow the parameters
        assert not torch.equal(block(x), y)
        block.use_int8_mlp(False)
        off = block(x)
        assert not torch.equal(off, y)
    # with gradients the block is what it is without
    x.requires_grad_()
    trained = block(x)
    assert torch.equal(block.use_int8_mlp()(x), trained)


def test_hooks_keep_the_module_in_its_own_types():
    announce("block, 8 bits, hook")
    block = make_block("transolver", torch.bfloat16).eval()
    x, seen = torch.randn(1, 40, 64, device=DEV, dtype=torch.bfloat16), []
    with torch.no_grad():
        plain = block(x)
        block.use_int8_mlp()
        handle = block.ln_mlp1[1].down.register_forward_hook(lambda *a: seen.append(1))
        hooked = block(x)
        assert seen
        handle.remove()
        assert not torch.equal(block(x), hooked)
        block.use_int8_mlp(False)
        assert torch.equal(block(x), plain)


def make_model(kind, act="swiglu", n_hidden=64):
    torch.manual_seed(8)
    if kind == "geotransolver":
        model = pn.GeoTransolver(functional_dim=3, out_dim=2, n_layers=2, n_hidden=n_hidden, n_head=4, dropout=0.2, act=act, mlp_ratio=2,
                                 slice_num=32, use_te=False, include_local_features=False)
    else:
        cls = pn.Transolver if kind == "transolver" else pn.FLAREModel
        model = cls(functional_dim=3, out_dim=2, embedding_dim=2, n_layers=2, n_hidden=n_hidden, n_head=4, dropout=0.2, act=act,
                    mlp_ratio=2, slice_num=32, use_te=False)
    return randomized(model, 9)


def call(model, fx, emb):
    return model(fx) if isinstance(model, pn.GeoTransolver) else model(fx, emb)


@pytest.mark.parametrize("kind", ["transolver", "flare", "geotransolver"])
def test_models_train_and_serve(kind):
    """A step with counter-based dropout and gated MLPs, repeatable from the saved counters, and then the model in 8 bits."""
    announce("model", kind)
    model = make_model(kind).to(DEV).train().use_counter_dropout(21)
    fx, emb = torch.randn(2, 70, 3, device=DEV), torch.randn(2, 70, 2, device=DEV)

    def step():
        model.zero_grad()
        with torch.autocast("cuda", dtype=torch.bfloat16):
            y = call(model, fx, emb)
        y.float().square().sum().backward()
        return [y.detach()] + [p.grad.clone() for p in model.parameters() if p.grad is not None]

    first, second = step(), step()
    assert all(bool(torch.isfinite(t).all()) for t in first)
    assert not torch.equal(first[0], second[0])
    assert [b.Attn.out_dropout.state.tolist() for b in model.blocks] == [[21, 2], [21 + (1 << 32), 2]]
    ones = torch.ones(64, 64, device=DEV)
    masks = [PF.dropout_add_norm(ones, None, 0.5, b.Attn.out_dropout.state) for b in model.blocks]
    assert 0.4 < float((masks[0] == masks[1]).float().mean()) < 0.6  # 4 096 fair coins: 0.5 within 0.1 by 12 of their deviations
    for b in model.blocks:
        b.Attn.out_dropout.state = b.Attn.out_dropout.state - torch.tensor([0, 2], device=DEV)
    again = step()
    assert len(again) == len(first) and all(torch.equal(a, b) for a, b in zip(again, first))
    model.eval()
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
        plain = call(model, fx, emb)
        served = call(model.use_int8_mlp(), fx, emb)
        assert not torch.equal(plain, served) and bool(torch.isfinite(served).all())
        assert torch.equal(call(model, fx, emb), served)
        assert torch.equal(call(model.use_int8_mlp(False), fx, emb), plain)


@pytest.mark.parametrize("act", ["swiglu", "geglu", "reglu", "glu"])
@pytest.mark.parametrize("kind", ["transolver", "flare", "geotransolver"])
def test_models_of_gated_blocks_are_their_tensor_ops(kind, act):
    """In float32, against the same model with hooks on its gated MLPs, which then run as tensor ops: within the 1e-4 that float32
    models are held to everywhere."""
    announce("model, gated", kind, act)
    model = make_model(kind, act).to(DEV).eval()
    fx, emb = torch.randn(2, 70, 3, device=DEV), torch.randn(2, 70, 2, device=DEV)
    with torch.no_grad():
        y, seen = call(model, fx, emb), []
        for b in model.blocks:
            b.ln_mlp1[1].gate.register_forward_hook(lambda *a: seen.append(1))
        want = call(model, fx, emb)
    assert len(seen) == len(model.blocks)
    assert float((y - want).norm()) <= 1e-4 * float(want.norm())


def test_a_captured_training_step_draws_new_masks():
    """Forward and backward of a block in a graph: every replay is the eager step of the same counter, bit for bit."""
    announce("block, captured training step")
    block = make_block("transolver", torch.bfloat16).train().use_counter_dropout(17)
    x = torch.randn(2, 64, 64, device=DEV, dtype=torch.bfloat16)
    dy = torch.randn_like(x)
    params = list(block.parameters())

    def step():
        y = block(x)
        return [y.detach(), *torch.autograd.grad(y, params, dy)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    state = block.Attn.out_dropout.state
    seen = []
    for offset in (40, 41, 42, 40):
        state.copy_(torch.tensor([17, offset]))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        assert state.tolist() == [17, offset + 1]
        state.copy_(torch.tensor([17, offset]))
        want = step()
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert torch.equal(g, w)
        seen.append(got[0])
        del want
    assert torch.equal(seen[0], seen[3]) and not torch.equal(seen[0], seen[1]) and not torch.equal(seen[1], seen[2])


def test_a_graph_serves_in_8_bits():
    announce("model, graph, 8 bits")
    model = make_model("transolver").to(DEV).eval().use_int8_mlp()

    def fwd(fx, emb):
        with torch.autocast("cuda", dtype=torch.bfloat16):
            return model(fx, emb)

    inputs = [(torch.randn(1, 300, 3, device=DEV), torch.randn(1, 300, 2, device=DEV)) for _ in range(3)]
    graphed = pn.GraphedForward(fwd, *inputs[0])
    with torch.no_grad():
        for fx, emb in inputs + inputs[:1]:
            got = graphed(fx, emb).clone()
            torch.cuda.synchronize()
            want = fwd(fx, emb)
            torch.cuda.synchronize()
            assert torch.equal(got, want)


def test_running_again_inside_a_backward_pass_is_refused():
    announce("block, recomputation")
    block = make_block("transolver", torch.float32).train().use_counter_dropout(2)
    x = torch.randn(1, 40, 64, device=DEV, requires_grad=True)
    y = torch.utils.checkpoint.checkpoint(block, x, use_reentrant=False)
    with pytest.raises(RuntimeError, match="another mask"):
        y.sum().backward()


@pytest.mark.parametrize("C,rows,tail", [(512, 4_300_000, 300_000), (256, 275 * 32_768, 32_768)])
def test_elements_past_32_bits(C, rows, tail):
    """The last rows of a call of more than 2^31 elements are those of a call of their own (of so many rows that the same kernels
    take them: every element is summed in the same order)."""
    announce("elements past 32 bits", C, rows)
    torch.manual_seed(10)
    F, dtype = 64, torch.bfloat16
    params = [torch.randn(F, C, device=DEV).to(dtype) / 16, torch.randn(F, device=DEV), torch.randn(F, C, device=DEV).to(dtype) / 16,
              torch.randn(F, device=DEV), torch.randn(C, F, device=DEV).to(dtype) / 8, torch.randn(C, device=DEV)]
    x = torch.empty(rows, C, device=DEV, dtype=dtype).normal_()
    last = x[-tail:].clone()
    y = PF.gated_mlp_forward(x, *params, residual=x)[-tail:].clone()
    assert torch.equal(y, PF.gated_mlp_forward(last, *params, residual=last))
    dx = PF.gated_mlp_backward(x, x, *params[:5], wanted=(True,) + (False,) * 6)[0][-tail:].clone()
    assert torch.equal(dx, PF.gated_mlp_backward(last, last, *params[:5], wanted=(True,) + (False,) * 6)[0])
    q = [t for k in (0, 2, 4) for t in (*PF.quantize_int8(params[k]), params[k + 1])]
    y = PF.gated_mlp_int8(x, *q, residual=x)[-tail:].clone()
    assert torch.equal(y, PF.gated_mlp_int8(last, *q, residual=last))
    del y, dx
    gamma, rng = torch.ones(C, device=DEV), torch.tensor([1, 2], device=DEV)
    _, n = PF.dropout_add_norm(x, x, 0.0, rng, gamma, gamma)
    assert torch.equal(n[-tail:], PF.dropout_add_norm(last, last, 0.0, rng, gamma, gamma)[1])
