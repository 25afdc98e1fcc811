"""The window attention layer in float16, which it computes as float32, and what a served block does around it."""
import pytest
import torch

import physicsnemo_amd as pn
from gpu_util import announce

pytestmark = pytest.mark.gpu
HALF = 2.0 ** -11


def model(blocks, **options):
    torch.manual_seed(3)
    return pn.Transolver(functional_dim=3, out_dim=2, embedding_dim=2, n_layers=3, n_hidden=64, n_head=4, slice_num=16, use_te=False, dropout=0.0,
                         window_blocks=blocks, window_options=dict(window=(30, 30), sinks=2, bias_buckets=8, max_distance=20), **options).cuda()


def rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


@pytest.mark.parametrize("blocks", [(0,), (0, 1, 2), (1,), (2,)])
def test_model_under_float16_autocast(blocks):
    """Served, also where the first block attends over a window, and as it is trained.  Against float32: every Linear of the way (preprocess 2, six in the
    blocks' MLPs, head) rounds its inputs and its result by 2^-11, nine of them, each once more for what comes from the one before."""
    announce("float16 autocast", blocks)
    net = model(blocks)
    fx, emb = (torch.randn(2, 300, n, device="cuda") for n in (3, 2))
    with torch.no_grad():
        want = net.eval()(fx, emb)
        with torch.autocast("cuda", torch.float16):
            served = net(fx, emb)
    with torch.autocast("cuda", torch.float16):
        trained = net.train()(fx, emb)
    assert rel(served, want) < 18 * HALF and rel(trained.detach(), want) < 18 * HALF
    trained.float().square().mean().backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in net.blocks.parameters())


def test_the_sum_with_the_residual_is_not_rounded():
    """float16 autocast: a float32 residual meets the layer's float32 result."""
    announce("residual")
    block = model((0,)).blocks[0].eval()
    x, residual = (torch.randn(2, 100, 64, device="cuda") for _ in range(2))
    with torch.no_grad():
        want = block.Attn.forward_block(x, residual, block.ln_mlp1[0])
        with torch.autocast("cuda", torch.float16):
            got = block.Attn.forward_block(x, residual, block.ln_mlp1[0])
            of_half = block.Attn.forward_block(x, residual.half(), block.ln_mlp1[0])
    assert all(a.dtype == torch.float32 and torch.equal(a, b) for a, b in zip(got, want))
    assert all(a.dtype == torch.float32 and rel(a, b) < 2 * HALF for a, b in zip(of_half, want))


@pytest.mark.parametrize("half", [False, True])
def test_hooks_of_the_layer(half):
    """They observe and change the layer's result in a served block as in a trained one."""
    announce("hooks", half)
    block = pn.TransolverBlock(4, 64, 0.0, use_te=False, window=dict(window=(12, 12))).cuda()
    fx, seen = torch.randn(2, 120, 64, device="cuda"), []
    def run():
        with torch.autocast("cuda", torch.float16, enabled=half):
            return block(fx)
    with torch.no_grad():
        plain = block.eval() and run()
        first = block.Attn.register_forward_hook(lambda m, i, o: seen.append(o.shape))
        assert torch.equal(run(), plain) and len(seen) == 1
        first.remove()
        block.Attn.register_forward_hook(lambda m, i, o: o * 0)
        block.Attn.register_forward_pre_hook(lambda m, i: seen.append(i[0].shape))
        served = run()
    trained = block.train()(fx) if not half else run()
    without = fx + block.ln_mlp1[1](block.ln_mlp1[0](fx))
    assert len(seen) == 3 and rel(served, without) < (18 * HALF if half else 1e-5) and rel(trained.detach(), without.detach()) < (18 * HALF if half else 1e-5)


@pytest.mark.parametrize("dim,heads,dim_head", [(48, 4, 16), (640, 4, 160 // 2), (64, 9, 64)])
@pytest.mark.parametrize("autocast", [False, True])
def test_layers_in_float16(autocast, dim, heads, dim_head):
    """Cast as a whole and given float16, or under autocast: float32 inside, results and gradients rounded once, by 2^-11 at most.  Layers of more
    inputs than the row kernels hold, too.  Float32 sums of up to 640 terms: 2 x 640 u on either side's results, which the bound leaves room for."""
    announce("float16", autocast, dim, heads, dim_head)
    torch.manual_seed(5)
    layer = pn.WindowAttention(dim, heads=heads, dim_head=dim_head, window=(20, 9), sinks=1, bias_buckets=8, max_distance=20).cuda()
    torch.nn.init.normal_(layer.bias)
    with torch.no_grad():
        for p in layer.parameters():
            p.copy_(p.half().float())
    x, dy = (torch.randn(2, 90, dim, device="cuda").half() for _ in range(2))
    lengths = torch.tensor([90, 41], dtype=torch.int32, device="cuda")

    def run(layer, x, **kw):
        with torch.no_grad():
            served = layer(x, **kw)
        x = x.detach().requires_grad_(True)
        out = layer(x, **kw)
        grads = torch.autograd.grad(out, [x, *layer.parameters()], dy.to(out.dtype))
        return served, out.detach(), grads
    want = run(layer, x.float(), lengths=lengths)
    if autocast:
        with torch.autocast("cuda", torch.float16):
            got = run(layer, x.float(), lengths=lengths)
    else:
        got = run(layer.half(), x, lengths=lengths)
    assert got[0].dtype == got[1].dtype == torch.float16
    assert rel(got[0], want[0]) < 1.5 * HALF and rel(got[1], want[1]) < 1.5 * HALF
    for (name, _), a, b in zip([("x", None), *layer.named_parameters()], got[2], want[2]):
        assert a.dtype == (torch.float32 if autocast else torch.float16) and rel(a, b) < 1.5 * HALF, (name, rel(a, b))


@pytest.mark.parametrize("autocast", [False, True])
def test_steps_in_float16(autocast):
    """A cache of float32, the rows of the whole layer, rounded once (float32 sums in another order: 2^-18 beside 2^-11)."""
    announce("float16 steps", autocast)
    torch.manual_seed(6)
    layer = pn.WindowAttention(64, heads=4, dim_head=32, window=(24, 0), sinks=2, kv_heads=2, bias_buckets=8, max_distance=20).cuda()
    torch.nn.init.normal_(layer.bias)
    layer = layer if autocast else layer.half()
    x = torch.randn(3, 40, 64, device="cuda")
    x = x if autocast else x.half()
    with torch.no_grad(), torch.autocast("cuda", torch.float16, enabled=autocast):
        whole, cache = layer(x), layer.cache(3, 40)
        rows = [layer.step(x[:, a:b], cache) for a, b in ((0, 17), (17, 18), (18, 18), (18, 19), (19, 40))]
    assert cache.k.dtype == torch.float32 and cache.lengths.tolist() == [40] * 3 and cache.used == 40
    assert all(r.dtype == torch.float16 for r in rows) and rel(torch.cat(rows, 1), whole) < HALF + 2.0 ** -18
    assert layer.cache(1, 1, torch.float16).k.dtype == torch.float32 and layer.cache(1, 1, torch.bfloat16).k.dtype == torch.bfloat16


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32, torch.bfloat16])
def test_steps_of_nothing(dtype):
    """No sequences or no new points: empty results, a cache as it was."""
    announce("nothing", dtype)
    layer = pn.WindowAttention(64, heads=4, dim_head=32, window=(24, 0)).cuda().to(dtype)
    for batch, points in ((0, 3), (2, 0), (0, 0)):
        cache = layer.cache(batch, 5)
        y = layer.step(torch.zeros(batch, points, 64, device="cuda", dtype=dtype), cache)
        assert y.shape == (batch, points, 64) and y.dtype == dtype and cache.used == 0 and not cache.lengths.any()


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32, torch.bfloat16])
def test_served_blocks_of_nothing(dtype):
    """The layer's part of a block without points, and a model on a grid without samples under float16 autocast, as with slices."""
    announce("block of nothing", dtype)
    block = pn.TransolverBlock(4, 64, 0.0, use_te=False, window=dict(window=(5, 5))).cuda().eval()
    x = torch.zeros(2, 0, 64, device="cuda", dtype=dtype)
    with torch.no_grad():
        for got in (*block.Attn.forward_block(x, x, block.ln_mlp1[0]), block.Attn.forward_block(x, x, None)):
            assert got.shape == x.shape and got.dtype == (torch.float32 if dtype == torch.float16 else dtype)
    for blocks in ((), (0, 2)):
        torch.manual_seed(1)
        net = pn.Transolver(functional_dim=3, out_dim=2, embedding_dim=2, n_layers=3, n_hidden=64, n_head=4, slice_num=16, use_te=False, structured_shape=(6, 7),
                            window_blocks=blocks, window_options=dict(window=(5, 5)) if blocks else None).cuda().eval()
        with torch.no_grad(), torch.autocast("cuda", torch.float16):
            assert net(torch.zeros(0, 42, 3, device="cuda"), torch.zeros(0, 42, 2, device="cuda")).shape == (0, 42, 2)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32, torch.bfloat16])
def test_projections_without_a_bias(dtype):
    """A layer whose Linears were exchanged for such serves as it trains."""
    announce("no biases", dtype)
    torch.manual_seed(7)
    layer = pn.WindowAttention(32, heads=4, dim_head=8, window=(9, 9))
    layer.in_project_qkv, layer.out_linear = torch.nn.Linear(32, 96, bias=False), torch.nn.Linear(32, 32, bias=False)
    layer, x = layer.cuda().to(dtype), torch.randn(2, 50, 32, device="cuda").to(dtype)
    with torch.no_grad():
        served = layer(x)
    trained = layer(x)
    assert trained.requires_grad and rel(served, trained.detach()) < 8 * torch.finfo(dtype).eps  # two products' roundings, and what they do to a softmax
