"""The window attention layer, its blocks and its cache on the GPU: its operators together, as a model runs them.

Values against the layer's formula in float64.  Layers of two projections, norm, rotation and attention: every product rounds its results by r = eps / 2
of the type, and the relative errors of a chain of five of them add up; with the factor 2 for sums in which terms cancel, rel-L2 stays
below 10 r (float32: below 64 r, sums of up to 256 terms)."""
import pytest
import torch

import physicsnemo_amd as pn
import window_oracle as wo
from gpu_util import announce
from test_gpu_rotate import turned

pytestmark = pytest.mark.gpu
BOUND = {torch.bfloat16: 10 * 2.0 ** -8, torch.float32: 64 * 2.0 ** -24}


def formula(layer, x, positions=None, lengths=None):
    """The layer in float64 with autograd."""
    p = {n: t.detach().double().requires_grad_(True) for n, t in layer.named_parameters()}
    B, N, _ = x.shape
    H, Hk, D = layer.heads, layer.kv_heads, layer.dim_head
    qkv = torch.nn.functional.linear(x, p["in_project_qkv.weight"], p["in_project_qkv.bias"]).view(B, N, H + 2 * Hk, D)
    q, k, v = qkv.split([H, Hk, Hk], 2)
    if layer.qk_norm:
        q, k = (t * (t.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * p[w] for t, w in ((q, "q_norm_weight"), (k, "k_norm_weight")))
    if layer.frequencies is not None:
        pos = torch.arange(N, device=x.device) if positions is None else positions
        pos = pos.double().reshape(*((1, N) if pos.shape[0] == N and pos.ndim < 3 and pos.shape != (B, N) else (B, N)), -1)
        angle = (pos[..., None] * layer.frequencies.double()).sum(-2)[:, :, None]
        q, k = turned(q, angle, False), turned(k, angle, False)
    n = torch.full((B,), N, device=x.device) if lengths is None else lengths.long()
    ok = wo.visible(N, N, torch.zeros(B, dtype=torch.long, device=x.device), *layer.window, layer.sinks, n)[:, None]
    q, k, v = q.transpose(1, 2), *(t.transpose(1, 2).repeat_interleave(H // Hk, 1) for t in (k, v))
    s = q @ k.mT * D ** -0.5
    if layer.bias is not None:
        s = s + wo.bias_of(p["bias"], N, N, torch.zeros(B, dtype=torch.long, device=x.device), layer.window[1], layer.max_distance)
    w = torch.softmax(s.masked_fill(~ok, -1e300), -1) * ok
    y = (w @ v).transpose(1, 2).flatten(2)
    return torch.nn.functional.linear(y, p["out_linear.weight"], p["out_linear.bias"]), p


LAYERS = [dict(window=(20, 20)), dict(window=(40, 0), sinks=3, kv_heads=2, bias_buckets=12, max_distance=30), dict(window=(None, None), qk_norm=False),
          dict(window=(15, 30), axes=3, bias_buckets=8, max_distance=20), dict(window=(9, 9), rotary_base=None)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("options", LAYERS)
def test_layer_and_its_gradients(options, dtype):
    announce("layer", options, dtype)
    torch.manual_seed(1)
    layer = pn.WindowAttention(48, heads=4, dim_head=16, **options).cuda()
    if layer.bias is not None:
        torch.nn.init.normal_(layer.bias)
    layer = layer.to(dtype) if dtype == torch.bfloat16 else layer
    layer.frequencies = None if layer.frequencies is None else layer.frequencies.float()
    B, N = 2, 133
    x = torch.randn(B, N, 48, device="cuda").to(dtype)
    positions = torch.rand(B, N, 3, device="cuda") * 10 if options.get("axes") == 3 else None
    lengths = torch.tensor([133, 70], dtype=torch.int32, device="cuda")
    dy = torch.randn(B, N, 48, device="cuda").to(dtype)
    xd = x.double().requires_grad_(True)
    want, p = formula(layer, xd, positions, lengths)
    grads = torch.autograd.grad(want, [xd, *p.values()], dy.double())
    with torch.no_grad():
        served = layer(x, positions, lengths)
    x.requires_grad_(True)
    got = layer(x, positions, lengths)
    own = torch.autograd.grad(got, [x, *layer.parameters()], dy)
    rel = lambda a, b: float((a.double() - b).norm() / b.norm())
    assert rel(served, want.detach()) < BOUND[dtype] and rel(got.detach(), want.detach()) < BOUND[dtype]
    for name, a, b in zip(["x", *p], own, grads):
        if float(b.norm()) > 1e-6 * float(grads[0].norm()):  # the key's bias has no gradient without a norm and a rotation: a score's shift by row
            assert rel(a, b) < 2 * BOUND[dtype], (name, rel(a, b))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_steps_of_a_cache_are_the_layer(dtype):
    """Sequences of their own lengths fed in pieces: a prompt, single points, a few at once; captured and replayed as well."""
    announce("steps", dtype)
    torch.manual_seed(2)
    layer = pn.WindowAttention(64, heads=4, dim_head=32, window=(24, 0), sinks=2, kv_heads=2, bias_buckets=8, max_distance=20).cuda()
    torch.nn.init.normal_(layer.bias)
    layer = layer.to(dtype)
    layer.frequencies = layer.frequencies.float()
    x = torch.randn(3, 60, 64, device="cuda").to(dtype)
    with torch.no_grad():
        whole = layer(x)
        cache = layer.cache(3, 60)
        rows = [layer.step(x[:, a:b], cache) for a, b in ((0, 17), (17, 18), (18, 19), (19, 24), (24, 25))]
        piece = x[:, 25:26].clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):  # outside the cache's count: what it leaves behind is taken back
            before = cache.lengths.clone()
            layer.step(piece, cache)
            cache.reset(before)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = layer.step(piece, cache)
        cache.reset(before)
        for t in range(25, 60):
            piece.copy_(x[:, t:t + 1])
            graph.replay()
            rows.append(out.clone())
    rel = float((torch.cat(rows, 1).double() - whole.double()).norm() / whole.double().norm())
    assert rel < BOUND[dtype], rel
    assert cache.lengths.tolist() == [60] * 3


@pytest.mark.parametrize("autocast", [False, True])
def test_model_with_window_blocks(autocast):
    """Blocks of both kinds in one model: served as trained, and gradients for every parameter of the blocks."""
    announce("model", autocast)
    torch.manual_seed(3)
    model = pn.Transolver(functional_dim=3, out_dim=2, embedding_dim=2, n_layers=3, n_hidden=128, n_head=4, slice_num=16, use_te=False, dropout=0.0,
                          window_blocks=(1, 2), window_options=dict(window=(30, 30), sinks=2, bias_buckets=8, max_distance=20)).cuda()
    fx, emb = torch.randn(2, 500, 3, device="cuda"), torch.randn(2, 500, 2, device="cuda")
    with torch.autocast("cuda", torch.bfloat16, enabled=autocast):
        with torch.no_grad():
            served = model.eval()(fx, emb)
        out = model.train()(fx, emb)
    assert float((served.float() - out.float()).norm() / out.float().norm()) < (4 * BOUND[torch.bfloat16] if autocast else 1e-4)
    out.float().square().mean().backward()
    for name, p in model.blocks[1].named_parameters():
        assert p.grad is not None and torch.isfinite(p.grad).all() and p.grad.any(), name


def test_model_cast_to_bfloat16():
    """Weights cast as a whole: the angles stay float32, the model runs and trains."""
    announce("bf16 model")
    torch.manual_seed(4)
    model = pn.Transolver(functional_dim=3, out_dim=2, embedding_dim=2, n_layers=2, n_hidden=128, n_head=4, slice_num=16, use_te=False, dropout=0.0,
                          window_blocks=(1,), window_options=dict(window=(30, 0), bias_buckets=8, max_distance=20)).cuda().to(torch.bfloat16)
    fx, emb = (torch.randn(2, 300, n, device="cuda", dtype=torch.bfloat16) for n in (3, 2))
    with torch.no_grad():
        assert torch.isfinite(model.eval()(fx, emb)).all()
    model.train()(fx, emb).float().square().mean().backward()
    for name, p in model.blocks[1].named_parameters():
        assert p.grad is not None and torch.isfinite(p.grad).all() and p.grad.any(), name


def test_block_with_counter_dropout_and_structured_points():
    announce("block")
    torch.manual_seed(4)
    block = pn.TransolverBlock(4, 64, 0.2, use_te=False, spatial_shape=(10, 12), window=dict(window=(12, 12))).cuda().use_counter_dropout(7)
    fx = torch.randn(2, 120, 64, device="cuda", requires_grad=True)
    out = block.train()(fx)
    out.sum().backward()
    assert torch.isfinite(fx.grad).all() and fx.grad.any()
    with torch.no_grad():
        a, b = block.eval()(fx), block(fx)
    assert torch.equal(a, b)
