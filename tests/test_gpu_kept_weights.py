"""Models evaluated between optimiser steps answer with their present weights, whatever the optimiser."""
import copy

import pytest
import torch

import physicsnemo_amd as pn
from gpu_util import announce

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("fused", [False, True])
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("kind", ["transolver", "flare", "geotransolver"])
def test_evaluation_follows_training(kind, int8, fused):
    announce("evaluation between steps", kind, int8, fused)
    torch.manual_seed(0)
    common = dict(functional_dim=3, out_dim=2, n_layers=2, n_hidden=64, n_head=4, mlp_ratio=2, slice_num=32, use_te=False)
    if kind == "geotransolver":
        model = pn.GeoTransolver(include_local_features=False, **common)
    else:
        model = (pn.Transolver if kind == "transolver" else pn.FLAREModel)(embedding_dim=2, **common)
    model = model.to(DEV)
    if int8:
        model.use_int8_mlp()
    optimizer = torch.optim.AdamW([p for p in model.parameters() if p.numel()], lr=0.05, fused=fused)
    fx, emb = torch.randn(2, 70, 3, device=DEV), torch.randn(2, 70, 2, device=DEV)

    def call(m):
        with torch.autocast("cuda", dtype=torch.bfloat16):
            return (m(fx) if kind == "geotransolver" else m(fx, emb)).float()

    outs = []
    for _ in range(3):
        model.train()
        optimizer.zero_grad()
        call(model).square().mean().backward()
        optimizer.step()
        model.eval()
        with torch.no_grad():
            outs.append(call(model))
            fresh = copy.deepcopy(model)
            for m in fresh.modules():  # nothing kept
                for name in ("_kernel_cache", "_mlp_cache", "_kernel_param_cache", "_cache", "_linear_cache", "_preprocess_cache"):
                    if name in m.__dict__:
                        m.__dict__[name] = {}
            assert torch.equal(outs[-1], call(fresh))
    assert not torch.equal(outs[0], outs[1]) and not torch.equal(outs[1], outs[2])
