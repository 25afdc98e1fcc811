"""Weights that modules keep in the kernels' layout are made again after every optimiser step, also of optimisers that write
parameters without a new version (fused ones), on the CPU."""
import pytest
import torch

import physicsnemo_amd as pn

CPU = torch.device("cpu")


def block():
    return pn.TransolverBlock(4, 64, 0.0, mlp_ratio=2, slice_num=32, use_te=False)


CASES = {
    "mlp": (lambda: pn.Mlp(4, 32, 8), lambda m: m._kernel_params(torch.float32, CPU)),
    "block": (block, lambda m: m._mlp_kernel_params(CPU, torch.float32)),
    "attention": (lambda: block().Attn, lambda m: m.kernel_params(torch.float32, CPU)),
    "flare": (lambda: pn.FLARE(64, heads=4, dim_head=16, n_global_queries=32), lambda m: m.kernel_params(torch.float32, CPU)),
    "context": (lambda: pn.ContextProjector(64, heads=4, dim_head=16, slice_num=32, use_te=False),
                lambda m: m.kernel_params(torch.float32, CPU)),
    "preprocess": (lambda: pn.Transolver(functional_dim=3, out_dim=2, embedding_dim=2, n_layers=1, n_hidden=64, n_head=4, slice_num=32,
                                         use_te=False), lambda m: m._preprocess_params(torch.float32, CPU)),
}


def tensors(params):
    return [t.clone() for t in (params.values() if isinstance(params, dict) else params) if t is not None]


@pytest.mark.parametrize("fused", [False, True])
@pytest.mark.parametrize("name", list(CASES))
def test_an_optimiser_step_is_noticed(name, fused):
    make, kept = CASES[name]
    torch.manual_seed(0)
    module = make()
    optimizer = torch.optim.AdamW(module.parameters(), lr=0.1, fused=fused)
    for _ in range(3):
        with torch.no_grad():
            before = tensors(kept(module))
            assert all(a is b for a, b in zip(list(kept(module)), list(kept(module))))  # kept as long as nothing happens
        for p in module.parameters():
            p.grad = torch.randn_like(p)
        optimizer.step()
        fresh = make()
        fresh.load_state_dict(module.state_dict())
        with torch.no_grad():
            after = tensors(kept(module))
            assert all(torch.equal(a, b) for a, b in zip(after, tensors(kept(fresh))))
            assert not all(torch.equal(a, b) for a, b in zip(before, after))


def test_other_parameters_stay_as_they_are():
    """A captured graph may read what is kept of them."""
    served, trained = block(), block()
    optimizer = torch.optim.AdamW(trained.parameters(), fused=True)
    with torch.no_grad():
        kept = served._mlp_kernel_params(CPU, torch.float32)
    for p in trained.parameters():
        p.grad = torch.randn_like(p)
    optimizer.step()
    with torch.no_grad():
        assert served._mlp_kernel_params(CPU, torch.float32) is kept


def test_optimisers_of_others_count_as_fused():
    class Unseen(torch.optim.Optimizer):
        def __init__(self, params):
            super().__init__(params, {})

        def step(self):
            for group in self.param_groups:
                for p in group["params"]:
                    p.data.mul_(2)

    mlp = pn.Mlp(4, 32, 8)
    optimizer = Unseen(mlp.parameters())
    with torch.no_grad():
        before = tensors(mlp._kernel_params(torch.float32, CPU))
        optimizer.step()
        assert all(torch.equal(b, 2 * a) for a, b in zip(before, mlp._kernel_params(torch.float32, CPU)))
