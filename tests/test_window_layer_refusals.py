"""What the window attention layer, its cache and the models around it refuse beforehand, without a GPU."""
import pytest
import torch

import physicsnemo_amd as pn


def test_blocks_have_no_positions_of_several_axes():
    """Blocks pass none, so that such a model could not run."""
    options = dict(functional_dim=3, out_dim=2, embedding_dim=2, n_layers=2, n_hidden=32, n_head=4, use_te=False)
    with pytest.raises(ValueError, match="axes has to be 1"):
        pn.Transolver(**options, window_blocks=(1,), window_options=dict(axes=2))
    with pytest.raises(ValueError, match="axes has to be 1"):
        pn.TransolverBlock(4, 32, 0.0, use_te=False, spatial_shape=(4, 5), window=dict(axes=2))
    model = pn.Transolver(**options, window_blocks=(1,), window_options=dict(axes=2, rotary_base=None))  # no positions needed
    assert model.blocks[1].Attn.frequencies is None


@pytest.mark.parametrize("options", [dict(sinks=129), dict(sinks=-1), dict(sinks=1.5), dict(sinks=None), dict(dim_head=129), dict(dim_head=0), dict(axes=0), dict(axes=-1),
                                     dict(axes=9, dim_head=32), dict(rotary_base=0.0), dict(rotary_base=-3.0)])
def test_layers_that_no_call_could_run(options):
    with pytest.raises(ValueError):
        pn.WindowAttention(32, **{"heads": 4, "dim_head": 8, **options})
    if "sinks" in options or "axes" in options:
        with pytest.raises(ValueError):
            pn.Transolver(functional_dim=3, out_dim=2, embedding_dim=2, n_layers=2, n_hidden=32, n_head=4, use_te=False, window_blocks=(0,),
                          window_options={k: v for k, v in options.items() if k != "dim_head"})


def test_layers_at_the_limits():
    for options in (dict(sinks=128), dict(sinks=0), dict(dim_head=128), dict(dim_head=1, rotary_base=None), dict(dim_head=16, axes=8), dict(axes=0, rotary_base=None)):
        layer = pn.WindowAttention(32, **{"heads": 4, "dim_head": 8, **options})
        assert layer.frequencies is None or torch.isfinite(layer.frequencies).all()
