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


def test_rows_that_do_not_go_into_a_cache():
    """Refused, and the cache is as it was: rows of one sequence went into the first for all of them."""
    cache = pn.WindowCache(2, 5, 3, 4, torch.float32, "cpu")
    cache.append(torch.ones(2, 1, 3, 4), torch.ones(2, 1, 3, 4))
    good = torch.full((2, 2, 3, 4), 7.0)
    for bad in (good[:1], good[:, :, :1], good[..., :2], good[0], torch.zeros(3, 2, 3, 4)):
        for k, v in ((bad, bad), (good, bad), (bad, good)):
            with pytest.raises(ValueError, match="keys and values"):
                cache.append(k, v)
    assert cache.used == 1 and cache.lengths.tolist() == [1, 1] and not cache.k[:, 1:].any() and not cache.v[:, 1:].any()
    cache.append(good, good)
    assert cache.lengths.tolist() == [3, 3] and bool(cache.k[:, 1:3].eq(7).all())


def test_steps_that_are_refused_leave_the_cache():
    layer = pn.WindowAttention(32, heads=128, dim_head=2, kv_heads=1, window=(9, 0), rotary_base=None, qk_norm=False, bias_buckets=256, max_distance=2048)
    cache = layer.cache(1, 4)
    with pytest.raises(ValueError, match="biases"):
        layer.step(torch.zeros(1, 1, 32), cache)
    assert cache.used == 0 and not cache.lengths.any()


def test_frequencies_of_the_callers_stay():
    """Those that a user sets go along with the layer like its weights."""
    layer = pn.WindowAttention(32, heads=4, dim_head=16)
    own = torch.linspace(0.1, 2.0, 8)[None]
    layer.frequencies = own.clone()
    for _ in (layer.to(torch.bfloat16), layer.half(), layer.double(), layer.cpu()):
        assert layer.frequencies.dtype == torch.float32 and torch.equal(layer.frequencies, own)
    model = torch.nn.Sequential(layer).to(torch.bfloat16)
    assert torch.equal(model[0].frequencies, own)
