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
