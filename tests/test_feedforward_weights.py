"""Which weights the feed-forward modules hand to the kernels: those of the moment of the call, however they were written."""
import pytest
import torch

import physicsnemo_amd as pn

CPU = torch.device("cpu")


@pytest.mark.parametrize("kept", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_gated_mlp_serves_its_present_weights(kept, dtype):
    """Writes through `.data` (averaged weights copied in and out) change neither a parameter's address nor its version."""
    torch.manual_seed(0)
    mlp = pn.GatedMlp(8, 12).to(kept)

    def now():
        return [p.detach().to(dtype if p.ndim == 2 else torch.float32) for p in mlp.parameters_in_order()]

    with torch.no_grad():
        first = [p.clone() for p in mlp._kernel_params(dtype, CPU)]
        assert all(torch.equal(a, b) for a, b in zip(first, now()))
        for p in mlp.parameters():
            p.data.mul_(2)
        second = mlp._kernel_params(dtype, CPU)
        assert all(torch.equal(b, 2 * a) and torch.equal(b, c) for a, b, c in zip(first, second, now()))


def test_a_gated_mlp_holds_no_second_copy_of_its_weights():
    mlp = pn.GatedMlp(8, 12, bias=False)
    with torch.no_grad():
        got = mlp._kernel_params(torch.float32, CPU)
    assert [None if p is None else p.data_ptr() for p in got] == [None if p is None else p.data_ptr() for p in mlp.parameters_in_order()]
    assert not [k for k in vars(mlp) if "cache" in k]
