"""Which weights the feed-forward modules hand to the kernels: those of the moment of the call, however they were written."""
import copy
import pickle

import pytest
import torch

import physicsnemo_amd as pn
from physicsnemo_amd import _lib
from physicsnemo_amd import functional as PF
from physicsnemo_amd.feedforward import Int8Mlp

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


class Stream:
    """A stream's part in keeping codes, on the CPU."""

    def __init__(self):
        self.synchronized = 0

    def synchronize(self):
        self.synchronized += 1


@pytest.fixture
def on_cpu(monkeypatch):
    """The library's rounding and torch's streams replaced by stand-ins: what is kept, and what calls do with it."""
    here = type("Here", (), {"stream": Stream(), "capturing": False, "made": 0, "recorded": []})()

    def quantize(w):
        here.made += 1
        scale = w.abs().amax(-1) / 127
        return (w / scale[:, None]).round().to(torch.int8), scale

    monkeypatch.setattr(PF, "quantize_int8", quantize)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: CPU.index)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: here.stream)
    monkeypatch.setattr(_lib, "current_stream_ptr", lambda device: id(here.stream))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: here.capturing)
    monkeypatch.setattr(torch.Tensor, "record_stream", lambda t, stream: here.recorded.append((t.data_ptr(), stream)))
    return here


def test_codes_follow_the_parameters(on_cpu):
    mlp, codes = pn.GatedMlp(8, 12), Int8Mlp()
    lins, of = mlp.linears(), lambda: codes._of(mlp.linears(), CPU)
    first = of()
    assert of() is first and on_cpu.made == 3
    scales = [s.clone() for _, s, _ in first]
    with torch.no_grad():
        lins[0].weight.mul_(2)  # noticed
    assert torch.equal(of()[0][1], 2 * scales[0]) and on_cpu.made == 6
    for lin in lins:
        lin.weight.data.mul_(4)
    codes.refresh()
    assert all(torch.equal(w[1], k * s) for w, s, k in zip(of(), (2 * scales[0], *scales[1:]), (4, 4, 4))) and on_cpu.made == 9
    for k in range(20):  # freed parameters' addresses come again
        lins[2].weight = None
        lins[2].weight = torch.nn.Parameter(torch.full((8, 12), float(k + 1)))
        assert torch.equal(of()[2][1], torch.full((8,), (k + 1) / 127))


def test_codes_are_complete_before_another_stream_reads_them(on_cpu):
    codes, lins = Int8Mlp(), pn.GatedMlp(8, 12).linears()
    first = on_cpu.stream
    weights = codes._of(lins, CPU)
    assert first.synchronized == 1 and not on_cpu.recorded
    on_cpu.stream = other = Stream()
    assert codes._of(lins, CPU) is weights and codes._of(lins, CPU) is weights
    assert sorted(p for p, _ in on_cpu.recorded) == sorted(t.data_ptr() for w in weights for t in w)  # once each
    assert all(s is other for _, s in on_cpu.recorded) and first.synchronized == 1


def test_codes_of_a_capture(on_cpu):
    """Made inside it they lie in the graph's memory, which holds nothing before a replay; made before it they are the graph's as
    long as it may replay."""
    codes, lins = Int8Mlp(), pn.GatedMlp(8, 12).linears()
    on_cpu.capturing = True
    inside = codes._of(lins, CPU)
    assert codes._of(lins, CPU) is not inside and on_cpu.stream.synchronized == 0
    on_cpu.capturing = False
    kept = codes._of(lins, CPU)
    assert kept is not inside and not codes.of_graphs
    on_cpu.capturing = True
    assert codes._of(lins, CPU) is kept and codes._of(lins, CPU) is kept
    assert len(codes.of_graphs) == 1 and codes.of_graphs[0] is kept and not on_cpu.recorded
    on_cpu.capturing = False
    with torch.no_grad():
        lins[0].weight.mul_(2)
    assert codes._of(lins, CPU) is not kept and codes.of_graphs[0] is kept


def test_blocks_keep_what_graphs_read_and_copies_make_their_own(on_cpu):
    block = pn.TransolverBlock(4, 32, 0.0, act="swiglu", use_te=False).use_int8_mlp()
    lins, codes = block.ln_mlp1[1].linears(), block.int8_mlp
    kept = codes._of(lins, CPU)
    on_cpu.capturing = True
    codes._of(lins, CPU)
    on_cpu.capturing = False
    made = on_cpu.made
    assert block.use_int8_mlp().int8_mlp is codes and codes._of(lins, CPU) is not kept and on_cpu.made == made + 3
    twin = copy.deepcopy(block)
    again = pickle.loads(pickle.dumps(codes))
    assert twin.int8_mlp is not codes and not twin.int8_mlp.of_graphs and not again.of_graphs
    assert block.use_int8_mlp(False).int8_mlp is None and block._int8_of_graphs[0] is kept


class Halved(pn.Mlp):
    def forward(self, x):
        return super().forward(x) / 2


class Skipping(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.layers = torch.nn.ModuleList([torch.nn.Linear(32, 64), torch.nn.GELU(), torch.nn.Linear(64, 32)])

    def forward(self, x):
        return x + self.layers[2](self.layers[1](self.layers[0](x)))


@pytest.mark.parametrize("replaced", [Halved(32, 64, 32), Skipping(), torch.nn.Sequential(torch.nn.Linear(32, 32))])
def test_only_the_blocks_own_mlps_run_in_8_bits(replaced):
    """A module that computes something else from three layers keeps its own forward."""
    assert Int8Mlp.linears(replaced) is None
    block = pn.TransolverBlock(4, 32, 0.0, use_te=False)
    assert Int8Mlp.linears(block.ln_mlp1[1])[1] == "gelu"
    block.ln_mlp1[1] = replaced
    with pytest.raises(ValueError, match="not Linear, activation, Linear"):
        block.use_int8_mlp()


def test_counters_do_not_move_inside_a_capture(monkeypatch):
    """The copy to the GPU belongs before the capture: in it the state would be a copy of the graph, set back by every replay."""
    rows = type("Rows", (), {"is_cuda": True, "device": torch.device("cuda", 0)})()
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    drop = pn.CounterDropout(0.5, seed=3)
    with pytest.raises(RuntimeError, match="before the capture"):
        drop._next(rows)
    assert drop.state.tolist() == [3, 0]


@pytest.mark.parametrize("fused", [False, True])
def test_codes_follow_an_optimiser(on_cpu, fused):
    """Fused optimisers write parameters without a new version."""
    mlp, codes = pn.GatedMlp(8, 12), Int8Mlp()
    optimizer = torch.optim.AdamW(mlp.parameters(), lr=0.1, fused=fused)
    for _ in range(3):
        codes._of(mlp.linears(), CPU)
        for p in mlp.parameters():
            p.grad = torch.randn_like(p)
        optimizer.step()
        for (q, s, _), lin in zip(codes._of(mlp.linears(), CPU), mlp.linears()):
            assert torch.equal(s, lin.weight.detach().abs().amax(-1) / 127)
