"""Attention over a window at its edges: rows behind sequences, scores out of the ordinary, means far from zero, scales of the caller's."""
import pytest
import torch

import window_oracle as wo
from gpu_util import announce
from physicsnemo_amd import autograd as PA
from physicsnemo_amd import functional as PF
from test_gpu_window import BF, F32, compare, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("buckets", [0, 8])
@pytest.mark.parametrize("D", [32, 40, 64, 128])
def test_rows_behind_sequences_are_not_read(D, buckets, dtype):
    """NaN or zeros behind sequences whose last tiles are not whole: the same bits.  A NaN that came in would be multiplied by a weight of zero, and the sums
    it spoils formed again row by row, in other roundings."""
    announce("behind", D, buckets, dtype)
    N = 330
    q, k, v, dy, bias = make(4, N, 4, 2, D, dtype, buckets, seed=D)
    lengths = (1, 70, 201, 323)  # behind a tile's first row, behind its first rows, in the middle, short of the buffer's end
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    call = dict(window=(90, 0), sinks=3, lengths=n, bias=bias, max_distance=20)

    def all_of_it(behind):
        ts = [t.clone() for t in (q, k, v, dy)]
        for t in ts:
            for b, m in enumerate(lengths):
                t[b, m:] = behind
        y, stats = PF.window_attention(*ts[:3], return_stats=True, **call)
        grads = PF.window_attention_backward(ts[3], *ts[:3], y, stats, **call)
        first = [max(0, m - 5) for m in lengths]
        newest = torch.stack([q[b, f:f + 5] for b, f in enumerate(first)])
        step = PF.window_attention_step(newest, *ts[1:3], n, left=90, sinks=3, bias=bias, max_distance=20)
        return [t for t in (y, stats, *grads, step) if t is not None]

    for a, b in zip(all_of_it(0.0), all_of_it(float("nan"))):
        assert torch.isfinite(a[a != float("inf")]).all() and torch.equal(a, b)
