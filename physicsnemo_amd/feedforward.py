"""Feed-forward parts that blocks take on request: the gated MLP, dropout from a counter-based generator, and the block MLP's
products in 8 bits.  None of them has a counterpart in the reference; a block without them runs as before."""
from __future__ import annotations

from contextlib import contextmanager

import torch
import torch.nn as nn

from . import _lib
from . import autograd as PA
from . import functional as PF
from . import versions

__all__ = ["GatedMlp", "CounterDropout"]

# block activations that make the MLP a gated one, and what they apply to the gate (the preprocess Mlp applies it, too)
GATED_ACTS = {"swiglu": "silu", "geglu": "gelu", "reglu": "relu", "glu": "sigmoid"}

_FUNCTIONS = {"silu": nn.functional.silu, "gelu": nn.functional.gelu, "relu": nn.functional.relu, "sigmoid": torch.sigmoid,
              "tanh": torch.tanh, None: lambda t: t}
_NAMES = {nn.SiLU: "silu", nn.GELU: "gelu", nn.ReLU: "relu", nn.Sigmoid: "sigmoid", nn.Tanh: "tanh"}


def plain_act(act: str) -> str:
    """The activation by name that a plain Mlp beside gated ones uses: a gated name's own, any other name itself."""
    return GATED_ACTS.get(act.lower(), act)


class GatedMlp(nn.Module):
    """y = down(act(gate(x)) * up(x)) [+ residual], three Linears on rows of `features` channels.

    On the GPU in float32 or bfloat16 (also under bf16 autocast) forward and backward are the library's kernels
    (`functional.gated_mlp_forward`, `autograd.gated_mlp`), which keep the hidden layer out of the graph; on the CPU, in other
    types and with hooked or replaced Linears it is tensor ops."""

    def __init__(self, features: int, hidden_features: int, act: str | None = "silu", bias: bool = True):
        super().__init__()
        act = act.lower() if act is not None else None
        if act not in _FUNCTIONS:
            raise KeyError(f"Activation function {act} not found. Available options are: {list(_FUNCTIONS)}")
        self.act = act
        self.gate = nn.Linear(features, hidden_features, bias=bias)
        self.up = nn.Linear(features, hidden_features, bias=bias)
        self.down = nn.Linear(hidden_features, features, bias=bias)

    def extra_repr(self) -> str:
        return f"act={self.act!r}"

    def linears(self):
        return self.gate, self.up, self.down

    def parameters_in_order(self):
        return [p for lin in self.linears() for p in (lin.weight, lin.bias)]

    def _kernel_params(self, dtype: torch.dtype, device: torch.device):
        """The six parameters for the kernels, weights in `dtype` and biases in float32: themselves where they are that, else
        cast for this call.  Nothing is kept: writes through `.data` would leave what is kept behind, unseen."""
        return [None if p is None else p.to(device=device, dtype=dtype if p.ndim == 2 else torch.float32).contiguous()
                for p in self.parameters_in_order()]

    def forward(self, x: torch.Tensor, residual: torch.Tensor | None = None) -> torch.Tensor:
        dtype = PA.compute_dtype(x)
        if not (x.numel() > 0 and PA._linears_served(dtype, *self.linears()) and x.shape[-1] == self.gate.in_features):
            y = self.down(_FUNCTIONS[self.act](self.gate(x)) * self.up(x))
            return y if residual is None else y + residual
        within = residual if residual is not None and residual.shape == x.shape and residual.dtype == dtype else None
        x = x.to(dtype)
        tensors = (x, residual, *self.parameters_in_order())
        if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
            y = PA.gated_mlp(x, *self.parameters_in_order(), act=self.act, residual=within)
        else:
            y = PF.gated_mlp_forward(x.contiguous(), *self._kernel_params(dtype, x.device), act=self.act,
                                     residual=None if within is None else within.contiguous())
        return y if residual is None or within is not None else y + residual


class CounterDropout(nn.Dropout):
    """Dropout whose mask is a function of (seed, offset) and of the element's place (`functional.dropout_add_norm`): it is never
    stored, the backward pass forms it again, and every call takes the next offset, in a captured graph every replay.

    `state` is the int64 pair (seed, next offset); masks come again after 2^32 calls.  It is no entry of the state dict; to go on after a restart with the masks
    that would have come next, save it and set it again.  It moves to the input's device with the first call, which a capture
    refuses.  Processes that train together take different seeds.  Calls of one module run on one stream at a time.  A backward pass that runs the module again (activation checkpointing) would draw
    another mask and is refused."""

    def __init__(self, p: float = 0.5, seed: int = 0, offset: int = 0):
        super().__init__(p)
        self.state = torch.tensor([seed, offset], dtype=torch.int64)
        self._left_out = False

    def extra_repr(self) -> str:
        return f"p={self.p}, counter-based"

    @property
    def active(self) -> bool:
        return self.training and self.p > 0

    def _next(self, x: torch.Tensor) -> torch.Tensor:
        if not x.is_cuda:
            raise RuntimeError("CounterDropout draws on GPU tensors only (no CPU fallback)")
        if torch._C._current_graph_task_id() != -1:
            raise RuntimeError("CounterDropout ran again inside a backward pass, where it would draw another mask")
        if self.state.device != x.device:
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError(f"CounterDropout's state is on {self.state.device}: run the module once on {x.device}, or move "
                                   "its state there, before the capture")
            self.state = self.state.to(x.device)
        return PF.dropout_advance(self.state)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if not self.active or self._left_out:
            return x
        if x.dtype in (torch.float16, torch.float64):
            return self.forward(x.float()).to(x.dtype)
        return PA.dropout_add_norm(x, None, self.p, self._next(x))

    @contextmanager
    def left_out(self):
        """Inside, calls return their argument: the caller applies the dropout itself, with the sum and LayerNorm behind it."""
        self._left_out = True
        try:
            yield
        finally:
            self._left_out = False

    def add_norm(self, x: torch.Tensor, residual: torch.Tensor, ln: nn.LayerNorm):
        """(residual + self(x), ln of it): one kernel where types, shapes and the LayerNorm allow, else one after the other."""
        fused = (self.active and x.is_cuda and x.dtype in (torch.float32, torch.bfloat16) and residual.dtype == x.dtype and
                 residual.shape == x.shape and type(ln) is nn.LayerNorm and ln.elementwise_affine and ln.bias is not None and
                 tuple(ln.normalized_shape) == (x.shape[-1],) and PA.unhooked(self, ln))
        if fused:
            return PA.dropout_add_norm(x, residual, self.p, self._next(x), ln.weight, ln.bias, ln.eps)
        normed, y = PA.layer_norm_residual(self(x) + residual, ln)
        return y, normed


def counter_dropout(attn: nn.Module) -> CounterDropout | None:
    """The layer's output dropout where it is an active `CounterDropout`, which the block then applies itself."""
    drop = getattr(attn, "out_dropout", None)
    return drop if isinstance(drop, CounterDropout) and drop.active and PA.unhooked(drop) else None


class Int8Mlp:
    """8-bit weights of a block's Mlp or GatedMlp, made once per parameter set, and the MLP on them.  A GatedMlp's hidden layer goes
    from float32 to codes; an Mlp is two Linears, between which it is rounded to the rows' type.

    A set is told by its parameters (`versions.stamp`) and holds them, so that no address comes twice.  Writes through `.data` or by
    a replayed graph are not noticed: `refresh` after them.  The codes are complete before the call that makes
    them returns, for streams and captures that use them later; a set that a capture meets unmade is made in the graph, on
    every replay, and not kept; one that a graph reads stays allocated (`of_graphs`).  Copies start without codes."""

    def __init__(self):
        self.of_graphs: list = []  # codes that a captured graph reads
        self._stamp = self._weights = self._held = None
        self._streams: set = set()

    def __reduce__(self):
        return Int8Mlp, ()

    def refresh(self):
        """Round the weights again on the next call."""
        self._stamp = None

    @staticmethod
    def linears(mlp: nn.Module):
        """(Linears, activation's name) of an MLP that runs in 8 bits, or None: hooks, replaced modules, other activations."""
        from .transolver import Mlp  # which imports this file

        if type(mlp) is GatedMlp:
            lins, act, modules = mlp.linears(), mlp.act, (mlp,)
        else:
            if type(mlp) is not Mlp:
                return None
            layers = mlp.layers
            if len(layers) != 3 or type(layers[1]) not in _NAMES or getattr(layers[1], "approximate", "none") != "none":
                return None
            lins, act, modules = (layers[0], layers[2]), _NAMES[type(layers[1])], (mlp, layers, layers[1])
        if not (all(type(lin) is nn.Linear for lin in lins) and PA.unhooked(*modules, *lins)):
            return None
        return lins, act

    def _of(self, lins, device):
        params = [p for lin in lins for p in (lin.weight, lin.bias)]
        stamp = (device,) + versions.stamp(*params)
        if torch.cuda.current_device() != device.index:
            with torch.cuda.device(device):
                return self._of_current_device(lins, device, params, stamp)
        return self._of_current_device(lins, device, params, stamp)

    def _of_current_device(self, lins, device, params, stamp):
        stream, capturing = _lib.current_stream_ptr(device), torch.cuda.is_current_stream_capturing()
        if self._stamp != stamp:
            with torch.no_grad():
                weights = [
                    (*PF.quantize_int8(lin.weight.detach().to(device=device, dtype=torch.float32).contiguous()),
                     None if lin.bias is None else lin.bias.detach().to(device=device, dtype=torch.float32).contiguous().clone())
                    for lin in lins]
            if capturing:
                return weights
            torch.cuda.current_stream(device).synchronize()
            self._weights, self._held, self._streams = weights, [None if p is None else p.detach() for p in params], {stream}
            self._stamp = stamp
        elif capturing:
            if not any(w is self._weights for w in self.of_graphs):
                self.of_graphs.append(self._weights)
        elif stream not in self._streams:  # the codes' memory is not reused before this stream's work on them is done
            for t in (t for w in self._weights for t in w if t is not None):
                t.record_stream(torch.cuda.current_stream(device))
            self._streams.add(stream)
        return self._weights

    def __call__(self, mlp: nn.Module, x: torch.Tensor, residual: torch.Tensor | None) -> torch.Tensor | None:
        """mlp(x) [+ residual], or None where x or the module does not run in 8 bits."""
        found = self.linears(mlp)
        if found is None or not x.is_cuda or x.dtype not in (torch.float32, torch.bfloat16) or x.numel() == 0:
            return None
        lins, act = found
        weights = self._of(lins, x.device)
        x = x.contiguous()
        residual = None if residual is None else residual.contiguous()
        if type(mlp) is GatedMlp:
            return PF.gated_mlp_int8(x, *(t for w in weights for t in w), act=act, residual=residual)
        return PF.linear_int8(PF.linear_int8(x, *weights[0], act=act), *weights[1], residual=residual)
