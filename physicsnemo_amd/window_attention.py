"""Attention of points over their neighbours in an order of the points: rows of a mesh file, a space-filling curve, a grid's rows, time steps.
Beside the slice attention, which every point shares with all others through a few tokens, it keeps what is near apart.  It has no
counterpart among the reference's attention layers; `Transolver(window_blocks=...)` puts it in the blocks that are named."""
from __future__ import annotations

import torch
import torch.nn as nn

from . import autograd as PA
from . import functional as PF

__all__ = ["WindowAttention", "WindowCache"]


class WindowCache:
    """Keys and values of `batch` sequences of up to `capacity` points that `WindowAttention.step` adds to, and how many points each holds
    (`lengths`, int32 on the device)."""

    def __init__(self, batch: int, capacity: int, heads: int, dim_head: int, dtype: torch.dtype, device):
        self.k = torch.zeros(batch, capacity, heads, dim_head, dtype=dtype, device=device)
        self.v = torch.zeros_like(self.k)
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=device)
        self.used = 0  # points added so far, as the host knows it: replays of a captured step are not counted

    @property
    def capacity(self) -> int:
        return self.k.shape[1]

    def reset(self, lengths: torch.Tensor | None = None) -> None:
        """Empties the cache, or sets how many of each sequence's points (from the first on) go on counting."""
        if lengths is None:
            self.lengths.zero_()
            self.used = 0
        else:
            if lengths.shape != self.lengths.shape:
                raise ValueError(f"lengths have to be of shape {tuple(self.lengths.shape)}, got {tuple(lengths.shape)}")
            low, high = (int(n) for n in lengths.aminmax()) if lengths.numel() else (0, 0)
            if low < 0 or high > self.capacity:
                raise ValueError(f"lengths have to be between 0 and {self.capacity}, got {low} to {high}")
            self.lengths.copy_(lengths)
            self.used = high

    def append(self, k: torch.Tensor, v: torch.Tensor) -> None:
        """k, v (B, T, heads, dim_head) behind what each sequence holds."""
        batch, _, heads, channels = self.k.shape
        T = k.shape[1] if k.ndim == 4 else 0
        if k.shape != v.shape or k.shape != (batch, T, heads, channels):
            raise ValueError(f"keys and values have to be {(batch, 'T', heads, channels)}, got {tuple(k.shape)} and {tuple(v.shape)}")
        if self.used + T > self.capacity:
            raise ValueError(f"the cache holds {self.used} of {self.capacity} points: no room for {T} more")
        rows = self.lengths[:, None].long() + torch.arange(T, device=k.device)
        rows = rows.clamp_(max=self.capacity - 1)  # replays past the capacity write the last row again and nothing outside
        which = torch.arange(k.shape[0], device=k.device)[:, None]
        self.k.index_put_((which, rows), k.to(self.k.dtype))
        self.v.index_put_((which, rows), v.to(self.v.dtype))
        self.lengths.add_(T).clamp_(max=self.capacity)
        self.used += T


class WindowAttention(nn.Module):
    """y = out_linear(attention of q, k, v = in_project_qkv(x) over the window), x (B, N, dim) in the order of the points.

    A point sees those from `window[0]` before it to `window[1]` behind it (None: no bound) and the first `sinks` points.  `kv_heads` key
    and value heads serve `heads` query heads.  Queries and keys are normalised per head (`qk_norm`) and, with a `rotary_base`, turned by
    their positions: by default their places in the order, else what `forward` is given, `axes` numbers a point, to each of which an equal share
    of the channel pairs belongs.  `bias_buckets` adds a learned bias by distance (`functional.relative_buckets`).  float32 and bfloat16 on the
    GPU, bf16 autocast as for the other layers, float16 as float32.  The output dropout is the blocks' (`out_dropout`)."""

    fp8_weights = False

    def __init__(self, dim: int, heads: int = 8, dim_head: int = 64, dropout: float = 0.0, window=(128, 128), sinks: int = 0,
                 kv_heads: int | None = None, qk_norm: bool = True, rotary_base: float | None = 10_000.0, axes: int = 1,
                 bias_buckets: int = 0, max_distance: int = 128):
        super().__init__()
        kv_heads = heads if kv_heads is None else kv_heads
        if kv_heads < 1 or heads % kv_heads:
            raise ValueError(f"heads have to be a multiple of kv_heads, got {heads} and {kv_heads}")
        self.window = tuple(window)
        if len(self.window) != 2:
            raise ValueError(f"window has to be (back, ahead), got {window!r}")
        for reach, what in zip(self.window, ("reach back", "reach ahead")):
            PF._bound(reach, f"the window's {what}")
        limits = PF._SEQ_LIMITS
        if not 1 <= dim_head <= limits["D"]:
            raise ValueError(f"heads of 1 to {limits['D']} channels are served, got {dim_head}")
        if PF._bound(sinks, "the number of first points") not in range(limits["sinks"] + 1):
            raise ValueError(f"0 to {limits['sinks']} first points can stay visible, got {sinks}")
        if rotary_base is not None and (rotary_base <= 0 or axes not in range(1, limits["axes"] + 1)):
            raise ValueError(f"a rotation has a positive base and one to {limits['axes']} axes, got {rotary_base} and {axes}")
        self.heads, self.kv_heads, self.dim_head, self.sinks, self.axes, self.max_distance = heads, kv_heads, dim_head, sinks, axes, max_distance
        if bias_buckets:
            PF.relative_buckets((), bias_buckets, max_distance, both=self.window[1] != 0)
        self.in_project_qkv = nn.Linear(dim, (heads + 2 * kv_heads) * dim_head)
        self.out_linear = nn.Linear(heads * dim_head, dim)
        self.out_dropout = nn.Dropout(dropout)
        self.qk_norm = qk_norm
        if qk_norm:
            self.q_norm_weight = nn.Parameter(torch.ones(dim_head))
            self.k_norm_weight = nn.Parameter(torch.ones(dim_head))
        self.bias = nn.Parameter(torch.zeros(bias_buckets, heads)) if bias_buckets else None
        self.rotary_base = rotary_base
        if rotary_base is not None and dim_head // 2 < axes:
            raise ValueError(f"{dim_head} channels a head have {dim_head // 2} pairs, too few for {axes} axes")
        self.register_buffer("frequencies", None if rotary_base is None else self._frequencies(), persistent=False)

    def _frequencies(self) -> torch.Tensor:
        each = self.dim_head // 2 // self.axes
        frequencies = torch.zeros(self.axes, each * self.axes)
        for a in range(self.axes):
            frequencies[a, a * each:(a + 1) * each] = float(self.rotary_base) ** (-torch.arange(each, dtype=torch.float64) / each)
        return frequencies

    def _apply(self, fn, recurse=True):
        own = self.frequencies
        super()._apply(fn, recurse)
        if own is not None:  # float32 whatever type the weights are cast to; on the meta device they have no values to keep
            self.frequencies = (self._frequencies() if own.is_meta else own).to(self.frequencies.device)
        return self

    def extra_repr(self) -> str:
        return f"heads={self.heads}, kv_heads={self.kv_heads}, window={self.window}, sinks={self.sinks}"

    def use_fp8_weights(self, enabled: bool = True):
        if enabled:
            raise ValueError("fp8 weights are for the slice attention layers")
        return self

    def _needs_grad(self, x: torch.Tensor) -> bool:
        return torch.is_grad_enabled() and (x.requires_grad or any(p.requires_grad for p in self.parameters()))

    def _projected(self, lin: nn.Linear, x: torch.Tensor, needs_grad: bool) -> torch.Tensor:
        if (x.dtype == torch.float32 and type(lin) is nn.Linear and lin.weight.dtype == torch.float16 and PA.unhooked(lin) and
                not torch.is_autocast_enabled("cuda")):  # weights of a float16 layer, which is computed in float32
            if needs_grad or lin.in_features > 512:
                return nn.functional.linear(x, lin.weight.float(), None if lin.bias is None else lin.bias.float())
        if needs_grad:
            return PA.linear_as_autocast(x, lin)
        if x.dtype in (torch.float32, torch.bfloat16) and type(lin) is nn.Linear and lin.in_features <= 512 and PA.unhooked(lin):
            bias = lin.weight.new_zeros(lin.out_features, dtype=torch.float32) if lin.bias is None else lin.bias.float().contiguous()
            return PF.linear(x, lin.weight.to(x.dtype).contiguous(), bias)
        return lin(x).to(x.dtype)

    def _qkv(self, x: torch.Tensor, positions, needs_grad: bool):
        """(q, k, v) as the attention takes them."""
        B, N, _ = x.shape
        H, Hk, D = self.heads, self.kv_heads, self.dim_head
        qkv = self._projected(self.in_project_qkv, x, needs_grad).view(B, N, H + 2 * Hk, D)
        q, k, v = qkv[:, :, :H], qkv[:, :, H:H + Hk], qkv[:, :, H + Hk:]
        if self.qk_norm or self.frequencies is not None:
            weights = (self.q_norm_weight, self.k_norm_weight) if self.qk_norm else (None, None)
            if not needs_grad:
                weights = tuple(None if w is None else w.detach().float().contiguous() for w in weights)
            turn = PA.norm_rotate if needs_grad else PF.norm_rotate
            rotary = (positions, self.frequencies) if self.frequencies is not None else (None, None)
            q, k = turn(q, k, *weights, *rotary, norm=self.qk_norm)
        return q, k, v

    def _positions(self, x: torch.Tensor, positions):
        if self.frequencies is None:
            if positions is not None:
                raise ValueError("positions are for a layer with rotary_base")
            return None
        if positions is None:
            if self.axes != 1:
                raise ValueError(f"positions of {self.axes} numbers a point are needed")
            return torch.arange(x.shape[1], device=x.device)
        if positions.dtype not in (torch.int32, torch.int64):
            positions = positions.float()
        return positions.to(x.device).contiguous()

    def _prepared(self, x: torch.Tensor) -> torch.Tensor:
        if x.ndim != 3:
            raise ValueError(f"Expected 3D input tensor (B, N, C), got {x.ndim}D tensor with shape {tuple(x.shape)}")
        if not x.is_cuda:
            raise RuntimeError("physicsnemo_amd runs on GPU tensors only (there is no CPU path)")
        if torch.is_autocast_enabled("cuda") and torch.get_autocast_dtype("cuda") == torch.bfloat16:
            x = x.to(torch.bfloat16)
        return x.contiguous()

    def _in_float32(self, x: torch.Tensor) -> bool:
        return x.dtype == torch.float16 or (torch.is_autocast_enabled("cuda") and torch.get_autocast_dtype("cuda") == torch.float16)

    def forward(self, x: torch.Tensor, positions: torch.Tensor | None = None, lengths: torch.Tensor | None = None) -> torch.Tensor:
        """positions (N) or (B, N), with several axes (N, axes) or (B, N, axes); lengths (B) int32: points of each sequence, those behind
        them come out as the bias of out_linear."""
        if x.is_cuda and self._in_float32(x):
            with torch.autocast("cuda", enabled=False):
                return self.forward(x.float(), positions, lengths).to(torch.float16)
        x = self._prepared(x)
        if x.numel() == 0:
            return x.new_zeros(*x.shape[:-1], self.out_linear.out_features)
        needs_grad = self._needs_grad(x)
        q, k, v = self._qkv(x, self._positions(x, positions), needs_grad)
        call = dict(window=self.window, sinks=self.sinks, lengths=lengths, max_distance=self.max_distance)
        if needs_grad:
            y = PA.window_attention(q, k, v, bias=self.bias, **call)
        else:
            y = PF.window_attention(q, k, v, bias=None if self.bias is None else self.bias.detach().float().contiguous(), **call)
        return self.out_dropout(self._projected(self.out_linear, y.flatten(2), needs_grad))

    def forward_block(self, x: torch.Tensor, residual: torch.Tensor, ln: nn.LayerNorm | None):
        """self(x) + residual and, with `ln`, its LayerNorm, for a block that is served."""
        if x.is_cuda and self._in_float32(x):
            with torch.autocast("cuda", enabled=False):  # the sum as well, as in the other layers
                return self.forward_block(x.float(), residual.float(), ln)
        if x.numel() == 0:
            y = self(x)
            y = y + residual.to(y.dtype)
            return y if ln is None else (y, y.clone())
        y = self(x).to(residual.dtype).contiguous()
        if ln is None:
            return PF.residual_layernorm(y, residual=residual.contiguous())
        return PF.residual_layernorm(y, residual=residual.contiguous(), ln_weight=ln.weight.detach().float().contiguous(),
                                     ln_bias=ln.bias.detach().float().contiguous(), ln_eps=ln.eps)

    def cache(self, batch: int, capacity: int, dtype: torch.dtype | None = None) -> WindowCache:
        """An empty cache for `step`, in the type that the layer's inputs will have, by default its weights' (float32 for float16)."""
        weight = self.in_project_qkv.weight
        dtype = dtype or weight.dtype
        return WindowCache(batch, capacity, self.kv_heads, self.dim_head, torch.float32 if dtype == torch.float16 else dtype, weight.device)

    @torch.no_grad()
    def step(self, x: torch.Tensor, cache: WindowCache, positions: torch.Tensor | None = None) -> torch.Tensor:
        """The next T points (B, T, dim) of every sequence: adds their keys and values to the cache and returns their rows of `forward` over
        all points so far.  For layers that look back only (window[1] = 0); positions as for `forward`, by default the places behind the cache."""
        if self.window[1] != 0:
            raise ValueError("step is for a layer whose window has no reach ahead")
        shared = self.heads // self.kv_heads
        if self.bias is not None and self.bias.shape[0] * shared > PF.MAX_STEP_BIASES:  # before the cache changes
            raise ValueError(f"step takes {PF.MAX_STEP_BIASES} biases a key head, got {self.bias.shape[0]} of {shared} query heads")
        if x.is_cuda and self._in_float32(x):
            with torch.autocast("cuda", enabled=False):
                return self.step(x.float(), cache, positions).to(torch.float16)
        x = self._prepared(x)
        if x.numel() == 0:
            return x.new_zeros(*x.shape[:-1], self.out_linear.out_features)
        if self.frequencies is not None and positions is None and self.axes == 1:
            positions = cache.lengths[:, None].long() + torch.arange(x.shape[1], device=x.device)
        q, k, v = self._qkv(x, self._positions(x, positions), False)
        if k.dtype != cache.k.dtype or k.shape[0] != cache.k.shape[0]:
            raise ValueError(f"the cache is for {cache.k.dtype} and {cache.k.shape[0]} sequences, the input for {k.dtype} and {k.shape[0]}")
        cache.append(k, v)
        bias = None if self.bias is None else self.bias.detach().float().contiguous()
        y = PF.window_attention_step(q, cache.k, cache.v, cache.lengths, left=self.window[0], sinks=self.sinks, bias=bias,
                                     max_distance=self.max_distance)
        return self._projected(self.out_linear, y.flatten(2), False)
