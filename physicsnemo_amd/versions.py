"""What tells whether parameters have changed since something was made of them."""
from __future__ import annotations

from torch.optim.optimizer import register_optimizer_step_post_hook

# id of a parameter -> steps of optimisers that may write it without a new version: torch's fused ones do, and others' may
_written: dict[int, int] = {}


def _count(optimizer, args, kwargs) -> None:
    groups = optimizer.param_groups
    if type(optimizer).__module__.startswith("torch.optim.") and not any(g.get("fused") for g in groups):
        return
    for group in groups:
        for p in group["params"]:
            _written[id(p)] = _written.get(id(p), 0) + 1


register_optimizer_step_post_hook(_count)


def stamp(*params) -> tuple:
    """The parameters' addresses, versions, types and fused optimiser steps (None stays None).  What writes them through `.data`, or in a
    replayed graph, changes none of these."""
    return tuple(None if p is None else (p.data_ptr(), p._version, p.dtype, _written.get(id(p), 0)) for p in params)
