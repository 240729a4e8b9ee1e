"""Test infrastructure: what users put round a model's modules (hooks, wrappers, sharding)."""
from __future__ import annotations

import torch
from torch import nn


class Round(nn.Module):
    """Calls the module it holds, and counts; attributes are those of the module inside."""

    def __init__(self, inner):
        super().__init__()
        self.inner, self.calls = inner, 0

    def forward(self, *args, **kw):
        self.calls += 1
        return self.inner(*args, **kw)

    def __getattr__(self, name):
        try:
            return super().__getattr__(name)
        except AttributeError:
            return getattr(super().__getattr__("inner"), name)


def shard(module, but=()):
    """The parameters of `module` hold their values only between its forward's start and end, as
    those of sharded modules do; modules in `but` keep theirs.  Returns a function that restores them."""
    held = [(p, p.detach().clone()) for n, p in module.named_parameters() if not n.startswith(tuple(but))]

    def gather(*_):
        with torch.no_grad():
            for p, v in held:
                p.data = v.clone()

    def spoil(*_):
        with torch.no_grad():
            for p, v in held:
                p.data = torch.full_like(v, float("nan"))

    spoil()
    handles = [module.register_forward_pre_hook(gather), module.register_forward_hook(spoil)]

    def restore():
        for h in handles:
            h.remove()
        gather()

    return restore


class Adapted(nn.Module):
    """A head with a low-rank addition; `weight` is the base's, as adapter libraries have it."""

    def __init__(self, base, rank=2):
        super().__init__()
        self.base = base
        g = torch.Generator().manual_seed(0)
        self.a = nn.Parameter(torch.randn(rank, base.in_features, generator=g).to(base.weight))
        self.b = nn.Parameter(torch.randn(base.out_features, rank, generator=g).to(base.weight))

    @property
    def weight(self):
        return self.base.weight

    def forward(self, x):
        return self.base(x) + (x @ self.a.T) @ self.b.T
