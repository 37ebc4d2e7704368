"""Pieces of the operators' metadata contracts that hold for eager and for traced calls.

A traced call (torch.compile, torch.export, torch.jit.trace) meets its contract twice: in the fake kernel, on whatever sizes
are known there, and in the operator that launches, on the tensors it is given.  The fake kernel must not pin a size that
is free (a comparison of a symbolic size would), so a check there only refuses what is certain.
"""
from __future__ import annotations

import torch

from . import _cabi


def certain(comparison) -> bool:
    """Is a comparison of sizes true?  One of free sizes that can go either way counts as false."""
    if isinstance(comparison, torch.SymBool):
        from torch.fx.experimental.symbolic_shapes import statically_known_true
        return statically_known_true(comparison)
    return bool(comparison)     # (a plain one, or under torch.jit.trace, where sizes are tensors)


def differs(shape, expected) -> bool:
    """Are two shapes certainly different?"""
    return len(shape) != len(expected) or any(certain(a != b) for a, b in zip(shape, expected))


def has_tangent(*tensors) -> bool:
    """Does any of them carry a forward-mode tangent?  No operator propagates one: a dual tensor is refused."""
    from torch.autograd import forward_ad
    if forward_ad._current_level < 0:
        return False
    functorch, native = torch._C._functorch, _cabi.native()
    for t in tensors:
        if not isinstance(t, torch.Tensor):
            continue
        while not native.has_tangent(t):    # (torch.func: of any level, which a dispatched call would not see)
            if not functorch.is_functorch_wrapped_tensor(t):
                break
            t = functorch.get_unwrapped(t)
        else:
            return True
    return False


NO_TANGENT = "there is no forward-mode derivative"


def refuse(operator, res):
    """Raise for a failed ``SupportResult``."""
    if not res.supported:
        raise ValueError(f"{operator} unsupported [{res.code}]: {res.reason}")
