"""``turbo_dropout``: dropout on B200 whose mask is never stored, with the residual added in the same pass.

Operator contract:

* ``x``: bf16, fp16 or fp32 ``[*]``.  Dimensions that lie at few strides (slices, transposed pair tensors) are read in place, other
  layouts through a contiguous copy.  The result does not depend on strides.  Fewer than 2^36 elements.
* ``p``: probability of an element to be dropped, held as ``round(65536 p) / 65536``.  ``out = residual + (kept ? x / (1 - p) : 0)``, one
  rounding; a dropped infinity or NaN is a zero.
* ``seed``: an ``int``, a pair ``(seed, offset)`` of them, an int64 tensor ``[2]`` on x's device that holds the pair (a captured
  graph reads it at every replay; do not change it between a forward and its backward), or ``None``: drawn from torch's
  generator of the device.  The same seed gives the same mask.  Take another seed, or another offset, for every call.
* ``shared_dim``: a dimension, not the last one, along which all elements share one mask (the row-wise dropout of a pair
  tensor ``[*, N, N, C]`` has -3); ``None``: every element has its own.  It has fewer than 2^31 elements, and so have the dimensions
  before it together.
* ``residual``: added, of x's shape and type.  ``training=False``: nothing is dropped, and the result is ``x``
  itself or ``residual + x``.
* returns x's type and shape, contiguous in training; autograd for x and the residual, first order, reverse mode only.  Between the passes
  nothing is kept but the seed.

The random bits: element m of the mask (row-major in x's shape with 1 in the place of the shared dimension) is dropped where half word
``m & 7`` of Philox 4x32-10 (Salmon, Moraes, Dror, Shaw 2011) with key ``seed`` and counter ``(m >> 3, offset)`` is below
``round(65536 p)``.

Unsupported inputs raise ``ValueError("turbo_dropout unsupported [code]: reason")``, in a traced call when it is traced or, for
sizes that are free there, when it runs.  The reference's counterpart is the dropout of its pair block
(openfold3/core/model/primitives/dropout.py, called from openfold3/core/model/latent/base_blocks.py:433-534).
"""
from __future__ import annotations

import math
from typing import Optional

import torch

from . import _cabi as C
from ._checks import NO_TANGENT, certain, differs, has_tangent, refuse
from .layer_norm import ROW_DTYPES
from .trimul import SupportResult

_STEPS = 65536
_MOST_ELEMENTS = 2 ** 36
_MOST = 2 ** 31     # of a shared dimension, and of those before it


def _is_int(n):
    return isinstance(n, (int, torch.SymInt)) and not isinstance(n, bool)


def _seed_numbers(seed):
    """``(seed, offset)`` as signed 64-bit numbers, or ``None``."""
    pair = (seed, 0) if _is_int(seed) else seed
    if not (isinstance(pair, (tuple, list)) and len(pair) == 2 and all(map(_is_int, pair))):
        return None
    if not all(-2 ** 63 <= n < 2 ** 64 for n in pair):
        return None
    return tuple(n - 2 ** 64 if n >= 2 ** 63 else n for n in pair)


def check_dropout_support(x, p, seed=None, shared_dim=None, residual=None, *, check_device=True) -> SupportResult:
    """Metadata-only contract check; returns the first failure."""
    if not isinstance(x, torch.Tensor):
        return SupportResult(False, "x_type", "x must be a torch.Tensor")
    if x.ndim < 1:
        return SupportResult(False, "x_shape", "x must have a dimension")
    if x.dtype not in ROW_DTYPES:
        return SupportResult(False, "x_dtype", "x must be BF16, FP16 or FP32")
    if certain(x.numel() >= _MOST_ELEMENTS):
        return SupportResult(False, "x_shape", "x must have fewer than 2^36 elements")
    if not (isinstance(p, (int, float)) and 0 <= p <= 1):
        return SupportResult(False, "p", "p must be a number in 0 .. 1")
    if isinstance(seed, torch.Tensor):
        if seed.dtype != torch.int64 or differs(seed.shape, (2,)):
            return SupportResult(False, "seed", "a seed tensor must be INT64 [2]: seed and offset")
        if seed.device != x.device:
            return SupportResult(False, "seed", "a seed tensor must live on x's device")
    elif seed is not None and _seed_numbers(seed) is None:
        return SupportResult(False, "seed", "seed must be a 64-bit int, a pair of them, an INT64 tensor [2], or None")
    if shared_dim is not None and not (_is_int(shared_dim) and -x.ndim <= shared_dim < x.ndim
                                       and shared_dim % x.ndim != x.ndim - 1):
        return SupportResult(False, "shared_dim", "shared_dim must be a dimension of x but the last one")
    if shared_dim is not None:
        shared = shared_dim % x.ndim
        if certain(x.shape[shared] >= _MOST) or certain(math.prod(x.shape[:shared]) >= _MOST):
            return SupportResult(False, "shared_dim", "a shared dimension, and those before it together, must be below 2^31")
    if residual is not None:
        if not isinstance(residual, torch.Tensor) or differs(residual.shape, tuple(x.shape)):
            return SupportResult(False, "residual_shape", "residual must have x's shape")
        if residual.dtype != x.dtype or residual.device != x.device:
            return SupportResult(False, "residual_dtype", "residual must have x's type and device")
    if has_tangent(x, residual):
        return SupportResult(False, "tangent", NO_TANGENT)
    if check_device:
        if not x.is_cuda:
            return SupportResult(False, "device", "x must be a CUDA tensor")
        if torch.cuda.get_device_capability(x.device)[0] != 10:
            return SupportResult(False, "device_arch", "these kernels require a Blackwell sm_100a device")
    return SupportResult(True, "ok", "supported")


def _check_op(x, residual, seed_tensor, threshold, shared, check_device):
    res = check_dropout_support(x, threshold / _STEPS, seed_tensor if seed_tensor is not None else 0,
                                shared if shared >= 0 else None, residual, check_device=check_device)
    refuse("turbo_dropout", res)


# --------------------------------------------------------------------------------------
# custom op: what a traced graph holds.  An eager call on plain CUDA tensors goes to `_native.dropout`.
# --------------------------------------------------------------------------------------
@torch.library.custom_op("tpf_b200::dropout", mutates_args=())
def _dropout(x: torch.Tensor, residual: Optional[torch.Tensor], seed_tensor: Optional[torch.Tensor], seed: int, offset: int,
             threshold: int, shared: int) -> torch.Tensor:
    _check_op(x, residual, seed_tensor, threshold, shared, True)
    return C.native().dropout_op(x, residual, seed_tensor, seed, offset, threshold, shared)


@_dropout.register_fake
def _(x, residual, seed_tensor, seed, offset, threshold, shared):
    _check_op(x, residual, seed_tensor, threshold, shared, False)
    return torch.empty_like(x, memory_format=torch.contiguous_format)


def _setup_context(ctx, inputs, output):
    x, residual, seed_tensor, *ctx.numbers = inputs
    ctx.save_for_backward(seed_tensor)
    ctx.has_residual = residual is not None


def _backward(ctx, d_out):
    d_x = torch.ops.tpf_b200.dropout(d_out, None, ctx.saved_tensors[0], *ctx.numbers)
    return d_x, d_out if ctx.has_residual else None, None, None, None, None, None


_dropout.register_autograd(_backward, setup_context=_setup_context)


def turbo_dropout(x, p, seed=None, *, shared_dim=None, residual=None, training=True):
    """Dropout of ``x``, with ``residual`` added; see the module docstring for the contract."""
    tracing = torch.compiler.is_compiling()
    known = isinstance(x, torch.Tensor) and isinstance(p, (int, float)) and 0 <= p <= 1
    if known and training and not tracing:
        numbers = (0, 0) if seed is None or isinstance(seed, torch.Tensor) else _seed_numbers(seed)
        if numbers is not None and (shared_dim is None or (_is_int(shared_dim) and -x.ndim <= shared_dim < x.ndim)):
            if seed is None and x.is_cuda:
                seed = _draw(x)
            out = C.native().dropout(x, residual, seed if isinstance(seed, torch.Tensor) else None, *numbers, round(_STEPS * p),
                                     -1 if shared_dim is None else shared_dim % x.ndim)
            if out is not None:
                return out
    refuse("turbo_dropout", check_dropout_support(x, p, seed, shared_dim, residual, check_device=not tracing))
    if not training:
        return x if residual is None else residual + x
    if seed is None:
        seed = _draw(x)
    numbers = (0, 0) if isinstance(seed, torch.Tensor) else _seed_numbers(seed)
    return torch.ops.tpf_b200.dropout(x, residual, seed if isinstance(seed, torch.Tensor) else None, *numbers, round(_STEPS * p),
                                      -1 if shared_dim is None else shared_dim % x.ndim)


def _draw(x):
    return torch.randint(-2 ** 63, 2 ** 63 - 1, (2,), dtype=torch.int64, device=x.device)
