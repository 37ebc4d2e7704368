"""``turbo_layer_norm``: layer norm of rows on B200, forward and backward.

Operator contract:

* ``x``: bf16, fp16 or fp32 ``[*, C]``, ``1 <= C <= 8192``.  Rows that lie at one pitch (slices of the last dimension, rows
  that are expanded) are read in place, other layouts through a contiguous copy.
* ``weight``, ``bias``: ``[C]`` of any of these types, or ``None`` (ones, zeros).
* ``checkpoint``: ``None`` keeps ``x`` for the backward pass.  ``"int8"`` keeps it in the 8-bit format of
  :func:`pack_activation` instead (one byte an element and a scale per 128 in place of two or four); the statistics are
  those of the true ``x``, the gradients are computed from the kept values.  The format is relative to the largest
  magnitude of a group, so rows whose mean is large against their spread lose more.
* returns ``x``'s type and shape, contiguous; autograd for x, weight and bias (a gradient has its parameter's type), first
  order, reverse mode only.  Statistics and sums are fp32 in a fixed order: the same inputs give the same bits.

A row that holds an infinity or a NaN is NaN; the others are not touched by it.  Unsupported inputs raise
``ValueError("turbo_layer_norm unsupported [code]: reason")``, in a traced call when it is traced (inside the compiler's own
exception) or, for sizes that are free there, when it runs.  There is no counterpart among the reference's kernels (it
calls torch's LayerNorm, openfold3/core/model/primitives/normalization.py).
"""
from __future__ import annotations

import math
from typing import Optional

import torch

from . import _cabi as C
from ._checks import NO_TANGENT, certain, differs, has_tangent, refuse
from .trimul import SupportResult

ROW_DTYPES = (torch.bfloat16, torch.float16, torch.float32)
MAX_COLUMNS = 8192
MAX_EPS = torch.finfo(torch.float32).max
CHECKPOINTS = (None, "int8")


def check_parameter(name, p, cols, x):
    """The first failure of an optional ``[C]`` parameter, or ``None``."""
    if p is None:
        return None
    if not isinstance(p, torch.Tensor) or differs(p.shape, (cols,)):
        return SupportResult(False, "weight_shape", f"{name} must have shape ({cols},)")
    if p.dtype not in ROW_DTYPES:
        return SupportResult(False, "weight_dtype", f"{name} must be BF16, FP16 or FP32")
    if p.device != x.device:
        return SupportResult(False, "weight_device", f"{name} must live on x's device")
    return None


def check_rows(x, eps, checkpoint, check_device):
    """Checks that the row-wise operators share; the first failure, or ``None``."""
    if not isinstance(x, torch.Tensor):
        return SupportResult(False, "x_type", "x must be a torch.Tensor")
    if x.ndim < 1 or certain(x.shape[-1] < 1):
        return SupportResult(False, "x_shape", "x must have shape [*,C], C >= 1")
    if certain(x.shape[-1] > MAX_COLUMNS):
        return SupportResult(False, "columns", f"C={x.shape[-1]} exceeds {MAX_COLUMNS}")
    if checkpoint not in CHECKPOINTS:
        return SupportResult(False, "checkpoint", "checkpoint must be None or 'int8'")
    if not (isinstance(eps, (int, float)) and 0 <= eps <= MAX_EPS):
        return SupportResult(False, "eps", "eps must be a finite FP32 number, not negative")
    if check_device:
        if not x.is_cuda:
            return SupportResult(False, "device", "x must be a CUDA tensor")
        if torch.cuda.get_device_capability(x.device)[0] != 10:
            return SupportResult(False, "device_arch", "these kernels require a Blackwell sm_100a device")
    return None


def check_layer_norm_support(x, weight=None, bias=None, eps=1e-5, checkpoint=None, *, check_device=True) -> SupportResult:
    """Metadata-only contract check; returns the first failure."""
    bad = check_rows(x, eps, checkpoint, check_device)
    if bad is not None:
        return bad
    if x.dtype not in ROW_DTYPES:
        return SupportResult(False, "x_dtype", "x must be BF16, FP16 or FP32")
    for name, p in (("weight", weight), ("bias", bias)):
        bad = check_parameter(name, p, x.shape[-1], x)
        if bad is not None:
            return bad
    if has_tangent(x, weight, bias):
        return SupportResult(False, "tangent", NO_TANGENT)
    return SupportResult(True, "ok", "supported")


def check_kept(d_out, rows_shape, cols, x, stats, codes, scales):
    """What a backward pass is given of its forward: ``x`` or its codes, and the statistics; the first failure, or ``None``."""
    rows = math.prod(rows_shape)
    if any(t is not None and t.device != d_out.device for t in (x, stats, codes, scales)):
        return SupportResult(False, "device", "all tensors must share one device")
    if stats.dtype != torch.float32 or differs(stats.shape, (2, rows)):
        return SupportResult(False, "stats", "stats must be FP32 [2, rows]")
    if x is not None:
        if differs(x.shape, tuple(rows_shape) + (cols,)):
            return SupportResult(False, "x_shape", "x does not belong to this gradient")
        return None
    if codes.dtype != torch.int8 or differs(codes.shape, (rows, -(-cols // 16) * 16)):
        return SupportResult(False, "codes", "codes must be INT8, rows at a pitch of C rounded up to 16")
    if scales.dtype != torch.float32 or differs(scales.shape, (rows, -(-cols // 128))):
        return SupportResult(False, "scales", "scales must be FP32 [rows, ceil(C / 128)]")
    return None


def _check_backward(dy, x, stats, codes, scales, weight, bias, check_device):
    res = check_layer_norm_support(dy, weight, bias, check_device=check_device)
    if not res.supported:
        return res
    if x is not None and x.dtype != dy.dtype:
        return SupportResult(False, "x_dtype", "x and its gradient must have one type")
    return check_kept(dy, dy.shape[:-1], dy.shape[-1], x, stats, codes, scales) or res


# --------------------------------------------------------------------------------------
# custom ops: what a traced graph holds.  An eager call on plain CUDA tensors goes to `_native.layer_norm`.
# --------------------------------------------------------------------------------------
def kept_like(x, int8):
    """Shapes of what a forward keeps: statistics, codes, scales (empty unless ``int8``)."""
    cols = x.shape[-1]
    rows = math.prod(x.shape[:-1])
    return [x.new_empty((2, rows), dtype=torch.float32),
            x.new_empty((rows, -(-cols // 16) * 16) if int8 else (0,), dtype=torch.int8),
            x.new_empty((rows, -(-cols // 128)) if int8 else (0,), dtype=torch.float32)]


@torch.library.custom_op("tpf_b200::layer_norm_fwd", mutates_args=())
def _layer_norm_fwd(x: torch.Tensor, weight: Optional[torch.Tensor], bias: Optional[torch.Tensor], eps: float,
                    int8: bool) -> list[torch.Tensor]:
    refuse("turbo_layer_norm", check_layer_norm_support(x, weight, bias, eps, "int8" if int8 else None))
    return C.native().layer_norm_fwd(x, weight, bias, eps, int8)


@_layer_norm_fwd.register_fake
def _(x, weight, bias, eps, int8):
    refuse("turbo_layer_norm", check_layer_norm_support(x, weight, bias, eps, check_device=False))
    return [torch.empty_like(x, memory_format=torch.contiguous_format), *kept_like(x, int8)]


@torch.library.custom_op("tpf_b200::layer_norm_bwd", mutates_args=())
def _layer_norm_bwd(dy: torch.Tensor, x: Optional[torch.Tensor], stats: torch.Tensor, codes: torch.Tensor,
                    scales: torch.Tensor, weight: Optional[torch.Tensor],
                    bias: Optional[torch.Tensor]) -> list[torch.Tensor]:
    refuse("layer norm backward", _check_backward(dy, x, stats, codes, scales, weight, bias, True))
    return C.native().layer_norm_bwd(dy, x, stats, codes, scales, weight, bias)


@_layer_norm_bwd.register_fake
def _(dy, x, stats, codes, scales, weight, bias):
    refuse("layer norm backward", _check_backward(dy, x, stats, codes, scales, weight, bias, False))
    none = lambda: dy.new_empty((0,), dtype=torch.float32)  # noqa: E731
    return [torch.empty_like(dy, memory_format=torch.contiguous_format),
            none() if weight is None else weight.new_empty(weight.shape),
            none() if bias is None else bias.new_empty(bias.shape)]


def _setup_context(ctx, inputs, output):
    x, weight, bias, _, int8 = inputs
    _, stats, codes, scales = output
    ctx.save_for_backward(None if int8 else x, stats, codes, scales, weight, bias)
    ctx.dtype = x.dtype
    ctx.set_materialize_grads(False)


def _backward(ctx, grads):
    dy = grads[0]
    if dy is None:
        return (None,) * 5
    x, stats, codes, scales, weight, bias = ctx.saved_tensors
    dx, dw, db = torch.ops.tpf_b200.layer_norm_bwd(dy.to(ctx.dtype), x, stats, codes, scales, weight, bias)
    return dx, None if weight is None else dw, None if bias is None else db, None, None


_layer_norm_fwd.register_autograd(_backward, setup_context=_setup_context)


def turbo_layer_norm(x, weight=None, bias=None, *, eps=1e-5, checkpoint=None):
    """Layer norm over the last dimension; see the module docstring for the contract."""
    if not torch.compiler.is_compiling():
        if checkpoint in CHECKPOINTS and isinstance(eps, (int, float)) and eps <= MAX_EPS:
            y = C.native().layer_norm(x, weight, bias, eps, checkpoint == "int8")
            if y is not None:
                return y
        refuse("turbo_layer_norm", check_layer_norm_support(x, weight, bias, eps, checkpoint))
    return torch.ops.tpf_b200.layer_norm_fwd(x, weight, bias, eps, checkpoint == "int8")[0]
