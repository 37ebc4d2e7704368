"""``turbo_norm_linear``: a layer norm and the bias-free Linear that follows it, on B200.

    out = layer_norm(x; norm_weight, norm_bias, eps) @ weight^T

Operator contract:

* ``x``: bf16 ``[*, C]``, C a multiple of 8 up to 8192; ``weight``: ``[O, C]``, O a multiple of 8, bf16, fp16 or fp32
  (rounded to bf16 inside, like the projections of :func:`turbo_trimul`); ``norm_weight``, ``norm_bias``: as in
  :func:`turbo_layer_norm`.  Projections that share an input (q, k, v, gate) go into one weight.  Fewer than 2^31 - 256
  rows, at most 2^30 outputs.
* ``checkpoint``: as in :func:`turbo_layer_norm`.  Only x is kept, whole or in 8 bits: the normalised rows are made again
  in the backward pass, for the weight's gradient too.
* returns bf16 ``[*, O]``; autograd for x, norm_weight, norm_bias and weight (first order, reverse mode only).  The
  normalised rows are rounded to bf16 on their way to the tensor cores (but in the forward of four rows and fewer), sums are
  fp32.  The gradients of weight and, where rows are narrow, of norm_weight are made of rows rounded that way.  The gradient
  that reaches the normalised rows is rounded to bf16 on its way to the layer norm's backward, as a bf16 Linear would leave
  it, but where rows are narrow (up to 128 columns, a weight of up to 128 KB).

Unsupported inputs raise ``ValueError("turbo_norm_linear unsupported [code]: reason")``, traced ones as in
:func:`turbo_layer_norm`.  There is no counterpart among the reference's kernels (it calls torch's LayerNorm and Linear).
"""
from __future__ import annotations

import math
from typing import Optional

import torch

from . import _cabi as C
from ._checks import NO_TANGENT, certain, differs, has_tangent, refuse
from .layer_norm import CHECKPOINTS, MAX_EPS, ROW_DTYPES, check_kept, check_parameter, check_rows, kept_like
from .trimul import SupportResult

MAX_ROWS = 2 ** 31 - 256
MAX_OUTPUTS = 2 ** 30


def check_norm_linear_support(x, norm_weight, norm_bias, weight, eps=1e-5, checkpoint=None, *,
                              check_device=True) -> SupportResult:
    """Metadata-only contract check; returns the first failure."""
    bad = check_rows(x, eps, checkpoint, check_device)
    if bad is not None:
        return bad
    if x.dtype != torch.bfloat16:
        return SupportResult(False, "x_dtype", "x must be BF16")
    cols = x.shape[-1]
    if certain(cols % 8 != 0):
        return SupportResult(False, "columns", f"C={cols} is not a multiple of 8")
    if not isinstance(weight, torch.Tensor) or weight.ndim != 2 or certain(weight.shape[1] != cols):
        return SupportResult(False, "weight_shape", f"weight must have shape (O, {cols})")
    if certain(math.prod(x.shape[:-1]) >= MAX_ROWS) or certain(weight.shape[0] > MAX_OUTPUTS):
        return SupportResult(False, "extent", f"at most {MAX_ROWS - 1} rows and {MAX_OUTPUTS} outputs")
    if certain(weight.shape[0] < 8) or certain(weight.shape[0] % 8 != 0):
        return SupportResult(False, "outputs", f"O={weight.shape[0]} is not a positive multiple of 8")
    if weight.dtype not in ROW_DTYPES:
        return SupportResult(False, "weight_dtype", "weight must be BF16, FP16 or FP32")
    if weight.device != x.device:
        return SupportResult(False, "weight_device", "weight must live on x's device")
    for name, p in (("norm_weight", norm_weight), ("norm_bias", norm_bias)):
        bad = check_parameter(name, p, cols, x)
        if bad is not None:
            return bad
    if has_tangent(x, norm_weight, norm_bias, weight):
        return SupportResult(False, "tangent", NO_TANGENT)
    return SupportResult(True, "ok", "supported")


def _check_backward(d_out, x, stats, codes, scales, norm_weight, norm_bias, weight, check_device):
    # x's part of the contract, on a stand-in of x's type and shape where only its codes are left
    like = d_out.new_empty((1,), dtype=torch.bfloat16).expand(d_out.shape[:-1] + weight.shape[1:]) if x is None else x
    res = check_norm_linear_support(like, norm_weight, norm_bias, weight, check_device=check_device)
    if not res.supported:
        return res
    if has_tangent(d_out):
        return SupportResult(False, "tangent", NO_TANGENT)
    if differs(d_out.shape, tuple(like.shape[:-1]) + (weight.shape[0],)):
        return SupportResult(False, "d_out_shape", "d_out does not belong to these rows and this weight")
    return check_kept(d_out, d_out.shape[:-1], weight.shape[1], x, stats, codes, scales) or res


# --------------------------------------------------------------------------------------
# custom ops: what a traced graph holds.  An eager call on plain CUDA tensors goes to `_native.norm_linear`.
# --------------------------------------------------------------------------------------
@torch.library.custom_op("tpf_b200::norm_linear_fwd", mutates_args=())
def _norm_linear_fwd(x: torch.Tensor, norm_weight: Optional[torch.Tensor], norm_bias: Optional[torch.Tensor],
                     weight: torch.Tensor, eps: float, int8: bool) -> list[torch.Tensor]:
    refuse("turbo_norm_linear",
           check_norm_linear_support(x, norm_weight, norm_bias, weight, eps, "int8" if int8 else None))
    return C.native().norm_linear_fwd(x, norm_weight, norm_bias, weight, eps, int8)


@_norm_linear_fwd.register_fake
def _(x, norm_weight, norm_bias, weight, eps, int8):
    refuse("turbo_norm_linear", check_norm_linear_support(x, norm_weight, norm_bias, weight, eps, check_device=False))
    return [x.new_empty(x.shape[:-1] + (weight.shape[0],)), *kept_like(x, int8)]


@torch.library.custom_op("tpf_b200::norm_linear_bwd", mutates_args=())
def _norm_linear_bwd(d_out: torch.Tensor, x: Optional[torch.Tensor], stats: torch.Tensor, codes: torch.Tensor,
                     scales: torch.Tensor, norm_weight: Optional[torch.Tensor], norm_bias: Optional[torch.Tensor],
                     weight: torch.Tensor) -> list[torch.Tensor]:
    refuse("normalised projection backward",
           _check_backward(d_out, x, stats, codes, scales, norm_weight, norm_bias, weight, True))
    return C.native().norm_linear_bwd(d_out, x, stats, codes, scales, norm_weight, norm_bias, weight)


@_norm_linear_bwd.register_fake
def _(d_out, x, stats, codes, scales, norm_weight, norm_bias, weight):
    refuse("normalised projection backward",
           _check_backward(d_out, x, stats, codes, scales, norm_weight, norm_bias, weight, False))
    none = lambda: d_out.new_empty((0,), dtype=torch.float32)  # noqa: E731
    return [d_out.new_empty(d_out.shape[:-1] + (weight.shape[1],)), weight.new_empty(weight.shape),
            none() if norm_weight is None else norm_weight.new_empty(norm_weight.shape),
            none() if norm_bias is None else norm_bias.new_empty(norm_bias.shape)]


def _setup_context(ctx, inputs, output):
    x, norm_weight, norm_bias, weight, _, int8 = inputs
    _, stats, codes, scales = output
    ctx.save_for_backward(None if int8 else x, stats, codes, scales, norm_weight, norm_bias, weight)
    ctx.set_materialize_grads(False)


def _backward(ctx, grads):
    d_out = grads[0]
    if d_out is None:
        return (None,) * 6
    x, stats, codes, scales, norm_weight, norm_bias, weight = ctx.saved_tensors
    dx, dw, dnw, dnb = torch.ops.tpf_b200.norm_linear_bwd(d_out.to(torch.bfloat16), x, stats, codes, scales, norm_weight,
                                                          norm_bias, weight)
    return dx, None if norm_weight is None else dnw, None if norm_bias is None else dnb, dw, None, None


_norm_linear_fwd.register_autograd(_backward, setup_context=_setup_context)


def turbo_norm_linear(x, norm_weight, norm_bias, weight, *, eps=1e-5, checkpoint=None):
    """Layer norm and Linear in one operator; see the module docstring for the contract."""
    if not torch.compiler.is_compiling():
        if checkpoint in CHECKPOINTS and isinstance(eps, (int, float)) and eps <= MAX_EPS:
            out = C.native().norm_linear(x, norm_weight, norm_bias, weight, eps, checkpoint == "int8")
            if out is not None:
                return out
        refuse("turbo_norm_linear", check_norm_linear_support(x, norm_weight, norm_bias, weight, eps, checkpoint))
    return torch.ops.tpf_b200.norm_linear_fwd(x, norm_weight, norm_bias, weight, eps, checkpoint == "int8")[0]
