"""``turbo_window_attention``: attention of a sequence over a sliding window and a few first tokens (sinks), on B200.

Operator contract:

* ``q``: bf16 or fp16 ``[*, N, H, D]``; ``k, v``: ``[*, M, HK, D]`` of q's type.  D is a multiple of 8 up to 128; H is a multiple of HK,
  and query head h reads key head ``h // (H / HK)``.  Tensors whose strides are multiples of 8 elements are read in place
  (slices of a stacked projection or of a cache), others through a copy.
* query i stands at position ``query_offset + i`` and sees key j where ``j < key_lengths``, ``j <= position + right``, and
  ``j >= position - left`` or ``j < sinks``, with ``window = (left, right)``; ``None`` for either: no limit.  ``(n, 0)`` is causal.
* ``sinks``: 0 .. 64.
* ``query_offset``: an ``int`` (within 2^28), or an int32 or int64 tensor ``[*]``, one for each sequence (clamped to +-2^29).
* ``key_lengths``: ``None`` (M), or an int32 or int64 tensor ``[*]`` (clamped to 0 .. M).  What lies behind the last key is not
  looked at and may be anything.  A query that sees no key gives zeros and has no gradient.
* ``scale``: positive, ``D ** -0.5`` where it is ``None``.
* returns q's type, ``[*, N, H, D]`` contiguous, with ``return_lse=True`` also the log-sum-exp, fp32 ``[*, H, N]`` (``-inf`` where
  nothing is seen).  Autograd for q, k and v, first order, reverse mode only; the gradients of shared key heads are summed in
  fp32.  The same inputs give the same bits.

A single token over its cache is ``N = 1`` with ``query_offset = key_lengths - 1``.  Probabilities and their gradients are rounded
to q's type as operands of the products, in fp16 within its range as well (a loss scale keeps them there).  Calls of few queries, and
gradients of at most 128 queries and 128 keys, take them in two parts: their results are off by 0.42 half steps of their norm, others
by 0.60.  Sums and the softmax are fp32, and a probability below 2^-126 is zero.  The log-sum-exp has no gradient.  A key or value inside the sequence that is infinite or NaN reaches every query whose 128 neighbours see it, as a
product of zero with it does elsewhere.

Unsupported inputs raise ``ValueError("turbo_window_attention unsupported [code]: reason")``, in a traced call when it is traced or,
for sizes that are free there, when it runs.  The reference has no counterpart.
"""
from __future__ import annotations

import math
from typing import Optional

import torch

from . import _cabi as C
from ._checks import NO_TANGENT, certain, differs, has_tangent, refuse
from .trimul import SupportResult

MAX_HEAD_DIM = 128
MAX_SINKS = 64
_MOST = 2 ** 28     # tokens, keys, reach of a limited window, magnitude of an offset


def _is_int(n):
    return isinstance(n, (int, torch.SymInt)) and not isinstance(n, bool)


def check_window_attention_support(q, k, v, *, window, sinks=0, query_offset=0, key_lengths=None, scale=None,
                                   check_device=True) -> SupportResult:
    """Metadata-only contract check; returns the first failure."""
    for name, t in (("q", q), ("k", k), ("v", v)):
        if not isinstance(t, torch.Tensor) or t.ndim < 3:
            return SupportResult(False, "shape", f"{name} must have shape [*,N,H,D]")
    if q.dtype not in (torch.bfloat16, torch.float16):
        return SupportResult(False, "dtype", "q must be BF16 or FP16")
    if k.dtype != q.dtype or v.dtype != q.dtype:
        return SupportResult(False, "dtype", "k and v must have q's type")
    if k.device != q.device or v.device != q.device:
        return SupportResult(False, "device", "all operands must share one device")
    if differs(v.shape, tuple(k.shape)) or differs(k.shape[:-3] + k.shape[-1:], tuple(q.shape[:-3] + q.shape[-1:])):
        return SupportResult(False, "shape", "k and v must have one shape, and q's batch and head size")
    D, H, HK = q.shape[-1], q.shape[-2], k.shape[-2]
    if certain(D < 8) or certain(D > MAX_HEAD_DIM) or certain(D % 8 != 0):
        return SupportResult(False, "head_dim", f"the head size must be a multiple of 8 up to {MAX_HEAD_DIM}")
    if certain(HK < 1) or certain(H < 1) or certain(H % HK != 0):
        return SupportResult(False, "heads", "q's heads must be a multiple of k's")
    if certain(q.shape[-3] > _MOST) or certain(k.shape[-3] > _MOST) or certain(math.prod(q.shape[:-3]) > 65535) or certain(H > 65535):
        return SupportResult(False, "size", "too many tokens, heads or sequences")
    if not (isinstance(window, (tuple, list)) and len(window) == 2
            and all(n is None or (_is_int(n) and 0 <= n < _MOST) for n in window)):
        return SupportResult(False, "window", "window must be (left, right), each None or an int in 0 .. 2^28 - 1")
    if not (_is_int(sinks) and 0 <= sinks <= MAX_SINKS):
        return SupportResult(False, "sinks", f"sinks must be an int in 0 .. {MAX_SINKS}")
    for name, t in (("query_offset", query_offset), ("key_lengths", key_lengths)):
        if isinstance(t, torch.Tensor):
            if t.dtype not in (torch.int32, torch.int64) or t.device != q.device:
                return SupportResult(False, name, f"{name} must be INT32 or INT64, on q's device")
            if differs(t.shape, tuple(q.shape[:-3])):
                return SupportResult(False, name, f"{name} must have one entry for each sequence")
    if not isinstance(query_offset, torch.Tensor) and not (_is_int(query_offset) and -_MOST <= query_offset <= _MOST):
        return SupportResult(False, "query_offset", "query_offset must be a tensor or an int within 2^28")
    if key_lengths is not None and not isinstance(key_lengths, torch.Tensor):
        return SupportResult(False, "key_lengths", "key_lengths must be a tensor or None")
    if scale is not None and not (isinstance(scale, (int, float)) and 2.0 ** -100 <= scale <= 2.0 ** 100):
        return SupportResult(False, "scale", "scale must be a positive number (2^-100 .. 2^100)")
    if has_tangent(q, k, v):
        return SupportResult(False, "tangent", NO_TANGENT)
    if check_device:
        if not q.is_cuda:
            return SupportResult(False, "device", "operands must be CUDA tensors")
        if torch.cuda.get_device_capability(q.device)[0] != 10:
            return SupportResult(False, "device_arch", "these kernels require a Blackwell sm_100a device")
    return SupportResult(True, "ok", "supported")


# --------------------------------------------------------------------------------------
# custom ops: what a traced graph holds.  An eager call on plain CUDA tensors goes to `_native.window_attention`.
# --------------------------------------------------------------------------------------
def _refuse_op(q, k, v, offsets, lengths, offset, left, right, sinks, scale, check_device):
    reach = lambda n: None if n < 0 else n  # noqa: E731
    check = lambda device: check_window_attention_support(  # noqa: E731
        q, k, v, window=(reach(left), reach(right)), sinks=sinks, query_offset=offset if offsets is None else offsets,
        key_lengths=lengths, scale=scale, check_device=device)
    refuse("turbo_window_attention", check(False))
    if any(t is not None and t.dtype != torch.int32 for t in (offsets, lengths)):
        refuse("turbo_window_attention", SupportResult(False, "key_lengths", "the operator takes INT32 offsets and lengths"))
    if check_device:
        refuse("turbo_window_attention", check(True))


@torch.library.custom_op("tpf_b200::window_attn_fwd", mutates_args=())
def _window_fwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, offsets: Optional[torch.Tensor], lengths: Optional[torch.Tensor],
                offset: int, left: int, right: int, sinks: int, scale: float) -> tuple[torch.Tensor, torch.Tensor]:
    _refuse_op(q, k, v, offsets, lengths, offset, left, right, sinks, scale, True)
    return C.native().window_attn_fwd(q, k, v, offsets, lengths, offset, left, right, sinks, scale)


def _lse_like(q):
    return q.new_empty((*q.shape[:-3], q.shape[-2], q.shape[-3]), dtype=torch.float32)


@_window_fwd.register_fake
def _(q, k, v, offsets, lengths, offset, left, right, sinks, scale):
    _refuse_op(q, k, v, offsets, lengths, offset, left, right, sinks, scale, False)
    return q.new_empty(q.shape), _lse_like(q)


@torch.library.custom_op("tpf_b200::window_attn_bwd", mutates_args=())
def _window_bwd(d_out: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor, lse: torch.Tensor,
                offsets: Optional[torch.Tensor], lengths: Optional[torch.Tensor], offset: int, left: int, right: int, sinks: int,
                scale: float) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    _refuse_bwd(d_out, q, k, v, out, lse, offsets, lengths, offset, left, right, sinks, scale, True)
    return C.native().window_attn_bwd(d_out, q, k, v, out, lse, offsets, lengths, offset, left, right, sinks, scale)


def _refuse_bwd(d_out, q, k, v, out, lse, offsets, lengths, offset, left, right, sinks, scale, check_device):
    _refuse_op(q, k, v, offsets, lengths, offset, left, right, sinks, scale, False)
    if any(t.dtype != q.dtype or t.device != q.device or differs(t.shape, tuple(q.shape)) for t in (d_out, out)):
        refuse("window attention backward", SupportResult(False, "out", "the output and its gradient must be as q"))
    if lse.dtype != torch.float32 or lse.device != q.device or differs(lse.shape, (*q.shape[:-3], q.shape[-2], q.shape[-3])):
        refuse("window attention backward", SupportResult(False, "lse", "the log-sum-exp must be FP32 [*,H,N]"))
    if check_device:
        _refuse_op(q, k, v, offsets, lengths, offset, left, right, sinks, scale, True)


@_window_bwd.register_fake
def _(d_out, q, k, v, out, lse, offsets, lengths, offset, left, right, sinks, scale):
    _refuse_bwd(d_out, q, k, v, out, lse, offsets, lengths, offset, left, right, sinks, scale, False)
    return q.new_empty(q.shape), k.new_empty(k.shape), v.new_empty(v.shape)


def _setup_context(ctx, inputs, output):
    q, k, v, offsets, lengths, *ctx.numbers = inputs
    out, lse = output
    ctx.save_for_backward(q, k, v, out, lse, offsets, lengths)
    ctx.mark_non_differentiable(lse)


def _backward(ctx, d_out, d_lse):
    q, k, v, out, lse, offsets, lengths = ctx.saved_tensors
    dq, dk, dv = torch.ops.tpf_b200.window_attn_bwd(d_out, q, k, v, out, lse, offsets, lengths, *ctx.numbers)
    return dq, dk, dv, *(None,) * 7


_window_fwd.register_autograd(_backward, setup_context=_setup_context)


def _int32(t):
    """int32, contiguous.  (Values beyond 32 bits are brought to the ends that they count as.)"""
    if t is None or not isinstance(t, torch.Tensor):
        return None
    if t.dtype == torch.int64:
        t = t.clamp(-2 ** 29, 2 ** 29).to(torch.int32)
    return t.contiguous()


def turbo_window_attention(q, k, v, *, window, sinks=0, query_offset=0, key_lengths=None, scale=None, return_lse=False):
    """``softmax(scale q k^T) v`` over the window and the sinks; see the module docstring for the contract."""
    tracing = torch.compiler.is_compiling()
    if not tracing:
        out = C.native().window_attention(q, k, v, window, sinks, query_offset, key_lengths, scale, return_lse)
        if out is not None:
            return out
    refuse("turbo_window_attention", check_window_attention_support(
        q, k, v, window=window, sinks=sinks, query_offset=query_offset, key_lengths=key_lengths, scale=scale,
        check_device=not tracing))
    offsets, lengths = _int32(query_offset), _int32(key_lengths)
    scale = float(q.shape[-1] ** -0.5 if scale is None else scale)
    if not tracing:     # the same with numbers and tensors in the form that the native route takes
        out = C.native().window_attention(q, k, v, tuple(window), sinks, query_offset if offsets is None else offsets, lengths, scale,
                                          return_lse)
        if out is not None:
            return out
    left, right = (-1 if n is None else n for n in window)
    out, lse = torch.ops.tpf_b200.window_attn_fwd(q, k, v, offsets, lengths, 0 if offsets is not None else query_offset, left, right,
                                                  sinks, scale)
    return (out, lse) if return_lse else out
