"""``turbo_rotary`` and ``turbo_qk_norm_rotary``: the position rotation of attention heads on B200, alone or behind an RMS norm of
every head of q and k in the same pass.

Operator contract:

* ``x``, ``q``, ``k``: bf16, fp16 or fp32 ``[*, N, H, D]``, ``2 <= D <= 256``; k has q's sizes but for its heads.  Slices of a stacked
  projection (any strides of the tokens and heads) are read in place.
* ``frequencies``: from :func:`rotary_frequencies`, for the first R elements of a head; the others are not rotated.
* ``positions``: ``None`` (0, 1, ...), an ``int`` (the first token's), or an integer tensor that broadcasts to ``[*, N]``.
* ``layout``: ``"half"`` rotates element i with i + R / 2, ``"interleaved"`` 2 i with 2 i + 1.
* the norm: ``x / sqrt(mean(x^2) + eps) * weight``, ``weight`` ``[D]`` of any of the three types or ``None`` (ones).
* returns x's type, contiguous; autograd for x, q, k and the weights (a gradient has its parameter's type), first order,
  reverse mode only.  The norm keeps q and k for the backward pass, the rotation alone nothing.  All arithmetic is fp32, sums have a
  fixed order: the same inputs give the same bits.
* angles: position times ``turns`` is exact modulo a turn, at any position; what goes to the sine and cosine is that number rounded to
  fp32, off by 2^-26 of a turn at most.  The ``turns`` that :func:`rotary_frequencies` makes are off by what it computes in 64-bit
  floats, about 2^-51 of themselves, which a position multiplies (below 2^-26 of a turn up to position 2^26).

Unsupported inputs raise ``ValueError("turbo_rotary unsupported [code]: reason")`` (``turbo_qk_norm_rotary`` likewise), in a traced
call when it is traced or, for sizes that are free there, when it runs.  The reference has no counterpart.
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional

import torch

from . import _cabi as C
from ._checks import NO_TANGENT, certain, differs, has_tangent, refuse
from .layer_norm import MAX_EPS, ROW_DTYPES, check_parameter
from .trimul import SupportResult

MAX_HEAD_DIM = 256
_MOST_ROWS = 2 ** 31 - 256   # tokens of all batches times heads
_MOST_HEADS = 2 ** 24 - 1    # of q and k together
LAYOUTS = ("half", "interleaved")
SCALINGS = (None, "linear", "ntk", "yarn")


class RotaryFrequencies(NamedTuple):
    """``turns``: int64 ``[R / 2]``, what a pair turns from one position to the next, as a fraction of 2^64 of a turn.
    ``magnitude``: the factor of the rotated elements."""

    turns: torch.Tensor
    magnitude: float = 1.0


def rotary_frequencies(dim, base=10000.0, *, scaling=None, factor=1.0, original_length=None, beta_fast=32.0, beta_slow=1.0,
                       magnitude=None, device=None) -> RotaryFrequencies:
    """Frequencies ``base ** (-2 i / dim)`` radians a position, of ``dim`` rotated elements.

    For contexts longer than the ``original_length`` that a model was trained with, by ``factor`` (>= 1): ``"linear"`` divides every
    frequency; ``"ntk"`` raises the base so that the slowest pair is slowed down by the factor; ``"yarn"`` (Peng et al. 2023)
    keeps pairs that turn more than ``beta_fast`` times over the original length, divides those that turn less than
    ``beta_slow`` times, with a ramp between, and has the magnitude ``0.1 ln(factor) + 1``.  ``magnitude`` replaces the factor of
    the rotated elements.
    """
    number = lambda n: isinstance(n, (int, float)) and not isinstance(n, bool) and math.isfinite(n)  # noqa: E731
    if not (isinstance(dim, int) and dim >= 2 and dim % 2 == 0):
        raise ValueError("rotary_frequencies: dim must be even and positive")
    if not (number(base) and base > 1):
        raise ValueError("rotary_frequencies: base must be above 1")
    if scaling not in SCALINGS:
        raise ValueError(f"rotary_frequencies: scaling must be one of {SCALINGS}")
    if not (number(factor) and factor >= 1):
        raise ValueError("rotary_frequencies: factor must be at least 1")
    if magnitude is not None and not number(magnitude):
        raise ValueError("rotary_frequencies: magnitude must be a number")
    if scaling == "ntk" and dim > 2:
        base = base * factor ** (dim / (dim - 2))
    radians = [base ** (-2.0 * i / dim) for i in range(dim // 2)]
    default = 1.0
    if scaling == "linear":
        radians = [f / factor for f in radians]
    elif scaling == "yarn":
        if not (number(original_length) and original_length >= 1):
            raise ValueError("rotary_frequencies: yarn needs the original_length")
        if not (number(beta_fast) and number(beta_slow) and beta_fast > beta_slow > 0):
            raise ValueError("rotary_frequencies: beta_fast must be above beta_slow, both positive")
        pair = lambda turns: dim * math.log(original_length / (2 * math.pi * turns)) / (2 * math.log(base))  # noqa: E731
        low, high = max(math.floor(pair(beta_fast)), 0), min(math.ceil(pair(beta_slow)), dim - 1)
        slowed = [min(max((i - low) / max(high - low, 1e-3), 0.0), 1.0) for i in range(dim // 2)]
        radians = [f * (1 - s) + f / factor * s for f, s in zip(radians, slowed)]
        default = 0.1 * math.log(factor) + 1.0
    turns = [round(f / (2 * math.pi) * 2.0 ** 64) for f in radians]
    turns = torch.tensor([t - 2 ** 64 if t >= 2 ** 63 else t for t in turns], dtype=torch.int64, device=device)
    return RotaryFrequencies(turns, default if magnitude is None else float(magnitude))


# --------------------------------------------------------------------------------------
# contract
# --------------------------------------------------------------------------------------
def _check(named, weights, turns, magnitude, positions, layout, eps, check_device):
    """``named``: [(name, tensor)], the first one sets type and device; the first failure."""
    first_name, x = named[0]
    for name, t in named:
        if not isinstance(t, torch.Tensor) or t.ndim < 3:
            return SupportResult(False, "x_shape", f"{name} must have shape [*,N,H,D]")
    if x.dtype not in ROW_DTYPES:
        return SupportResult(False, "x_dtype", f"{first_name} must be BF16, FP16 or FP32")
    if certain(x.shape[-1] < 2) or certain(x.shape[-1] > MAX_HEAD_DIM):
        return SupportResult(False, "head_dim", f"heads of 2 to {MAX_HEAD_DIM} elements")
    for name, t in named[1:]:
        if t.dtype != x.dtype or t.device != x.device:
            return SupportResult(False, "x_dtype", f"{name} must have {first_name}'s type and device")
        if t.ndim != x.ndim or differs(t.shape[:-2] + t.shape[-1:], x.shape[:-2] + x.shape[-1:]):
            return SupportResult(False, "x_shape", f"{name} must have {first_name}'s sizes but for the heads")
    if any(certain(math.prod(t.shape[:-1]) > _MOST_ROWS) for _, t in named) or certain(sum(t.shape[-2] for _, t in named) > _MOST_HEADS):
        return SupportResult(False, "tokens", "too many tokens and heads")
    for name, w in weights:
        bad = check_parameter(name, w, x.shape[-1], x)
        if bad is not None:
            return bad
    if not isinstance(turns, torch.Tensor) or turns.dtype != torch.int64 or turns.ndim != 1 or certain(turns.shape[0] < 1):
        return SupportResult(False, "frequencies", "frequencies must come from rotary_frequencies")
    if certain(2 * turns.shape[0] > x.shape[-1]):
        return SupportResult(False, "frequencies", "the rotated part must not exceed a head")
    if turns.device != x.device:
        return SupportResult(False, "frequencies", f"frequencies must live on {first_name}'s device")
    if not (isinstance(magnitude, (int, float)) and -MAX_EPS <= magnitude <= MAX_EPS):
        return SupportResult(False, "frequencies", "the magnitude must be a finite number")
    if positions is not None:
        if not isinstance(positions, torch.Tensor) or positions.dtype not in (torch.int32, torch.int64):
            return SupportResult(False, "positions", "positions must be None, an int, or an INT32 or INT64 tensor")
        if positions.device != x.device:
            return SupportResult(False, "positions", f"positions must live on {first_name}'s device")
        lead = tuple(x.shape[:-2])
        if positions.ndim > len(lead) or any(certain(a != 1) and certain(a != b)
                                             for a, b in zip(positions.shape[::-1], lead[::-1])):
            return SupportResult(False, "positions", "positions must broadcast to [*,N]")
    if layout not in LAYOUTS:
        return SupportResult(False, "layout", f"layout must be one of {LAYOUTS}")
    if not (isinstance(eps, (int, float)) and 0 <= eps <= MAX_EPS):
        return SupportResult(False, "eps", "eps must be a finite FP32 number, not negative")
    if has_tangent(*(t for _, t in named), *(w for _, w in weights)):
        return SupportResult(False, "tangent", NO_TANGENT)
    if check_device:
        if not x.is_cuda:
            return SupportResult(False, "device", f"{first_name} must be a CUDA tensor")
        if torch.cuda.get_device_capability(x.device)[0] != 10:
            return SupportResult(False, "device_arch", "these kernels require a Blackwell sm_100a device")
    return SupportResult(True, "ok", "supported")


def _parts(frequencies, positions):
    """``(turns, magnitude, positions tensor or None, first position)``."""
    turns, magnitude = frequencies if isinstance(frequencies, tuple) and len(frequencies) == 2 else (None, 1.0)
    if not isinstance(magnitude, (int, float)):
        turns = None
    if positions is None:
        return turns, magnitude, None, 0
    if isinstance(positions, (int, torch.SymInt)) and not isinstance(positions, bool) and -2 ** 62 <= positions <= 2 ** 62:
        return turns, magnitude, None, positions
    return turns, magnitude, positions, 0


def check_rotary_support(x, frequencies, positions=None, *, layout="half", check_device=True) -> SupportResult:
    """Metadata-only contract check of :func:`turbo_rotary`; returns the first failure."""
    turns, magnitude, positions, _ = _parts(frequencies, positions)
    return _check([("x", x)], [], turns, magnitude, positions, layout, 0.0, check_device)


def check_qk_norm_rotary_support(q, k, q_weight, k_weight, frequencies, positions=None, *, eps=1e-6, layout="half",
                                 check_device=True) -> SupportResult:
    """Metadata-only contract check of :func:`turbo_qk_norm_rotary`; returns the first failure."""
    turns, magnitude, positions, _ = _parts(frequencies, positions)
    return _check([("q", q), ("k", k)], [("q_weight", q_weight), ("k_weight", k_weight)], turns, magnitude, positions, layout, eps,
                  check_device)


# --------------------------------------------------------------------------------------
# custom ops: what a traced graph holds.  An eager call on plain CUDA tensors goes to `_native.rotary`.
# --------------------------------------------------------------------------------------
def _refuse_op(named, qw, kw, turns, positions, magnitude, half, norm, eps, check_device):
    name = "turbo_qk_norm_rotary" if norm else "turbo_rotary"
    check = lambda device: _check(named, [("q_weight", qw), ("k_weight", kw)], turns, magnitude, positions,  # noqa: E731
                                  "half" if half else "interleaved", eps, device)
    refuse(name, check(False))
    if positions is not None and (positions.dtype != torch.int64 or differs(positions.shape, tuple(named[0][1].shape[:-2]))):
        refuse(name, SupportResult(False, "positions", "the operator takes INT64 positions of q's tokens"))
    if check_device:
        refuse(name, check(True))


@torch.library.custom_op("tpf_b200::rotary_fwd", mutates_args=())
def _rotary_fwd(q: torch.Tensor, k: Optional[torch.Tensor], qw: Optional[torch.Tensor], kw: Optional[torch.Tensor],
                turns: torch.Tensor, positions: Optional[torch.Tensor], first: int, magnitude: float, half: bool, norm: bool,
                eps: float) -> list[torch.Tensor]:
    _refuse_op([("q", q)] + ([("k", k)] if k is not None else []), qw, kw, turns, positions, magnitude, half, norm, eps, True)
    return C.native().rotary_fwd(q, k, qw, kw, turns, positions, first, magnitude, half, norm, eps)


@_rotary_fwd.register_fake
def _(q, k, qw, kw, turns, positions, first, magnitude, half, norm, eps):
    _refuse_op([("q", q)] + ([("k", k)] if k is not None else []), qw, kw, turns, positions, magnitude, half, norm, eps, False)
    return [q.new_empty(q.shape), q.new_empty((0,)) if k is None else k.new_empty(k.shape)]


@torch.library.custom_op("tpf_b200::rotary_bwd", mutates_args=())
def _rotary_bwd(dq: Optional[torch.Tensor], dk: Optional[torch.Tensor], q: Optional[torch.Tensor], k: Optional[torch.Tensor],
                qw: Optional[torch.Tensor], kw: Optional[torch.Tensor], turns: torch.Tensor, positions: Optional[torch.Tensor],
                first: int, magnitude: float, half: bool, norm: bool, eps: float) -> list[torch.Tensor]:
    _refuse_bwd(dq, dk, q, k, qw, kw, turns, positions, magnitude, half, norm, eps, True)
    return C.native().rotary_bwd(dq, dk, q, k, qw, kw, turns, positions, first, magnitude, half, norm, eps)


def _refuse_bwd(dq, dk, q, k, qw, kw, turns, positions, magnitude, half, norm, eps, check_device):
    named = [(n, t) for n, t in (("dq", dq), ("dk", dk)) if t is not None]
    if not named:
        refuse("rotary backward", SupportResult(False, "d_out", "a gradient is needed"))
    for d, x in ((dq, q), (dk, k)):
        if norm and d is not None and (x is None or x.dtype != d.dtype or differs(x.shape, tuple(d.shape))
                                       or x.device != d.device):
            refuse("rotary backward", SupportResult(False, "x_shape", "x does not belong to this gradient"))
    _refuse_op(named, qw, kw, turns, positions, magnitude, half, norm, eps, check_device)


@_rotary_bwd.register_fake
def _(dq, dk, q, k, qw, kw, turns, positions, first, magnitude, half, norm, eps):
    _refuse_bwd(dq, dk, q, k, qw, kw, turns, positions, magnitude, half, norm, eps, False)
    some = dq if dq is not None else dk
    like = lambda t, e: e.new_empty((0,)) if t is None else t.new_empty(t.shape)  # noqa: E731
    f32 = some.new_empty((0,), dtype=torch.float32)
    return [like(dq, some), like(dk, some), like(qw, f32), like(kw, f32)]


def _setup_context(ctx, inputs, output):
    q, k, qw, kw, turns, positions, *ctx.numbers = inputs
    norm = ctx.numbers[3]
    ctx.save_for_backward(q if norm else None, k if norm else None, qw, kw, turns, positions)
    ctx.has_k = k is not None
    ctx.set_materialize_grads(False)


def _backward(ctx, grads):
    dq, dk = grads[0], grads[1] if ctx.has_k else None
    if dq is None and dk is None:
        return (None,) * 11
    q, k, qw, kw, turns, positions = ctx.saved_tensors
    gq, gk, gqw, gkw = torch.ops.tpf_b200.rotary_bwd(dq, dk, q, k, qw, kw, turns, positions, *ctx.numbers)
    return (gq if dq is not None else None, gk if dk is not None else None, None if qw is None else gqw, None if kw is None else gkw,
            *(None,) * 7)


_rotary_fwd.register_autograd(_backward, setup_context=_setup_context)


# --------------------------------------------------------------------------------------
# public operators
# --------------------------------------------------------------------------------------
def _full_positions(positions, x):
    """int64, contiguous, one for each token."""
    lead = x.shape[:-2]
    if positions is None or (positions.dtype == torch.int64 and positions.shape == lead and positions.is_contiguous()):
        return positions
    return positions.to(torch.int64).expand(lead).contiguous()


def turbo_rotary(x, frequencies, positions=None, *, layout="half"):
    """The position rotation of ``x [*, N, H, D]``; see the module docstring for the contract."""
    turns, magnitude, positions, first = _parts(frequencies, positions)
    tracing = torch.compiler.is_compiling()
    if not tracing and turns is not None and layout in LAYOUTS and (positions is None or isinstance(positions, torch.Tensor)):
        out = C.native().rotary(x, None, None, None, turns, positions, first, magnitude, layout == "half", False, 0.0)
        if out is not None:
            return out
    refuse("turbo_rotary", _check([("x", x)], [], turns, magnitude, positions, layout, 0.0, not tracing))
    positions = _full_positions(positions, x)
    if not tracing:
        out = C.native().rotary(x, None, None, None, turns, positions, first, magnitude, layout == "half", False, 0.0)
        if out is not None:
            return out
    return torch.ops.tpf_b200.rotary_fwd(x, None, None, None, turns, positions, first, magnitude, layout == "half", False, 0.0)[0]


def turbo_qk_norm_rotary(q, k, q_weight, k_weight, frequencies, positions=None, *, eps=1e-6, layout="half"):
    """RMS norm of every head of q and k and the position rotation, in one pass: ``(q, k)``; see the module docstring."""
    turns, magnitude, positions, first = _parts(frequencies, positions)
    tracing = torch.compiler.is_compiling()
    good = isinstance(eps, (int, float)) and eps <= MAX_EPS and layout in LAYOUTS and k is not None
    if not tracing and good and turns is not None and (positions is None or isinstance(positions, torch.Tensor)):
        out = C.native().rotary(q, k, q_weight, k_weight, turns, positions, first, magnitude, layout == "half", True, eps)
        if out is not None:
            return out
    refuse("turbo_qk_norm_rotary", _check([("q", q), ("k", k)], [("q_weight", q_weight), ("k_weight", k_weight)], turns, magnitude,
                                          positions, layout, eps, not tracing))
    positions = _full_positions(positions, q)
    if not tracing:
        out = C.native().rotary(q, k, q_weight, k_weight, turns, positions, first, magnitude, layout == "half", True, eps)
        if out is not None:
            return out
    return tuple(torch.ops.tpf_b200.rotary_fwd(q, k, q_weight, k_weight, turns, positions, first, magnitude, layout == "half", True,
                                               float(eps)))
