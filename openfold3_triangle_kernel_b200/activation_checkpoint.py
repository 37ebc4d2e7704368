"""Activations kept in 8 bits between a forward and a backward pass.

Format: groups of 128 consecutive elements of a row (the last one ragged) share an fp32 scale.  With ``a`` the largest
magnitude of a group, ``code = rint(x * fl32(127 / a))`` (ties to even, the product exact), ``scale = fl32(a / 127)`` and
``value = code * scale``.  (The scale of ``a = FLT_MAX`` is one step less, so that no value overflows.)  A value is off by half a
step of the codes, ``a / 254``, and by the roundings of the two factors and the product, ``a 2^-21``, at most; one that is
given back in 16 bits is rounded to them, half a step of that type on top.  Groups with ``a < 2**-119`` are kept as zeros; a group
that holds an infinity or a NaN comes back as NaN.

* :func:`pack_activation` / :func:`unpack_activation`: the two directions, for any ``[*, C]`` in bf16, fp16 or fp32.
* :func:`int8_activations`: a context inside which autograd keeps large 16-bit activations in this format.
* ``checkpoint="int8"`` of :func:`turbo_layer_norm` and :func:`turbo_norm_linear`, whose kernels write the codes in the
  forward pass and read them in the backward pass, without a pass of their own.

None of them is differentiated.  Unsupported inputs raise ``ValueError("... unsupported [code]: reason")``, traced ones as in
:func:`turbo_layer_norm`.  The reference
has no counterpart: it keeps activations whole or computes them again (openfold3/core/utils/checkpointing.py).
"""
from __future__ import annotations

import torch

from . import _cabi as C
from ._checks import certain, differs, refuse
from .layer_norm import ROW_DTYPES
from .trimul import SupportResult

GROUP = 128
_MAX_GROUPS = 2 ** 31 - 1024
_SCALAR_TYPES = {torch.float16: 5, torch.float32: 6, torch.bfloat16: 15}  # c10::ScalarType


def _groups(cols):
    return -(-cols // GROUP)


def _countable(x):
    cols = x.shape[-1]
    if isinstance(cols, torch.SymInt):
        return True     # (a free size: the launch sees to it)
    return cols == 0 or (cols < 2 ** 31 - GROUP and not certain(x.numel() // cols * _groups(cols) >= _MAX_GROUPS))


def check_pack_support(x, *, check_device=True) -> SupportResult:
    """Metadata-only contract check of :func:`pack_activation`."""
    if not isinstance(x, torch.Tensor):
        return SupportResult(False, "x_type", "x must be a torch.Tensor")
    if x.ndim < 1:
        return SupportResult(False, "x_shape", "x must have shape [*,C]")
    if x.dtype not in ROW_DTYPES:
        return SupportResult(False, "x_dtype", "x must be BF16, FP16 or FP32")
    if not _countable(x):
        return SupportResult(False, "extent", "x must have fewer than 2^31 groups of 128 elements")
    if check_device:
        if not x.is_cuda:
            return SupportResult(False, "device", "x must be a CUDA tensor")
        if torch.cuda.get_device_capability(x.device)[0] != 10:
            return SupportResult(False, "device_arch", "these kernels require a Blackwell sm_100a device")
    return SupportResult(True, "ok", "supported")


def check_unpack_support(codes, scales, dtype, *, check_device=True) -> SupportResult:
    """Metadata-only contract check of :func:`unpack_activation`."""
    if not isinstance(codes, torch.Tensor) or not isinstance(scales, torch.Tensor):
        return SupportResult(False, "x_type", "codes and scales must be torch.Tensor instances")
    if codes.dtype != torch.int8 or scales.dtype != torch.float32:
        return SupportResult(False, "x_dtype", "codes must be int8 and scales FP32")
    if codes.ndim >= 1 and not _countable(codes):
        return SupportResult(False, "extent", "codes must have fewer than 2^31 groups of 128 elements")
    if codes.ndim < 1 or differs(scales.shape, tuple(codes.shape[:-1]) + (_groups(codes.shape[-1]),)):
        return SupportResult(False, "x_shape", "scales must have one entry per 128 elements of a row of codes")
    if dtype not in ROW_DTYPES:
        return SupportResult(False, "dtype", "dtype must be torch.bfloat16, float16 or float32")
    if scales.device != codes.device:
        return SupportResult(False, "device", "codes and scales must share one device")
    if check_device:
        if not codes.is_cuda:
            return SupportResult(False, "device", "codes and scales must be CUDA tensors")
        if torch.cuda.get_device_capability(codes.device)[0] != 10:
            return SupportResult(False, "device_arch", "these kernels require a Blackwell sm_100a device")
    return SupportResult(True, "ok", "supported")


@torch.library.custom_op("tpf_b200::int8_pack", mutates_args=())
def _int8_pack(x: torch.Tensor) -> list[torch.Tensor]:
    refuse("pack_activation", check_pack_support(x))
    return C.native().int8_pack_op(x)


@_int8_pack.register_fake
def _(x):
    refuse("pack_activation", check_pack_support(x, check_device=False))
    return [x.new_empty(x.shape, dtype=torch.int8),
            x.new_empty(x.shape[:-1] + (_groups(x.shape[-1]),), dtype=torch.float32)]


@torch.library.custom_op("tpf_b200::int8_unpack", mutates_args=())
def _int8_unpack(codes: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    refuse("unpack_activation", check_unpack_support(codes, scales, dtype))
    return C.native().int8_unpack_op(codes, scales, _SCALAR_TYPES[dtype])


@_int8_unpack.register_fake
def _(codes, scales, dtype):
    refuse("unpack_activation", check_unpack_support(codes, scales, dtype, check_device=False))
    return codes.new_empty(codes.shape, dtype=dtype)


def pack_activation(x):
    """``x [*, C]`` -> ``(codes int8 [*, C], scales fp32 [*, ceil(C / 128)])``."""
    if not torch.compiler.is_compiling():
        packed = C.native().int8_pack(x)
        if packed is not None:
            return packed
        refuse("pack_activation", check_pack_support(x))
    codes, scales = torch.ops.tpf_b200.int8_pack(x.detach())
    return codes, scales


def unpack_activation(codes, scales, dtype=torch.bfloat16):
    """The values that ``(codes, scales)`` of :func:`pack_activation` stand for, in ``dtype``."""
    if not torch.compiler.is_compiling():
        x = C.native().int8_unpack(codes, scales, dtype)
        if x is not None:
            return x
        refuse("unpack_activation", check_unpack_support(codes, scales, dtype))
    return torch.ops.tpf_b200.int8_unpack(codes, scales.detach(), dtype)


class _Packed:
    """A kept activation: its memory, flat, in 8 bits, and the size and strides to give it back with."""

    __slots__ = ("codes", "scales", "dtype", "size", "stride")

    def __init__(self, t):
        flat = t.as_strided((t.numel(),), (1,))
        self.codes, self.scales = pack_activation(flat.view(-1, GROUP) if flat.numel() % GROUP == 0 else flat)
        self.dtype, self.size, self.stride = t.dtype, t.size(), t.stride()

    def tensor(self):
        return unpack_activation(self.codes, self.scales, self.dtype).as_strided(self.size, self.stride)


def _is_dense(t):
    """Do the elements fill one stretch of memory, each once, in some order of the dimensions?"""
    expected = 1
    for stride, size in sorted((st, sz) for st, sz in zip(t.stride(), t.shape) if sz != 1):
        if stride != expected:
            return False
        expected *= size
    return True


# what makes a copy of a tensor in another type or arrangement (autograd numbers the overloads)
_COPIES = frozenset(n + "Backward" for n in ("ToCopy", "Clone", "T", "Transpose", "Permute", "View", "UnsafeView", "ReshapeAlias",
                                             "Expand", "Squeeze", "Unsqueeze", "Slice", "Select", "Split", "SplitWithSizes",
                                             "Unbind", "AsStrided", "Cat", "Stack"))
_MOST_COPIES = 256


def _is_parameter(t):
    """A parameter, trained or frozen; a view of one; a copy of trained ones (autocast and stacked projections make some)."""
    base = t if t._base is None else t._base
    if isinstance(base, torch.nn.Parameter) or (base.is_leaf and base.requires_grad):
        return True
    nodes, count = [t.grad_fn], 0
    while nodes:
        node, count = nodes.pop(), count + 1
        if node is None or node.name().rstrip("0123456789") not in _COPIES or count > _MOST_COPIES:
            return False
        nodes.extend(n for n, _ in node.next_functions if n is not None and n.name() != "torch::autograd::AccumulateGrad")
    return True


def _packable(t, min_elements):
    return (type(t) in (torch.Tensor, torch.nn.Parameter) and t.is_cuda and t.dtype in (torch.bfloat16, torch.float16)
            and t.layout == torch.strided and t.numel() >= min_elements and not _is_parameter(t)
            and not t.is_conj() and not t.is_neg() and _is_dense(t)
            and (t.numel() % GROUP == 0 or t.numel() < 2 ** 31 - GROUP)
            and torch.cuda.get_device_capability(t.device)[0] == 10)


def int8_activations(min_elements=65536, keep_whole=None):
    """Context manager: what autograd keeps inside it for the backward pass, it keeps in 8 bits and gives back as the values
    these stand for.

    A 16-bit tensor then takes 1 + 4 / 128 bytes an element in the place of 2, once for each node that keeps it: nothing is
    looked up by a tensor's address, which kernels and replayed graphs write to without autograd's knowledge.  What one node
    keeps (layer norm, activation function, one stacked projection) takes half; what two keep takes what it took, and an input
    of separate q, k, v and gate projections, which autograd holds once for all, twice that: stack them, or name it in
    ``keep_whole``.  The TriMul and the pair-stack block hold their intermediates in byte buffers of their own; of theirs,
    inputs and outputs are reached.

    This is done to bf16 and fp16 CUDA tensors of at least ``min_elements`` elements (the groups follow their memory order).
    fp32 tensors (statistics, log-sum-exps), parameters (``nn.Parameter``, frozen ones too, leaves that require gradients, views
    of either, and casts, transposes or concatenations of trained ones), tensors whose elements overlap or leave gaps, and
    tensors for which ``keep_whole(t)`` is true are kept as they are.  What else takes no gradient cannot be told from an
    activation: name a large constant table and a 16-bit copy of a frozen fp32 weight, as autocast makes it, in ``keep_whole``
    (or freeze the weight in 16 bits).  An activation that holds an infinity (logits behind a mask) would come back as NaN in
    its groups: keep such tensors whole.  An attention makes its probabilities again from the kept q and k, so what these are
    off by grows with the logits: gradients of :func:`turbo_attention` are off by 1.5 % of their norm at logits of a standard
    deviation of 1, 5 % at 4, 9 % at 8.
    """
    def pack(t):
        if not _packable(t, min_elements) or (keep_whole is not None and keep_whole(t)):
            return t
        return _Packed(t.detach())

    def unpack(kept):
        return kept.tensor() if isinstance(kept, _Packed) else kept

    return torch.autograd.graph.saved_tensors_hooks(pack, unpack)
