"""B200 (sm_100a) triangle attention and triangle multiplicative update.

Public operators: :func:`turbo_attention`, :func:`turbo_trimul` (same contracts as
the TurboPairFormer operators of the same names), and the row-wise operators around them in training:
:func:`turbo_layer_norm`, :func:`turbo_norm_linear` and activations kept in 8 bits (:func:`pack_activation`,
:func:`unpack_activation`, :func:`int8_activations`).  The device is reached only
through ``libtpf_b200.so`` (C ABI, ``include/tpf_b200.h``); there is no fallback.
"""
from . import _cabi
from .activation_checkpoint import int8_activations, pack_activation, unpack_activation
from .attention import is_turbo_attention_supported, turbo_attention
from .layer_norm import check_layer_norm_support, turbo_layer_norm
from .norm_linear import check_norm_linear_support, turbo_norm_linear
from .trimul import check_trimul_support, turbo_trimul

__all__ = ["turbo_attention", "turbo_trimul", "turbo_layer_norm", "turbo_norm_linear", "pack_activation",
           "unpack_activation", "int8_activations", "is_turbo_attention_supported", "check_trimul_support",
           "check_layer_norm_support", "check_norm_linear_support", "_cabi"]
