"""B200 (sm_100a) triangle attention and triangle multiplicative update.

Public operators: :func:`turbo_attention`, :func:`turbo_trimul` (same contracts as
the TurboPairFormer operators of the same names), and the row-wise operators around them in training:
:func:`turbo_layer_norm`, :func:`turbo_norm_linear` and activations kept in 8 bits (:func:`pack_activation`,
:func:`unpack_activation`, :func:`int8_activations`); dropout with the residual (:func:`turbo_dropout`), and
the operators of a sequence attention (:func:`turbo_rotary`, :func:`turbo_qk_norm_rotary`, :func:`turbo_window_attention`).
:func:`pair_stack_block` composes the pair stack of the first two, with or without dropout.  The device is reached only
through ``libtpf_b200.so`` (C ABI, ``include/tpf_b200.h``); there is no fallback.
"""
from . import _cabi
from .activation_checkpoint import int8_activations, pack_activation, unpack_activation
from .attention import is_turbo_attention_supported, turbo_attention
from .dropout import check_dropout_support, turbo_dropout
from .layer_norm import check_layer_norm_support, turbo_layer_norm
from .norm_linear import check_norm_linear_support, turbo_norm_linear
from .pair_block import pair_stack_block
from .rotary import (RotaryFrequencies, check_qk_norm_rotary_support, check_rotary_support, rotary_frequencies,
                     turbo_qk_norm_rotary, turbo_rotary)
from .trimul import check_trimul_support, turbo_trimul
from .window_attention import check_window_attention_support, turbo_window_attention

__all__ = ["turbo_attention", "turbo_trimul", "turbo_layer_norm", "turbo_norm_linear", "pack_activation",
           "unpack_activation", "int8_activations", "is_turbo_attention_supported", "check_trimul_support",
           "check_layer_norm_support", "check_norm_linear_support", "turbo_dropout", "check_dropout_support",
           "pair_stack_block", "turbo_rotary", "turbo_qk_norm_rotary", "RotaryFrequencies", "rotary_frequencies", "check_rotary_support",
           "check_qk_norm_rotary_support", "turbo_window_attention", "check_window_attention_support", "_cabi"]
