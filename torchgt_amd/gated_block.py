"""A pre-norm gated encoder layer: root-mean-square norm, gated projections, linears with activation and residual.

The reference's layers have LayerNorm and a feed-forward block of one projection and a GELU
(models/graphormer_dist_node_level.py:27-39, :276-314); what is here stands beside ``EncoderLayer`` and
``FeedForwardNetwork`` for models of any width, with the same ``forward`` signatures.  ``Graphormer(..., gated=True)``
builds its layers of it.  All of it runs on the library's kernels through ``torch.ops.torchgt.*``.

float32 or bfloat16, all tensors of one call of one type; sums and statistics in float32.  The ``_8bit`` functions take
rows of OCP e4m3 codes with a scale per row (``add_rms_norm_8bit`` for activations, ``quantize_rows`` for weights, once)
and have no gradients; their sums are off by at most 2^-10 of the largest of every eight neighbouring products (the matrix
instruction's alignment), far below what a code of four bits rounds.  Second derivatives and forward-mode tangents are refused.
"""
import torch
import torch.nn as nn

from . import _ext
from .module_tree import at_work
from .multi_head_attention import MultiHeadAttention

ACTIVATIONS = {None: 0, "gelu": 1, "relu": 2, "silu": 3}      # TGT_ACT_* of include/torchgt_hip.h


def _act(name, op):
    if name not in ACTIVATIONS:
        raise ValueError(f"{op}: unknown activation {name!r} (None, 'gelu', 'relu' or 'silu')")
    return ACTIVATIONS[name]


def add_rms_norm(x, residual, weight, eps=1e-6):
    """``(s, y)`` with ``s = x + residual`` in x's type and ``y = s / sqrt(mean(s * s) + eps) * weight`` over the last dimension.
    ``residual`` may be None (s is x then).  1 to 16384 features."""
    return _ext.op("add_rms_norm")(x, residual, weight, float(eps))


def add_rms_norm_8bit(x, residual, weight, eps=1e-6):
    """``(s, codes, scales)``: the same with ``y`` as float8_e4m3fn codes and one float32 scale per row,
    ``y ~ codes * scales[..., None]``.  A scale is the smallest power of two that brings the row's largest magnitude to at
    most 448 (1 for a row of zeros, never below 2^-126)."""
    return _ext.op("add_rms_norm_8bit")(x, residual, weight, float(eps))


def quantize_rows(w):
    """``(codes, scales)`` of a float32 or bfloat16 matrix, row by row, as ``add_rms_norm_8bit`` makes them."""
    return _ext.op("quantize_rows")(w)


def gated_linear(x, gate_weight, up_weight, gate_bias=None, up_bias=None, activation="silu"):
    """``act(x gate_weight^T + gate_bias) * (x up_weight^T + up_bias)`` for x ``[..., in]`` and weights ``[out, in]``: both
    products, the activation and the product of the two in one kernel.  Kept for the backward: the inputs, and from 512 features
    on (float32: 128; except for small weights) both projections, 2 ``out`` values a row; else the backward forms them again.
    activation: 'silu', 'gelu' (exact erf form), 'relu' or None."""
    return _ext.op("gated_linear")(x, gate_weight, up_weight, gate_bias, up_bias, _act(activation, "gated_linear"))


def gated_linear_8bit(x, x_scales, gate_weight, gate_scales, up_weight, up_scales, gate_bias=None, up_bias=None, activation="silu",
                      dtype=torch.bfloat16):
    """``gated_linear`` on codes with scales: x ``[..., in]`` with x_scales ``[...]``, weights ``[out, in]`` with scales ``[out]``.
    Biases and the result are of ``dtype`` (bfloat16 or float32); ``in`` is a multiple of 16."""
    return _ext.op("gated_linear_8bit")(x, x_scales, gate_weight, gate_scales, up_weight, up_scales, gate_bias, up_bias,
                                        _act(activation, "gated_linear_8bit"), dtype)


def linear_act(x, weight, bias=None, activation=None, residual=None):
    """``act(x weight^T + bias) + residual`` for x ``[..., in]``, weight ``[out, in]``, residual ``[..., out]``, in one kernel."""
    return _ext.op("linear_act")(x, weight, bias, residual, _act(activation, "linear_act"))


def linear_act_8bit(x, x_scales, weight, weight_scales, bias=None, activation=None, residual=None, dtype=torch.bfloat16):
    """``linear_act`` on codes with scales; bias, residual and the result are of ``dtype``; ``in`` is a multiple of 16."""
    return _ext.op("linear_act_8bit")(x, x_scales, weight, weight_scales, bias, residual, _act(activation, "linear_act_8bit"), dtype)


class RMSNorm(nn.Module):
    """``add_rms_norm`` with its weight: ``forward(x, residual=None)`` gives y, or (s, y) with a residual."""

    def __init__(self, hidden_size, eps=1e-6):
        super().__init__()
        self.weight = nn.Parameter(torch.ones(hidden_size))
        self.eps = eps

    def forward(self, x, residual=None):
        s, y = add_rms_norm(x, residual, self.weight, self.eps)
        return y if residual is None else (s, y)


class GatedFeedForwardNetwork(nn.Module):
    """``down(act(gate(x)) * up(x))``; ``forward(x, residual)`` adds the residual in the last product's kernel."""

    def __init__(self, hidden_size, ffn_size, activation="silu", bias=True):
        super().__init__()
        _act(activation, "GatedFeedForwardNetwork")
        self.gate = nn.Linear(hidden_size, ffn_size, bias=bias)
        self.up = nn.Linear(hidden_size, ffn_size, bias=bias)
        self.down = nn.Linear(ffn_size, hidden_size, bias=bias)
        self.activation = activation

    def forward(self, x, residual=None):
        h = gated_linear(x, self.gate.weight, self.up.weight, self.gate.bias, self.up.bias, self.activation)
        return linear_act(h, self.down.weight, self.down.bias, residual=residual)


class GatedEncoderLayer(nn.Module):
    """``EncoderLayer`` with RMSNorm and the gated feed-forward block, called in the same way.

    Where no dropout is at work behind the block its residual is added in the last product, also with
    ``defer_residual=True``: (sum, None) comes back then, and the next norm has one tensor less to read and to write."""

    def __init__(self, hidden_size, ffn_size, dropout_rate, attention_dropout_rate, num_heads, attn_bias_dim, activation="silu"):
        super().__init__()
        self.self_attention_norm = RMSNorm(hidden_size)
        self.self_attention = MultiHeadAttention(hidden_size, attention_dropout_rate, num_heads, attn_bias_dim)
        self.self_attention_dropout = nn.Dropout(dropout_rate)
        self.ffn_norm = RMSNorm(hidden_size)
        self.ffn = GatedFeedForwardNetwork(hidden_size, ffn_size, activation)
        self.ffn_dropout = nn.Dropout(dropout_rate)

    def forward(self, x, attn_bias=None, edge_index=None, attn_type=None, residual=None, defer_residual=False):
        n1, n2 = self.self_attention_norm, self.ffn_norm
        x, y = add_rms_norm(x, residual, n1.weight, n1.eps)
        y = self.self_attention(y, attn_bias, edge_index, attn_type=attn_type)
        y = self.self_attention_dropout(y)
        x, y = add_rms_norm(x, y, n2.weight, n2.eps)
        if not at_work(self.ffn_dropout):
            x = self.ffn(y, residual=x)
            return (x, None) if defer_residual else x
        y = self.ffn_dropout(self.ffn(y))
        return (x, y) if defer_residual else x + y
