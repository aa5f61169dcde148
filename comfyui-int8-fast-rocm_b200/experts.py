"""Mixture-of-experts feed-forward on quantised weights: the router, the
experts' two products and the weighted sum, composed from the operators of
:mod:`library`.  No counterpart in the reference, whose linears are dense.

Weights are per-expert stacks of the package's own formats: int8 with one
scale a row (``int8_tensorwise``), or packed int4 with one scale a row or per
128 k.  ConvRot layers work the same way: the weights are rotated when they
are quantised (``rot=(kind, group)``) and the activation before each product.
"""
from __future__ import annotations

import torch
from torch import Tensor

from . import library as kops  # the kernels as registered torch.library operators


def quantize_experts_int8(weight: Tensor, rot=None):
    """[E, N, K] float -> (int8 [E, N, K], float32 [E, N]), each expert as
    ``quantize_int8_axiswise(dim=1)`` of its (rotated) weight."""
    E, Nn, K = weight.shape
    q, s = kops.quant_weight_int8(weight.reshape(E * Nn, K), rot)
    return q.reshape(E, Nn, K), s.reshape(E, Nn)


def quantize_experts_int4(weight: Tensor, rot=None, group: int = 0):
    """[E, N, K] float -> (packed int4 [E, N, K/2], scales float32 [E, N] for
    group 0 or [E, N, K/128] for group 128)."""
    E, Nn, K = weight.shape
    p, s = kops.quant_weight_int4(weight.reshape(E * Nn, K), rot, group)
    return p.reshape(E, Nn, K // 2), s.reshape((E, Nn) if group == 0 else (E, Nn, K // 128))


def _tokens(x: Tensor, logits: Tensor, residual):
    x2 = x.reshape(-1, x.shape[-1])
    l2 = logits.reshape(-1, logits.shape[-1])
    if l2.shape[0] != x2.shape[0]:
        raise ValueError(f"{x2.shape[0]} tokens but {l2.shape[0]} rows of logits")
    if residual is not None:  # (-1 stands for any number where there are no tokens)
        residual = residual.reshape(x2.shape[0], -1 if x2.shape[0] else residual.shape[-1])
    return x2, l2, residual


@torch.no_grad()
def int8_forward_experts(x: Tensor, logits: Tensor, up: Tensor, up_scale: Tensor, down: Tensor, down_scale: Tensor,
                         top_k: int, *, scoring: str = "softmax", renormalize: bool = True, up_bias=None,
                         down_bias=None, residual=None, rot=None, down_rot=None) -> Tensor:
    """W8A8 mixture-of-experts feed-forward with the SiTU gated activation:
    per token ``sum_e weight_e * down_e(situ(up_e(x)))`` (+ ``residual``)
    over its ``top_k`` experts, ``x`` [..., K] (bf16/f16), ``logits`` [..., E],
    ``up`` [E, 2F, K] ([hidden | gate] rows), ``down`` [E, K', F] int8.  The
    tokens are quantised once and gathered by the first product; the
    activation is part of the second product's quantiser."""
    x2, l2, res = _tokens(x, logits, residual)
    _, weights, offsets, rows, pos = kops.route_experts(l2, top_k, scoring, renormalize)
    xq, xs = kops.quant_act_int8(x2, rot)
    h = kops.gemm_w8a8_grouped(xq, xs, up, up_scale, offsets, rows, up_bias, x.dtype)
    hq, hs = kops.quant_act_int8_situ(h, down_rot)
    y = kops.gemm_w8a8_grouped(hq, hs, down, down_scale, offsets, None, down_bias, x.dtype)
    return kops.combine_experts(y, weights, pos, res).reshape(*x.shape[:-1], down.shape[1])


@torch.no_grad()
def w4_forward_experts(x: Tensor, logits: Tensor, up: Tensor, up_scale: Tensor, down: Tensor, down_scale: Tensor,
                       top_k: int, *, scoring: str = "softmax", renormalize: bool = True, up_bias=None,
                       down_bias=None, residual=None, rot=None, down_rot=None) -> Tensor:
    """:func:`int8_forward_experts` for few tokens on packed 4-bit weights
    (``up`` [E, 2F, K/2], ``down`` [E, K', F/2]), the activations kept in
    their dtype (bf16/f16/f32)."""
    x2, l2, res = _tokens(x, logits, residual)
    _, weights, offsets, rows, pos = kops.route_experts(l2, top_k, scoring, renormalize)
    if rot is not None:
        x2 = kops.rotate(x2, *rot)
    h = kops.situ(kops.matvec_w4(x2, up, up_scale, up_bias, offsets, rows))
    if down_rot is not None:
        h = kops.rotate(h, *down_rot)
    y = kops.matvec_w4(h, down, down_scale, down_bias, offsets)
    return kops.combine_experts(y, weights, pos, res).reshape(*x.shape[:-1], down.shape[1])
