"""Routing, grouped products and their sum for layers of quantized experts.

The reference runs a mixture-of-experts layer as a loop over its experts
(QATMoELayer.forward, src/qat/qat_moe_layer.py:85-116): each expert picks its
tokens, multiplies by its quantized weights and adds its part.  Here a layer is

    route = moe_route(router_logits, top_k)
    h = grouped_matmul(x, W_gate_up, route.offsets, rows=route.rows, slots=route.slots)
    ...
    y = grouped_matmul(h, W_down, route.offsets)
    out = moe_combine(y, route.weights, route.rows, route.slots)

with W (E, out, in) the stacked results of bcjr_quantize_experts.  All of it is
on the device, sized by T * top_k alone: no count is read back, so a step can be
captured into a graph.  Every operator is differentiable; equal calls give equal
bits.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib

_ops = _lib.load_ops()


class MoERoute(NamedTuple):
    """T tokens' choice of experts, sorted by expert (M = T * top_k places)."""
    weights: torch.Tensor  # (T, top_k) float32, differentiable; 0 where there is no expert
    experts: torch.Tensor  # (T, top_k) int32, by descending logit; -1 for none
    offsets: torch.Tensor  # (E + 1,) int32: expert e has the places [offsets[e], offsets[e + 1])
    rows: torch.Tensor     # (M,) int32: token of each place, -1 behind offsets[E]
    slots: torch.Tensor    # (T, top_k) int32: place of each pair, -1 for none


def _gpu(what: str, t: torch.Tensor) -> None:
    if not t.is_cuda:
        raise AssertionError(f"{what} runs on the GPU; got a tensor on {t.device}")


def moe_route(logits, top_k, *, renormalize=False, valid=None):
    """Send every token to its top_k experts.

    logits: (T, E) router logits, float32, bfloat16 or float16, E <= 1024; a logit
            of -inf is never chosen.
    top_k:  1 <= top_k <= min(E, 64).
    renormalize: weights are the softmax over the chosen experts, not over all.
    valid:  (T,) bool or None: a token that is False (padding) gets no expert.

    Ties go to the lowest expert.  A token with fewer than top_k experts above
    -inf has -1 (weight 0, slot -1) for the rest.  The choice itself has no
    gradient; weights have."""
    _gpu("moe_route", logits)
    if logits.dim() != 2:
        raise AssertionError(f"logits must be (T, E); got {tuple(logits.shape)}")
    if not 1 <= top_k <= logits.shape[1]:
        raise AssertionError(f"top_k={top_k} outside [1, E={logits.shape[1]}]")
    if valid is not None and (valid.dtype != torch.bool or tuple(valid.shape) != (logits.shape[0],)):
        raise AssertionError(f"valid must be ({logits.shape[0]},) bool; got {tuple(valid.shape)} {valid.dtype}")
    return MoERoute(*_lib.run_op(_ops.moe_route, logits, valid, top_k, renormalize))


def grouped_matmul(x, w, offsets, *, rows=None, slots=None):
    """y (M, N): row p of y is w[e] times row p of x, e the expert whose places
    [offsets[e], offsets[e + 1]) hold p; zeros behind offsets[E].

    x:       (M, K) bfloat16 or float16 in sorted order or, with rows, (T, K):
             place p takes row rows[p] (a place outside [0, T) a row of zeros).
    w:       (E, N, K), x's type or float32 (rounded to x's type as it is read;
             its gradient stays float32).  A program that serves fixed
             float32 weights rounds them once itself: half the bytes a call.
    offsets: (E + 1,) int32 on the device, ascending, from 0.
    rows, slots: of moe_route; slots (T, k), the places of each row, are needed
             for the gradient of a gathered x.

    Products are summed in float32 and rounded once."""
    _gpu("grouped_matmul", x)
    if x.dim() != 2 or w.dim() != 3 or x.shape[1] != w.shape[2]:
        raise AssertionError(f"x must be (rows, K) and w (E, N, K); got {tuple(x.shape)}, {tuple(w.shape)}")
    if tuple(offsets.shape) != (w.shape[0] + 1,):
        raise AssertionError(f"offsets must be (E+1={w.shape[0] + 1},); got {tuple(offsets.shape)}")
    if w.dtype != x.dtype and w.dtype != torch.float32:
        raise AssertionError(f"w must be {x.dtype} like x, or float32; got {w.dtype}")
    return _lib.run_op(_ops.grouped_matmul, x, w, offsets, rows, slots)


def moe_combine(y, weights, rows, slots):
    """out (T, N): out[t] = sum_j weights[t, j] * y[slots[t, j]], summed in float32
    in the order of j; a slot of -1 adds nothing.  y (M, N) float32, bfloat16 or
    float16; weights (T, k); rows, slots of moe_route (rows for the gradient)."""
    _gpu("moe_combine", y)
    if y.dim() != 2 or slots.dim() != 2 or weights.shape != slots.shape:
        raise AssertionError(f"y must be (M, N), weights and slots (T, k); got {tuple(y.shape)}, "
                             f"{tuple(weights.shape)}, {tuple(slots.shape)}")
    if not y.shape[0] == rows.numel() == slots.numel():
        raise AssertionError(f"y has {y.shape[0]} rows, rows {rows.numel()} and slots {slots.numel()} places: "
                             "all must be T * k")
    return _lib.run_op(_ops.moe_combine, y, weights, rows, slots)


__all__ = ["MoERoute", "moe_route", "grouped_matmul", "moe_combine"]
