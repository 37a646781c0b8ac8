"""Distillation from a teacher's top logits.

The reference trains quantized layers against the full-precision model by a KL
divergence over the whole vocabulary (the drivers in src/qat).  A teacher run
once stores its top K logits per position; these operators take the divergence
from them, without a (T, V) probability tensor.
"""
from __future__ import annotations

import torch

from . import _lib

_ops = _lib.load_ops()


def _check(logits, values, indices, temperature, teacher_lse):
    if not logits.is_cuda:
        raise AssertionError(f"topk_distill_loss runs on the GPU; logits are on {logits.device}")
    if logits.dim() != 2 or values.dim() != 2 or values.shape[0] != logits.shape[0] or indices.shape != values.shape:
        raise AssertionError(f"logits must be (T, V), teacher values and indices (T, K); got {tuple(logits.shape)}, "
                             f"{tuple(values.shape)}, {tuple(indices.shape)}")
    if teacher_lse is not None and tuple(teacher_lse.shape) != (logits.shape[0],):
        raise AssertionError(f"teacher_lse must be ({logits.shape[0]},); got {tuple(teacher_lse.shape)}")
    if not temperature > 0:
        raise AssertionError(f"temperature must be > 0; got {temperature}")


def topk_distill_loss(logits, teacher_values, teacher_indices, *, temperature=1.0, teacher_lse=None):
    """Divergence (T,) float32 of each row's student distribution from its teacher's.

    logits:  (T, V) float32, bfloat16 or float16, V <= 2^20; differentiable.
    teacher_values, teacher_indices: (T, K): the teacher's logits and the
             vocabulary entries they belong to, in any order, each entry once
             (a repeated one counts as entries of its own); an index outside
             [0, V) is no entry, so rows may have fewer than K.
    temperature: both sides' logits are divided by it.  (The usual factor
             temperature^2 is the caller's.)
    teacher_lse: (T,) logsumexp(teacher logits / temperature) over the
             teacher's whole vocabulary, or None.

    With p = softmax(logits / temperature): without teacher_lse the teacher q is
    the softmax over its entries and the loss sum q (log q - log p).  With it
    q = exp(values / temperature - teacher_lse), and the mass outside the
    entries counts as one event more: r (log r - log p_r), r = 1 - sum q (none
    under 1e-6), p_r the student's mass there.

    A row without entries has loss and gradient 0; a row whose gradient is 0
    (masked out of the batch's loss) gets zeros whatever its logits are.  A
    student logit of -inf on an entry with mass makes the loss inf; NaN, +inf or
    nothing but -inf make it NaN.  The teacher's side has no gradient."""
    _check(logits, teacher_values, teacher_indices, temperature, teacher_lse)
    return _lib.run_op(_ops.topk_distill_loss, logits, teacher_values, teacher_indices, teacher_lse,
                       float(temperature))


def topk_distill_loss_and_grad(logits, teacher_values, teacher_indices, row_weights, *, temperature=1.0,
                               teacher_lse=None):
    """(loss (T,) float32, g (T, V) in logits' type): topk_distill_loss and
    g = d sum(row_weights * loss) / d logits in one launch, for a step that knows
    its rows' weights (T,) beforehand (the mean over unmasked positions, a loss
    scale).  Continue with logits.backward(g).  Not recorded by autograd."""
    _check(logits, teacher_values, teacher_indices, temperature, teacher_lse)
    if tuple(row_weights.shape) != (logits.shape[0],):
        raise AssertionError(f"row_weights must be ({logits.shape[0]},); got {tuple(row_weights.shape)}")
    with torch.no_grad():
        return _lib.run_op(_ops.topk_distill_both, logits.detach(), teacher_values, teacher_indices, row_weights,
                           teacher_lse, float(temperature))


__all__ = ["topk_distill_loss", "topk_distill_loss_and_grad"]
