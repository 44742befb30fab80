"""Distillation from a teacher's top logits, forward and backward, on the GPU.

``distill_loss`` trains a student (such as ``RNNMemoryTransformer``, whose ``forward`` takes ``teacher=``) on the few
largest logits that a teacher left per position. Kernels: ``atlas_distill_forward`` / ``_backward`` (csrc/distill.cuh).
No reference counterpart (its loss is the next-token cross-entropy, rnn_transformer.py:852-860).
"""
from __future__ import annotations

import struct

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from . import _lib
from .selective_scan import _IO, _check, _need_cuda, _run

MAX_ENTRIES = 1024  # teacher entries per row

# struct AtlasDistill of include/atlas_mem.h in native alignment (checked against the header by the tests)
_DISTILL = struct.Struct("@8P4qfi")


def _operands(logits, teacher_values, teacher_indices, temperature):
    """The arguments of distill_loss, checked and laid out: rows of logits, of values and of indices. Part of the autograd
    function, so that a traced call checks the inputs that it is run with."""
    what = "distill_loss"
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError(f"atlas_rnn_b200.{what}: expected logits [..., V], got {tuple(logits.shape)}")
    if logits.dtype not in _IO:
        raise TypeError(f"atlas_rnn_b200.{what}: logits must be float32 or bfloat16, not {logits.dtype}")
    if teacher_values.dim() < 1 or not 1 <= teacher_values.shape[-1] <= MAX_ENTRIES:
        raise ValueError(f"atlas_rnn_b200.{what}: expected teacher_values [..., K] with K from 1 to {MAX_ENTRIES}, got "
                         f"{tuple(teacher_values.shape)}")
    if not teacher_values.is_floating_point():
        raise TypeError(f"atlas_rnn_b200.{what}: teacher_values must be a floating type, not {teacher_values.dtype}")
    if teacher_indices.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"atlas_rnn_b200.{what}: teacher_indices must be int32 or int64, not {teacher_indices.dtype}")
    if not 1e-6 <= temperature <= 1e6:
        raise ValueError(f"atlas_rnn_b200.{what}: temperature must be from 1e-6 to 1e6, not {temperature}")
    lead, V, K = logits.shape[:-1], logits.shape[-1], teacher_values.shape[-1]
    if V > 0x7ffffff0:
        raise ValueError(f"atlas_rnn_b200.{what}: {V} tokens are too many")
    _check(what, "teacher_values", teacher_values, (*lead, K), None, logits.device)
    _check(what, "teacher_indices", teacher_indices, (*lead, K), None, logits.device)
    _need_cuda(logits, what)
    x = logits.reshape(-1, V)
    x = x if x.stride(1) == 1 or V == 1 else x.contiguous()
    return (x, teacher_values.to(torch.float32).reshape(-1, K).contiguous(),
            teacher_indices.to(torch.int64).reshape(-1, K).contiguous())


class DistillLossFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, teacher_values, teacher_indices, temperature):
        x, values, indices = _operands(logits, teacher_values, teacher_indices, temperature)
        rows, V = x.shape
        dev = x.device
        loss = torch.empty(logits.shape[:-1], dtype=torch.float32, device=dev)
        valid = torch.empty(logits.shape[:-1], dtype=torch.float32, device=dev)
        stats = torch.empty(rows, 4, dtype=torch.float32, device=dev)
        if rows:
            _run("distill_loss forward", _lib.lib().atlas_distill_forward, dev,
                 _DISTILL.pack(x.data_ptr(), values.data_ptr(), indices.data_ptr(), loss.data_ptr(), valid.data_ptr(),
                               stats.data_ptr(), 0, 0, rows, V, values.shape[1], x.stride(0), temperature, _IO[x.dtype]))
        ctx.save_for_backward(x, values, indices, stats)
        ctx.temperature, ctx.shape = temperature, logits.shape
        ctx.mark_non_differentiable(valid)
        return loss, valid

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss, _):
        x, values, indices, stats = ctx.saved_tensors
        rows, V = x.shape
        dev = x.device
        dlogits = torch.empty(ctx.shape, dtype=x.dtype, device=dev)
        dloss = dloss.contiguous()
        if rows:
            _run("distill_loss backward", _lib.lib().atlas_distill_backward, dev,
                 _DISTILL.pack(x.data_ptr(), values.data_ptr(), indices.data_ptr(), 0, 0, stats.data_ptr(),
                               dloss.data_ptr(), dlogits.data_ptr(), rows, V, values.shape[1], x.stride(0),
                               ctx.temperature, _IO[x.dtype]))
        return dlogits, None, None, None


def distill_loss(logits: Tensor, teacher_values: Tensor, teacher_indices: Tensor, *, temperature: float = 1.0,
                 reduction: str = "mean") -> Tensor:
    """KL divergence of the student's softmax from a teacher's, over the teacher's top logits.

    logits [..., V] (float32 or bfloat16); teacher_values [..., K] (a floating type) and teacher_indices [..., K] (int32 or
    int64), K up to 1024: the teacher's logits and their tokens. Entries whose index is outside 0 .. V - 1 (-1, say), or
    whose value is -inf or NaN, are absent, so rows may have fewer than K; tokens may repeat. Per row, with
    p = softmax(teacher_values / temperature) over the entries and q = softmax(logits / temperature), temperature from
    1e-6 to 1e6:

        loss = temperature^2 sum_k p_k (log p_k - log q[index_k])

    and 0 (without a gradient) for a row that has no entries. reduction 'none' returns float32 [...]; 'sum' the sum; 'mean'
    the mean over the rows with entries (0 when there are none). Gradients go to the logits alone. Sums and logarithms
    are float32: a row's loss is exact to about temperature^2 log2(V) 2^-22, which counts where high temperatures make p and q alike."""
    if reduction not in ("none", "mean", "sum"):
        raise ValueError(f"atlas_rnn_b200.distill_loss: reduction must be 'none', 'mean' or 'sum', not {reduction!r}")
    loss, valid = DistillLossFn.apply(logits, teacher_values.detach(), teacher_indices, float(temperature))
    if reduction == "none":
        return loss
    return loss.sum() if reduction == "sum" else loss.sum() / valid.sum().clamp(min=1.0)
