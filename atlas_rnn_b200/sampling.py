"""Token sampling on the GPU: the filters and the draw of ``RNNMemoryTransformer.generate`` as one kernel.

``sample_tokens`` fuses ``min_p_filter`` and ``gumbel_sample`` (rnn_transformer.py:42-59) with top-k and top-p
(nucleus) filters, drawing from uniforms that the caller gives. Kernel: ``atlas_sample_tokens`` (csrc/sample.cuh).
"""
from __future__ import annotations

import operator
import struct

import torch
from torch import Tensor

from . import _lib
from .selective_scan import _IO, _check, _need_cuda, _ptr, _run

MAX_VOCAB = (1 << 24) - 16  # tokens per row

# struct AtlasSample of include/atlas_mem.h in native alignment (checked against the header by the tests)
_SAMPLE = struct.Struct("@3P4q3dq4Pi4x")


def _setting(name: str, value, lead: tuple, device, dtype, lowest, highest):
    """(one value, None) or (0, a tensor with one per row)."""
    if not isinstance(value, Tensor):
        if dtype == torch.int32:
            value = operator.index(value)  # TypeError for what is no integer
        if not (value >= lowest and (highest is None or value <= highest)):  # a NaN fails too
            raise ValueError(f"atlas_rnn_b200.sample_tokens: {name} must be at least {lowest}"
                             + (f" and at most {highest}" if highest is not None else "") + f", not {value}")
        return value, None
    if value.is_floating_point() != (dtype == torch.float32) or value.dtype == torch.bool:
        raise TypeError(f"atlas_rnn_b200.sample_tokens: {name} per row must be "
                        + ("a floating type" if dtype == torch.float32 else "an integer type") + f", not {value.dtype}")
    _check("sample_tokens", name, value, lead, None, device)
    if value.dtype == torch.int64 and dtype == torch.int32:
        value = value.clamp(0, 0x7fffffff)
    return 0, value.to(dtype).contiguous()


def _sample(logits, noise, temperature, top_k, top_p, min_p) -> Tensor:
    what = "sample_tokens"
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError(f"atlas_rnn_b200.{what}: expected logits [..., V], got {tuple(logits.shape)}")
    if logits.dtype not in _IO:
        raise TypeError(f"atlas_rnn_b200.{what}: logits must be float32 or bfloat16, not {logits.dtype}")
    dev, lead, V = logits.device, logits.shape[:-1], logits.shape[-1]
    if V > MAX_VOCAB:
        raise ValueError(f"atlas_rnn_b200.{what}: at most {MAX_VOCAB} tokens, not {V}")
    _check(what, "noise", noise, logits.shape, torch.float32, dev)
    t, t_row = _setting("temperature", temperature, lead, dev, torch.float32, 0.0, None)
    k, k_row = _setting("top_k", top_k, lead, dev, torch.int32, 0, None)
    p, p_row = _setting("top_p", top_p, lead, dev, torch.float32, 0.0, 1.0)
    m, m_row = _setting("min_p", min_p, lead, dev, torch.float32, 0.0, 1.0)
    _need_cuda(logits, what)
    out = torch.empty(lead, dtype=torch.int64, device=dev)
    if out.numel() == 0:
        return out
    x, u = logits.detach().reshape(-1, V), noise.detach().reshape(-1, V)
    x = x if x.stride(1) == 1 or V == 1 else x.contiguous()
    u = u if u.stride(1) == 1 or V == 1 else u.contiguous()
    _run(what, _lib.lib().atlas_sample_tokens, dev,
         _SAMPLE.pack(x.data_ptr(), u.data_ptr(), out.data_ptr(), x.shape[0], V, x.stride(0), u.stride(0), t, p, m,
                      min(k, 0x7fffffff), _ptr(t_row), _ptr(p_row), _ptr(m_row), _ptr(k_row), _IO[x.dtype]))
    return out


class SampleTokensFn(torch.autograd.Function):
    """``sample_tokens`` for torch.jit.trace, which sees no calls of the library outside such a function."""

    @staticmethod
    def forward(ctx, *args):
        out = _sample(*args)
        ctx.mark_non_differentiable(out)
        return out

    @staticmethod
    def backward(ctx, _):
        return (None,) * 6


def sample_tokens(logits: Tensor, noise: Tensor, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0) -> Tensor:
    """One token per row of ``logits`` [..., V] (float32 or bfloat16), drawn with the uniforms ``noise`` [..., V]
    (float32 in [0, 1)). In the order of descending logit, ties by lowest index, the filters are, on softmax(logits):

        top_k   the first top_k tokens (0: all)
        top_p   of those, the ones with less than top_p of their probability before them, the first always (1: all)
        min_p   of those, the ones with at least min_p times the first one's probability

    and the token is the kept one with the largest logits / temperature - log(-log(noise)); temperature 0 (or below
    1e-30) gives the first token. The filters see the logits without the temperature, as ``min_p_filter`` before ``gumbel_sample`` does: divide
    the logits beforehand for filters on the tempered distribution. Each setting is a number or a tensor with one value
    per row (a row with a NaN among them gets its first token). Masked tokens are -inf (NaN counts as -inf); a row with
    nothing above -inf gives 0.
    V up to 2^24 - 16. Returns int64 [...], the same whatever the batch: scores are compared in float64; the probabilities
    that the filters add up are float32 exponentials, each exact to 2^-21 of the largest one (a token d below the maximum to
    (d + 1) 2^-22 of its own and 2^-40 of the largest), and are added exactly."""
    call = SampleTokensFn.apply if torch._C._is_tracing() else _sample
    return call(logits, noise, temperature, top_k, top_p, min_p)
