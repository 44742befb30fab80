"""Selective state space scan and the short causal convolution in front of it, on the GPU.

Beside ``AssocScan`` and ``memory_recurrence``, whose recurrences carry one scalar gate per step,
``selective_scan`` decays every (channel, state) pair at its own rate, as the mixing layer of a state
space language model does; ``causal_conv1d`` is that layer's depthwise convolution with its activation.
Both take prompts and training sequences of any length (with gradients), rows of their own lengths, and a
carried state, so that a prompt can be cut anywhere; a single step without gradients runs one small
kernel each. Kernels: ``atlas_sscan_*`` (csrc/sscan.cuh) and ``atlas_causal_conv_*`` (csrc/causal_conv.cuh).
No reference counterpart.
"""
from __future__ import annotations

import ctypes
import functools
import struct

import torch
from torch import Tensor
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from .ops import _has_tangent

MAX_STATE = 64     # states per channel
MAX_CONV_K = 8     # taps
MAX_BATCH, MAX_STEPS, MAX_CHANNELS, MAX_CONV_CHANNELS = 1 << 24, (1 << 31) - 1, 1 << 30, 1 << 20

_IO = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16}

# struct AtlasSelScan of include/atlas_mem.h in native alignment (checked against the header by the tests)
_SCAN = struct.Struct("@2q6i5P12q4PP2P2P2NP2qP9P")


def _ptr(t: Tensor | None) -> int:
    return 0 if t is None else t.data_ptr()


def _need_cuda(t: Tensor, what: str):
    if not t.is_cuda:
        raise RuntimeError(f"atlas_rnn_b200.{what}: tensors must be on a CUDA device (no CPU path)")


def _check(what: str, name: str, t: Tensor, shape: tuple, dtype, device):
    if t.shape != shape:
        raise ValueError(f"atlas_rnn_b200.{what}: {name} must have shape {tuple(shape)}, not {tuple(t.shape)}")
    if dtype is not None and t.dtype != dtype:
        raise TypeError(f"atlas_rnn_b200.{what}: {name} must be {dtype}, not {t.dtype}")
    if t.device != device:
        raise RuntimeError(f"atlas_rnn_b200.{what}: {name} is on {t.device}, expected {device}")


def _check_sizes(what: str, b: int, t: int, channels: int, most: int):
    if b > MAX_BATCH or t > MAX_STEPS or channels > most:
        raise ValueError(f"atlas_rnn_b200.{what}: at most {MAX_BATCH} rows of {MAX_STEPS} steps of {most} channels, not "
                         f"{(b, t, channels)}")


def _f32(what: str, name: str, t: Tensor | None, shape: tuple, device) -> Tensor | None:
    """A parameter or state as dense fp32."""
    if t is None:
        return None
    _check(what, name, t, shape, None, device)
    if t.dtype != torch.float32:
        if not t.is_floating_point():
            raise TypeError(f"atlas_rnn_b200.{what}: {name} must be a floating type, not {t.dtype}")
        t = t.to(torch.float32)
    return t if t.is_contiguous() else t.contiguous()


def _rows(t: Tensor) -> Tensor:
    """Rows whose last dimension is dense (other strides are passed on)."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _lengths(what: str, lengths, batch: int, device) -> Tensor | None:
    if lengths is None:
        return None
    if not isinstance(lengths, Tensor) or lengths.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"atlas_rnn_b200.{what}: lengths must be an int32 or int64 tensor")
    _check(what, "lengths", lengths, (batch,), None, device)
    return lengths.clamp(0, 0x7fffffff).to(torch.int32).contiguous() if lengths.dtype == torch.int64 \
        else lengths.contiguous()


def _through_autograd(*tensors) -> bool:
    """Whether a call goes through its autograd function: for a backward pass; with a forward-mode tangent, which the
    function refuses (a call past it would drop the tangent); and for a trace, which would have no more of a call past it than
    the allocation of the outputs. Else the call itself saves the detour's time. The function holds the checks and layouts
    too: a traced call does them on the inputs that it is run with."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return torch._C._is_tracing() or (forward_ad._current_level >= 0 and _has_tangent(*tensors))


def _run(what: str, fn, device, *args):
    """fn(*args, current stream of device) with ``device`` current: kernels launch on the current device."""
    index = device.index
    if index == torch.cuda.current_device():
        code = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(device):
            code = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if code:
        _lib.check(code, what)


# ---- selective scan --------------------------------------------------------------------------

@functools.lru_cache(maxsize=256)
def _scan_workspaces(device, b, t, d, n, g, io, chunk):
    """Bytes of the kept states, and of a forward's and a backward's scratch: they go by the sizes (and the device) alone."""
    sizes = [ctypes.c_size_t() for _ in range(3)]
    record = _SCAN.pack(b, t, d, n, g, 0, io, chunk, *[0] * 41)
    with torch.cuda.device(device):
        _lib.check(_lib.lib().atlas_sscan_workspace(record, *[ctypes.byref(s) for s in sizes]),
                   "selective_scan workspace")
    return tuple(s.value for s in sizes)


class _Scan:
    """The operands of one scan call, ready for the C ABI."""

    __slots__ = ("u", "delta", "z", "B", "C", "A", "D", "bias", "h0", "lengths", "softplus", "chunk")

    def __init__(self, u, delta, A, B, C, D, z, bias, h0, lengths, softplus, chunk):
        self.u, self.delta, self.A, self.B, self.C, self.D = u, delta, A, B, C, D
        self.z, self.bias, self.h0, self.lengths, self.softplus, self.chunk = z, bias, h0, lengths, softplus, chunk

    def pack(self, out=None, hT=None, saved=None, scratch=None, dout=None, dhT=None, du=None, ddelta=None, dz=None,
             dB=None, dC=None, dA=None, dD=None, dbias=None, dh0=None) -> bytes:
        u, d, z, B, C = self.u, self.delta, self.z, self.B, self.C
        zs = (0, 0) if z is None else (z.stride(0), z.stride(1))
        os = (0, 0) if dout is None else (dout.stride(0), dout.stride(1))
        return _SCAN.pack(
            u.shape[0], u.shape[1], u.shape[2], B.shape[3], B.shape[2], int(self.softplus), _IO[u.dtype], self.chunk,
            u.data_ptr(), d.data_ptr(), _ptr(z), B.data_ptr(), C.data_ptr(), u.stride(0), u.stride(1), d.stride(0),
            d.stride(1), *zs, *B.stride()[:3], *C.stride()[:3], self.A.data_ptr(), _ptr(self.D), _ptr(self.bias),
            _ptr(self.h0), _ptr(self.lengths), _ptr(out), _ptr(hT), _ptr(saved), _ptr(scratch),
            0 if saved is None else saved.numel(), 0 if scratch is None else scratch.numel(), _ptr(dout), *os, _ptr(dhT),
            _ptr(du), _ptr(ddelta), _ptr(dz), _ptr(dB), _ptr(dC), _ptr(dA), _ptr(dD), _ptr(dbias), _ptr(dh0))

    def workspaces(self):
        u = self.u
        sizes = map(int, (*u.shape, self.B.shape[3], self.B.shape[2]))  # while a trace is taken they are tensors
        return _scan_workspaces(u.device.index, *sizes, _IO[u.dtype], self.chunk)

    def forward(self, keep: bool):
        """(out, final state, kept states or None)."""
        u = self.u
        dev = u.device
        if u.numel() == 0:  # nothing to walk (no rows or no steps): the state passes through
            hT = u.new_zeros(u.shape[0], u.shape[2], self.B.shape[3], dtype=torch.float32) if self.h0 is None else self.h0.clone()
            return torch.empty_like(u, memory_format=torch.contiguous_format), hT, None
        out = torch.empty(u.shape, dtype=u.dtype, device=dev)
        hT = torch.empty(u.shape[0], u.shape[2], self.B.shape[3], dtype=torch.float32, device=dev)
        saved = scratch = None
        if keep or u.shape[1] > 1:
            ns, nf, _ = self.workspaces()
            saved = torch.empty(ns, dtype=torch.uint8, device=dev) if keep else None
            scratch = torch.empty(nf, dtype=torch.uint8, device=dev) if nf else None
        _run("selective_scan forward", _lib.lib().atlas_sscan_forward, dev, self.pack(out, hT, saved, scratch))
        return out, hT, saved


def _scan_operands(u, delta, A, B, C, D, z, bias, h0, lengths, softplus, chunk) -> _Scan:
    """The arguments of selective_scan, checked and laid out."""
    what = "selective_scan"
    if u.dim() != 3 or B.dim() not in (3, 4) or C.dim() != B.dim():
        raise ValueError(f"atlas_rnn_b200.{what}: expected u [b, t, d] and B, C [b, t, n] or [b, t, g, n], got "
                         f"{tuple(u.shape)}, {tuple(B.shape)}, {tuple(C.shape)}")
    if u.dtype not in _IO:
        raise TypeError(f"atlas_rnn_b200.{what}: u must be float32 or bfloat16, not {u.dtype}")
    if B.dim() == 3:
        B, C = B.unsqueeze(2), C.unsqueeze(2)
    b, t, d = u.shape
    g, n = B.shape[2], B.shape[3]
    dev = u.device
    _check_sizes(what, b, t, d, MAX_CHANNELS)
    if not 1 <= n <= MAX_STATE:
        raise ValueError(f"atlas_rnn_b200.{what}: 1 to {MAX_STATE} states per channel, not {n}")
    if g < 1 or d % g:
        raise ValueError(f"atlas_rnn_b200.{what}: {d} channels do not split into {g} groups")
    if chunk < 0 or chunk % 32:
        raise ValueError(f"atlas_rnn_b200.{what}: chunk must be a multiple of 32, not {chunk}")
    _check(what, "delta", delta, (b, t, d), u.dtype, dev)
    _check(what, "B", B, (b, t, g, n), u.dtype, dev)
    _check(what, "C", C, (b, t, g, n), u.dtype, dev)
    if z is not None:
        _check(what, "z", z, (b, t, d), u.dtype, dev)
    A = _f32(what, "A", A, (d, n), dev)
    D, bias = _f32(what, "D", D, (d,), dev), _f32(what, "delta_bias", bias, (d,), dev)
    h0 = _f32(what, "initial_state", h0, (b, d, n), dev)
    lengths = _lengths(what, lengths, b, dev)
    _need_cuda(u, what)
    return _Scan(_rows(u), _rows(delta), A, _rows(B), _rows(C), D, None if z is None else _rows(z), bias, h0, lengths,
                 bool(softplus), chunk)


class SelectiveScanFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, u, delta, A, B, C, D, z, bias, h0, lengths, softplus, chunk):
        ctx.set_materialize_grads(False)
        s = _scan_operands(u, delta, A, B, C, D, z, bias, h0, lengths, softplus, chunk)
        out, hT, saved = s.forward(keep=any(ctx.needs_input_grad))
        ctx.save_for_backward(s.u, s.delta, s.A, s.B, s.C, s.D, s.z, s.bias, s.h0, s.lengths, saved)
        ctx.softplus, ctx.chunk, ctx.shapes = s.softplus, chunk, (B.shape, C.shape)
        return out, hT

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, dhT):
        u, delta, A, B, C, D, z, bias, h0, lengths, saved = ctx.saved_tensors
        need = ctx.needs_input_grad  # (u, delta, A, B, C, D, z, bias, h0, ...)
        s = _Scan(u, delta, A, B, C, D, z, bias, h0, lengths, ctx.softplus, ctx.chunk)
        dev = u.device
        if u.numel() == 0:  # the state passed through
            zeros = [None if t is None else torch.zeros_like(t) for t in (u, delta, A, B, C, D, z, bias, h0)]
            zeros[3], zeros[4] = zeros[3].view(ctx.shapes[0]), zeros[4].view(ctx.shapes[1])
            return *zeros[:8], zeros[8] if dhT is None else dhT, None, None, None
        dout = torch.zeros(u.shape, dtype=u.dtype, device=dev) if dout is None else _rows(dout)
        dhT = None if dhT is None else dhT.contiguous()
        rows = lambda: torch.empty(u.shape, dtype=u.dtype, device=dev)
        du, ddelta, dz = rows(), rows(), rows() if z is not None else None
        dB = torch.empty(B.shape, dtype=u.dtype, device=dev) if need[3] or need[4] else None
        dC = torch.empty(C.shape, dtype=u.dtype, device=dev) if need[3] or need[4] else None
        f32 = lambda t, flag: torch.empty(t.shape, dtype=torch.float32, device=dev) if t is not None and flag else None
        dA, dD, dbias, dh0 = f32(A, True), f32(D, need[5]), f32(bias, need[7]), f32(h0, need[8])
        scratch = torch.empty(s.workspaces()[2], dtype=torch.uint8, device=dev)
        packed = s.pack(saved=saved, scratch=scratch, dout=dout, dhT=dhT, du=du, ddelta=ddelta, dz=dz, dB=dB, dC=dC,
                        dA=dA, dD=dD, dbias=dbias, dh0=dh0)
        _run("selective_scan backward", _lib.lib().atlas_sscan_backward, dev, packed)
        if dB is not None:
            dB, dC = dB.view(ctx.shapes[0]), dC.view(ctx.shapes[1])
        return du, ddelta, dA, dB, dC, dD, dz, dbias, dh0, None, None, None


def selective_scan(u: Tensor, delta: Tensor, A: Tensor, B: Tensor, C: Tensor, D: Tensor | None = None,
                   z: Tensor | None = None, *, delta_bias: Tensor | None = None, delta_softplus: bool = False,
                   initial_state: Tensor | None = None, lengths: Tensor | None = None, chunk: int = 0):
    """Selective state space scan over [batch, steps, channels].

    Per batch row, channel d (of group g) and state n:

        dt_t = softplus(delta_t + delta_bias)   (delta_softplus False: delta_t + delta_bias)
        h_t  = exp(dt_t A[d, n]) h_{t-1} + dt_t u_t B_t[g, n],   h_0 = initial_state (or 0)
        out_t = (sum_n C_t[g, n] h_t + D u_t) silu(z_t)          (D, z None: left out)

    u, delta, z [b, t, d] and B, C [b, t, n] or [b, t, g, n] (d a multiple of g, n up to 64) are all float32 or all
    bfloat16, of any batch and step strides (halves of one projection are taken as they are); A [d, n],
    D, delta_bias [d] and initial_state [b, d, n] are computed in float32, as is the state (an A of -inf as the lowest finite
    value, so that a step with dt = 0 leaves the state). lengths [b] (int32 or
    int64): steps at or past a row's length are not read, leave its state alone and give 0.
    Returns (out [b, t, d] in u's type, final state [b, d, n] float32); both carry gradients to every
    floating input. The sums over steps, states and channels are in float32 and in a fixed order, so the same call gives the
    same bits. A training call keeps the states of every 8th step for its backward (d / 8 floats a step for each
    state, n counted as 8, 16, 32 or 64).
    One step without gradients runs one small kernel. chunk: steps per piece of a cut time axis (a multiple
    of 32, lengthened where t takes more than 65535 pieces; 0 lets the library choose)."""
    if _through_autograd(u, delta, A, B, C, D, z, delta_bias, initial_state):
        return SelectiveScanFn.apply(u, delta, A, B, C, D, z, delta_bias, initial_state, lengths, delta_softplus, chunk)
    return _scan_operands(u, delta, A, B, C, D, z, delta_bias, initial_state, lengths, delta_softplus,
                          chunk).forward(keep=False)[:2]


# ---- causal convolution ----------------------------------------------------------------------

def _conv_operands(x, weight, bias, init, lengths, activation):
    """The arguments of causal_conv1d, checked and laid out."""
    what = "causal_conv1d"
    if x.dim() != 3:
        raise ValueError(f"atlas_rnn_b200.{what}: expected x [b, t, c], got {tuple(x.shape)}")
    if x.dtype not in _IO:
        raise TypeError(f"atlas_rnn_b200.{what}: x must be float32 or bfloat16, not {x.dtype}")
    if activation not in (None, "silu"):
        raise ValueError(f"atlas_rnn_b200.{what}: activation must be None or 'silu', not {activation!r}")
    B, T, C = x.shape
    _check_sizes(what, B, T, C, MAX_CONV_CHANNELS)
    K = weight.shape[-1]
    if not 2 <= K <= MAX_CONV_K:
        raise ValueError(f"atlas_rnn_b200.{what}: 2 to {MAX_CONV_K} taps, not {K}")
    dev = x.device
    w = _f32(what, "weight", weight, (C, 1, K) if weight.dim() == 3 else (C, K), dev)
    bias = _f32(what, "bias", bias, (C,), dev)
    if init is not None:
        _check(what, "initial_state", init, (B, K - 1, C), x.dtype, dev)
        if not init.is_contiguous():
            init = init.contiguous()
    lengths = _lengths(what, lengths, B, dev)
    _need_cuda(x, what)
    return _rows(x), w, bias, init, lengths, int(activation == "silu")


def _conv_forward(x, w, bias, init, lengths, silu):
    B, T, C = x.shape
    K = w.shape[-1]
    if x.numel() == 0:
        final = x.new_zeros(B, K - 1, C) if init is None else init.clone()
        return torch.empty_like(x, memory_format=torch.contiguous_format), final
    y = torch.empty(B, T, C, dtype=x.dtype, device=x.device)
    final = torch.empty(B, K - 1, C, dtype=x.dtype, device=x.device)
    _run("causal_conv1d forward", _lib.lib().atlas_causal_conv_forward, x.device, x.data_ptr(), x.stride(0),
         x.stride(1), w.data_ptr(), _ptr(bias), _ptr(init), _ptr(lengths), y.data_ptr(), final.data_ptr(), K, silu,
         _IO[x.dtype], B, T, C)
    return y, final


class CausalConv1dFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, bias, init, lengths, activation):
        ctx.set_materialize_grads(False)
        *tensors, ctx.silu = _conv_operands(x, w, bias, init, lengths, activation)
        y, final = _conv_forward(*tensors, ctx.silu)
        ctx.save_for_backward(*tensors)
        return y, final

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, d_final):
        x, w, bias, init, lengths = ctx.saved_tensors
        B, T, C = x.shape
        K = w.shape[-1]
        dev = x.device
        if x.numel() == 0:  # the state passed through
            dx, dw, dbias, d_init = (None if t is None else torch.zeros_like(t) for t in (x, w, bias, init))
            return dx, dw, dbias, d_init if d_final is None or init is None else d_final, None, None
        dy = torch.zeros(B, T, C, dtype=x.dtype, device=dev) if dy is None else _rows(dy)
        d_final = None if d_final is None else d_final.contiguous()
        dx = torch.empty(B, T, C, dtype=x.dtype, device=dev)
        d_init = torch.empty_like(init) if init is not None and ctx.needs_input_grad[3] else None
        dw = torch.empty(w.shape, dtype=torch.float32, device=dev)
        dbias = torch.empty(C, dtype=torch.float32, device=dev) if bias is not None else None
        L = _lib.lib()
        scratch = torch.empty(L.atlas_causal_conv_scratch(B, T, C, K), dtype=torch.uint8, device=dev)
        _run("causal_conv1d backward", L.atlas_causal_conv_backward, dev, x.data_ptr(), x.stride(0), x.stride(1),
             w.data_ptr(), _ptr(bias), _ptr(init), _ptr(lengths), dy.data_ptr(), dy.stride(0), dy.stride(1),
             _ptr(d_final), dx.data_ptr(), _ptr(d_init), dw.data_ptr(), _ptr(dbias), scratch.data_ptr(),
             scratch.numel(), K, ctx.silu, _IO[x.dtype], B, T, C)
        return dx, dw, dbias, d_init, None, None


def causal_conv1d(x: Tensor, weight: Tensor, bias: Tensor | None = None, *, activation: str | None = None,
                  initial_state: Tensor | None = None, lengths: Tensor | None = None):
    """Causal depthwise convolution over [batch, steps, channels], with its activation and a carried state:

        y_t = act(bias + sum_j weight[:, j] x_{t + j - (K - 1)})

    x [b, t, c] float32 or bfloat16 (any batch and step strides); weight [c, K] or a Conv1d's [c, 1, K], 2 <= K <= 8, and bias
    [c] are computed in float32; activation None or 'silu'. initial_state [b, K - 1, c] in x's type holds the inputs
    before the first step (None: zeros). lengths [b]: steps at or past a row's length are not read and give 0.
    Returns (y, final state [b, K - 1, c]: the last K - 1 inputs of each row, the next call's
    initial_state), both with gradients to x, weight, bias and initial_state."""
    if _through_autograd(x, weight, bias, initial_state):
        return CausalConv1dFn.apply(x, weight, bias, initial_state, lengths, activation)
    return _conv_forward(*_conv_operands(x, weight, bias, initial_state, lengths, activation))
