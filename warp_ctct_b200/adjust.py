"""Adjustment of raw logits: penalties for repeated tokens, additive biases, masks of allowed tokens.

For a token v that occurs c times in the history of a row with logit x::

    z = x;  if c > 0: z = x / repetition_penalty if x > 0 else x * repetition_penalty
    z -= presence_penalty * (c > 0) + frequency_penalty * c
    z += bias[v]
    out = z if v is allowed else -inf

``adjust_logits`` is the step of a decoder: (R, V) logits, a history per row.  ``adjust_joint_logits`` and
``adjust_joint_logits_packed`` do the same to every row of a joint tensor before ``ctct_loss_from_logits`` or
``ctct_loss_packed(from_logits=True)`` (the reference takes the joint tensor as it is, warp_ctct/__init__.py:97-100): the
history of a row is its context's labels.  Gradients flow to the logits and to the bias.
"""
from __future__ import annotations

from collections import namedtuple
from math import inf
from typing import Optional, Union

import torch
from torch.autograd.function import once_differentiable

from . import _lib

T = torch.Tensor


def pack_token_mask(mask: T) -> T:
    """(..., V) truth values -> (..., ceil(V / 32)) int32 words, bit v % 32 of word v // 32: the ``allowed`` argument of
    the functions below."""
    V = mask.size(-1)
    words = (V + 31) // 32
    bits = torch.nn.functional.pad(mask.to(torch.int64), (0, words * 32 - V)).view(*mask.shape[:-1], words, 32)
    packed = (bits << torch.arange(32, device=mask.device)).sum(-1)
    return torch.where(packed >= 1 << 31, packed - (1 << 32), packed).to(torch.int32)


def _penalty(name: str, value: Union[float, T], N: int, device, positive: bool):
    """(scalar, tensor or None) of a penalty given as a number or as (N,) float32."""
    if not isinstance(value, torch.Tensor):
        value = float(value)
        if not (0.0 < value < inf if positive else -inf < value < inf):
            raise RuntimeError(f"{name} must be a finite number{' above 0' if positive else ''}, not {value}")
        return value, None
    if value.dim() != 1 or value.size(0) != N:
        raise RuntimeError(f"{name} must be a number or have shape ({N},)")
    if value.dtype != torch.float32 or value.device != device:
        raise RuntimeError(f"{name} must be float32 on {device}")
    if value.requires_grad:
        raise RuntimeError(f"{name} is not differentiated: detach it")
    return 1.0, value if value.is_contiguous() else value.contiguous()


def _kind(name: str, t: Optional[T], N: int, U1: int, last: int, step: bool, device) -> int:
    """0 none, 1 (last), 2 (N, last), 3 (N, U1, last)."""
    if t is None:
        return 0
    if t.device != device:
        raise RuntimeError(f"{name} must be on {device}, not on {t.device}")
    kind = t.dim()
    if 1 <= kind <= (2 if step else 3) and t.size(-1) == last and (kind == 1 or t.size(0) == N) and (kind < 3 or t.size(1) == U1):
        return kind
    per_context = "" if step else f" or ({N}, {U1}, {last})"
    raise RuntimeError(f"{name} must have shape ({last},), ({N}, {last}){per_context}, not {tuple(t.shape)}")


# What both directions of a call have in common.  shape: (N, T, U1, V, rows), rows < 0 for the padded layout and the
# step; bias: (kind, 1 if float32); scalars, tensors: the penalties as `_penalty` gives them.
_Call = namedtuple("_Call", "shape row_stride code tokens pitch lengths lx ly bias allowed mask_kind scalars tensors")


def _forward(c: _Call, logits: T, bias: Optional[T]):
    N, Tm, U1, V, rows = c.shape
    dev = logits.device
    prev = _lib.enter_device(dev)
    try:
        out = torch.empty_like(logits) if c.row_stride == 0 else logits.new_empty(logits.shape)
        cu = torch.empty((N + 1,), dtype=torch.int64, device=dev) if rows >= 0 else None
        tokens, lengths, lx, ly, allowed = c.tokens, c.lengths, c.lx, c.ly, c.allowed
        rn, pn, qn = c.tensors
        rc = _lib.lib().ctct_b200_adjust_forward(
            logits.data_ptr(), c.row_stride, c.code, None if tokens is None else tokens.data_ptr(), c.pitch,
            None if lengths is None else lengths.data_ptr(), None if lx is None else lx.data_ptr(),
            None if ly is None else ly.data_ptr(), N, Tm, U1, V, rows, None if cu is None else cu.data_ptr(),
            None if bias is None else bias.data_ptr(), *c.bias, None if allowed is None else allowed.data_ptr(), c.mask_kind,
            *c.scalars, None if rn is None else rn.data_ptr(), None if pn is None else pn.data_ptr(),
            None if qn is None else qn.data_ptr(), out.data_ptr(), _lib.raw_stream(dev))
    finally:
        _lib.leave_device(prev)
    if rc:
        _lib.check(rc, "ctct_b200_adjust_forward")
    return out, cu


def _backward(ctx, dy: T):
    logits, tokens, lengths, lx, ly, cu, allowed, rn = ctx.saved_tensors
    shape, row_stride, code, pitch, bias_meta, mask_kind, repetition = ctx.call
    out_shape, dtype, dev, bias_shape, bias_dtype = ctx.like
    N, Tm, U1, V, rows = shape
    lib = _lib.lib()
    if not dy.is_contiguous():
        dy = dy.contiguous()
    need_x, need_b = ctx.needs_input_grad[:2]
    prev = _lib.enter_device(dev)
    try:
        dx = torch.empty(out_shape, dtype=dtype, device=dev) if need_x else None
        db = torch.empty(bias_shape, dtype=bias_dtype, device=dev) if need_b else None
        ws, nbytes = None, 0
        if need_b:
            nbytes = lib.ctct_b200_adjust_workspace_bytes(N, Tm, U1, V, code, int(rows >= 0), bias_meta[0])
            ws = torch.empty((nbytes,), dtype=torch.uint8, device=dev)
        rc = lib.ctct_b200_adjust_backward(
            dy.data_ptr(), _lib.ptr(logits), row_stride, code, _lib.ptr(tokens), pitch, _lib.ptr(lengths), _lib.ptr(lx),
            _lib.ptr(ly), N, Tm, U1, V, rows, _lib.ptr(cu), *bias_meta, _lib.ptr(allowed), mask_kind, repetition, _lib.ptr(rn),
            _lib.ptr(dx), _lib.ptr(db), _lib.ptr(ws), nbytes, _lib.raw_stream(dev))
    finally:
        _lib.leave_device(prev)
    if rc:
        _lib.check(rc, "ctct_b200_adjust_backward")
    return dx, db, None


class AdjustLogits(torch.autograd.Function):
    """Keeps the logits only if a repetition penalty scales some of them."""

    @staticmethod
    def forward(ctx, logits: T, bias: Optional[T], c: _Call):
        out, cu = _forward(c, logits, bias)
        scaled = c.tokens is not None and (c.tensors[0] is not None or c.scalars[0] != 1.0)
        # tensors that a caller could change in between go through save_for_backward, which notices
        ctx.save_for_backward(logits if scaled else None, c.tokens, c.lengths, c.lx, c.ly, cu, c.allowed, c.tensors[0])
        ctx.call = (c.shape, c.row_stride, c.code, c.pitch, c.bias, c.mask_kind, c.scalars[0])
        ctx.like = (logits.shape, logits.dtype, logits.device, *((None, None) if bias is None else (bias.shape, bias.dtype)))
        return out

    @staticmethod
    def backward(ctx, dy: T):
        # a graph of the gradient is only asked for with create_graph: the guard against a second
        # differentiation costs nothing otherwise
        return _backward_once(ctx, dy) if torch.is_grad_enabled() else _backward(ctx, dy)


_backward_once = once_differentiable(_backward)


def _apply(logits: T, N: int, Tm: int, U1: int, rows: int, row_stride: int, tokens: Optional[T], pitch: int, lengths: Optional[T],
           lx: Optional[T], ly: Optional[T], bias: Optional[T], allowed: Optional[T], repetition, presence, frequency,
           step: bool) -> T:
    dev, dtype = logits.device, logits.dtype
    V = logits.size(-1)
    if V < 1:
        raise RuntimeError("logits must have at least one token")
    bias_kind = _kind("bias", bias, N, U1, V, step, dev)
    bias_f32 = 0
    if bias_kind:
        bias_f32 = int(bias.dtype == torch.float32)
        if not bias_f32 and bias.dtype != dtype:
            raise RuntimeError(f"bias must be float32 or of the logits' type {dtype}, not {bias.dtype}")
        if not bias.is_contiguous():
            bias = bias.contiguous()
    mask_kind = _kind("allowed", allowed, N, U1, (V + 31) // 32, step, dev)
    if mask_kind:
        if allowed.dtype != torch.int32:
            raise RuntimeError("allowed must be int32 words (pack_token_mask)")
        if not allowed.is_contiguous():
            allowed = allowed.contiguous()
    r, rn = _penalty("repetition_penalty", repetition, N, dev, True)
    p, pn = _penalty("presence_penalty", presence, N, dev, False)
    q, qn = _penalty("frequency_penalty", frequency, N, dev, False)
    c = _Call((N, Tm, U1, V, rows), row_stride, _lib.dtype_code(dtype), tokens, pitch, lengths, lx, ly, (bias_kind, bias_f32), allowed,
              mask_kind, (r, p, q), (rn, pn, qn))
    if torch.is_grad_enabled() and (logits.requires_grad or (bias is not None and bias.requires_grad)):
        return AdjustLogits.apply(logits, bias, c)
    return _forward(c, logits, bias)[0]


def _int_on(name: str, t: T, device) -> T:
    if t.device != device:
        raise RuntimeError(f"{name} must be on {device}, not on {t.device}")
    if t.dtype == torch.int32:
        return t if t.is_contiguous() else t.contiguous()
    if t.is_floating_point() or t.is_complex() or t.dtype == torch.bool:
        raise RuntimeError(f"{name} must hold integers, not {t.dtype}")
    if t.dtype == torch.int64:   # what 32 bits do not hold is out of every range, and stays so
        t = t.clamp(-1, 2 ** 31 - 1)
    return t.to(torch.int32).contiguous()


def adjust_logits(logits: T, tokens: Optional[T] = None, tokens_lengths: Optional[T] = None, bias: Optional[T] = None,
                  allowed: Optional[T] = None, repetition_penalty: Union[float, T] = 1.0,
                  presence_penalty: Union[float, T] = 0.0, frequency_penalty: Union[float, T] = 0.0) -> T:
    """One decoding step: the adjusted logits of R rows.

    Args:
        logits: (R, V) float32, float16 or bfloat16 on the GPU; rows may be apart (``scores[:, -1]`` is read in place).
        tokens: (R, L) integer history of every row (None: no history); entries outside [0, V) are ignored.
        tokens_lengths: (R,) tokens of each history, the first ones of its row (None: all L).
        bias: (V,) or (R, V), float32 or the logits' type.
        allowed: (ceil(V/32),) or (R, ceil(V/32)) int32 words of allowed tokens (``pack_token_mask``).
        repetition_penalty, presence_penalty, frequency_penalty: numbers, or (R,) float32 tensors.
    Returns (R, V), contiguous, in the type of the logits; -inf where a token is not allowed.
    """
    if not logits.is_cuda:
        raise RuntimeError("logits must be located in the CUDA")
    _lib.dtype_code(logits.dtype)
    if logits.dim() != 2:
        raise RuntimeError("logits must have 2 dims.")
    R, V = logits.shape
    dev = logits.device
    if (logits.stride(1) != 1 and V > 1) or logits.stride(0) < V:
        logits = logits.contiguous()
    if tokens is not None:
        if tokens.dim() != 2 or tokens.size(0) != R:
            raise RuntimeError(f"tokens must have shape ({R}, L)")
        L = tokens.size(1)
        tokens = _int_on("tokens", tokens, dev)
        if tokens_lengths is None:
            tokens_lengths = torch.full((R,), L, dtype=torch.int32, device=dev)
        elif tokens_lengths.dim() != 1 or tokens_lengths.size(0) != R:
            raise RuntimeError(f"tokens_lengths must have shape ({R},)")
        else:
            tokens_lengths = _int_on("tokens_lengths", tokens_lengths, dev)
    elif tokens_lengths is not None:
        raise RuntimeError("tokens_lengths without tokens")
    else:
        L = 0
    return _apply(logits, R, 1, 1, -1, 0 if logits.is_contiguous() else logits.stride(0), tokens, L, tokens_lengths, None, None, bias,
                  allowed, repetition_penalty, presence_penalty, frequency_penalty, True)


def _joint_args(logits: T, labels: T, frames_lengths: Optional[T], labels_lengths: Optional[T]):
    if not logits.is_cuda:
        raise RuntimeError("logits must be located in the CUDA")
    _lib.dtype_code(logits.dtype)
    if labels.dim() != 2:
        raise RuntimeError("labels must have 2 dims.")
    N = labels.size(0)
    for name, t in (("frames_lengths", frames_lengths), ("labels_lengths", labels_lengths)):
        if t is not None and (t.dim() != 1 or t.size(0) != N):
            raise RuntimeError(f"{name} must have shape ({N},)")
    dev = logits.device
    return (_int_on("labels", labels, dev), None if frames_lengths is None else _int_on("frames_lengths", frames_lengths, dev),
            None if labels_lengths is None else _int_on("labels_lengths", labels_lengths, dev))


def adjust_joint_logits(logits: T, labels: T, frames_lengths: Optional[T] = None, labels_lengths: Optional[T] = None,
                        bias: Optional[T] = None, allowed: Optional[T] = None, repetition_penalty: Union[float, T] = 1.0,
                        presence_penalty: Union[float, T] = 0.0, frequency_penalty: Union[float, T] = 0.0) -> T:
    """The adjusted logits of a joint tensor, for ``ctct_loss_from_logits`` on the same labels and lengths.

    Args:
        logits: (N, T, U, V) raw scores, U = max labels + 1; float32, float16 or bfloat16.
        labels: (N, U-1); the history of rows [n, :, u] is labels[n, :u].
        frames_lengths, labels_lengths: (N,); rows beyond them are zeros and take no part in any gradient.
            None: all rows are valid.
        bias: (V,), (N, V) or (N, U, V), float32 or the logits' type.
        allowed: (ceil(V/32),), (N, ceil(V/32)) or (N, U, ceil(V/32)) int32 words (``pack_token_mask``): a grammar's
            state for each context.
        repetition_penalty, presence_penalty, frequency_penalty: numbers, or (N,) float32 tensors.
    """
    labels, lx, ly = _joint_args(logits, labels, frames_lengths, labels_lengths)
    if logits.dim() != 4 or logits.size(0) != labels.size(0) or logits.size(2) != labels.size(1) + 1:
        raise RuntimeError("logits must have shape (N, T, U, V), labels (N, U - 1)")
    logits = logits.contiguous()
    N, Tm, U1, _ = logits.shape
    return _apply(logits, N, Tm, U1, -1, 0, labels, U1 - 1, None, lx, ly, bias, allowed, repetition_penalty, presence_penalty,
                  frequency_penalty, False)


def adjust_joint_logits_packed(logits: T, labels: T, frames_lengths: T, labels_lengths: T, max_frames: Optional[int] = None,
                               bias: Optional[T] = None, allowed: Optional[T] = None, repetition_penalty: Union[float, T] = 1.0,
                               presence_penalty: Union[float, T] = 0.0, frequency_penalty: Union[float, T] = 0.0) -> T:
    """``adjust_joint_logits`` on a packed (rows, V) joint tensor (``pack_joint``), for ``ctct_loss_packed(from_logits=True)``.

    max_frames: an upper bound of frames_lengths known on the host; omitted, it is read back from the device (one
    synchronisation).  Rows that the lengths place beyond the tensor are not touched, surplus rows are zeros.
    """
    labels, lx, ly = _joint_args(logits, labels, frames_lengths, labels_lengths)
    if logits.dim() != 2:
        raise RuntimeError("packed logits must have 2 dims.")
    if max_frames is None:
        max_frames = int(lx.max().item()) if lx.numel() else 0
    if max_frames < 0:
        raise RuntimeError("max_frames must not be negative")
    logits = logits.contiguous()
    U1 = labels.size(1) + 1
    return _apply(logits, labels.size(0), int(max_frames), U1, logits.size(0), 0, labels, U1 - 1, None, lx, ly, bias, allowed,
                  repetition_penalty, presence_penalty, frequency_penalty, False)
