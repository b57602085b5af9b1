"""Layer norm, and the layer norm of an additive joiner, with their backward passes.

The reference scores a joint tensor that its caller builds (warp_ctct/__init__.py:97-100); these are the norms that
such a joiner has: over the rows of the encoder's and the predictor's outputs (``layer_norm``), and over
``f[n, t] + g[n, u]`` for every row of the joint tensor (``joint_layer_norm``), in the padded and the packed layout of
the losses.  The sum ``f + g`` never lies in memory: forward writes the joint tensor once, backward reads its
gradient once.  All sums are float32 and taken in a fixed order, so results are the same bits every time.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import _lib

T = torch.Tensor


def _check_params(x: T, weight: Optional[T], bias: Optional[T], H: int) -> int:
    """Checks weight and bias against activations `x`; 1 if they are float32, 0 if they have x's type."""
    f32 = None
    for name, p in (("weight", weight), ("bias", bias)):
        if p is None:
            continue
        if p.dim() != 1 or p.size(0) != H:
            raise RuntimeError(f"{name} must have shape ({H},)")
        if p.dtype != x.dtype and p.dtype != torch.float32:
            raise RuntimeError(f"{name} must be float32 or of the activations' type {x.dtype}, not {p.dtype}")
        if p.device != x.device:
            raise RuntimeError(f"{name} must be on {x.device}, not on {p.device}")
        is_f32 = p.dtype == torch.float32
        if f32 is not None and f32 != is_f32:
            raise RuntimeError("weight and bias must have the same type")
        f32 = is_f32
    return int(bool(f32))


def _check_eps(eps: float) -> float:
    eps = float(eps)
    if not 0.0 <= eps < float("inf"):
        raise RuntimeError(f"eps must be a finite number that is not negative, not {eps}")
    return eps


def _dense(p: Optional[T]) -> Optional[T]:
    return p if p is None or p.is_contiguous() else p.contiguous()


def _as_rows(x: T) -> T:
    """`x` as (rows, H) with adjacent elements in a row and one stride between rows; a copy if it has no such form."""
    H = x.size(-1)
    if x.dim() == 2 and (x.stride(1) == 1 or H == 1) and x.stride(0) >= 0:
        return x
    if x.is_contiguous():
        return x.view(-1, H)
    if x.dim() == 2 or x.stride(-1) != 1:
        return x.contiguous().view(-1, H)
    try:
        return x.view(-1, H)
    except RuntimeError:
        return x.contiguous().view(-1, H)


def _ln_forward(rows: T, weight: Optional[T], bias: Optional[T], p_f32: int, eps: float, want_grad: bool):
    R, H = rows.shape
    dev = rows.device
    with _lib.on_device(dev):
        y = torch.empty((R, H), dtype=rows.dtype, device=dev)
        stats = torch.empty((R, 2), dtype=torch.float32, device=dev) if want_grad else None
        rc = _lib.lib().ctct_b200_layer_norm_forward(
            rows.data_ptr(), rows.stride(0), _lib.dtype_code(rows.dtype), R, H, _lib.ptr(weight), _lib.ptr(bias), p_f32, eps,
            y.data_ptr(), _lib.ptr(stats), _lib.raw_stream(dev))
    _lib.check(rc, "ctct_b200_layer_norm_forward")
    return y, stats


class LayerNorm(torch.autograd.Function):
    """(rows, H) -> (rows, H); x is kept for the backward pass, with 8 bytes of statistics per row."""

    @staticmethod
    def forward(ctx, rows: T, weight: Optional[T], bias: Optional[T], p_f32: int, eps: float):
        y, stats = _ln_forward(rows, weight, bias, p_f32, eps, True)
        ctx.save_for_backward(rows, weight, stats)
        ctx.meta = (p_f32, None if bias is None else bias.dtype)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy: T):
        rows, weight, stats = ctx.saved_tensors
        p_f32, bias_dtype = ctx.meta
        R, H = rows.shape
        dev = rows.device
        lib = _lib.lib()
        code = _lib.dtype_code(rows.dtype)
        dy = _as_rows(dy)
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        with _lib.on_device(dev):
            dx = torch.empty((R, H), dtype=rows.dtype, device=dev) if need_x else None
            dw = torch.empty((H,), dtype=weight.dtype, device=dev) if need_w else None
            db = torch.empty((H,), dtype=bias_dtype, device=dev) if need_b else None
            ws, nbytes = None, 0
            if need_w or need_b:
                nbytes = lib.ctct_b200_layer_norm_workspace_bytes(R, H, code)
                ws = torch.empty((nbytes,), dtype=torch.uint8, device=dev)
            rc = lib.ctct_b200_layer_norm_backward(
                dy.data_ptr(), dy.stride(0), rows.data_ptr(), rows.stride(0), code, R, H, _lib.ptr(weight), p_f32,
                stats.data_ptr(), _lib.ptr(dx), _lib.ptr(dw), _lib.ptr(db), _lib.ptr(ws), nbytes, _lib.raw_stream(dev))
        _lib.check(rc, "ctct_b200_layer_norm_backward")
        return dx, dw, db, None, None


def layer_norm(x: T, weight: Optional[T] = None, bias: Optional[T] = None, eps: float = 1e-5) -> T:
    """Layer norm over the last dimension: ``(x - mean) / sqrt(var + eps) * weight + bias``.

    Args:
        x: (..., H) float32, float16 or bfloat16 on the GPU.  Rows may be apart (a slice of a wider
            tensor is read in place); statistics are float32.
        weight, bias: (H,) in float32 or in the type of ``x`` (both the same); None: ones, zeros.
        eps: added to the variance.
    Returns a contiguous tensor of the shape and type of ``x``.  Gradients flow to x, weight and bias, once.
    """
    if not x.is_cuda:
        raise RuntimeError("x must be located in the CUDA")
    _lib.dtype_code(x.dtype)
    if x.dim() < 1 or x.size(-1) < 1:
        raise RuntimeError("x must have at least one dimension, with at least one element")
    p_f32 = _check_params(x, weight, bias, x.size(-1))
    eps = _check_eps(eps)
    rows, weight, bias = _as_rows(x), _dense(weight), _dense(bias)
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)
                                    or (bias is not None and bias.requires_grad)):
        y = LayerNorm.apply(rows, weight, bias, p_f32, eps)
    else:
        y, _ = _ln_forward(rows, weight, bias, p_f32, eps, False)
    return y if x.dim() == 2 else y.view(x.shape)


def _joint_forward(f: T, g: T, lx: Optional[T], ly: Optional[T], weight: Optional[T], bias: Optional[T], p_f32: int, eps: float,
                   rows: int, want_grad: bool):
    """rows < 0: padded.  Returns (y, saved): `saved` holds what the backward pass needs besides the inputs."""
    N, Tm, H = f.shape
    U1 = g.size(1)
    dev = f.device
    lib = _lib.lib()
    with _lib.on_device(dev):
        y = torch.empty((rows, H) if rows >= 0 else (N, Tm, U1, H), dtype=f.dtype, device=dev)
        saved, nbytes = None, 0
        if want_grad or rows >= 0:
            nbytes = lib.ctct_b200_joint_norm_saved_bytes(N, Tm, U1, rows, int(want_grad))
            saved = torch.empty((nbytes,), dtype=torch.uint8, device=dev)
        rc = lib.ctct_b200_joint_norm_forward(
            f.data_ptr(), f.stride(0), f.stride(1), g.data_ptr(), g.stride(0), g.stride(1), _lib.dtype_code(f.dtype),
            _lib.ptr(lx), _lib.ptr(ly), N, Tm, U1, H, rows, _lib.ptr(weight), _lib.ptr(bias), p_f32, eps, y.data_ptr(),
            int(want_grad), _lib.ptr(saved), nbytes, _lib.raw_stream(dev))
    _lib.check(rc, "ctct_b200_joint_norm_forward")
    return y, saved


class JointLayerNorm(torch.autograd.Function):
    """y = LN(f[:, :, None] + g[:, None]) on the valid rows; keeps f, g and 4 bytes per row."""

    @staticmethod
    def forward(ctx, f: T, g: T, weight: Optional[T], bias: Optional[T], lx: Optional[T], ly: Optional[T], p_f32: int, eps: float,
                rows: int):
        y, saved = _joint_forward(f, g, lx, ly, weight, bias, p_f32, eps, rows, True)
        ctx.save_for_backward(f, g, weight, lx, ly, saved)
        ctx.meta = (p_f32, rows, None if bias is None else bias.dtype)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy: T):
        f, g, weight, lx, ly, saved = ctx.saved_tensors
        p_f32, rows, bias_dtype = ctx.meta
        N, Tm, H = f.shape
        U1 = g.size(1)
        dev = f.device
        lib = _lib.lib()
        dy = dy.contiguous()
        need_f, need_g, need_w, need_b = ctx.needs_input_grad[:4]
        with _lib.on_device(dev):
            df = torch.empty((N, Tm, H), dtype=f.dtype, device=dev) if need_f else None
            dg = torch.empty((N, U1, H), dtype=f.dtype, device=dev) if need_g else None
            dw = torch.empty((H,), dtype=weight.dtype, device=dev) if need_w else None
            db = torch.empty((H,), dtype=bias_dtype, device=dev) if need_b else None
            nbytes = lib.ctct_b200_joint_norm_workspace_bytes(N, Tm, U1, H)
            ws = torch.empty((nbytes,), dtype=torch.uint8, device=dev)
            rc = lib.ctct_b200_joint_norm_backward(
                dy.data_ptr(), f.data_ptr(), f.stride(0), f.stride(1), g.data_ptr(), g.stride(0), g.stride(1),
                _lib.dtype_code(f.dtype), _lib.ptr(lx), _lib.ptr(ly), N, Tm, U1, H, rows, _lib.ptr(weight), p_f32,
                saved.data_ptr(), saved.numel(), _lib.ptr(df), _lib.ptr(dg), _lib.ptr(dw), _lib.ptr(db), ws.data_ptr(), nbytes,
                _lib.raw_stream(dev))
        _lib.check(rc, "ctct_b200_joint_norm_backward")
        return df, dg, dw, db, None, None, None, None, None


def _joint(f: T, g: T, lx: Optional[T], ly: Optional[T], weight: Optional[T], bias: Optional[T], eps: float, rows: int) -> T:
    from . import _as_int
    for name, t in (("f", f), ("g", g)):
        if not t.is_cuda:
            raise RuntimeError(f"{name} must be located in the CUDA")
    _lib.dtype_code(f.dtype)
    if f.dim() != 3 or g.dim() != 3 or f.size(0) != g.size(0) or f.size(2) != g.size(2):
        raise RuntimeError("f and g must have shapes (N, T, H) and (N, U, H)")
    if g.dtype != f.dtype or g.device != f.device:
        raise RuntimeError("f and g must have the same type and device")
    N, _, H = f.shape
    if H < 1 or g.size(1) < 1:
        raise RuntimeError("f and g must have at least one element per row, g at least one context")
    for name, t in (("frames_lengths", lx), ("labels_lengths", ly)):
        if t is not None and (t.dim() != 1 or t.size(0) != N):
            raise RuntimeError(f"{name} must have shape ({N},)")
        if t is not None and t.device != f.device:
            raise RuntimeError(f"{name} must be on {f.device}, not on {t.device}")
    p_f32 = _check_params(f, weight, bias, H)
    eps = _check_eps(eps)
    if f.stride(2) != 1 and H > 1:
        f = f.contiguous()
    if g.stride(2) != 1 and H > 1:
        g = g.contiguous()
    weight, bias = _dense(weight), _dense(bias)
    lx = None if lx is None else _as_int(lx)
    ly = None if ly is None else _as_int(ly)
    if torch.is_grad_enabled() and (f.requires_grad or g.requires_grad or (weight is not None and weight.requires_grad)
                                    or (bias is not None and bias.requires_grad)):
        return JointLayerNorm.apply(f, g, weight, bias, lx, ly, p_f32, eps, rows)
    return _joint_forward(f, g, lx, ly, weight, bias, p_f32, eps, rows, False)[0]


def joint_layer_norm(f: T, g: T, frames_lengths: Optional[T] = None, labels_lengths: Optional[T] = None,
                     weight: Optional[T] = None, bias: Optional[T] = None, eps: float = 1e-5) -> T:
    """``layer_norm(f[:, :, None] + g[:, None], weight, bias, eps)`` for every row of the joint tensor.

    Args:
        f: (N, T, H) encoder frames, g: (N, U, H) predictor states (U = max labels + 1), the same type: float32,
            float16 or bfloat16.  Both may be slices or expanded, as long as a row's elements are adjacent.
        frames_lengths, labels_lengths: (N,) as in ``ctct_loss``; rows beyond them are zeros and take no
            part in any gradient.  None: all rows are valid.
        weight, bias, eps: as in ``layer_norm``.
    Returns (N, T, U, H).  One step of a decoder is T = 1, with U hypotheses.
    """
    return _joint(f, g, frames_lengths, labels_lengths, weight, bias, eps, -1)


def joint_layer_norm_packed(f: T, g: T, frames_lengths: T, labels_lengths: T, weight: Optional[T] = None,
                            bias: Optional[T] = None, eps: float = 1e-5, rows: Optional[int] = None) -> T:
    """``pack_joint(joint_layer_norm(...), frames_lengths, labels_lengths)`` without the padded tensor.

    rows: the number of valid rows, sum of frames_lengths[n] * (labels_lengths[n] + 1), known where the batch was
    put together; omitted, it is read back from the device (one synchronisation).  With another number, rows
    beyond it are not computed, and surplus rows are zeros.
    """
    if rows is None:
        rows = int((frames_lengths.clamp(0, f.size(1)).long() * (labels_lengths.clamp(0, g.size(1) - 1).long() + 1)).sum().item())
    if rows < 0:
        raise RuntimeError("rows must not be negative")
    return _joint(f, g, frames_lengths, labels_lengths, weight, bias, eps, int(rows))
