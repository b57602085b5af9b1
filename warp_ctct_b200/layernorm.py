"""Layer norm, and the layer norm of an additive joiner, with their backward passes.

The reference scores a joint tensor that its caller builds (warp_ctct/__init__.py:97-100); these are the norms that
such a joiner has: over the rows of the encoder's and the predictor's outputs (``layer_norm``), and over
``f[n, t] + g[n, u]`` for every row of the joint tensor (``joint_layer_norm``), in the padded and the packed layout of
the losses.  The sum ``f + g`` never lies in memory: forward writes the joint tensor once, backward reads its
gradient once.  All sums are float32 and taken in a fixed order, so results are the same bits every time.
"""
from __future__ import annotations

from math import inf
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import _as_int, _lib

T = torch.Tensor


def _check_params(x: T, weight: Optional[T], bias: Optional[T], H: int) -> int:
    """Checks weight and bias against activations `x`; 1 if they are float32, 0 if they have x's type."""
    f32 = None
    dtype, device = x.dtype, x.device
    for name, p in (("weight", weight), ("bias", bias)):
        if p is None:
            continue
        if p.dim() != 1 or p.size(0) != H:
            raise RuntimeError(f"{name} must have shape ({H},)")
        pd = p.dtype
        if pd != dtype and pd != torch.float32:
            raise RuntimeError(f"{name} must be float32 or of the activations' type {dtype}, not {pd}")
        if p.device != device:
            raise RuntimeError(f"{name} must be on {device}, not on {p.device}")
        if f32 is not None and f32 != (pd == torch.float32):
            raise RuntimeError("weight and bias must have the same type")
        f32 = pd == torch.float32
    return 1 if f32 else 0


def _check_eps(eps: float) -> float:
    eps = float(eps)
    if not 0.0 <= eps < inf:
        raise RuntimeError(f"eps must be a finite number that is not negative, not {eps}")
    return eps


def _dense(p: Optional[T]) -> Optional[T]:
    return p if p is None or p.is_contiguous() else p.contiguous()


def _wants_grad(*tensors: Optional[T]) -> bool:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


def _as_rows(x: T) -> T:
    """`x` as (rows, H) with adjacent elements in a row and one stride between rows; a copy if it has no such form."""
    if x.dim() == 2 and (x.stride(1) == 1 or x.size(1) == 1):
        return x
    H = x.size(-1)
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
    prev = _lib.enter_device(dev)
    try:
        y = torch.empty_like(rows) if rows.is_contiguous() else rows.new_empty((R, H))
        stats = torch.empty((R, 2), dtype=torch.float32, device=dev) if want_grad else None
        rc = _lib.lib().ctct_b200_layer_norm_forward(
            rows.data_ptr(), rows.stride(0), _lib.dtype_code(rows.dtype), R, H, None if weight is None else weight.data_ptr(),
            None if bias is None else bias.data_ptr(), p_f32, eps, y.data_ptr(), stats.data_ptr() if want_grad else None,
            _lib.raw_stream(dev))
    finally:
        _lib.leave_device(prev)
    if rc:
        _lib.check(rc, "ctct_b200_layer_norm_forward")
    return y, stats


def _ln_backward(ctx, dy: T):
    rows, weight, stats = ctx.saved_tensors
    p_f32, bias_dtype = ctx.meta
    R, H = rows.shape
    dev = rows.device
    lib = _lib.lib()
    code = _lib.dtype_code(rows.dtype)
    dy = _as_rows(dy)
    need_x, need_w, need_b = ctx.needs_input_grad[:3]
    prev = _lib.enter_device(dev)
    try:
        dx = dw = db = ws = None
        nbytes = 0
        if need_x:
            dx = torch.empty_like(rows) if rows.is_contiguous() else rows.new_empty((R, H))
        if need_w:
            dw = torch.empty_like(weight)
        if need_b:
            db = torch.empty((H,), dtype=bias_dtype, device=dev) if dw is None else torch.empty_like(dw)
        if need_w or need_b:
            nbytes = lib.ctct_b200_layer_norm_workspace_bytes(R, H, code)
            ws = torch.empty((nbytes,), dtype=torch.uint8, device=dev)
        rc = lib.ctct_b200_layer_norm_backward(
            dy.data_ptr(), dy.stride(0), rows.data_ptr(), rows.stride(0), code, R, H, _lib.ptr(weight), p_f32, stats.data_ptr(),
            _lib.ptr(dx), _lib.ptr(dw), _lib.ptr(db), _lib.ptr(ws), nbytes, _lib.raw_stream(dev))
    finally:
        _lib.leave_device(prev)
    if rc:
        _lib.check(rc, "ctct_b200_layer_norm_backward")
    return dx, dw, db, None, None


class LayerNorm(torch.autograd.Function):
    """(rows, H) -> (rows, H); x is kept for the backward pass, with 8 bytes of statistics per row."""

    @staticmethod
    def forward(ctx, rows: T, weight: Optional[T], bias: Optional[T], p_f32: int, eps: float):
        y, stats = _ln_forward(rows, weight, bias, p_f32, eps, True)
        ctx.save_for_backward(rows, weight, stats)
        ctx.meta = (p_f32, None if bias is None else bias.dtype)
        return y

    @staticmethod
    def backward(ctx, dy: T):
        # a graph of the gradient is only asked for with create_graph: the guard against a second
        # differentiation costs nothing otherwise
        return _ln_backward_once(ctx, dy) if torch.is_grad_enabled() else _ln_backward(ctx, dy)


_ln_backward_once = once_differentiable(_ln_backward)


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
    dims = x.dim()
    if dims < 1 or x.size(-1) < 1:
        raise RuntimeError("x must have at least one dimension, with at least one element")
    p_f32 = _check_params(x, weight, bias, x.size(-1))
    eps = _check_eps(eps)
    rows, weight, bias = _as_rows(x), _dense(weight), _dense(bias)
    if _wants_grad(x, weight, bias):
        y = LayerNorm.apply(rows, weight, bias, p_f32, eps)
    else:
        y, _ = _ln_forward(rows, weight, bias, p_f32, eps, False)
    return y if dims == 2 else y.view(x.shape)


def _joint_forward(f: T, g: T, lx: Optional[T], ly: Optional[T], weight: Optional[T], bias: Optional[T], p_f32: int, eps: float,
                   rows: int, want_grad: bool):
    """rows < 0: padded.  Returns (y, saved): `saved` holds what the backward pass needs besides the inputs."""
    N, Tm, H = f.shape
    U1 = g.size(1)
    dev = f.device
    lib = _lib.lib()
    prev = _lib.enter_device(dev)
    try:
        y = f.new_empty((rows, H) if rows >= 0 else (N, Tm, U1, H))
        saved, saved_ptr, nbytes = None, None, 0
        if want_grad or rows >= 0:
            nbytes = lib.ctct_b200_joint_norm_saved_bytes(N, Tm, U1, rows, int(want_grad))
            saved = torch.empty((nbytes,), dtype=torch.uint8, device=dev)
            saved_ptr = saved.data_ptr()
        rc = lib.ctct_b200_joint_norm_forward(
            f.data_ptr(), f.stride(0), f.stride(1), g.data_ptr(), g.stride(0), g.stride(1), _lib.dtype_code(f.dtype),
            None if lx is None else lx.data_ptr(), None if ly is None else ly.data_ptr(), N, Tm, U1, H, rows,
            None if weight is None else weight.data_ptr(), None if bias is None else bias.data_ptr(), p_f32, eps, y.data_ptr(),
            want_grad, saved_ptr, nbytes, _lib.raw_stream(dev))
    finally:
        _lib.leave_device(prev)
    if rc:
        _lib.check(rc, "ctct_b200_joint_norm_forward")
    return y, saved


def _joint_backward(ctx, dy: T):
    f, g, weight, lx, ly, saved = ctx.saved_tensors
    p_f32, rows, bias_dtype = ctx.meta
    N, Tm, H = f.shape
    U1 = g.size(1)
    dev = f.device
    lib = _lib.lib()
    code = _lib.dtype_code(f.dtype)
    if not dy.is_contiguous():
        dy = dy.contiguous()
    need_f, need_g, need_w, need_b = ctx.needs_input_grad[:4]
    prev = _lib.enter_device(dev)
    try:
        df = None if not need_f else torch.empty_like(f) if f.is_contiguous() else f.new_empty((N, Tm, H))
        dg = None if not need_g else torch.empty_like(g) if g.is_contiguous() else g.new_empty((N, U1, H))
        dw = torch.empty_like(weight) if need_w else None
        db = None if not need_b else torch.empty((H,), dtype=bias_dtype, device=dev) if dw is None else torch.empty_like(dw)
        nbytes = lib.ctct_b200_joint_norm_workspace_bytes(N, Tm, U1, H, code)
        ws = torch.empty((nbytes,), dtype=torch.uint8, device=dev)
        rc = lib.ctct_b200_joint_norm_backward(
            dy.data_ptr(), f.data_ptr(), f.stride(0), f.stride(1), g.data_ptr(), g.stride(0), g.stride(1), code,
            _lib.ptr(lx), _lib.ptr(ly), N, Tm, U1, H, rows, _lib.ptr(weight), p_f32, saved.data_ptr(), saved.numel(),
            _lib.ptr(df), _lib.ptr(dg), _lib.ptr(dw), _lib.ptr(db), ws.data_ptr(), nbytes, _lib.raw_stream(dev))
    finally:
        _lib.leave_device(prev)
    if rc:
        _lib.check(rc, "ctct_b200_joint_norm_backward")
    return df, dg, dw, db, None, None, None, None, None


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
    def backward(ctx, dy: T):
        return _joint_backward_once(ctx, dy) if torch.is_grad_enabled() else _joint_backward(ctx, dy)


_joint_backward_once = once_differentiable(_joint_backward)


def _joint(f: T, g: T, lx: Optional[T], ly: Optional[T], weight: Optional[T], bias: Optional[T], eps: float, rows: int) -> T:
    if not f.is_cuda:
        raise RuntimeError("f must be located in the CUDA")
    if not g.is_cuda:
        raise RuntimeError("g must be located in the CUDA")
    _lib.dtype_code(f.dtype)
    if f.dim() != 3 or g.dim() != 3:
        raise RuntimeError("f and g must have shapes (N, T, H) and (N, U, H)")
    N, _, H = f.shape
    Ng, U1, Hg = g.shape
    if N != Ng or H != Hg:
        raise RuntimeError("f and g must have shapes (N, T, H) and (N, U, H)")
    if g.dtype != f.dtype or g.device != f.device:
        raise RuntimeError("f and g must have the same type and device")
    if H < 1 or U1 < 1:
        raise RuntimeError("f and g must have at least one element per row, g at least one context")
    for name, t in (("frames_lengths", lx), ("labels_lengths", ly)):
        if t is None:
            continue
        if t.dim() != 1 or t.size(0) != N:
            raise RuntimeError(f"{name} must have shape ({N},)")
        if t.device != f.device:
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
    if _wants_grad(f, g, weight, bias):
        return JointLayerNorm.apply(f, g, weight, bias, lx, ly, p_f32, eps, rows)
    return _joint_forward(f, g, lx, ly, weight, bias, p_f32, eps, rows, False)[0]


def joint_layer_norm(f: T, g: T, frames_lengths: Optional[T] = None, labels_lengths: Optional[T] = None,
                     weight: Optional[T] = None, bias: Optional[T] = None, eps: float = 1e-5) -> T:
    """``layer_norm(f[:, :, None] + g[:, None], weight, bias, eps)`` for every row of the joint tensor.

    Args:
        f: (N, T, H) encoder frames, g: (N, U, H) predictor states (U = max labels + 1), the same type: float32,
            float16 or bfloat16, H up to 8192.  Both may be slices or expanded, as long as a row's elements are adjacent.
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
