"""Products with bias, activation and residual in their epilogue on the gfx950
GEMM core (``csrc/linear.hip``, ``include/mm1_linear.h``): how a sublayer's
output joins the residual stream in one launch, where the reference runs a
torch product and an addition (CODE/mimans/model/attention_tilelang.py:518,
swiglu_tilelang.py:284-286, block.py:81-92).

* ``fused_linear(x, w, bias, activation, residual, out_dtype)``:
  ``act(x w^T + bias) + residual``, differentiable once in every tensor
  (in reverse; forward-mode tangents are refused);
* ``Linear``: an ``nn.Linear`` with an activation whose forward takes a residual.

``Attention`` and ``SwiGLU`` call it for their last product when they are given
the residual stream (``forward(x, residual=...)``).

x and w enter the product in bf16 (fp32 ones are rounded, as under bf16
autocast), sums and epilogue are fp32, the output is rounded once.  Any sizes
and strides: operands that the tiles do not take as they lie (fp32, widths that 8
does not divide, odd starts) are copied with zeros behind their rows.  The
backward keeps z in bf16 where there is an activation; its output gradient
enters the products in bf16, and the bias's gradient is summed before that
rounding.  Results are bitwise repeatable.
"""
from __future__ import annotations

import functools

import torch
import torch.nn as nn

from . import _lib
from .calls import F32, call, refuse_tangents, workspace

DTYPE = torch.bfloat16
ROW, COL = 0, 1                 # MM1_GEMM_ROW, MM1_GEMM_COL
MAX_WIDTH = 4_000_000           # N and K whose rows the tiles' offsets reach, forward and backward
MAX_ROWS = 1 << 28
MAX_LD = 1 << 21                # longest row stride that the tiles' 32-bit offsets are sure to take
ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}      # MM1_ACT_*


@functools.lru_cache(maxsize=1024)
def _product_bytes(m, n, k, w_layout, act):
    return _lib.load().mm1_linear_workspace_size(m, n, k, ROW, w_layout, act)


@functools.lru_cache(maxsize=1024)
def _backward_bytes(m, n, k, dz, dx, dw, db):
    return _lib.load().mm1_linear_backward_workspace_size(m, n, k, dz, dx, dw, db)


def _row_stride(t):
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _operand(t):
    """(tensor, row stride): `t` in bf16 with rows that the products read in
    pieces of 8 -- as it lies in memory, or a copy with zeros behind its rows."""
    rows, cols = t.shape
    if t.dtype is DTYPE and cols % 8 == 0 and t.is_contiguous() and t.data_ptr() % 16 == 0:
        return t, cols
    t = _rows(t)
    ld = t.stride(0) if rows > 1 else cols
    if t.dtype is DTYPE and cols % 8 == 0 and ld % 8 == 0 and ld <= MAX_LD and t.data_ptr() % 16 == 0:
        return t, ld
    width = -(-cols // 8) * 8
    packed = torch.empty(rows, width, dtype=DTYPE, device=t.device)
    call("mm1_pack_bf16", t.device, t.data_ptr(), F32[t.dtype], ld, rows, cols, packed.data_ptr(), width, rows)
    return packed, width


def _rows(t, longest=1 << 40):
    """The 2-D tensor `t` where it has rows of consecutive values that do not
    overlap, at most `longest` apart, else a copy that has."""
    rows, cols = t.shape
    if (cols > 1 and t.stride(1) != 1) or (rows > 1 and not cols <= t.stride(0) <= longest):
        return t.contiguous()
    return t


def _forward(x, w, bias, act, residual, out_dtype, train):
    """(output, x and its row stride, w, its layout and row stride, z in bf16 or
    None): the product and what its backward reads; operands None for no rows."""
    n, k = w.shape
    device = x.device
    x2 = x if x.dim() == 2 else x.reshape(-1, k)
    m = x2.shape[0]
    out = torch.empty(m, n, dtype=out_dtype, device=device)
    shaped = out if x.dim() == 2 else out.view(*x.shape[:-1], n)
    if m == 0:
        return shaped, None, 0, None, ROW, 0, None
    layout = ROW
    if k > 1 and w.stride(1) != 1 and (n == 1 or w.stride(0) == 1):
        w, layout = w.t(), COL
    x2, ldx = _operand(x2)
    w2, ldw = _operand(w)
    pre = torch.empty(m, n, dtype=DTYPE, device=device) if train and act else None
    if residual is not None:
        residual = _rows(residual if residual.dim() == 2 else residual.reshape(m, n), MAX_LD)
    keep, ws, ws_bytes = workspace(_product_bytes(m, n, k, layout, act), device)
    call("mm1_linear", device, x2.data_ptr(), ROW, ldx, w2.data_ptr(), layout, ldw,
         None if bias is None else bias.data_ptr(), 0 if bias is None else F32[bias.dtype], act,
         None if residual is None else residual.data_ptr(), 0 if residual is None else F32[residual.dtype],
         0 if residual is None else _row_stride(residual), None if pre is None else pre.data_ptr(), n, out.data_ptr(),
         F32[out_dtype], n, ws, ws_bytes, m, n, k)
    return shaped, x2, ldx, w2, layout, ldw, pre


class FusedLinear(torch.autograd.Function):
    """fused_linear on checked arguments."""

    @staticmethod
    def forward(ctx, x, w, bias, act, residual, out_dtype):
        out, x2, ldx, w2, layout, ldw, pre = _forward(x, w, bias, act, residual, out_dtype, True)
        ctx.save_for_backward(x2, w2, pre)
        ctx.meta = (x.shape, w.shape, act, ldx, layout, ldw, x.dtype, w.dtype, None if bias is None else bias.dtype,
                    None if residual is None else residual.dtype)
        return out

    @staticmethod
    def backward(ctx, dy):
        return _recorded_gradients(ctx, dy) if torch.is_grad_enabled() else _gradients(ctx, dy)


def _gradients(ctx, dy):
    """FusedLinear's backward: one call of the library."""
    x_shape, (n, k), act, ldx, layout, ldw, x_dtype, w_dtype, b_dtype, r_dtype = ctx.meta
    need_x, need_w, need_b, _, need_r, _ = ctx.needs_input_grad
    device, dtype = dy.device, dy.dtype
    dr = None if not need_r else dy if dtype is r_dtype else dy.to(r_dtype)
    dy2 = _rows(dy if dy.dim() == 2 else dy.reshape(-1, n), MAX_LD)
    m = dy2.shape[0]
    new = torch.empty if m else torch.zeros
    dx = new(x_shape, dtype=x_dtype, device=device) if need_x else None
    # in w's own layout, as the [N, K] that it is a view of
    dw = new((n, k) if layout == ROW else (k, n), dtype=w_dtype, device=device) if need_w else None
    db = new(n, dtype=b_dtype, device=device) if need_b else None
    if m and (need_x or need_w or need_b):
        x2, w2, pre = ctx.saved_tensors
        ldy, at = _row_stride(dy2), dy2.data_ptr()
        form = act != 0 or dtype is not DTYPE or n % 8 != 0 or ldy % 8 != 0 or at % 16 != 0
        keep, ws, ws_bytes = workspace(_backward_bytes(m, n, k, form, need_x, need_w, need_b), device)
        call("mm1_linear_backward", device, at, F32[dtype], ldy, None if pre is None else pre.data_ptr(), n, act,
             x2.data_ptr(), ldx, w2.data_ptr(), layout, ldw, None if dx is None else dx.data_ptr(), F32[x_dtype],
             None if dw is None else dw.data_ptr(), F32[w_dtype], None if db is None else db.data_ptr(),
             0 if db is None else F32[b_dtype], ws, ws_bytes, m, n, k)
    return dx, dw if dw is None or layout == ROW else dw.t(), db, None, dr, None


# under create_graph: a second derivative raises
_recorded_gradients = torch.autograd.function.once_differentiable(_gradients)


def _check(t, name, device, shape=None):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not t.is_cuda or t.device != device:
        raise ValueError(f"{name} must be a CUDA (HIP) tensor on x's device, got device {t.device}")
    if t.dtype not in F32:
        raise TypeError(f"{name} must be fp32 or bf16, got {t.dtype}")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")


def _check_sizes(rows, n, k):
    """What the library takes, before its 32-bit arguments."""
    if n > MAX_WIDTH or k > MAX_WIDTH:
        raise ValueError(f"N and K are at most {MAX_WIDTH:,}, got {n:,} and {k:,}")
    if rows > MAX_ROWS:
        raise ValueError(f"x has {rows:,} rows, at most {MAX_ROWS:,} are taken")


def fused_linear(x, w, bias=None, activation="none", residual=None, out_dtype=None):
    """``act(x w^T + bias) + residual`` [..., N]: x [..., K] and w [N, K]
    (nn.Linear's layout, or the transposed view of a [K, N] matrix), bias [N]
    and residual [..., N] in fp32 or bf16; activation "none", "relu", "gelu",
    "gelu_tanh" or "silu".  The output is in ``out_dtype``, by default the
    residual's, without one bf16.  N and K are at most 4,000,000, rows 2^28."""
    refuse_tangents("fused_linear", (x, w, bias, residual))
    device = getattr(x, "device", None)
    _check(x, "x", device)
    _check(w, "w", device)
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"unknown activation {activation!r}")
    x_shape, w_shape = x.shape, w.shape
    if len(w_shape) != 2 or not x_shape or x_shape[-1] != w_shape[1] or 0 in w_shape:
        raise ValueError(f"x has shape {tuple(x_shape)}, w {tuple(w_shape)}: [..., K] and [N, K] expected")
    n, k = w_shape
    _check_sizes(x.numel() // k, n, k)
    needs_grad = x.requires_grad or w.requires_grad
    if bias is not None:
        _check(bias, "bias", device, w_shape[:1])
        bias = bias if bias.is_contiguous() else bias.contiguous()
        needs_grad = needs_grad or bias.requires_grad
    if residual is not None:
        _check(residual, "residual", device, (*x_shape[:-1], w_shape[0]))
        needs_grad = needs_grad or residual.requires_grad
    if out_dtype is None:
        out_dtype = DTYPE if residual is None else residual.dtype
    elif out_dtype not in F32:
        raise TypeError(f"out_dtype must be fp32 or bf16, got {out_dtype}")
    if needs_grad and torch.is_grad_enabled():
        return FusedLinear.apply(x, w, bias, act, residual, out_dtype)
    return _forward(x, w, bias, act, residual, out_dtype, False)[0]


class Linear(nn.Linear):
    """``nn.Linear`` (same parameters, state and initialisation) on
    ``fused_linear``: ``forward(x, residual=None)`` is
    ``act(x weight^T + bias) + residual``.  The arithmetic is ``fused_linear``'s
    whatever the parameters' type: fp32 ones enter the product rounded to bf16,
    under autocast or not, and their gradients come from bf16 operands."""

    def __init__(self, in_features, out_features, bias=True, activation="none", device=None, dtype=None):
        super().__init__(in_features, out_features, bias, device=device, dtype=dtype)
        if activation not in ACTIVATIONS:
            raise ValueError(f"unknown activation {activation!r}")
        self.activation = activation

    def forward(self, x, residual=None):
        return fused_linear(x, self.weight, self.bias, self.activation, residual)

    def extra_repr(self):
        return f"{super().extra_repr()}, activation={self.activation}"
