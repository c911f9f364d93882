"""Embedding lookup with a scale and its gradient on the gfx950 kernels of
``csrc/embedding.hip`` (``include/mm1_embedding.h``): how tokens enter the model
whose tied output head (``lm_head.py``) reads the same matrix.  The reference
uses torch's ``nn.Embedding`` there (CODE/mimans/model/model.py:53-127).

* ``embed(ids, weight, scale, padding_idx, out_dtype)``: rows of ``weight``
  times ``scale``, differentiable in ``weight`` (any number of times,
  in reverse; forward-mode tangents are refused);
* ``embedding_grad(ids, grad_out, vocab, ...)``: the matrix's gradient, new or
  added to one that is there (the tied head's);
* ``Embedding``: an ``nn.Embedding`` whose lookup runs here, to be handed to
  ``LMHead`` like any other.

ids: int64 or int32 of any shape.  An id outside [0, vocab) -- a padded batch's
fill, such as ``IGNORE_INDEX`` -- gives a row of zeros and no gradient.  Values
are fp32 or bf16, sums fp32; the gradient adds each row's tokens in their order,
so it is bitwise repeatable.
"""
from __future__ import annotations

import torch
import torch.nn as nn

from . import _lib
from .calls import F32, call, refuse_tangents, workspace, written

MAX_VOCAB, MAX_DIM = 1 << 30, (1 << 31) - 1     # what the library's 32-bit arguments hold


def _check_sizes(vocab, dim):
    if not 1 <= vocab <= MAX_VOCAB or not 1 <= dim <= MAX_DIM:
        raise ValueError(f"a matrix of {vocab:,} rows and {dim:,} columns: 1 to {MAX_VOCAB:,} rows are taken, of 1 to "
                         f"{MAX_DIM:,} columns")


def _check_ids(ids):
    if not isinstance(ids, torch.Tensor):
        raise TypeError("ids must be a torch.Tensor")
    if not ids.is_cuda:
        raise ValueError(f"ids must be a CUDA (HIP) tensor, got device {ids.device}")
    if ids.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"ids must be int64 or int32, got {ids.dtype}")


def _check_rows(t, name, device, shape=None):
    """A 2-D fp32 or bf16 tensor on `device` whose rows are consecutive values."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.device != device:
        raise ValueError(f"{name} must be on {device}, got device {t.device}")
    if t.dtype not in F32:
        raise TypeError(f"{name} must be fp32 or bf16, got {t.dtype}")
    if t.dim() != 2 or (shape is not None and tuple(t.shape) != tuple(shape)):
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape) if shape else '[vocab, dim]'}")
    _check_sizes(*t.shape)
    if (t.shape[1] > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < t.shape[1]):
        raise ValueError(f"{name} must have rows of consecutive values that do not overlap, got strides {t.stride()}")


def _row_stride(t):
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _span(t):
    """The bytes from a tensor's first value to behind its last."""
    return (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()


def _shares(out, t):
    """Whether `out`, rows of values, may share memory with `t`: their spans meet
    and they are not different columns of rows equally far apart."""
    a0, b0 = out.data_ptr(), t.data_ptr()
    if (b0 >= a0 + _span(out) if b0 >= a0 else a0 >= b0 + _span(t)) or not t.numel():
        return False
    pitch, width = out.stride(0) * out.element_size(), out.shape[1] * out.element_size()
    steps = [(n, s) for n, s in zip(t.shape, t.stride()) if n > 1]
    cols = steps.pop()[0] if steps and steps[-1][1] == 1 else 1
    if pitch == 0 or any(s * t.element_size() % pitch for _, s in steps):
        return True
    at, wide = (b0 - a0) % pitch, cols * t.element_size()      # t's columns seen from out's first
    return at < width or at + wide > pitch


def _padding(padding_idx, vocab):
    """-1 for none; a negative index counts from the end, as in nn.Embedding."""
    if padding_idx is None:
        return -1
    if not -vocab <= padding_idx < vocab:
        raise ValueError(f"padding_idx {padding_idx} is outside a vocabulary of {vocab}")
    return padding_idx % vocab


def _lookup(ids, weight, scale, out_dtype):
    vocab, dim = weight.shape
    out = torch.empty(*ids.shape, dim, dtype=out_dtype, device=ids.device)
    flat = ids if ids.is_contiguous() else ids.contiguous()
    call("mm1_embedding", ids.device, flat.data_ptr(), int(flat.dtype is torch.int64), weight.data_ptr(),
         F32[weight.dtype], _row_stride(weight), out.data_ptr(), F32[out_dtype], dim, scale, flat.numel(), vocab, dim)
    return out


def _gradient(ids, grad_out, scale, padding, out, accumulate):
    """The kernels on checked arguments; `out` [vocab, dim] is written."""
    vocab, dim = out.shape
    flat = ids if ids.is_contiguous() else ids.contiguous()
    rows = grad_out.reshape(-1, dim)
    # one stored row for all tokens is read as such; anything else that is not rows of values is copied
    if (dim > 1 and rows.stride(1) != 1) or (rows.shape[0] > 1 and 0 != rows.stride(0) < dim):
        rows = rows.contiguous()
    keep, ws, ws_bytes = workspace(_lib.load().mm1_embedding_grad_workspace_size(flat.numel(), vocab, dim), ids.device)
    call("mm1_embedding_grad", ids.device, flat.data_ptr(), int(flat.dtype is torch.int64), rows.data_ptr(),
         F32[rows.dtype], _row_stride(rows), out.data_ptr(), F32[out.dtype], _row_stride(out), scale, padding,
         int(accumulate), ws, ws_bytes, flat.numel(), vocab, dim)
    return out


def embedding_grad(ids, grad_out, vocab, scale=1.0, padding_idx=None, dtype=torch.float32, out=None,
                   accumulate=False):
    """[vocab, dim]: row v is ``scale`` times the sum of ``grad_out`` [..., dim]
    over the tokens whose id is v.  Written to ``out`` (its own dtype; a row
    stride of its own) or to a new tensor of ``dtype``; with ``accumulate`` the
    sums are added to ``out``, whose other rows are left as they are.  ``out``
    shares no memory with the inputs.  Leaves no autograd graph."""
    refuse_tangents("embedding_grad", (grad_out, out))
    _check_ids(ids)
    if not isinstance(grad_out, torch.Tensor):
        raise TypeError("grad_out must be a torch.Tensor")
    if grad_out.device != ids.device:
        raise ValueError(f"grad_out must be on {ids.device}, got device {grad_out.device}")
    if grad_out.dtype not in F32:
        raise TypeError(f"grad_out must be fp32 or bf16, got {grad_out.dtype}")
    if grad_out.dim() < 1 or grad_out.shape[:-1] != ids.shape or grad_out.shape[-1] < 1:
        raise ValueError(f"grad_out has shape {tuple(grad_out.shape)}, expected {tuple(ids.shape)} and a width")
    dim = grad_out.shape[-1]
    _check_sizes(vocab, dim)
    padding = _padding(padding_idx, vocab)
    if out is None:
        if accumulate:
            raise ValueError("accumulate adds to `out`, which is missing")
        if dtype not in F32:
            raise TypeError(f"dtype must be fp32 or bf16, got {dtype}")
        out = torch.empty(vocab, dim, dtype=dtype, device=ids.device)
        return _gradient(ids, grad_out.detach(), scale, padding, out, False)
    _check_rows(out, "out", ids.device, (vocab, dim))
    if out.requires_grad:
        raise ValueError("out must not require a gradient: it is written in place")
    if _shares(out, grad_out) or _shares(out, ids):
        raise ValueError("out must not share memory with grad_out or ids: it is written while they are read")
    _gradient(ids, grad_out.detach(), scale, padding, out, accumulate)
    written(out)
    return out


class EmbeddingGrad(torch.autograd.Function):
    """embedding_grad as a function of grad_out, whose own derivative is a
    lookup: what a recorded backward of FusedEmbedding leaves in the graph."""

    @staticmethod
    def forward(ctx, grad_out, ids, vocab, scale, padding, dtype):
        ctx.save_for_backward(ids)
        ctx.scale, ctx.padding, ctx.grad_dtype = scale, padding, grad_out.dtype
        out = torch.empty(vocab, grad_out.shape[-1], dtype=dtype, device=ids.device)
        return _gradient(ids, grad_out, scale, padding, out, False)

    @staticmethod
    def backward(ctx, grad):
        (ids,) = ctx.saved_tensors
        if ctx.padding >= 0:       # the padding row takes no gradient, so it hands none on
            ids = torch.where(ids == ctx.padding, -1, ids)
        return FusedEmbedding.apply(ids, grad.contiguous(), ctx.scale, -1, ctx.grad_dtype), None, None, None, None, None


class FusedEmbedding(torch.autograd.Function):
    """scale * weight[ids]; see ``embed``."""

    @staticmethod
    def forward(ctx, ids, weight, scale, padding, out_dtype):
        ctx.save_for_backward(ids)
        ctx.meta = (weight.shape[0], scale, padding, weight.dtype)
        return _lookup(ids, weight, scale, out_dtype)

    @staticmethod
    def backward(ctx, grad_out):
        (ids,) = ctx.saved_tensors
        vocab, scale, padding, dtype = ctx.meta
        if not torch.is_grad_enabled():
            out = torch.empty(vocab, grad_out.shape[-1], dtype=dtype, device=ids.device)
            return None, _gradient(ids, grad_out, scale, padding, out, False), None, None, None
        return None, EmbeddingGrad.apply(grad_out, ids, vocab, scale, padding, dtype), None, None, None


def embed(ids, weight, scale=1.0, padding_idx=None, out_dtype=None):
    """``scale * weight[ids]`` [*ids.shape, dim] in ``out_dtype`` (default: the
    weight's), from a [vocab, dim] matrix in fp32 or bf16.  ``padding_idx``:
    the row that takes no gradient (it is looked up like any other)."""
    refuse_tangents("embed", (weight,))
    _check_ids(ids)
    _check_rows(weight, "weight", ids.device)
    out_dtype = weight.dtype if out_dtype is None else out_dtype
    if out_dtype not in F32:
        raise TypeError(f"out_dtype must be fp32 or bf16, got {out_dtype}")
    padding = _padding(padding_idx, weight.shape[0])
    if torch.is_grad_enabled() and weight.requires_grad:
        return FusedEmbedding.apply(ids, weight, scale, padding, out_dtype)
    return _lookup(ids, weight, scale, out_dtype)


class Embedding(nn.Embedding):
    """``nn.Embedding`` (same parameter, state and initialisation) whose lookup
    is ``embed``: rows times ``scale`` in ``out_dtype`` (default: the weight's)."""

    def __init__(self, num_embeddings, embedding_dim, padding_idx=None, scale=1.0, out_dtype=None, device=None,
                 dtype=None):
        super().__init__(num_embeddings, embedding_dim, padding_idx, device=device, dtype=dtype)
        if out_dtype is not None and out_dtype not in F32:
            raise TypeError(f"out_dtype must be fp32 or bf16, got {out_dtype}")
        self.scale, self.out_dtype = scale, out_dtype

    def forward(self, ids):
        return embed(ids, self.weight, self.scale, self.padding_idx, self.out_dtype)

    def extra_repr(self):
        return f"{super().extra_repr()}, scale={self.scale}"
