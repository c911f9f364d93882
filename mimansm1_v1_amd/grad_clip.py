"""The global norm of gradients and their clipping on the gfx950 kernels of
``csrc/grad_clip.hip`` (``include/mm1_clip.h``): what the reference's training
step does between the backward and the optimizer
(CODE/mimans/training/optim.py:114-179) with torch.

* ``grad_norm(tensors, norm_type)``: one norm over every value of every tensor;
* ``clip_grads(tensors, max_norm, norm_type, out)``: the tensors times
  min(1, max_norm / (norm + 1e-6)), new or in ``out``, and the norm;
* ``clip_grad_norm_(parameters, max_norm, ...)``: the same on the parameters'
  ``.grad`` in place, as torch's function.

Tensors: fp32 and bf16 in any mix, on one device, of any shape whose memory is
one run of values or equally spaced runs (a transposed matrix, some columns of
one).  Norms are fp32 on the device, from fp64 sums in a fixed order; nothing is
copied to the host unless ``error_if_nonfinite`` asks for it.
"""
from __future__ import annotations

import math
import operator
from array import array

import torch

from . import _lib
from .calls import F32, call, refuse_tangents, workspace, written

EPS = 1e-6
NORMS = {2.0: 0, math.inf: 1}        # MM1_NORM_2, MM1_NORM_MAX


def _norm_code(norm_type):
    code = NORMS.get(float(norm_type))
    if code is None:
        raise ValueError(f"norm_type must be 2 or inf, got {norm_type}")
    return code


def _runs(t):
    """(order of the dimensions in memory, rows, cols, distance of the rows) of
    a tensor that is `rows` runs of `cols` consecutive values, or None."""
    order = sorted((i for i in range(t.dim()) if t.shape[i] != 1), key=lambda i: -t.stride(i))
    groups = []                       # [values, stride] from the outermost on
    for i in order:
        if groups and groups[-1][1] == t.shape[i] * t.stride(i):
            groups[-1] = [groups[-1][0] * t.shape[i], t.stride(i)]
        else:
            groups.append([t.shape[i], t.stride(i)])
    if not groups:
        return order, 1, 1, 1
    if groups[-1][1] != 1:
        groups.append([1, 1])         # single values, equally spaced
    if len(groups) > 2:
        return None
    cols = groups[-1][0]
    rows, distance = groups[0] if len(groups) == 2 else (1, cols)
    return None if distance < cols else (order, rows, cols, distance)


_address, _numel, _whole, _device, _same_size = (getattr(torch.Tensor, n) for n in (
    "data_ptr", "numel", "is_contiguous", "get_device", "is_same_size"))
_dtype, _needs_grad = (operator.attrgetter(n) for n in ("dtype", "requires_grad"))


def _described(tensors, name, device):
    """(addresses, dtypes, all contiguous) of a list: a few passes of C calls, for
    a step's hundreds of gradients."""
    try:
        found = list(map(_address, tensors)), list(map(_dtype, tensors)), all(map(_whole, tensors))
        devices = set(map(_device, tensors))
    except TypeError:
        raise TypeError(f"{name} must be torch.Tensors") from None
    except RuntimeError as error:            # no address: not a dense tensor
        raise TypeError(f"{name} must be dense tensors ({error})") from None
    if devices != {device.index} or device.type != "cuda":
        raise ValueError(f"{name} must be CUDA (HIP) tensors on one device")
    return found


class _Table:
    """The host arrays that describe a list of tensors to the library.  out:
    None (read only), the tensors themselves (in place) or others."""

    def __init__(self, tensors, out=None):
        self.count = len(tensors)
        if not isinstance(tensors[0], torch.Tensor):
            raise TypeError("gradients must be torch.Tensors")
        self.device = tensors[0].device
        address, dtypes, whole = _described(tensors, "gradients", self.device)
        numel = list(map(_numel, tensors))
        self.output = self.rows = self.ld = self.ld_out = None
        try:
            self.f32 = bytes(map(F32.__getitem__, dtypes))
        except KeyError as kind:
            raise TypeError(f"gradients must be fp32 or bf16, got {kind}") from None
        if out is not None and out is not tensors:
            if len(out) != self.count:
                raise ValueError(f"out has {len(out)} tensors for {self.count} gradients")
            target, kinds, out_whole = _described(out, "out", self.device)
            if kinds != dtypes or not all(map(_same_size, out, tensors)):
                raise ValueError("out must have the gradients' shapes and dtypes")
            if target == address and all(a.stride() == b.stride() for a, b in zip(tensors, out)):
                out = tensors                # other views of the same memory: in place
            else:
                if not set(address).isdisjoint(target):
                    self._refuse_shared(tensors, out)
                whole = whole and out_whole
                self.output = array("Q", target)
        if out is not None:
            some = address if self.output is None else target
            if len(set(some)) < len(some):       # empty tensors may share an address
                some = [p for p, n in zip(some, numel) if n]
            if len(set(some)) < len(some):
                raise ValueError("a tensor to be written appears twice")
        self.input = array("Q", address)
        if whole:
            self.cols = array("l", numel)
        else:
            self._strided(tensors, out if self.output is not None else None)

    @staticmethod
    def _refuse_shared(tensors, out):
        """An output may be its own gradient and nobody else's: another's would be
        overwritten before or after it is read, as the workgroups happen to run."""
        read = {}                         # the gradients at an address: the same one may be given twice
        for i, t in enumerate(tensors):
            if t.numel():
                read.setdefault(t.data_ptr(), []).append(i)
        for i, o in enumerate(out):
            for j in read.get(o.data_ptr(), ()) if o.numel() else ():
                if j != i or tensors[i].stride() != o.stride():
                    raise ValueError(f"out[{i}] lies in the memory of gradient {j}")

    def _strided(self, tensors, out):
        empty = ([], 0, 0, 0)
        runs = [_runs(t) if t.numel() else empty for t in tensors]
        to = runs if out is None else [_runs(t) if t.numel() else empty for t in out]
        for t, a, b in zip(tensors, runs, to):
            if a is None or b is None:
                raise ValueError(f"a tensor of shape {tuple(t.shape)} and strides {t.stride()} is not equally spaced "
                                 "runs of values")
            if a[0] != b[0]:
                raise ValueError("out must lie in memory in the order of its gradient")
        # a run that one side holds whole and the other in rows is rows on both
        for i, (a, b) in enumerate(zip(runs, to)):
            if a[1:3] != b[1:3]:
                rows, cols = max(a[1], b[1]), min(a[2], b[2])
                split = lambda r: (r[0], rows, cols, r[3] if r[1] == rows else cols)
                if a[1] * a[2] != rows * cols or min(a[1], b[1]) != 1:
                    raise ValueError("out must lie in memory in the runs of its gradient")
                runs[i], to[i] = split(a), split(b)
        self.rows = array("l", [r[1] for r in runs])
        self.cols = array("l", [r[2] for r in runs])
        self.ld = array("l", [r[3] for r in runs])
        self.ld_out = array("l", [r[3] for r in to])

    def run(self, norm, norm_code, max_norm=None, known=False):
        at = lambda a: None if a is None else a.buffer_info()[0]
        keep, ws, ws_bytes = workspace(_lib.load().mm1_grad_norm_workspace_size(self.count), self.device)
        shape = (at(self.rows), at(self.cols), at(self.ld))
        if max_norm is None:
            call("mm1_grad_norm", self.device, self.count, at(self.input), *shape, self.f32, norm_code,
                 norm.data_ptr(), ws, ws_bytes)
        else:
            call("mm1_grad_clip", self.device, self.count, at(self.input), at(self.output), *shape, at(self.ld_out),
                 self.f32, norm_code, max_norm, EPS, int(known), norm.data_ptr(), ws, ws_bytes)


def _list(tensors):
    return [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)


def _any_needs_grad(tensors):
    try:
        return any(map(_needs_grad, tensors))
    except AttributeError:
        raise TypeError("gradients must be torch.Tensors") from None


def _unrecorded(tensors):
    refuse_tangents("the norm", tensors)
    if torch.is_grad_enabled() and _any_needs_grad(tensors):
        raise RuntimeError("the norm and the clipped gradients leave no autograd graph: call under torch.no_grad()")


def _max_norm(max_norm):
    max_norm = float(max_norm)
    if not max_norm >= 0:
        raise ValueError(f"max_norm must be at least 0, got {max_norm}")
    return max_norm


def grad_norm(tensors, norm_type=2.0):
    """The norm of all values of `tensors` together (norm_type 2, or inf for
    the largest magnitude): a 0-dim fp32 tensor on their device."""
    tensors, code = _list(tensors), _norm_code(norm_type)
    if not tensors:
        return torch.tensor(0.0)
    _unrecorded(tensors)
    table = _Table(tensors)
    norm = torch.empty((), dtype=torch.float32, device=table.device)
    table.run(norm, code)
    return norm


def clip_grads(tensors, max_norm, norm_type=2.0, out=None):
    """(clipped, norm): each tensor times min(1, max_norm / (norm + 1e-6)),
    rounded once to its dtype, and the norm before clipping.  The results are
    new tensors, or those of ``out``: of the same shapes and dtypes, each in memory
    of its own or its gradient's (in place; ``out`` may be `tensors`)."""
    out = out if out is None or out is tensors else _list(out)
    same = out is tensors
    tensors, code, max_norm = _list(tensors), _norm_code(norm_type), _max_norm(max_norm)
    if not tensors:
        return [], torch.tensor(0.0)
    _unrecorded(tensors)
    to = tensors if same else out if out is not None else [torch.empty_like(t) for t in tensors]
    refuse_tangents("the norm", to)
    if out is not None and _any_needs_grad(to):
        raise ValueError("out must not require a gradient: it is written in place")
    table = _Table(tensors, to)
    norm = torch.empty((), dtype=torch.float32, device=table.device)
    table.run(norm, code, max_norm)
    if out is not None:
        written(*to)
    return to, norm


@torch.no_grad()
def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False):
    """torch.nn.utils.clip_grad_norm_ (without ``foreach``) on these kernels: scales
    the gradients of `parameters` in place so that their norm is at most max_norm,
    and returns the norm before.  No two of them share memory.  ``error_if_nonfinite`` waits for the norm on the host and
    raises before anything is scaled."""
    grads = [p.grad for p in _list(parameters) if p.grad is not None]
    code, max_norm = _norm_code(norm_type), _max_norm(max_norm)
    refuse_tangents("the norm", grads)
    if not grads:
        return torch.tensor(0.0)
    table = _Table(grads, grads)
    norm = torch.empty((), dtype=torch.float32, device=table.device)
    if error_if_nonfinite:
        table.run(norm, code)
        if not math.isfinite(norm.item()):
            raise RuntimeError(f"the norm of order {norm_type} of the gradients is not finite")
    table.run(norm, code, max_norm, known=error_if_nonfinite)
    written(*grads)
    return norm
