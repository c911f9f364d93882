"""Calls of the C ABI on the device that the tensors are on."""
from __future__ import annotations

import torch
from torch.autograd import forward_ad

from . import _lib

F32 = {torch.float32: 1, torch.bfloat16: 0}     # the types the operators hold values in, as the *_f32 arguments


_entries: dict = {}


def call(name: str, device, *args) -> None:
    """The entry point `name` with `args` and the current stream of `device`,
    launched with that device current; raises what a nonzero code names."""
    fn = _entries.get(name)
    if fn is None:
        fn = _entries[name] = getattr(_lib.load(), name)
    index = device.index
    stream = torch._C._cuda_getCurrentRawStream(index)
    if torch._C._cuda_getDevice() == index:
        rc = fn(*args, stream)
    else:
        with torch.cuda.device(index):
            rc = fn(*args, stream)
    if rc:
        _lib.check(rc, name)


def refuse_tangents(name: str, tensors) -> None:
    """Raises where a tensor (None is none) carries a forward-mode tangent, as an
    autograd.Function without a jvp does: a call that goes to the kernels past
    autograd would drop it."""
    if forward_ad._current_level >= 0 and any(
            isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError(f"{name} has no forward-mode derivative")


def workspace(nbytes: int, device):
    """(tensor that keeps the memory, address, bytes); no memory for 0 bytes."""
    if nbytes == 0:
        return None, None, 0
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
    return ws, ws.data_ptr(), nbytes


def written(*tensors) -> None:
    """Tells autograd that kernels have changed these tensors in place."""
    try:
        torch.autograd.graph.increment_version(tensors)
    except RuntimeError:             # tensors of inference mode keep no version
        torch.autograd.graph.increment_version([t for t in tensors if not t.is_inference()])
