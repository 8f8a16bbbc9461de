"""Helpers shared by the torch custom-op wrappers."""
from __future__ import annotations

import ctypes
import contextlib

import torch
from torch.autograd import forward_ad

from .. import _lib


def ptr(t: torch.Tensor) -> ctypes.c_void_p:
    return ctypes.c_void_p(t.data_ptr())


def stream_of(t: torch.Tensor) -> ctypes.c_void_p:
    return ctypes.c_void_p(torch.cuda.current_stream(t.device).cuda_stream)


_ENTRIES: dict = {}
_get_device = getattr(torch._C, "_cuda_getDevice", None)
_get_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def launch(t: torch.Tensor, name: str, *args) -> None:
    """Call the vs_* function `name` with `args` and, as the last argument, the current stream of
    t's GPU, with that GPU as the current device.  Bound functions are kept and the device is only
    switched where it has to be: in a decoding loop the host's time per call counts."""
    fn = _ENTRIES.get(name)
    if fn is None:
        require_gpu_tensor(t, name)
        fn = _ENTRIES[name] = getattr(_lib.lib(), name)
    dev = t.get_device()
    if _get_device() != dev:
        with torch.cuda.device(dev):
            return _lib.call(name, *args, _get_stream(dev))
    if _lib._RANGES:
        return _lib.call(name, *args, _get_stream(dev))
    status = fn(*args, _get_stream(dev))
    if status:
        _lib.check(status, name)


_PLAIN = (torch.Tensor, torch.nn.Parameter)
_is_compiling = torch.compiler.is_compiling
_dispatch_modes = torch._C._len_torch_dispatch_stack
_tracer = torch._C._get_tracing_state
_functorch_level = torch._C._functorch.peek_interpreter_stack


def plain_tensors(*tensors) -> bool:
    """True when a call needs none of the dispatcher's services: ordinary tensors with data, nothing tracing.
    The implementation (or its autograd Function) is then called directly, which takes several
    microseconds of host time off a call, and about a hundred off a training pass."""
    if _is_compiling():
        return False
    plain = not _dispatch_modes() and _tracer() is None and _functorch_level() is None and not tensors[0].is_meta
    for t in tensors:
        if t is not None and type(t) not in _PLAIN:
            plain = False
    if forward_ad._current_level >= 0:
        _refuse_tangents(plain, tensors)
    return plain


def _refuse_tangents(plain, tensors) -> None:
    """Raise for tensors with a forward-mode tangent that a kernel or the dispatcher would drop (only the CPU
    definitions, called directly, carry it)."""
    for t in tensors:
        if t is not None and (t.is_cuda or not plain) and forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError("this operator has no forward-mode derivative")


def records(*tensors) -> bool:
    """True when autograd records a call on these tensors."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


@contextlib.contextmanager
def on_device(t: torch.Tensor):
    """Make t's GPU the current HIP device for the native launch."""
    if t.is_cuda:
        with torch.cuda.device(t.device):
            yield
    else:
        yield


def require_gpu_tensor(t: torch.Tensor, name: str) -> None:
    """GPU tensors must run the native kernels; fail loudly if unavailable."""
    if not _lib.available():
        raise _lib.NativeLibraryMissing(
            f"{name}: native library not built; refusing a silent fallback")
    if not _lib.gpu_available():
        raise _lib.VelesError(f"{name}: native library sees no GPU")


def contiguous_f32(t: torch.Tensor, name: str) -> torch.Tensor:
    if t.dtype != torch.float32:
        raise TypeError(f"{name}: expected float32, got {t.dtype}")
    return t.contiguous()
