"""What the multi-type operators (moe, int8) share on the host: argument checks
and the stream and workspace of a call.  These run on every call of a decode
step, beside kernels of a few microseconds, so they keep to a few attribute
reads and no temporary objects."""

from __future__ import annotations

import functools
import inspect
import threading

import torch

DTYPE_CODE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_raw_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else \
    (lambda index: torch.cuda.current_stream(index).cuda_stream)


_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def stream_argument(fn):
    """A function that finds the ``stream`` argument of a call of ``fn``."""
    params = list(inspect.signature(fn).parameters.values())
    at = next(i for i, p in enumerate(params) if p.name == "stream")
    at = at if params[at].kind is not inspect.Parameter.KEYWORD_ONLY else len(params)

    def find(args, kwargs):
        return args[at] if len(args) > at else kwargs.get("stream")
    return find


def _get_stream(index: int):
    """torch's current stream of a device: (id, device index, device type)."""
    return torch._C._cuda_getCurrentStream(index)


def _set_stream(stream):
    torch._C._cuda_setStream(stream_id=stream[0], device_index=stream[1], device_type=stream[2])


@functools.lru_cache(maxsize=256)
def _stream_of_handle(handle: int, index: int):
    # 0 and 1 are the handles of the legacy default stream
    s = torch.cuda.default_stream(index) if handle in (0, 1) else torch.cuda.ExternalStream(handle, device=index)
    return s.stream_id, s.device_index, s.device_type


@functools.lru_cache(maxsize=256)
def _stream_object(stream_id, device_index, device_type):
    return torch.cuda.Stream(stream_id=stream_id, device_index=device_index, device_type=device_type)


def run_on(stream: int, index: int, fn, args, kwargs):
    """``fn(*args, **kwargs)``, whose kernels go to the raw stream ``stream`` of
    device ``index``, with that stream current: what it copies and allocates on
    the way (an x with other strides, a workspace, y) is then ordered with the
    kernels and goes back to the stream's own memory.  What it allocated and
    returns may be used on the caller's stream, so its memory waits for that one
    too.  (torch.cuda.stream does the same switch, in 10 us more.)"""
    if index != _current_device():
        with torch.cuda.device(index):
            return run_on(stream, index, fn, args, kwargs)
    if stream == _raw_stream(index):
        return fn(*args, **kwargs)
    caller = _get_stream(index)
    _set_stream(_stream_of_handle(stream, index))
    try:
        out = fn(*args, **kwargs)
    finally:
        _set_stream(caller)
    for t in out if isinstance(out, tuple) else (out,):
        if not any(t is a for a in (*args, *kwargs.values())):
            t.record_stream(_stream_object(*caller))
    return out


def on_device_of_x(fn):
    """Runs ``fn(x, ...)`` with the device of its first argument current, which
    may be given by its name, too, and the raw ``stream`` where one is given."""
    name = next(iter(inspect.signature(fn).parameters))
    stream_of_call = stream_argument(fn)

    @functools.wraps(fn)
    def wrapper(*args, **kwargs):
        if not args and name not in kwargs:
            return fn(**kwargs)  # Python's own error
        x = args[0] if args else kwargs[name]
        index = x.get_device() if isinstance(x, torch.Tensor) else -1
        if index < 0:
            raise ValueError(f"{name} must be a CUDA tensor")
        stream = stream_of_call(args, kwargs)
        if stream is not None:
            return run_on(stream, index, fn, args, kwargs)
        if index == _current_device():
            return fn(*args, **kwargs)
        with torch.cuda.device(index):
            return fn(*args, **kwargs)
    return wrapper


def new(shape, dtype, device) -> torch.Tensor:
    """An uninitialised contiguous tensor [M] or [N, M] (two thirds of torch.empty's time)."""
    return torch.empty_strided(shape, (shape[1], 1) if len(shape) == 2 else (1,), dtype=dtype, device=device)


def rows_of(x: torch.Tensor, K: int):
    """x ([K] or [N, K]) as rows that the kernels can read (unit last stride,
    no overlap): (tensor, N, row stride, dtype code)."""
    code = DTYPE_CODE.get(x.dtype)
    if code is None:
        raise TypeError(f"x must be float32, bfloat16 or float16, got {x.dtype}")
    shape = x.shape
    if len(shape) > 2 or len(shape) == 0 or shape[-1] != K:
        raise ValueError(f"x must be [K={K}] or [N, K={K}], got {tuple(shape)}")
    if len(shape) == 1:
        return (x if x.stride(0) == 1 or K == 1 else x.contiguous()), 1, K, code
    N = shape[0]
    s0, s1 = x.stride()
    if (s1 != 1 and K > 1) or (s0 < K and N > 1):
        x, s0 = x.contiguous(), K
    return x, N, s0, code


def out_for(y, shape, dtype, device, vec: bool):
    """The output rows [N, M] of a call: (tensor to return, row stride)."""
    if y is None:
        return new(shape[1:] if vec else shape, dtype, device), shape[1]
    want = tuple(shape[1:] if vec else shape)
    if y.dtype != dtype or y.device != device or tuple(y.shape) != want:
        raise ValueError(f"y must be a {dtype} tensor {want} on {device}")
    if (y.stride(-1) != 1 and shape[1] > 1) or (not vec and shape[0] > 1 and y.stride(0) < shape[1]):
        raise ValueError("y must have unit last stride and rows that do not overlap")
    return y, (shape[1] if vec else y.stride(0))


def stream_of(stream, device) -> int:
    return _raw_stream(device.index) if stream is None else stream


class Workspaces(threading.local):
    """Buffers by (device, stream), grown on demand, of one host thread.  Calls
    of a thread on a stream are ordered and share a buffer; a call is several
    launches that pass data through it, and another thread's launches on the
    same stream may come between them (the C call runs without the GIL)."""

    def __init__(self):
        self.buffers: dict = {}


_WS = Workspaces()


def workspace(device, nbytes: int, stream):
    """(tensor, pointer, bytes) of a call's workspace.  Under capture a buffer
    of its own, from the graph's memory; for a raw stream handle none: the
    library's own of that stream, which it refuses under capture."""
    if stream is not None:
        return None, None, 0
    if torch.cuda.is_current_stream_capturing():
        ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
        return ws, ws.data_ptr(), nbytes
    key = (device.index, _raw_stream(device.index))
    buffers = _WS.buffers
    ws = buffers.get(key)
    if ws is None or ws[2] < nbytes:
        t = torch.empty(nbytes, dtype=torch.uint8, device=device)
        ws = buffers[key] = (t, t.data_ptr(), nbytes)
    return ws
