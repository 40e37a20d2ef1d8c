"""int8 matrix products with one scale per token and one per channel.

``y[n, m] = (sum_k xq[n, k] wq[m, k]) xs[n] ws[m] (+ bias[m])`` for any number of
tokens n, the sum exact: what serves a prompt or a large batch, beside the
GEMVs' few columns.  ``quantize_int8`` makes rows and scales (weights once,
activations per call), ``int8_matmul`` multiplies, ``int8_linear`` does both
for activations in fp32, bf16 or fp16.  As in ``gemv``, tensors must already be
on the GPU, work is enqueued on the current CUDA stream (or ``stream``), and
there is no CPU path.

The reference has no such operator: its weights are ggml blocks and its
products one vector wide (src/qgemv_kernels.cuh).
"""

from __future__ import annotations

import functools

import torch

from . import _lib
from ._tensors import DTYPE_CODE, new, on_device_of_x, out_for, rows_of, stream_of, workspace


@on_device_of_x
def quantize_int8(x: torch.Tensor, q: torch.Tensor | None = None, scales: torch.Tensor | None = None,
                  stream: int | None = None):
    """Rounds each row of x ([K] or [N, K]; fp32, bf16 or fp16) to int8 with its own scale.

    ``scales = max |x| / 127``, ``q = rint(x / scales)``, in fp32.  A zero row gets scale 0 and
    zeros, a row with a NaN or an infinity scale NaN and zeros.  Returns ``(q int8 like x,
    scales float32 [N])`` (a scalar tensor for a vector).
    """
    K = x.shape[-1] if x.dim() else 0
    if K < 1:
        raise ValueError("x must have at least one column")
    X, N, ldx, code = rows_of(x, K)
    vec = x.dim() == 1
    if q is None:
        q = new(x.shape, torch.int8, x.device)
    elif q.dtype != torch.int8 or q.shape != x.shape or q.device != x.device or \
            (q.stride(-1) != 1 and K > 1) or (not vec and N > 1 and q.stride(0) < K):
        raise ValueError("q must be an int8 tensor like x with unit last stride")
    want = x.shape[:-1]
    if scales is None:
        scales = torch.empty(want, dtype=torch.float32, device=x.device)
    elif scales.dtype != torch.float32 or scales.shape != want or scales.device != x.device or \
            not scales.is_contiguous():
        raise ValueError(f"scales must be a contiguous float32 tensor {tuple(want)}")
    _lib.call("qgemv_int8_quantize", X.data_ptr(), code, ldx, N, K, q.data_ptr(),
              K if vec else q.stride(0), scales.data_ptr(), stream_of(stream, x.device))
    return q, scales


def _weights(wq, ws, bias, K, device):
    shape = wq.shape
    if wq.dtype != torch.int8 or len(shape) != 2 or shape[1] != K or wq.get_device() != device.index or \
            wq.stride(1) != 1:
        raise ValueError(f"wq must be an int8 tensor [M, K={K}] with unit last stride on {device}")
    M = shape[0]
    if ws.dtype != torch.float32 or ws.shape != (M,) or ws.get_device() != device.index or not ws.is_contiguous():
        raise ValueError(f"ws must be a contiguous float32 tensor [{M}] on {device}")
    if bias is None:
        return M, None
    if bias.dtype != torch.float32 or bias.shape != (M,) or bias.device != device or \
            not bias.is_contiguous():
        raise ValueError(f"bias must be a contiguous float32 tensor [{M}] on {device}")
    return M, bias.data_ptr()


def _y_code(dtype):
    code = DTYPE_CODE.get(dtype)
    if code is None:
        raise TypeError(f"out_dtype must be float32, bfloat16 or float16, got {dtype}")
    return code


@on_device_of_x
def int8_matmul(xq: torch.Tensor, xs: torch.Tensor, wq: torch.Tensor, ws: torch.Tensor,
                bias: torch.Tensor | None = None, out_dtype: torch.dtype = torch.float32,
                y: torch.Tensor | None = None, stream: int | None = None) -> torch.Tensor:
    """y = (xq wq^T) * xs[:, None] * ws (+ bias), the int8 product summed exactly.

    xq int8 [N, K] with xs float32 [N] (or [K] with a scalar tensor), wq int8 [M, K] with ws
    float32 [M], bias float32 [M].  K is a multiple of 16 below 2^17; rows start on 16-byte
    boundaries (any such row stride).
    """
    shape = xq.shape
    if xq.dtype != torch.int8 or len(shape) not in (1, 2) or (xq.stride(-1) != 1 and shape[-1] > 1):
        raise ValueError("xq must be an int8 tensor [K] or [N, K] with unit last stride")
    vec = len(shape) == 1
    N, K = (1, shape[0]) if vec else shape
    device = xq.device
    if xs.dtype != torch.float32 or xs.shape != shape[:-1] or xs.get_device() != device.index or \
            not xs.is_contiguous():
        raise ValueError(f"xs must be a contiguous float32 tensor {tuple(shape[:-1])} on {device}")
    M, b = _weights(wq, ws, bias, K, device)
    code = _y_code(out_dtype)
    y, ldy = out_for(y, (N, M), out_dtype, device, vec)
    _lib.call("qgemv_int8_matmul", xq.data_ptr(), xs.data_ptr(), K if vec else xq.stride(0),
              wq.data_ptr(), ws.data_ptr(), wq.stride(0), b, N, M, K, y.data_ptr(), code, ldy,
              stream_of(stream, device))
    return y


@functools.lru_cache(maxsize=256)
def _ws_bytes(N, K):
    return _lib.lib().qgemv_int8_linear_workspace_bytes(N, K)


@on_device_of_x
def int8_linear(x: torch.Tensor, wq: torch.Tensor, ws: torch.Tensor, bias: torch.Tensor | None = None,
                out_dtype: torch.dtype | None = None, y: torch.Tensor | None = None,
                stream: int | None = None) -> torch.Tensor:
    """``int8_matmul(*quantize_int8(x), wq, ws, bias)`` in one call; y has x's type unless
    ``out_dtype`` says otherwise."""
    X, N, ldx, code = rows_of(x, x.shape[-1] if x.dim() else 0)
    K, device = x.shape[-1], x.device
    M, b = _weights(wq, ws, bias, K, device)
    dtype = out_dtype or x.dtype
    ycode = _y_code(dtype)
    y, ldy = out_for(y, (N, M), dtype, device, x.dim() == 1)
    _, ptr, nbytes = workspace(device, _ws_bytes(N, K), stream)
    _lib.call("qgemv_int8_linear", X.data_ptr(), code, ldx, wq.data_ptr(), ws.data_ptr(), wq.stride(0), b,
              N, M, K, y.data_ptr(), ycode, ldy, ptr, nbytes, stream_of(stream, device))
    return y
