"""Mixture-of-experts layers over q8_0 / q4_0 experts, for a few tokens.

``moe_layer`` is a whole layer (router, SwiGLU experts, weighted sum);
``moe_route`` its router alone, ``moe_experts`` its experts with the choice
made by the caller.  ``QuantizedExperts`` holds the experts' weights in the
layout the kernels stream (expert tiles, made once).  ``x`` is ``[K]`` or
``[N, K]`` in fp32, bf16 or fp16; ``y`` has its type and shape.  As in
``gemv``, tensors must already be on the GPU, work is enqueued on the current
CUDA stream (or ``stream``), and there is no CPU path.

The reference has no such operator: its kernels stop at one matrix
(src/qgemv_kernels.cuh).
"""

from __future__ import annotations

import ctypes
import functools

import torch

from . import _lib
from ._tensors import DTYPE_CODE, new, on_device_of_x, out_for, rows_of, stream_of, workspace
from .gemv import QuantizedMatrix
from .qformats import BLOCK_BYTES, QK

SCORING = {"softmax": 0, "sigmoid": 1}
MAX_EXPERTS, MAX_CHOICES = 1024, 32


def _router(router, top_k, scoring, bias, scale, normalize, device) -> _lib.MoeRouter:
    shape, code = router.shape, DTYPE_CODE.get(router.dtype)
    if len(shape) != 2 or code is None or router.get_device() != device.index:
        raise ValueError(f"router must be a float32, bfloat16 or float16 tensor [E, K] on {device}")
    ldw, last = router.stride()
    E = shape[0]
    if (last != 1 and shape[1] > 1) or (E > 1 and ldw < shape[1]):
        raise ValueError("router must have unit last stride and rows that do not overlap")
    if scoring not in SCORING:
        raise ValueError(f"scoring must be 'softmax' or 'sigmoid', got {scoring!r}")
    if not 1 <= top_k <= min(E, MAX_CHOICES):
        raise ValueError(f"top_k must be in [1, min(E={E}, {MAX_CHOICES})], got {top_k}")
    if bias is not None and (bias.dtype != torch.float32 or tuple(bias.shape) != (E,)
                             or bias.device != device or not bias.is_contiguous()):
        raise ValueError(f"bias must be a contiguous float32 tensor [{E}] on {device}")
    return _lib.MoeRouter(router.data_ptr(), code, E, ldw,
                          None if bias is None else bias.data_ptr(), top_k, SCORING[scoring],
                          bool(normalize), scale)


@on_device_of_x
def moe_route(x: torch.Tensor, router: torch.Tensor, top_k: int, *, scoring: str = "softmax",
              bias: torch.Tensor | None = None, scale: float = 1.0, normalize: bool = True,
              stream: int | None = None):
    """The ``top_k`` best experts of each token and their weights.

    ``logits = x router^T`` (``router`` [E, K]; 64-bit sums rounded to fp32 once), scores =
    softmax or sigmoid of the logits.  The experts are those of largest score, plus
    ``bias`` [E] where given (which steers the choice, not the weights); ties go to the
    lower index.  Their scores, divided by their sum if ``normalize``, times ``scale`` are
    the weights.  Returns ``(ids int32, weights float32)``, each [N, top_k] ([top_k] for a
    vector x), in descending order of score.
    """
    X, N, ldx, code = rows_of(x, router.shape[-1])
    device = x.device
    r = _router(router, top_k, scoring, bias, scale, normalize, device)
    shape = (N, top_k) if x.dim() == 2 else (top_k,)
    ids, weights = new(shape, torch.int32, device), new(shape, torch.float32, device)
    _lib.call("qgemv_moe_route", ctypes.byref(r), X.data_ptr(), code, ldx, N, X.shape[-1],
              ids.data_ptr(), weights.data_ptr(), stream_of(stream, device))
    return ids, weights


class QuantizedExperts:
    """E SwiGLU experts (gate, up [F, K]; down [K, F]) resident on one GPU as
    expert tiles.

    ``gate``, ``up`` and ``down`` are SoA planes ``(q, d)`` with a leading expert
    dimension: q int8 [E, rows, cols] (q8_0) or uint8 [E, rows, cols / 2] (q4_0),
    d float16 [E, rows, cols / 32].  gate and up share a format; down may have the
    other one.  The last ``n_shared`` experts take every token of ``moe_layer``
    with weight 1.  The planes are only read here; they may be freed afterwards.
    """

    def __init__(self, gate, up, down, n_shared: int = 0):
        fmt, E, F, K = self._planes("gate", gate)
        if self._planes("up", up) != (fmt, E, F, K):
            raise ValueError("gate and up must have the same format and shape")
        fmt_down, Ed, Kd, Fd = self._planes("down", down)
        if (Ed, Kd, Fd) != (E, K, F):
            raise ValueError(f"down must be [E={E}, K={K}, F={F}], got {(Ed, Kd, Fd)}")
        if not 1 <= E <= MAX_EXPERTS or not 0 <= n_shared <= min(E, MAX_CHOICES):
            raise ValueError(f"{E} experts, {n_shared} of them shared: at most {MAX_EXPERTS} and "
                             f"{MAX_CHOICES}")
        dev = gate[0].device
        if any(t.device != dev for t in (*gate, *up, *down)):
            raise ValueError("gate, up and down must be on one device")
        self.fmt, self.fmt_down = fmt, fmt_down
        self.n_experts, self.n_shared, self.hidden, self.ffn = E, n_shared, K, F
        with torch.cuda.device(dev):
            self.gate_up = self._tile(fmt, gate, up, E, F, K)
            self.down = self._tile(fmt_down, down, None, E, K, F)
        self.device = dev
        self._set = _lib.ExpertSet(_lib.FORMAT_CODE[fmt], _lib.FORMAT_CODE[fmt_down], E, n_shared,
                                   K, F, self.gate_up.data_ptr(), self.down.data_ptr())
        self._ref = ctypes.byref(self._set)

    @staticmethod
    def _planes(name, planes):
        q, d = planes
        fmt = {torch.int8: "q8_0", torch.uint8: "q4_0"}.get(q.dtype)
        if fmt is None or not q.is_cuda or q.dim() != 3 or not q.is_contiguous():
            raise ValueError(f"{name}: q must be a contiguous int8 (q8_0) or uint8 (q4_0) CUDA tensor "
                             "[E, rows, cols or cols / 2]")
        E, rows, cols = q.shape[0], q.shape[1], q.shape[2] * (1 if fmt == "q8_0" else 2)
        if not rows or not cols or rows % QK or cols % QK:
            raise ValueError(f"{name}: rows and columns must be positive multiples of {QK}, got "
                             f"{rows} x {cols}")
        if d.dtype != torch.float16 or tuple(d.shape) != (E, rows, cols // QK) or not d.is_contiguous():
            raise ValueError(f"{name}: d must be contiguous float16 [{E}, {rows}, {cols // QK}]")
        return fmt, E, rows, cols

    @staticmethod
    def _tile(fmt, planes, second, E, rows, cols):
        code = _lib.FORMAT_CODE[fmt]
        nbytes = _lib.lib().qgemv_moe_tiles_bytes(code, E, rows * (1 if second is None else 2), cols)
        out = torch.empty(nbytes, dtype=torch.uint8, device=planes[0].device)
        q2, d2 = (None, None) if second is None else (second[0].data_ptr(), second[1].data_ptr())
        _lib.call("qgemv_moe_tile", code, planes[0].data_ptr(), planes[1].data_ptr(), q2, d2, E, rows,
                  cols, out.data_ptr(), torch.cuda.current_stream(out.device).cuda_stream)
        return out

    @classmethod
    def from_float(cls, gate: torch.Tensor, up: torch.Tensor, down: torch.Tensor, fmt: str,
                   fmt_down: str | None = None, n_shared: int = 0) -> "QuantizedExperts":
        """Quantizes float32 weights gate, up [E, F, K] and down [E, K, F]."""
        from . import qformats

        def planes(w, f):
            quantize = qformats.quantize_q8_0 if f == "q8_0" else qformats.quantize_q4_0
            q, d = quantize(w.reshape(-1, w.shape[-1]))
            return q.view(*w.shape[:2], -1), d.view(*w.shape[:2], -1)
        return cls(planes(gate, fmt), planes(up, fmt), planes(down, fmt_down or fmt), n_shared)

    @classmethod
    def from_matrices(cls, gate: QuantizedMatrix, up: QuantizedMatrix, down: QuantizedMatrix,
                      n_experts: int, n_shared: int = 0) -> "QuantizedExperts":
        """From SoA matrices with the experts' rows one after the other: gate, up
        [E * F, K], down [E * K, F] (what ``GGUFReader.load`` gives for expert tensors)."""
        def planes(m):
            if m.layout != "soa":
                raise ValueError("gate, up and down must be SoA matrices")
            if n_experts < 1 or m.M % n_experts:
                raise ValueError(f"{m.M} rows do not divide over {n_experts} experts")
            return (m.q.view(n_experts, m.M // n_experts, -1), m.d.view(n_experts, m.M // n_experts, -1))
        return cls(planes(gate), planes(up), planes(down), n_shared)

    @property
    def nbytes(self) -> int:
        """Bytes of the quantized weights (the tiles pad columns to 128)."""
        n = self.n_experts * self.hidden * self.ffn // QK
        return n * (2 * BLOCK_BYTES[self.fmt] + BLOCK_BYTES[self.fmt_down])


def _experts_on(experts, x):
    device = x.device
    if experts.device != device:
        raise ValueError(f"the experts are on {experts.device}, x on {device}")
    return device


@functools.lru_cache(maxsize=256)
def _ws_bytes(N, slots, hidden, ffn):
    return _lib.lib().qgemv_moe_workspace_bytes(N, slots, hidden, ffn)


@on_device_of_x
def moe_experts(x: torch.Tensor, ids: torch.Tensor, weights: torch.Tensor,
                experts: QuantizedExperts, y: torch.Tensor | None = None,
                stream: int | None = None) -> torch.Tensor:
    """``y[n] = sum_j weights[n, j] * down_e (silu(gate_e x_n) * (up_e x_n))``, e = ids[n, j].

    ids int32 and weights float32 are [N, slots] ([slots] for a vector x).  An id outside
    [0, E), -1 for instance, selects no expert; one that a token names twice counts with
    the sum of its weights; a token without experts gets zeros.
    """
    device = _experts_on(experts, x)
    X, N, ldx, code = rows_of(x, experts.hidden)
    vec = x.dim() == 1
    slots = ids.shape[-1] if ids.dim() else 0
    want = (slots,) if vec else (N, slots)
    if (ids.shape != want or weights.shape != want or ids.dtype != torch.int32
            or weights.dtype != torch.float32 or ids.get_device() != device.index
            or weights.get_device() != device.index
            or not ids.is_contiguous() or not weights.is_contiguous()):
        raise ValueError(f"ids (int32) and weights (float32) must be contiguous [N={N}, slots] on {device}")
    if not 1 <= slots <= MAX_CHOICES:
        raise ValueError(f"1 to {MAX_CHOICES} choices per token, got {slots}")
    y, ldy = out_for(y, (N, experts.hidden), x.dtype, device, vec)
    if N == 0:
        return y
    _, ptr, nbytes = workspace(device, _ws_bytes(min(N, 64), slots, experts.hidden, experts.ffn), stream)
    _lib.call("qgemv_moe_experts", experts._ref, X.data_ptr(), code, ldx, ids.data_ptr(),
              weights.data_ptr(), slots, N, y.data_ptr(), ldy, ptr, nbytes, stream_of(stream, device))
    return y


@on_device_of_x
def moe_layer(x: torch.Tensor, router: torch.Tensor, experts: QuantizedExperts, top_k: int, *,
              scoring: str = "softmax", bias: torch.Tensor | None = None, scale: float = 1.0,
              normalize: bool = True, y: torch.Tensor | None = None,
              stream: int | None = None) -> torch.Tensor:
    """A whole mixture-of-experts layer: ``moe_route`` over the experts that are not
    shared, then ``moe_experts`` with these and the shared ones (weight 1)."""
    device = _experts_on(experts, x)
    X, N, ldx, code = rows_of(x, experts.hidden)
    if router.shape != (experts.n_experts - experts.n_shared, experts.hidden):
        raise ValueError(f"router must be [{experts.n_experts - experts.n_shared}, {experts.hidden}], "
                         f"got {tuple(router.shape)}")
    r = _router(router, top_k, scoring, bias, scale, normalize, device)
    slots = top_k + experts.n_shared
    if slots > MAX_CHOICES:
        raise ValueError(f"{slots} choices per token (shared experts included), at most {MAX_CHOICES}")
    y, ldy = out_for(y, (N, experts.hidden), x.dtype, device, x.dim() == 1)
    if N == 0:
        return y
    _, ptr, nbytes = workspace(device, _ws_bytes(min(N, 64), slots, experts.hidden, experts.ffn), stream)
    _lib.call("qgemv_moe_layer", experts._ref, ctypes.byref(r), X.data_ptr(), code, ldx, N,
              y.data_ptr(), ldy, ptr, nbytes, stream_of(stream, device))
    return y
