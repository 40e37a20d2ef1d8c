"""Calls with a raw stream handle while torch's current stream is another one: what
a call copies or allocates on the way belongs to the stream of its kernels."""

import contextlib
import types

import pytest
import torch

import qgemv_roofline_b200 as qg
from qgemv_roofline_b200 import _tensors, gemv

DEV = "cuda"


@pytest.mark.parametrize("wrap", [_tensors.on_device_of_x, gemv._on_tensor_device])
@pytest.mark.parametrize("handle,positional", [(9, False), (9, True), (0, False), (5, False), (None, False)])
def test_the_raw_stream_is_current_inside_the_call(wrap, handle, positional, monkeypatch):
    """Stand-ins for torch's streams (a stream's id is its handle): no GPU."""
    current, used = [5], []
    stream = lambda h, device=None: types.SimpleNamespace(stream_id=h, device_index=0, device_type=1)
    class Tensor(torch.Tensor):
        is_cuda, device = True, types.SimpleNamespace(index=0)

        def get_device(self):
            return 0

        def record_stream(self, s):
            used.append(s)

    monkeypatch.setattr(torch.cuda, "default_stream", lambda device=None: stream(0))
    monkeypatch.setattr(torch.cuda, "ExternalStream", stream)
    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    monkeypatch.setattr(_tensors, "_current_device", lambda: 0)
    monkeypatch.setattr(_tensors, "_raw_stream", lambda index: current[-1])
    monkeypatch.setattr(_tensors, "_get_stream", lambda index: (current[-1], index, 1))
    monkeypatch.setattr(_tensors, "_set_stream", lambda s: current.append(s[0]))
    monkeypatch.setattr(_tensors, "_stream_object", lambda h, index, kind: h)
    _tensors._stream_of_handle.cache_clear()
    x = torch.zeros(2).as_subclass(Tensor)
    seen = []

    @wrap
    def call(x, y=None, stream=None):
        seen.append(current[-1])
        if y is not None and (y == 7).all():
            raise ValueError
        return torch.zeros(2).as_subclass(Tensor) if y is None else y

    call(x, None, handle) if positional else call(x, stream=handle)
    here = 5 if handle is None else handle
    assert seen == [here] and current[-1] == 5
    assert used == ([5] if handle in (0, 9) else [])  # a new result waits for the caller's stream, too
    y = torch.zeros(2).as_subclass(Tensor)
    assert call(x, y, stream=handle) is y and used == ([5] if handle in (0, 9) else [])
    with pytest.raises(ValueError):
        call(x, y + 7, stream=handle)
    assert seen == [here] * 3 and current[-1] == 5  # whatever the call does
    _tensors._stream_of_handle.cache_clear()


def calls():
    g = torch.Generator(DEV).manual_seed(8)
    K = 256
    w = [torch.randn(6, *s, device=DEV, generator=g) * s[1] ** -0.5 for s in ((128, K), (128, K), (K, 128))]
    experts = qg.QuantizedExperts.from_float(*w, "q8_0")
    router = torch.randn(6, K, device=DEV, generator=g) * 0.2
    wq, ws = qg.quantize_int8(torch.randn(600, K, device=DEV, generator=g))
    m = qg.QuantizedMatrix.from_float(torch.randn(320, K, device=DEV, generator=g), "q4_0")
    ids = torch.randint(0, 6, (12, 2), device=DEV, generator=g).int()
    weights = torch.rand(12, 2, device=DEV, generator=g)
    return {
        "layer": lambda x, **kw: qg.moe_layer(x, router, experts, 2, **kw),
        "experts": lambda x, **kw: qg.moe_experts(x, ids, weights, experts, **kw),
        "route": lambda x, **kw: qg.moe_route(x, router, 2, **kw),
        "quantize": lambda x, **kw: qg.quantize_int8(x, **kw),
        "linear": lambda x, **kw: qg.int8_linear(x, wq, ws, **kw),
        "gemv": m, "tiled": m.to_tiled(), "tc": m.to_tc(),
    }


@pytest.mark.gpu
@pytest.mark.parametrize("op", ["layer", "experts", "route", "quantize", "linear", "gemv", "tiled", "tc"])
def test_a_transposed_x_on_a_raw_stream(op):
    call = calls()[op]
    flat = lambda out: out if isinstance(out, tuple) else (out,)
    x = torch.randn(256, 12, device=DEV, generator=torch.Generator(DEV).manual_seed(9)).t()
    want = flat(call(x.contiguous()))
    raw = torch.cuda.Stream()
    torch.cuda.synchronize()
    # the current stream is busy: a copy made there would come after the kernels
    torch.cuda._sleep(20_000_000)
    got = flat(call(x, stream=raw.cuda_stream))
    raw.synchronize()
    with torch.cuda.stream(raw):
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    torch.cuda.synchronize()
    # the raw stream is busy: what the call let go of must not be given away meanwhile
    with torch.cuda.stream(raw):
        torch.cuda._sleep(20_000_000)
    got = flat(call(x, stream=raw.cuda_stream))
    junk = [torch.full((n,), float("nan"), device=DEV) for n in (256 * 12, 1 << 14, 1 << 16, 1 << 18) for _ in range(8)]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    del junk


@pytest.mark.gpu
def test_the_default_stream_by_its_handle():
    call = calls()["linear"]
    x = torch.randn(256, 12, device=DEV).t()
    want = call(x)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = call(x, stream=torch.cuda.default_stream().cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(got, want)
