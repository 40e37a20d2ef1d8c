"""Several host threads on one stream: each thread's calls are ordered, the launches
of different threads come in any order, and no call reads another's workspace."""

import threading

import pytest
import torch

import qgemv_roofline_b200 as qg

pytestmark = pytest.mark.gpu
DEV = "cuda"


def in_threads(work, n, seconds=120):
    """Runs work(i) in n threads at once; raises what a thread raised."""
    errors, meet = [], threading.Barrier(n)

    def run(i):
        try:
            meet.wait(seconds)
            work(i)
        except BaseException as e:  # handed to the caller
            errors.append(e)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(n)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(seconds)
    if errors:
        raise errors[0]
    assert not any(t.is_alive() for t in threads)


def operators():
    """Calls of x [N, 256] that take a workspace."""
    g = torch.Generator(DEV).manual_seed(5)
    K = 256
    w = [torch.randn(6, *s, device=DEV, generator=g) * s[1] ** -0.5 for s in ((128, K), (128, K), (K, 128))]
    experts = qg.QuantizedExperts.from_float(*w, "q8_0")
    router = torch.randn(6, K, device=DEV, generator=g) * 0.2
    wq, ws = qg.quantize_int8(torch.randn(600, K, device=DEV, generator=g))
    m = qg.QuantizedMatrix.from_float(torch.randn(320, K, device=DEV, generator=g), "q4_0")
    tiles, tc = m.to_tiled(), m.to_tc()
    return [lambda x: qg.moe_layer(x, router, experts, 2), lambda x: qg.int8_linear(x, wq, ws), m, tiles, tc]


@pytest.mark.parametrize("op", range(5))
def test_threads_on_the_default_stream(op):
    call = operators()[op]
    sizes = (4, 13, 7)  # rows: other sizes, so other layouts of the workspace
    g = torch.Generator(DEV).manual_seed(6)
    xs = [torch.randn(n, 256, device=DEV, generator=g) for n in sizes]
    want = [call(x) for x in xs]
    torch.cuda.synchronize()
    got = [[] for _ in xs]

    def work(i):
        for _ in range(300):
            got[i].append(call(xs[i]))

    in_threads(work, len(xs))
    torch.cuda.synchronize()
    for ys, w in zip(got, want):
        assert len(ys) == 300 and all(torch.equal(y, w) for y in ys)


@pytest.mark.parametrize("op", [0, 1])
def test_threads_on_one_raw_stream(op):
    """The library's own workspace of a stream, which grows while another thread's calls use it."""
    g = torch.Generator(DEV).manual_seed(7)
    K = 256
    w = [torch.randn(6, *s, device=DEV, generator=g) * s[1] ** -0.5 for s in ((128, K), (128, K), (K, 128))]
    experts = qg.QuantizedExperts.from_float(*w, "q8_0")
    router = torch.randn(6, K, device=DEV, generator=g) * 0.2
    wq, ws = qg.quantize_int8(torch.randn(K, K, device=DEV, generator=g))
    call = [lambda x, **kw: qg.moe_layer(x, router, experts, 2, **kw), lambda x, **kw: qg.int8_linear(x, wq, ws, **kw)][op]
    sizes = (1, 6, 40, 64)
    xs = [torch.randn(n, K, device=DEV, generator=g) for n in sizes]
    want = [call(x) for x in xs]
    ys = [[torch.zeros_like(x) for _ in range(100)] for x in xs]
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()

    def work(i):
        for y in ys[i]:
            call(xs[i], y=y, stream=stream.cuda_stream)

    in_threads(work, len(xs))
    stream.synchronize()
    for got, w in zip(ys, want):
        assert all(torch.equal(y, w) for y in got)
