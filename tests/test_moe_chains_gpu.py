"""Expert calls one after the other on one stream, nothing waiting between them."""

import numpy as np
import pytest
import torch

import qgemv_roofline_b200 as qg
from test_moe_gpu import DEV, Layer, gpu

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("given", [False, True])
@pytest.mark.parametrize("N,k", [(1, 2), (1, 1), (3, 1)])
def test_choices_that_change_with_every_call(N, k, given):
    """Few units: gate and up run on a few SMs, and down's CTAs find the others free while
    the choices at the same addresses are still an earlier call's."""
    E, K, F, calls = 24, 512, 32, 64
    L = Layer(E, K, F, "q8_0", seed=40 + N + k)
    router = gpu((L.rng.standard_normal((E, K))).astype(np.float32))
    xs = [L.x(N)[0] for _ in range(calls)]
    routed = [qg.moe_route(x, router, k) for x in xs]
    ids, w = (torch.empty_like(t) for t in routed[0])

    def call(i):
        if given:
            ids.copy_(routed[i][0])
            w.copy_(routed[i][1])
            return qg.moe_experts(xs[i], ids, w, L.experts)
        return qg.moe_layer(xs[i], router, L.experts, k)

    want = []
    for i in range(calls):
        want.append(call(i))
        torch.cuda.synchronize()
    assert len({tuple(i.flatten().tolist()) for i, _ in routed}) > 4
    for _ in range(10):
        assert all(torch.equal(a, b) for a, b in zip([call(i) for i in range(calls)], want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = [call(i) for i in range(calls)]
    for _ in range(20):
        for y in got:
            y.zero_()
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
