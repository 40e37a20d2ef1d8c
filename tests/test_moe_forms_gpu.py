"""Expert layers in the forms that the kernels tell apart: every pair of formats and
type with one and two MMAs an entry and several entries an expert, columns that end
inside a slab, passes that shared memory shortens, and a layer's bias and scale."""

import numpy as np
import pytest
import torch

import qgemv_roofline_b200 as qg

import moe_reference as ref
from test_moe_gpu import DEV, TORCH, Layer, choose, gpu

pytestmark = pytest.mark.gpu
PAIRS = [(a, b) for a in ("q8_0", "q4_0") for b in ("q8_0", "q4_0")]


@pytest.mark.parametrize("fmt,down", PAIRS)
@pytest.mark.parametrize("dtype", list(TORCH))
@pytest.mark.parametrize("N,E,k,K,F", [
    (2, 2, 2, 416, 288),     # two tokens an expert: one MMA
    (3, 3, 3, 704, 160),     # three: two MMAs
    (13, 2, 2, 352, 608),    # 13: entries of 4, 4, 4 and 1
    (9, 1, 1, 1056, 1312),   # one expert
    (64, 6, 2, 288, 224),
    (67, 4, 2, 160, 96),     # a second pass of 3 tokens
])
def test_types_formats_and_entries(fmt, down, dtype, N, E, k, K, F):
    L = Layer(E, K, F, fmt, down, seed=N + K)
    x, x64 = L.x(N, dtype)
    ids, w = choose(L.rng, N, E, k)
    y = qg.moe_experts(x, gpu(ids), gpu(w), L.experts)
    L.check(y, x64, ids, w, dtype)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("N", [16, 33, 64, 70])
def test_passes_that_shared_memory_shortens(N, dtype):
    """1024 experts and 32 choices leave room for the entries of 32 tokens."""
    E, K, F, k = 1024, 64, 32, 32
    L = Layer(E, K, F, "q4_0", "q8_0", seed=N)
    x, x64 = L.x(N, dtype)
    ids, w = choose(L.rng, N, E, k)
    ids[::3, 4], ids[1::4, 7] = -1, ids[1::4, 8]  # dropped choices, and an expert twice
    y = qg.moe_experts(x, gpu(ids), gpu(w), L.experts)
    L.check(y, x64, ids, w, dtype)
    # each token by itself: the sum over its experts in another order
    one = torch.stack([qg.moe_experts(x[n], gpu(ids[n]), gpu(w[n]), L.experts) for n in range(0, N, 9)])
    L.check(one, x64[::9], ids[::9], w[::9], dtype)


@pytest.mark.parametrize("N,dtype", [(1, "bfloat16"), (2, "float32"), (9, "float16"), (40, "bfloat16"), (130, "float32")])
@pytest.mark.parametrize("scoring,shared,normalize", [("sigmoid", 1, True), ("softmax", 0, True), ("sigmoid", 2, False),
                                                      ("softmax", 1, False)])
def test_layer_with_bias_and_scale(N, dtype, scoring, shared, normalize):
    E, k = 24, 4
    L = Layer(E + shared, 320, 192, "q8_0", "q4_0", shared=shared, seed=N)
    x, x64 = L.x(N, dtype)
    r = (L.rng.standard_normal((E, 320)) * 0.2).astype(np.float32)
    bias = L.rng.standard_normal(E).astype(np.float32) * 0.3
    y = qg.moe_layer(x, gpu(r), L.experts, k, scoring=scoring, bias=gpu(bias), scale=2.5, normalize=normalize)
    ids, w, _ = ref.route(x64, r, k, scoring, bias, 2.5, normalize)
    assert (ids != ref.route(x64, r, k, scoring, None, 2.5, normalize)[0]).any()  # the bias changes the choice
    ids = np.concatenate([ids, np.tile(np.arange(E, E + shared), (N, 1))], 1)
    w = np.concatenate([w, np.ones((N, shared))], 1)
    L.check(y, x64, ids, w, dtype)


@pytest.mark.parametrize("N", [1, 5, 70])
def test_in_place(N):
    """y may be x: a pass reads its rows before it writes them."""
    L = Layer(5, 256, 128, "q8_0", seed=N)
    x, _ = L.x(N, "float16")
    router = gpu(L.rng.standard_normal((5, 256)).astype(np.float32))
    want = qg.moe_layer(x, router, L.experts, 2)
    z = x.clone()
    assert qg.moe_layer(z, router, L.experts, 2, y=z) is z and torch.equal(z, want)
    wq, ws = qg.quantize_int8(torch.randn(256, 256, device=DEV))
    want = qg.int8_linear(x, wq, ws)
    z = x.clone()
    assert qg.int8_linear(z, wq, ws, y=z) is z and torch.equal(z, want)
