"""Routing where few tests go: weights of small scores, loads by element and by type in
the many-token kernel, rows longer than one staged chunk."""

import numpy as np
import pytest
import torch

import qgemv_roofline_b200 as qg

import moe_reference as ref
from test_moe_gpu import DEV, TORCH, gpu

pytestmark = pytest.mark.gpu


def check(x, r, k, scoring="softmax", bias=None, scale=1.0, normalize=True, xt=None, rt=None):
    """x, r: fp32 values that the types of xt, rt (tensors on the GPU) hold."""
    ids, w = qg.moe_route(gpu(x) if xt is None else xt, gpu(r) if rt is None else rt, k, scoring=scoring,
                          bias=None if bias is None else gpu(bias), scale=scale, normalize=normalize)
    want, ww, tol = ref.route(x, r, k, scoring, bias, scale, normalize)
    assert np.array_equal(ids.cpu().numpy(), want)
    got = w.double().cpu().numpy()
    worst = (np.abs(got - ww) / (tol * ww + 1e-37)).max()
    assert worst <= 1, f"{worst:.3g} of the bound"


@pytest.mark.parametrize("N", [1, 2, 40])
@pytest.mark.parametrize("k", [1, 2, 5])
def test_normalised_weights_of_tiny_sigmoids(N, k):
    """A sum of scores below the smallest normal fp32 number is a sum like any other: a score
    of 6e-39 is held to 2^-22 of itself (fp32's subnormal step 2^-149 below 2^-126.9)."""
    logits = np.array([-88.0, -88.1, -88.2, -88.05, -88.3, -88.5], np.float32)
    x = np.ones((N, 1), np.float32)
    ids, w = qg.moe_route(gpu(x), gpu(logits[:, None]), k, scoring="sigmoid")
    s = np.exp(logits.astype(np.float64))  # sigmoid(l) = e^l / (1 + e^l), e^l < 2^-126
    order = np.argsort(-s, kind="stable")[:k]
    assert (ids.cpu().numpy() == order).all()
    want = s[order] / s[order].sum()
    # expf of a logit of 88.5 to 2 ulps, scores to 2^-21.8 each (2^-149 / 3.6e-39), a division
    assert np.abs(w.double().cpu().numpy() / want - 1).max() <= 2 * (2.0 ** -21.8 + 4 * 2.0 ** -24)


@pytest.mark.parametrize("N", [1, 2, 40])
@pytest.mark.parametrize("gap", [20.0, 90.0, 95.0, 200.0])
def test_a_bias_that_chooses_far_below_the_best(N, gap):
    r = np.array([0, -gap, -gap - 1, -gap - 3, -gap - 0.5], np.float32)[:, None]
    bias = np.array([0, 2, 2.5, 3, 0], np.float32)
    check(np.ones((N, 1), np.float32), r, 3, bias=bias, scale=1.5)
    ids, w = qg.moe_route(torch.ones(N, 1, device=DEV), gpu(r), 3, bias=gpu(bias))
    assert torch.allclose(w.sum(-1), torch.ones(N, device=DEV), atol=1e-6, rtol=0)


def test_chosen_experts_of_no_score():
    """Every chosen logit -inf beside a finite one: weights of zero."""
    x = torch.tensor([[1e30, 1.0]], device=DEV).expand(2, 2).contiguous()
    r = torch.tensor([[0.0, 1.0], [-1e30, 0.0], [-1e30, 0.0]], device=DEV)
    ids, w = qg.moe_route(x, r, 2, bias=torch.tensor([0.0, 2.0, 2.0], device=DEV))
    assert ids.tolist() == [[1, 2]] * 2 and (w == 0).all()


@pytest.mark.parametrize("dtype", list(TORCH))
@pytest.mark.parametrize("rdtype", list(TORCH))
@pytest.mark.parametrize("N,E,K", [(33, 20, 90), (50, 37, 256), (129, 300, 131), (40, 9, 7)])
def test_many_tokens_by_type_and_stride(dtype, rdtype, N, E, K):
    """Both matrices in vectors (rows of 16-byte multiples) and by element."""
    rng = np.random.default_rng(N + E)
    x = torch.from_numpy(rng.standard_normal((N, K)).astype(np.float32)).to(TORCH[dtype])
    r = torch.from_numpy((2 * K ** -0.5 * rng.standard_normal((E, K))).astype(np.float32)).to(TORCH[rdtype])
    for xo, ro, pad in ((0, 0, 0), (3, 0, 8), (0, 5, 9), (8, 8, 24)):
        xt, rt = (torch.full((t.shape[0], K + pad + o), float("nan"), dtype=t.dtype, device=DEV)
                  for t, o in ((x, xo), (r, ro)))
        xt[:, xo:xo + K], rt[:, ro:ro + K] = x.to(DEV), r.to(DEV)
        check(x.float().numpy(), r.float().numpy(), min(5, E), xt=xt[:, xo:xo + K], rt=rt[:, ro:ro + K])


@pytest.mark.parametrize("N", [1, 2, 7, 35])
@pytest.mark.parametrize("E,K", [(8, 5120), (160, 4100), (1024, 96), (700, 2052), (300, 7168), (1, 9000), (5, 4097)])
@pytest.mark.parametrize("dtype,rdtype", [("float32", "float32"), ("bfloat16", "float32"), ("float16", "bfloat16")])
def test_long_rows_and_many_experts(N, E, K, dtype, rdtype):
    """Rows longer than a staged chunk of x (4096 or 2048 columns), more tiles of experts than warps."""
    rng = np.random.default_rng(N + E + K)
    x = torch.from_numpy(rng.standard_normal((N, K)).astype(np.float32)).to(TORCH[dtype])
    r = torch.from_numpy((2 * K ** -0.5 * rng.standard_normal((E, K))).astype(np.float32)).to(TORCH[rdtype])
    bias = (rng.random(E) * 0.2).astype(np.float32)
    for scoring, b in (("softmax", None), ("sigmoid", bias)):
        check(x.float().numpy(), r.float().numpy(), min(E, 8), scoring, b, 2.5, xt=x.to(DEV), rt=r.to(DEV))
