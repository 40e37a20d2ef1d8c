"""Expert layers whose activations hold outliers, against 64-bit values and a bound per block of 32.

The kernels round a block of activations to integers X with |X| <= 0x7F7F7F = FX at the block's
largest value m.  With s = fl(FX / m) and scale = fl(m / FX):

    |X - v FX / m| <= 1/2 + |v| (FX / m) 2^-23 <= 1/2 + FX 2^-23 < 1.5   (rounding; s and the product)
    |X scale - v|  <= 1.5 m / FX + |v| 2^-24 < 2^-21.9 m

so a value moves by at most BLOCK = 2^-21.9 of its block's largest.  An outlier with a weight of zero
then leaves its neighbours 22 bits below it, whatever the type of x, where a norm-wise bound
(1e-5 |w| |x|) would let it cover them."""

import numpy as np
import pytest
import torch

import qgemv_roofline_b200 as qg
from oracle import qformats_oracle as o

import moe_reference as ref
from test_moe_gpu import DEV, TORCH, gpu

pytestmark = pytest.mark.gpu
BLOCK = 2.0 ** -21.9
EPS = 2.0 ** -24


def dot(w, x, dx):
    """w [rows, cols] x [cols] and a bound of its error for x off by dx."""
    a, blocks = np.abs(w), len(x) // 32
    m = np.repeat((np.abs(x) + dx).reshape(-1, 32).max(-1), 32)
    # fp32: a product of scales and a sum per block; a term is a block's low or high digits,
    # the low ones below 2^-7 of the block's largest
    tol = a @ (dx + BLOCK * m) + (blocks + 16) * EPS * (a @ (np.abs(x) + dx + 2.0 ** -7 * m))
    return w @ x, tol


def layer(x, ids, weights, gate, up, down, dtype):
    y, tol = np.zeros_like(x), np.zeros_like(x)
    for n in range(len(x)):
        for e, w in zip(ids[n], weights[n].astype(np.float64)):
            g, dg = dot(gate[e], x[n], np.zeros_like(x[n]))
            u, du = dot(up[e], x[n], np.zeros_like(x[n]))
            s = g * 0.5 * (1 + np.tanh(g / 2))
            h = w * s * u
            # |silu'| <= 1.1; expf to 2 ulps, a sum, a division and two products
            dh = abs(w) * (1.1 * dg * (np.abs(u) + du) + np.abs(s) * du) + 2.0 ** -20 * np.abs(h)
            part, dp = dot(down[e], h, dh)
            y[n] += part
            tol[n] += dp + 8 * EPS * np.abs(part)
    return y, tol + ref.HALF_STEP[dtype] * (np.abs(y) + tol) + 1e-7 * (dtype == "float16")


def planes(fmt, w):
    E, rows, cols = w.shape
    q, d = o.quantize(fmt, w.reshape(E * rows, cols).astype(np.float32))
    return q.reshape(E, rows, -1), d.view(np.float16).reshape(E, rows, -1)


@pytest.mark.parametrize("dtype", list(TORCH))
@pytest.mark.parametrize("fmt,down_fmt", [("q8_0", "q4_0"), ("q4_0", "q8_0")])
@pytest.mark.parametrize("N", [1, 3, 13])
@pytest.mark.parametrize("where", ["x", "h"])
def test_outliers_do_not_cover_their_neighbours(N, fmt, down_fmt, dtype, where):
    rng = np.random.default_rng(N)
    E, K, F, k, col = 3, 64, 96, 2, 5
    gate, up, down = (rng.standard_normal(s) * s[2] ** -0.5 for s in ((E, F, K), (E, F, K), (E, K, F)))
    x = torch.from_numpy(rng.standard_normal((N, K)).astype(np.float32))
    big = 2.0 ** 14 if dtype == "float16" else 2.0 ** 17
    if where == "x":      # a channel far above the others, which no row of gate and up reads
        x[:, col] = big
        gate[:, :, col] = up[:, :, col] = 0
    else:                 # a row of h far above the others, which no row of down reads
        x[:, col] = 16.0
        gate[:, :, col] = up[:, :, col] = 0
        gate[:, 40, col], up[:, 40, col] = 8.0, big / 128
        down[:, :, 40] = 0
    x = x.to(TORCH[dtype])
    parts = planes(fmt, gate), planes(fmt, up), planes(down_fmt, down)
    w64 = [ref.dequant(f, *p) for f, p in zip((fmt, fmt, down_fmt), parts)]
    ids = np.stack([rng.permutation(E)[:k] for _ in range(N)]).astype(np.int32)
    weights = (0.25 + rng.random((N, k))).astype(np.float32)
    experts = qg.QuantizedExperts(*[(gpu(q), gpu(d)) for q, d in parts])
    y = qg.moe_experts(x.to(DEV), gpu(ids), gpu(weights), experts)
    want, tol = layer(x.double().numpy(), ids, weights, *w64, dtype)
    worst = (np.abs(y.double().cpu().numpy() - want) / tol).max()
    assert worst <= 1, f"{worst:.3g} of the bound"
