"""Plain 64-bit restatement of the mixture-of-experts operators (numpy), with
the error bound of the kernels' arithmetic beside each result."""

import numpy as np

# The GEMVs' bound on a row's dot (block fixed point, fp32 block sums): the
# experts' products are the same arithmetic.
DOT = 1e-5
HALF_STEP = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}


def dequant(fmt, q, d):
    """Planes [..., rows, cols(/2)], scales [..., rows, cols/32] -> float64 weights."""
    d = d.astype(np.float64)
    if fmt == "q8_0":
        v = q.astype(np.float64)
    else:
        b = q.reshape(*d.shape, 16)
        v = np.concatenate([(b & 15).astype(np.float64), (b >> 4).astype(np.float64)], -1) - 8
        v = v.reshape(*d.shape[:-1], -1)
    return v * np.repeat(d, 32, -1)


def route(x, router, k, scoring="softmax", bias=None, scale=1.0, normalize=True):
    """ids, weights, relative bound of the weights; the logits are rounded to fp32."""
    logits = (x.astype(np.float64) @ router.astype(np.float64).T).astype(np.float32).astype(np.float64)
    mx = logits.max(-1, keepdims=True)
    if scoring == "softmax":
        p = np.exp(logits - mx)
        score = p / p.sum(-1, keepdims=True)
    else:
        score = 1 / (1 + np.exp(-logits))
    rank = logits if bias is None else score + bias.astype(np.float64)
    ids = np.argsort(-rank, axis=-1, kind="stable")[:, :k]
    w = np.take_along_axis(score, ids, -1)
    if normalize:
        w = w / w.sum(-1, keepdims=True)
    # expf of a rounded difference (its half step times the exponent) to 2 ulps, sums of up
    # to 1024 fp32 terms in a tree of 5 + 32 steps, a division and a product
    span = np.abs(logits - mx).max(-1, keepdims=True) if scoring == "softmax" else np.abs(logits).max(-1, keepdims=True)
    return ids.astype(np.int32), w * scale, (2 * span + 8 + 2 * 37 + 4) * 2.0 ** -24


def experts(x, ids, weights, gate, up, down, out_dtype="float32"):
    """y and its bound; gate, up [E, F, K] and down [E, K, F] in float64.

    With |dg| <= DOT |w_g| |x|, |du| alike, and |silu'| <= 1.1:
      |dh| <= |w| (1.1 |dg| (|u| + |du|) + |silu(g)| |du|) + 2^-20 |h|  (expf, division, products)
      |dy| <= sum_j |down_row| (|dh_j| + DOT |h_j + dh_j|) + (sum of <= 40 fp32 terms) + rounding."""
    N, K = x.shape
    y = np.zeros((N, K))
    tol = np.zeros((N, K))
    for n in range(N):
        xn = np.linalg.norm(x[n])
        mag = np.zeros(K)
        for j, e in enumerate(ids[n]):
            if not 0 <= e < gate.shape[0]:
                continue
            w = float(weights[n, j])
            g, u = gate[e] @ x[n], up[e] @ x[n]
            dg = DOT * np.linalg.norm(gate[e], axis=1) * xn
            du = DOT * np.linalg.norm(up[e], axis=1) * xn
            s = g * 0.5 * (1 + np.tanh(g / 2))
            h = s * u * w
            dh = abs(w) * (1.1 * dg * (np.abs(u) + du) + np.abs(s) * du) + 2.0 ** -20 * np.abs(h)
            dn = np.linalg.norm(down[e], axis=1)
            part = down[e] @ h
            y[n] += part
            mag += np.abs(part)
            tol[n] += dn * (np.linalg.norm(dh) + DOT * (np.linalg.norm(h) + np.linalg.norm(dh)))
        tol[n] += 40 * 2.0 ** -24 * mag
    tol += HALF_STEP[out_dtype] * (np.abs(y) + tol) + 1e-30
    return y, tol
