"""int8 products with a scale per token and channel, on the GPU against exact integers."""

import numpy as np
import pytest
import torch

import qgemv_roofline_b200 as qg
from qgemv_roofline_b200 import _lib

pytestmark = pytest.mark.gpu
DEV = "cuda"
TORCH = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
HALF_STEP = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}
TINY = {"float32": 1e-44, "bfloat16": 1e-40, "float16": 2.0 ** -25}  # half the smallest step


def gpu(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to(DEV)


def quantize(x):
    """The definition in fp32, as numpy rounds (IEEE division, half to even)."""
    x = x.astype(np.float32)
    s = (np.abs(x).max(-1) / np.float32(127)).astype(np.float32)
    with np.errstate(divide="ignore", invalid="ignore"):
        q = np.nan_to_num(np.where(s[..., None] > 0, np.rint(x / s[..., None]), 0))
    return np.clip(q, -127, 127).astype(np.int8), s


def product(xq, xs, wq, ws, bias):
    """y in float64 (integers below 2^53 are exact there) and the sum of its terms' sizes."""
    y = (xq.astype(np.float64) @ wq.astype(np.float64).T) * xs.astype(np.float64)[:, None] * ws.astype(np.float64)
    size = np.abs(y)
    if bias is not None:
        y, size = y + bias, size + np.abs(bias)
    return y, size


def check(y, want, size, dtype):
    """Four fp32 roundings (sum, two scales, bias), then y's own."""
    got = y.double().cpu().numpy()
    tol = 4.01 * 2.0 ** -24 * size
    tol = tol + HALF_STEP[dtype] * (np.abs(want) + tol) + TINY[dtype]
    worst = (np.abs(got - want) / tol).max()
    assert worst <= 1, f"{worst:.3g} of the bound"


SIZES = [(1, 1, 16), (1, 11008, 4096), (1, 300, 11008), (2, 130, 48), (3, 128, 128), (16, 128, 4096), (17, 257, 400),
         (32, 4096, 512), (33, 100, 2064), (64, 512, 1024), (65, 640, 320), (100, 1000, 160), (128, 129, 2048),
         (129, 300, 272), (256, 256, 256), (300, 5003, 2064), (513, 129, 4096), (1025, 2050, 528), (2100, 1024, 1040)]


@pytest.mark.parametrize("N,M,K", SIZES)
@pytest.mark.parametrize("dtype,biased", [("float32", True), ("bfloat16", False), ("float16", True)])
def test_matmul(N, M, K, dtype, biased):
    rng = np.random.default_rng(N + M + K)
    xq, wq = (rng.integers(-128, 128, s, dtype=np.int8) for s in ((N, K), (M, K)))
    xs, ws = (rng.random(n).astype(np.float32) * 1e-2 / K ** 0.5 for n in (N, M))
    xs, ws = xs.astype(np.float32), ws.astype(np.float32)
    bias = rng.standard_normal(M).astype(np.float32) if biased else None
    y = qg.int8_matmul(gpu(xq), gpu(xs), gpu(wq), gpu(ws), gpu(bias) if biased else None, TORCH[dtype])
    assert y.dtype == TORCH[dtype] and y.shape == (N, M)
    check(y, *product(xq, xs, wq, ws, bias), dtype)


@pytest.mark.parametrize("N,M,K", [
    (1, 9000, 1040), (16, 6100, 2064), (31, 3331, 3120), (32, 11001, 1088), (64, 11006, 1040), (64, 2501, 4112),
    (97, 4097, 2064), (127, 5003, 3088), (128, 8190, 1040), (129, 1001, 2576), (250, 1023, 4096), (257, 4000, 8208),
    (640, 129, 1040), (513, 515, 8208)])
@pytest.mark.parametrize("dtype", list(TORCH))
@pytest.mark.parametrize("shift,pad", [(0, 0), (1, 2), (4, 4)])
def test_splits_of_k(N, M, K, dtype, shift, pad):
    """Clusters of every size, into rows of y that start at any element and hold more
    than the product: what is beside it stays."""
    rng = np.random.default_rng(N * M + K)
    xq, wq = (torch.from_numpy(rng.integers(-128, 128, s, dtype=np.int8)).to(DEV) for s in ((N, K), (M, K)))
    xs, ws = (torch.from_numpy(rng.random(n).astype(np.float32) * 1e-2).to(DEV) for n in (N, M))
    bias = torch.from_numpy(rng.standard_normal(M).astype(np.float32)).to(DEV)
    whole = torch.full((N, shift + M + pad), 77.0, dtype=TORCH[dtype], device=DEV)
    y = whole[:, shift:shift + M]
    qg.int8_matmul(xq, xs, wq, ws, bias, TORCH[dtype], y)
    # integers below 2^53: exact in 64 bits in any order
    want = (xq.double() @ wq.double().T) * xs.double()[:, None] * ws.double()
    size = want.abs() + bias.double().abs()
    check(y, (want + bias.double()).cpu().numpy(), size.cpu().numpy(), dtype)
    assert (whole[:, :shift] == 77).all() and (whole[:, shift + M:] == 77).all()


@pytest.mark.parametrize("N", [1, 40, 300])
def test_sums_at_the_ends_of_int32(N):
    M, K = 130, 131056  # the largest K: 131056 * 128 * 128 = 2^31 - 2^18
    xq = np.full((N, K), -128, np.int8)
    wq = np.full((M, K), -128, np.int8)
    wq[1::2] = 127
    one = np.ones(max(N, M), np.float32)
    y = qg.int8_matmul(gpu(xq), gpu(one[:N]), gpu(wq), gpu(one[:M]), out_dtype=torch.float32)
    check(y, *product(xq, one[:N], wq, one[:M], None), "float32")


@pytest.mark.parametrize("N,K", [(1, 1), (1, 4096), (3, 100), (5, 11008), (700, 64), (2, 40000)])
@pytest.mark.parametrize("dtype", list(TORCH))
def test_quantize(N, K, dtype):
    rng = np.random.default_rng(N + K)
    x = torch.from_numpy((rng.standard_normal((N, K)) * 10.0 ** rng.uniform(-6, 3, (N, 1))).astype(np.float32))
    x = x.to(TORCH[dtype])
    q, s = qg.quantize_int8(x.to(DEV))
    wq, ws = quantize(x.float().numpy())
    assert np.array_equal(q.cpu().numpy(), wq) and np.array_equal(s.cpu().numpy(), ws)
    # strided rows in, padded rows out, nothing beside them written
    xs = torch.zeros(N, K + 9, dtype=x.dtype, device=DEV)
    xs[:, 5:5 + K] = x.to(DEV)
    out = torch.full((N, K + 32), 77, dtype=torch.int8, device=DEV)
    qg.quantize_int8(xs[:, 5:5 + K], q=out[:, 16:16 + K])
    assert torch.equal(out[:, 16:16 + K], q)
    assert (out[:, :16] == 77).all() and (out[:, 16 + K:] == 77).all()


def test_quantize_edges():
    tiny = np.float32(1e-45)
    x = np.zeros((9, 64), np.float32)
    x[1] = np.float32(3.4e38)
    x[2, 3] = np.nan
    x[3, 60] = -np.inf
    x[4, ::2] = tiny                       # the scale underflows to 0
    x[5, :3] = [200 * tiny, -190 * tiny, 100 * tiny]   # a subnormal scale: clipped at 127
    x[6] = np.arange(64) - 31.5            # ties: half to even
    x[7, 0], x[7, 1] = 127, 0.5
    x[8] = -0.0
    q, s = qg.quantize_int8(gpu(x))
    wq, ws = quantize(x)
    for r in (0, 1, 4, 5, 6, 7, 8):
        assert np.array_equal(q[r].cpu().numpy(), wq[r]) and s[r].item() == ws[r], r
    for r in (2, 3):
        assert torch.isnan(s[r]) and (q[r] == 0).all()
    # a row that is not finite gives NaN, the others are untouched
    wq = np.random.default_rng(1).integers(-127, 128, (33, 64), dtype=np.int8)
    y = qg.int8_linear(gpu(x), gpu(wq), torch.ones(33, device=DEV))
    assert torch.isnan(y[2]).all() and torch.isnan(y[3]).all()
    assert torch.isfinite(y[[0, 4, 5, 6, 7, 8]]).all() and (y[[0, 4, 8]] == 0).all()


@pytest.mark.parametrize("N,M,K", [(1, 257, 4096), (4, 1000, 160), (50, 384, 1040), (200, 513, 512), (777, 1030, 2048)])
@pytest.mark.parametrize("dtype", list(TORCH))
def test_linear(N, M, K, dtype):
    rng = np.random.default_rng(N + M + K)
    x = torch.from_numpy(rng.standard_normal((N, K)).astype(np.float32)).to(TORCH[dtype])
    W = (rng.standard_normal((M, K)) * K ** -0.5).astype(np.float32)
    wq, ws = qg.quantize_int8(gpu(W))
    bias = gpu(rng.standard_normal(M).astype(np.float32))
    y = qg.int8_linear(x.to(DEV), wq, ws, bias)
    assert y.dtype == x.dtype
    xq, xs = quantize(x.float().numpy())
    check(y, *product(xq, xs, wq.cpu().numpy(), ws.cpu().numpy(), bias.cpu().numpy()), dtype)
    # the same as its two halves, bit for bit, and another type out
    q, s = qg.quantize_int8(x.to(DEV))
    assert torch.equal(y, qg.int8_matmul(q, s, wq, ws, bias, x.dtype))
    y32 = qg.int8_linear(x.to(DEV), wq, ws, bias, out_dtype=torch.float32)
    assert torch.equal(y32.to(x.dtype), y)
    # how far int8 is from the product itself: every factor is off by half a step of its scale
    full = x.double().numpy() @ W.astype(np.float64).T + bias.double().cpu().numpy()
    ax, aw = np.abs(x.double().numpy()).max(-1) / 254, np.abs(W).max(-1) / 254
    far = (ax[:, None] * np.abs(W).sum(-1) + np.abs(x.double().numpy()).sum(-1)[:, None] * aw
           + K * ax[:, None] * aw) * 1.001
    assert (np.abs(y32.double().cpu().numpy() - full) <= far + 1e-4).all()


def test_vectors_strides_and_guard_bands():
    rng = np.random.default_rng(5)
    N, M, K = 70, 300, 208
    xq, wq = (rng.integers(-127, 128, s, dtype=np.int8) for s in ((N, K), (M, K)))
    xs, ws = rng.random(N).astype(np.float32), rng.random(M).astype(np.float32)
    X, W = torch.zeros(N, 256, dtype=torch.int8, device=DEV), torch.zeros(M, 512, dtype=torch.int8, device=DEV)
    X[:, 32:32 + K], W[:, 16:16 + K] = gpu(xq), gpu(wq)
    X[:, 32 + K:], W[:, 16 + K:] = 99, 98   # columns past K are not read into the sum
    want = product(xq, xs, wq, ws, None)
    for dtype in ("float32", "bfloat16"):
        out = torch.full((N + 2, M + 11), 5.0, dtype=TORCH[dtype], device=DEV)
        y = qg.int8_matmul(X[:, 32:32 + K], gpu(xs), W[:, 16:16 + K], gpu(ws), out_dtype=TORCH[dtype],
                           y=out[1:-1, 3:3 + M])
        check(y, *want, dtype)
        out[1:-1, 3:3 + M] = 5.0
        assert (out == 5.0).all()
    y = qg.int8_matmul(X[3, 32:32 + K], gpu(xs)[3], W[:, 16:16 + K], gpu(ws))
    check(y[None], want[0][3:4], want[1][3:4], "float32")
    x = torch.randn(K, device=DEV)
    assert torch.equal(qg.int8_linear(x, gpu(wq), gpu(ws)), qg.int8_linear(x[None], gpu(wq), gpu(ws))[0])
    t = torch.randn(K, 5, device=DEV).t()  # columns of a matrix: laid out anew
    assert torch.equal(qg.int8_linear(t, gpu(wq), gpu(ws)), qg.int8_linear(t.contiguous(), gpu(wq), gpu(ws)))
    assert qg.int8_linear(x[None][:0], gpu(wq), gpu(ws)).shape == (0, M)
    assert qg.int8_matmul(X[:, :K], gpu(xs), gpu(wq)[:0], gpu(ws)[:0]).shape == (N, 0)


@pytest.mark.parametrize("N", [1, 20, 400])
def test_weights_made_just_before(N):
    """The product may read its weights ahead of the previous launch, but not ahead of
    the one that writes them."""
    g = torch.Generator(DEV).manual_seed(N)
    M, K = 2000, 1024
    x = torch.randn(N, K, device=DEV, generator=g)
    q, s = torch.empty(M, K, dtype=torch.int8, device=DEV), torch.empty(M, device=DEV)
    want = []
    Ws = [torch.randn(M, K, device=DEV, generator=g) for _ in range(4)]
    for W in Ws:
        a, b = qg.quantize_int8(W)
        torch.cuda.synchronize()
        want.append(qg.int8_linear(x, a, b))
        torch.cuda.synchronize()
    xq, xs = qg.quantize_int8(x)
    for _ in range(5):
        for W, y in zip(Ws, want):
            qg.quantize_int8(W, q=q, scales=s)
            got = qg.int8_linear(x, q, s)
            qg.quantize_int8(Ws[0], q=q, scales=s)
            qg.quantize_int8(W, q=q, scales=s)
            also = qg.int8_matmul(xq, xs, q, s)
            assert torch.equal(got, y) and torch.equal(also, y)


def test_captured_replayed_and_on_two_streams():
    g = torch.Generator(DEV).manual_seed(2)
    wq, ws = qg.quantize_int8(torch.randn(1500, 768, device=DEV, generator=g))
    xs = [torch.randn(n, 768, device=DEV, generator=g) for n in (1, 130, 600)]
    want = [qg.int8_linear(x, wq, ws) for x in xs]
    static = [torch.zeros_like(x) for x in xs]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = [qg.int8_linear(x, wq, ws) for x in static]
    for s, x in zip(static, xs):
        s.copy_(x)
    for _ in range(3):
        graph.replay()
        eager = qg.int8_linear(xs[1], wq, ws)
        assert all(torch.equal(a, b) for a, b in zip(outs, want)) and torch.equal(eager, want[1])
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = [[] for _ in xs]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(qg.int8_linear(xs[i], wq, ws))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i]) for i in range(3) for y in got[i])
    y = torch.empty_like(want[2])
    qg.int8_linear(xs[2], wq, ws, y=y, stream=streams[0].cuda_stream)  # a raw handle
    streams[0].synchronize()
    assert torch.equal(y, want[2])


def test_a_wait_that_runs_out_is_reported():
    lib = _lib.lib()
    g = torch.Generator(DEV).manual_seed(3)
    wq, ws = qg.quantize_int8(torch.randn(16384, 8192, device=DEV, generator=g))
    for n in (1, 500):  # single CTAs, CTA pairs
        xq, xs = qg.quantize_int8(torch.randn(n, 8192, device=DEV, generator=g))
        want = qg.int8_matmul(xq, xs, wq, ws)
        torch.cuda.synchronize()
        seen = False
        for _ in range(20):
            assert lib.qgemv_set_wait_limit(1) == 0  # 1 us: shorter than a DRAM round trip under load
            try:
                qg.int8_matmul(xq, xs, wq, ws)
                torch.cuda.synchronize()
            finally:
                assert lib.qgemv_set_wait_limit(0) == 0
            if lib.qgemv_check_device_error(1, None) == 6:
                seen = True
                break
        assert seen, "no wait ran out under a 1 us limit"
        assert lib.qgemv_check_device_error(0, None) == 0
        assert torch.equal(qg.int8_matmul(xq, xs, wq, ws), want)
    assert lib.qgemv_check_device_error(0, None) == 0


def test_decode_and_prefill_steps_together():
    """A projection in int8, a mixture of experts, a GEMV head: the operators in a row, each
    reading the one before, for a prompt and then one token at a time."""
    g = torch.Generator(DEV).manual_seed(4)
    K, F, E, V = 256, 128, 6, 300
    proj = qg.quantize_int8(torch.randn(K, K, device=DEV, generator=g) * K ** -0.5)
    router = torch.randn(E, K, device=DEV, generator=g) * 0.2
    w = [torch.randn(E, *s, device=DEV, generator=g) * s[1] ** -0.5 for s in ((F, K), (F, K), (K, F))]
    experts = qg.QuantizedExperts.from_float(*w, "q8_0")
    head = qg.QuantizedMatrix.from_float(torch.randn(V, K, device=DEV, generator=g) * K ** -0.5, "q8_0")

    def step(x):
        h = x + qg.int8_linear(x, *proj)
        h = h + qg.moe_layer(h, router, experts, 2)
        return head(h)

    x = torch.randn(70, K, device=DEV, generator=g)
    whole = step(x)
    each = torch.stack([step(v) for v in x])
    # a token alone and in a batch differ by rounding only (other kernels take it): a
    # thousandth of the row's size is far above that and far below a wrong choice
    assert ((whole - each).norm(dim=1) <= 1e-3 * whole.norm(dim=1)).all()
    graph = torch.cuda.CUDAGraph()
    static = x[:5].clone()
    step(static)
    with torch.cuda.graph(graph):
        out = step(static)
    graph.replay()
    assert torch.equal(out, step(static))


def test_refusals():
    x = torch.zeros(2, 64, device=DEV)
    xq, xs = qg.quantize_int8(x)
    wq, ws = torch.zeros(10, 64, dtype=torch.int8, device=DEV), torch.zeros(10, device=DEV)
    for bad in (x.cpu(), x.double(), x[None], torch.zeros((), device=DEV), x[:, :0]):
        with pytest.raises((ValueError, TypeError)):
            qg.quantize_int8(bad)
    for kw in ({"q": xq[:1]}, {"q": xq.to(torch.uint8)}, {"scales": xs[:1]}, {"scales": xs.double()}):
        with pytest.raises(ValueError):
            qg.quantize_int8(x, **kw)
    for a in ((xq.float(), xs, wq, ws), (xq, xs[:1], wq, ws), (xq, xs, wq[:, :32], ws), (xq, xs, wq.cpu(), ws),
              (xq, xs, wq, ws[:4]), (xq, xs, wq, ws, ws[:4]), (xq.t(), xs, wq, ws), (xq, xs, wq.float(), ws)):
        with pytest.raises(ValueError):
            qg.int8_matmul(*a)
    with pytest.raises(TypeError):
        qg.int8_matmul(xq, xs, wq, ws, out_dtype=torch.int32)
    with pytest.raises(ValueError):
        qg.int8_matmul(xq, xs, wq, ws, y=torch.zeros(2, 9, device=DEV))
    with pytest.raises(ValueError):
        qg.int8_linear(x, wq, ws, y=torch.zeros(2, 10, dtype=torch.float16, device=DEV))
    # sizes and alignment that the tensor copies need
    for K in (8, 24, 1 << 17):
        z = torch.zeros(2, K, dtype=torch.int8, device=DEV)
        with pytest.raises(_lib.QGemvError):
            qg.int8_matmul(z, xs, z, xs)
    buf = torch.zeros(2, 128, dtype=torch.int8, device=DEV)
    for a in (buf[:, 8:72], buf.view(-1)[:2 * 72].view(2, 72)[:, :64]):
        with pytest.raises(_lib.QGemvError):
            qg.int8_matmul(a, xs, wq, ws)
