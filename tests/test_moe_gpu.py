"""Mixture-of-experts layers on the GPU against a plain 64-bit restatement."""

import numpy as np
import pytest
import torch

import qgemv_roofline_b200 as qg
from qgemv_roofline_b200 import _lib
from oracle import qformats_oracle as o

import moe_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
TORCH = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def planes(fmt, E, rows, cols, rng, scale=1.0):
    q, d = o.quantize(fmt, (rng.standard_normal((E * rows, cols)) * scale * cols ** -0.5).astype(np.float32))
    return q.reshape(E, rows, -1), d.view(np.float16).reshape(E, rows, -1)


def gpu(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to(DEV)


class Layer:
    """Experts on the GPU and their float64 weights."""

    def __init__(self, E, K, F, fmt, down=None, shared=0, seed=0):
        rng = np.random.default_rng(seed)
        down = down or fmt
        g, u, dn = (planes(fmt, E, F, K, rng), planes(fmt, E, F, K, rng), planes(down, E, K, F, rng))
        self.gate, self.up, self.down = ref.dequant(fmt, *g), ref.dequant(fmt, *u), ref.dequant(down, *dn)
        self.experts = qg.QuantizedExperts(*[(gpu(q), gpu(d)) for q, d in (g, u, dn)], n_shared=shared)
        self.rng, self.E, self.K, self.F, self.shared = rng, E, K, F, shared

    def x(self, N, dtype="float32"):
        t = torch.from_numpy(self.rng.standard_normal((N, self.K)).astype(np.float32)).to(TORCH[dtype])
        return t.to(DEV), t.double().numpy()

    def check(self, y, x64, ids, weights, dtype="float32"):
        want, tol = ref.experts(x64, ids, weights, self.gate, self.up, self.down, dtype)
        got = y.double().cpu().numpy()
        assert np.isfinite(got).all()
        worst = (np.abs(got - want) / tol).max()
        assert worst <= 1, f"{worst:.3g} of the bound"


def choose(rng, N, E, k):
    ids = np.stack([rng.permutation(E)[:k] for _ in range(N)]).astype(np.int32)
    return ids, rng.random((N, k)).astype(np.float32)


@pytest.mark.parametrize("fmt,down", [("q8_0", "q8_0"), ("q4_0", "q4_0"), ("q4_0", "q8_0"), ("q8_0", "q4_0")])
@pytest.mark.parametrize("N,E,k,K,F", [
    (1, 1, 1, 32, 32),        # the smallest
    (1, 8, 2, 256, 128),
    (2, 3, 3, 96, 160),       # two tokens of every expert; columns that end inside a group
    (5, 12, 4, 480, 352),
    (9, 2, 2, 128, 64),       # nine tokens of each expert: the 16-column form
    (33, 3, 2, 160, 96),      # more than 16 tokens of an expert: several entries
    (64, 16, 3, 512, 256),
    (70, 5, 1, 64, 96),       # two passes of tokens
    (3, 40, 8, 2048, 1056),   # several units per CTA
])
def test_experts(fmt, down, N, E, k, K, F):
    L = Layer(E, K, F, fmt, down, seed=N + E + K)
    x, x64 = L.x(N)
    ids, w = choose(L.rng, N, E, k)
    y = qg.moe_experts(x, gpu(ids), gpu(w), L.experts)
    L.check(y, x64, ids, w)


@pytest.mark.parametrize("dtype", list(TORCH))
@pytest.mark.parametrize("N", [1, 6, 20])
def test_experts_types(dtype, N):
    L = Layer(6, 288, 224, "q4_0", "q8_0", seed=N)
    x, x64 = L.x(N, dtype)
    ids, w = choose(L.rng, N, 6, 3)
    y = qg.moe_experts(x, gpu(ids), gpu(w), L.experts)
    assert y.dtype == TORCH[dtype]
    L.check(y, x64, ids, w, dtype)


def test_experts_choices_that_select_nothing_and_twice_the_same():
    L = Layer(5, 128, 96, "q8_0", seed=3)
    x, x64 = L.x(6)
    ids = np.array([[0, -1, 4], [-1, -1, -1], [2, 2, 2], [5, 1000000, -7], [3, 1, 3], [4, 0, 1]], np.int32)
    w = L.rng.random((6, 3)).astype(np.float32)
    y = qg.moe_experts(x, gpu(ids), gpu(w), L.experts)
    L.check(y, x64, ids, w)
    assert (y[1] == 0).all() and (y[3] == 0).all()


def test_experts_every_token_without_an_expert():
    L = Layer(3, 64, 32, "q4_0", seed=4)
    x, _ = L.x(4)
    y = torch.full((4, 64), 7.0, device=DEV)
    qg.moe_experts(x, torch.full((4, 2), -1, dtype=torch.int32, device=DEV), torch.ones(4, 2, device=DEV),
                   L.experts, y=y)
    assert (y == 0).all()


def test_non_finite_activations_stay_in_their_row():
    L = Layer(4, 256, 128, "q8_0", seed=5)
    x, x64 = L.x(5)
    ids, w = choose(L.rng, 5, 4, 2)
    x[1, 70] = float("nan")
    x[3, 255] = float("inf")
    y = qg.moe_experts(x, gpu(ids), gpu(w), L.experts)
    assert torch.isnan(y[1]).all() and torch.isnan(y[3]).all()
    keep = [0, 2, 4]
    L.check(y[keep], x64[keep], ids[keep], w[keep])
    w[2, 0] = np.nan  # a NaN weight too
    x, x64 = L.x(5)
    y = qg.moe_experts(x, gpu(ids), gpu(w), L.experts)
    assert torch.isnan(y[2]).all()
    keep = [0, 1, 3, 4]
    L.check(y[keep], x64[keep], ids[keep], w[keep])
    # and nothing of it stays in the workspace
    y = qg.moe_experts(x[keep], gpu(ids[keep]), gpu(w[keep]), L.experts)
    L.check(y, x64[keep], ids[keep], w[keep])


@pytest.mark.parametrize("F", [96, 128])
def test_a_stale_nan_in_the_workspace_does_not_reach_the_next_call(F):
    bad = Layer(2, 128, 256, "q8_0", seed=6)   # its h fills the blocks that F = 96 pads
    x, _ = bad.x(8)
    ids, w = choose(bad.rng, 8, 2, 2)
    qg.moe_experts(x * float("nan"), gpu(ids), gpu(w), bad.experts)
    L = Layer(2, 96, F, "q8_0", seed=7)
    x, x64 = L.x(8)
    L.check(qg.moe_experts(x, gpu(ids), gpu(w), L.experts), x64, ids, w)


@pytest.mark.parametrize("scale", [2.0 ** -60, 1e-12, 1e4, 2.0 ** 40])
def test_experts_scaled_activations(scale):
    # silu(g) u of a scaled token spans both ends of the float range of h
    L = Layer(2, 128, 64, "q8_0", seed=8)
    x, x64 = L.x(3)
    s = torch.tensor(scale, dtype=torch.float32)
    ids, w = choose(L.rng, 3, 2, 2)
    y = qg.moe_experts(x * s.to(DEV), gpu(ids), gpu(w), L.experts)
    L.check(y, x64 * float(s), ids, w)


def test_strided_rows_and_guard_bands():
    L = Layer(4, 160, 96, "q4_0", seed=9)
    x, x64 = L.x(3, "float16")
    ids, w = choose(L.rng, 3, 4, 2)
    buf = torch.full((5, 200), 3.0, dtype=torch.float16, device=DEV)
    buf[:3, 7:167] = x
    out = torch.full((5, 200), 5.0, dtype=torch.float16, device=DEV)
    y = qg.moe_experts(buf[:3, 7:167], gpu(ids), gpu(w), L.experts, y=out[1:4, 11:171])
    L.check(y, x64, ids, w, "float16")
    out[1:4, 11:171] = 5.0
    assert (out == 5.0).all()
    # a transposed x (stride 1 between tokens) is laid out anew
    y2 = qg.moe_experts(x.t().contiguous().t(), gpu(ids), gpu(w), L.experts)
    assert torch.equal(y2, qg.moe_experts(x, gpu(ids), gpu(w), L.experts))
    # a token repeated by a zero stride
    y3 = qg.moe_experts(x[:1].expand(3, 160), gpu(ids), gpu(w), L.experts)
    L.check(y3, np.repeat(x64[:1], 3, 0), ids, w, "float16")
    # a vector
    y4 = qg.moe_experts(x[0], gpu(ids[0]), gpu(w[0]), L.experts)
    assert y4.shape == (160,)
    L.check(y4[None], x64[:1], ids[:1], w[:1], "float16")
    assert qg.moe_experts(x[:0], gpu(ids[:0]), gpu(w[:0]), L.experts).shape == (0, 160)


@pytest.mark.parametrize("N,E,K,k", [(1, 1, 1, 1), (1, 8, 32, 2), (1, 128, 2048, 8), (2, 5, 37, 5), (8, 64, 4100, 6),
                                     (9, 320, 512, 12), (40, 1024, 96, 32), (300, 17, 1000, 4)])
@pytest.mark.parametrize("scoring,biased,normalize", [("softmax", False, True), ("softmax", True, False),
                                                      ("sigmoid", True, True), ("sigmoid", False, False)])
def test_route(N, E, K, k, scoring, biased, normalize):
    rng = np.random.default_rng(N + E + K)
    x = rng.standard_normal((N, K)).astype(np.float32)
    r = (rng.standard_normal((E, K)) * 2 * K ** -0.5).astype(np.float32)
    bias = (rng.random(E) * 0.2).astype(np.float32) if biased else None
    ids, w = qg.moe_route(gpu(x), gpu(r), k, scoring=scoring, bias=None if bias is None else gpu(bias),
                          scale=1.5, normalize=normalize)
    want, ww, tol = ref.route(x, r, k, scoring, bias, 1.5, normalize)
    assert ids.dtype == torch.int32 and np.array_equal(ids.cpu().numpy(), want)
    got = w.double().cpu().numpy()
    assert (np.abs(got - ww) <= tol * ww + 1e-37).all()


@pytest.mark.parametrize("dtype", list(TORCH))
@pytest.mark.parametrize("rdtype", list(TORCH))
def test_route_types_and_strides(dtype, rdtype):
    rng = np.random.default_rng(11)
    x = torch.from_numpy(rng.standard_normal((6, 90)).astype(np.float32)).to(TORCH[dtype])
    r = torch.from_numpy(rng.standard_normal((20, 90)).astype(np.float32)).to(TORCH[rdtype])
    xs, rs = torch.zeros(6, 101, dtype=x.dtype, device=DEV), torch.zeros(20, 97, dtype=r.dtype, device=DEV)
    xs[:, 3:93], rs[:, 5:95] = x.to(DEV), r.to(DEV)
    ids, w = qg.moe_route(xs[:, 3:93], rs[:, 5:95], 4)
    want, ww, tol = ref.route(x.float().numpy(), r.float().numpy(), 4)
    assert np.array_equal(ids.cpu().numpy(), want)
    assert (np.abs(w.double().cpu().numpy() - ww) <= tol * ww).all()
    i1, w1 = qg.moe_route(xs[2, 3:93], rs[:, 5:95], 4)
    assert torch.equal(i1, ids[2]) and torch.equal(w1, w[2])


def test_route_without_tokens():
    ids, w = qg.moe_route(torch.zeros(0, 64, device=DEV), torch.zeros(5, 64, device=DEV), 2)
    assert ids.shape == w.shape == (0, 2)


def test_route_ties_go_to_the_lower_index():
    rng = np.random.default_rng(12)
    r = rng.standard_normal((50, 64)).astype(np.float32)
    r[[7, 20, 45]] = r[30]
    x = rng.standard_normal((5, 64)).astype(np.float32)
    x[0] = r[30]
    x[1] = 0  # every logit equal
    for scoring in ("softmax", "sigmoid"):
        ids, w = qg.moe_route(gpu(x), gpu(r), 6, scoring=scoring)
        want, ww, tol = ref.route(x, r, 6, scoring)
        assert np.array_equal(ids.cpu().numpy(), want)
        assert ids[1].tolist() == list(range(6)) and ids[0].tolist()[:4] == [7, 20, 30, 45]


def test_route_non_finite_logits():
    x = torch.ones(4, 32, device=DEV)
    r = torch.randn(10, 32, device=DEV, generator=torch.Generator(DEV).manual_seed(1))
    x[1, 3] = float("nan")
    x[2, 5] = float("inf")
    for scoring in ("softmax", "sigmoid"):
        ids, w = qg.moe_route(x, r, 3, scoring=scoring)
        assert ((ids >= 0) & (ids < 10)).all()
        assert torch.isnan(w[1]).all() and torch.isfinite(w[[0, 3]]).all()
        if scoring == "softmax":
            assert torch.isnan(w[2]).all()   # exp(inf - inf)
    # a score of -inf is the lowest number, but a number
    r = torch.zeros(4, 2, device=DEV)
    r[:, 0] = torch.tensor([0.0, 1.0, -3e38, 2.0])
    ids, w = qg.moe_route(torch.tensor([10.0, 0.0], device=DEV), r, 4)
    assert ids.tolist() == [3, 1, 0, 2] and w[3] == 0 and torch.isfinite(w).all()
    # every chosen score underflows: weights of zero
    ids, w = qg.moe_route(torch.tensor([-300.0], device=DEV), torch.ones(3, 1, device=DEV), 2, scoring="sigmoid")
    assert (w == 0).all()


@pytest.mark.parametrize("scoring,shared,normalize", [("softmax", 0, True), ("sigmoid", 2, True), ("softmax", 1, False)])
@pytest.mark.parametrize("N,dtype", [(1, "bfloat16"), (4, "float32"), (19, "float16"), (66, "float32")])
def test_layer(N, dtype, scoring, shared, normalize):
    L = Layer(9 + shared, 256, 160, "q4_0", "q8_0", shared=shared, seed=N)
    x, x64 = L.x(N, dtype)
    r = (L.rng.standard_normal((9, 256)) * 0.2).astype(np.float32)
    y = qg.moe_layer(x, gpu(r), L.experts, 3, scoring=scoring, normalize=normalize, scale=1.25)
    ids, w, _ = ref.route(x64, r, 3, scoring, None, 1.25, normalize)
    ids = np.concatenate([ids, np.tile(np.arange(9, 9 + shared), (N, 1))], 1)
    w = np.concatenate([w, np.ones((N, shared))], 1)
    L.check(y, x64, ids, w, dtype)
    # the same as its two halves, bit for bit
    i2, w2 = qg.moe_route(x, gpu(r), 3, scoring=scoring, normalize=normalize, scale=1.25)
    i2 = torch.cat([i2, torch.arange(9, 9 + shared, device=DEV, dtype=torch.int32).expand(N, shared)], 1).contiguous()
    w2 = torch.cat([w2, torch.ones(N, shared, device=DEV)], 1).contiguous()
    assert torch.equal(y, qg.moe_experts(x, i2, w2, L.experts))


def test_same_bits_every_time_and_dependent_calls():
    L = Layer(12, 512, 256, "q8_0", shared=1, seed=20)
    r = gpu((L.rng.standard_normal((11, 512)) * 0.1).astype(np.float32))
    x, _ = L.x(5)
    first = qg.moe_layer(x, r, L.experts, 4)
    for _ in range(5):
        assert torch.equal(qg.moe_layer(x, r, L.experts, 4), first)
    # a chain of layers, nothing waits between: each reads the previous output
    def chain(sync):
        z = x
        for _ in range(6):
            z = qg.moe_layer(z, r, L.experts, 4) + z
            if sync:
                torch.cuda.synchronize()
        return z
    assert torch.equal(chain(False), chain(True))


def test_captured_and_replayed():
    L = Layer(10, 256, 128, "q4_0", seed=21)
    r = gpu((L.rng.standard_normal((10, 256)) * 0.1).astype(np.float32))
    x, _ = L.x(3)
    other, _ = L.x(3)
    want = [qg.moe_layer(v, r, L.experts, 2) for v in (x, other)]
    static = x.clone()
    graphs = []
    for _ in range(2):  # two graphs, each with its own workspace
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = qg.moe_layer(static, r, L.experts, 2)
        graphs.append((g, out))
    for g, out in graphs:
        for v, w in zip((x, other, x), (want[0], want[1], want[0])):
            static.copy_(v)
            g.replay()
            eager = qg.moe_layer(other, r, L.experts, 2)
            assert torch.equal(out, w) and torch.equal(eager, want[1])
    # both at once, on two streams
    static.copy_(x)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(20):
        for s, (g, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(out, want[0]) for _, out in graphs)


FIRST_CALLS = """
import torch, qgemv_roofline_b200 as qg
g = torch.Generator("cuda").manual_seed(1)
w = [torch.randn(4, *s, device="cuda", generator=g) for s in ((64, 128), (64, 128), (128, 64))]
experts = qg.QuantizedExperts.from_float(*w, "q8_0")
router = torch.randn(4, 128, device="cuda", generator=g)
wq, ws = qg.quantize_int8(w[0][0])
xs = [torch.randn(n, 128, device="cuda", generator=g) for n in (1, 9, 40, 200)]
calls = lambda: [f(x) for x in xs for f in (lambda x: qg.moe_layer(x, router, experts, 2), lambda x: qg.int8_linear(x, wq, ws))]
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = calls()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(out, calls()))
stream = torch.cuda.Stream()
with torch.cuda.stream(stream):
    graph = torch.cuda.CUDAGraph()
    graph.capture_begin()
    for f in (lambda s: qg.moe_layer(xs[0], router, experts, 2, stream=s), lambda s: qg.int8_linear(xs[0], wq, ws, stream=s)):
        try:
            f(stream.cuda_stream)
            raise SystemExit("a raw stream under capture was not refused")
        except qg.QGemvError as e:
            assert e.status == 5, e
    graph.capture_end()
print("first calls ok")
"""


def test_first_calls_of_a_process_are_captured():
    """Nothing that a first call sets up is missing under capture; a raw stream handle under
    capture, which would get the stream's shared workspace, is refused."""
    import subprocess
    import sys
    r = subprocess.run([sys.executable, "-c", FIRST_CALLS], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "first calls ok" in r.stdout, r.stdout + r.stderr


def test_two_streams_at_once():
    L = Layer(16, 512, 512, "q8_0", seed=22)
    r = gpu((L.rng.standard_normal((16, 512)) * 0.1).astype(np.float32))
    xs = [L.x(n)[0] for n in (1, 7)]
    want = [qg.moe_layer(x, r, L.experts, 4) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(30):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(qg.moe_layer(xs[i], r, L.experts, 4))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(y, want[i]) for y in got[i])
    # a raw stream handle
    y = torch.empty_like(want[1])
    qg.moe_layer(xs[1], r, L.experts, 4, y=y, stream=streams[0].cuda_stream)
    streams[0].synchronize()
    assert torch.equal(y, want[1])


def test_a_wait_that_runs_out_is_reported():
    lib = _lib.lib()
    L = Layer(4, 8192, 256, "q8_0", seed=23)  # half a megabyte per unit: its sums come microseconds late
    x, x64 = L.x(4)
    ids, w = choose(L.rng, 4, 4, 2)
    args = x, gpu(ids), gpu(w), L.experts
    want = qg.moe_experts(*args)
    torch.cuda.synchronize()
    seen = False
    for _ in range(30):
        assert lib.qgemv_set_wait_limit(1) == 0
        try:
            qg.moe_experts(*args)
            torch.cuda.synchronize()
        finally:
            assert lib.qgemv_set_wait_limit(0) == 0
        if lib.qgemv_check_device_error(1, None) == 6:
            seen = True
            break
    assert seen, "no wait ran out under a 1 us limit"
    assert lib.qgemv_check_device_error(0, None) == 0
    assert torch.equal(qg.moe_experts(*args), want)
    assert lib.qgemv_check_device_error(0, None) == 0


def test_experts_from_float_and_from_matrices():
    E, K, F = 3, 96, 64
    g = torch.Generator(DEV).manual_seed(3)
    gate, up, down = (torch.randn(E, *s, device=DEV, generator=g) for s in ((F, K), (F, K), (K, F)))
    a = qg.QuantizedExperts.from_float(gate, up, down, "q4_0", "q8_0")
    m = [qg.QuantizedMatrix.from_float(w.reshape(-1, w.shape[-1]), f)
         for w, f in ((gate, "q4_0"), (up, "q4_0"), (down, "q8_0"))]
    b = qg.QuantizedExperts.from_matrices(*m, n_experts=E)
    assert torch.equal(a.gate_up, b.gate_up) and torch.equal(a.down, b.down)
    assert a.nbytes == E * K * F // 32 * (2 * 18 + 34)
    x = torch.randn(2, K, device=DEV, generator=g)
    ids = torch.tensor([[0, 2], [1, 2]], dtype=torch.int32, device=DEV)
    w = torch.rand(2, 2, device=DEV, generator=g)
    y = qg.moe_experts(x, ids, w, b)
    dq = [ref.dequant(f, mm.q.cpu().numpy().reshape(E, -1, mm.q.shape[1]), mm.d.cpu().numpy().reshape(E, -1, mm.d.shape[1]))
          for mm, f in zip(m, ("q4_0", "q4_0", "q8_0"))]
    want, tol = ref.experts(x.double().cpu().numpy(), ids.cpu().numpy(), w.cpu().numpy(), *dq)
    assert (np.abs(y.double().cpu().numpy() - want) <= tol).all()


def test_experts_from_a_gguf_file(tmp_path):
    from qgemv_roofline_b200 import gguf
    E, K, F = 3, 96, 64
    rng = np.random.default_rng(4)
    parts = {"gate": ("q4_0", planes("q4_0", E, F, K, rng)), "up": ("q4_0", planes("q4_0", E, F, K, rng)),
             "down": ("q8_0", planes("q8_0", E, K, F, rng))}
    tensors = {}
    for name, (fmt, (q, d)) in parts.items():
        rows = q.shape[1]
        b = qg.to_aos(fmt, torch.from_numpy(q.reshape(E * rows, -1)), torch.from_numpy(d.reshape(E * rows, -1)))
        tensors[f"blk.0.ffn_{name}_exps.weight"] = (fmt, b.numpy().reshape(E, rows, *b.shape[1:]))
    path = str(tmp_path / "experts.gguf")
    gguf.write_gguf(path, tensors)
    names = list(tensors)
    r = gguf.GGUFReader(path)
    assert r.tensors[names[0]].dims == (K, F, E) and r.tensors[names[2]].dims == (F, K, E)
    a = r.load_experts(*names)
    with pytest.raises(ValueError):
        r.load_experts(names[0], names[2], names[1])
    b = qg.QuantizedExperts(*[(gpu(q), gpu(d)) for _, (q, d) in parts.values()])
    assert torch.equal(a.gate_up, b.gate_up) and torch.equal(a.down, b.down)
    assert (a.n_experts, a.hidden, a.ffn, a.fmt, a.fmt_down) == (E, K, F, "q4_0", "q8_0")


def test_refusals():
    L = Layer(4, 64, 32, "q8_0", shared=1, seed=30)
    x, _ = L.x(2)
    r = torch.zeros(3, 64, device=DEV)
    ids, w = torch.zeros(2, 2, dtype=torch.int32, device=DEV), torch.zeros(2, 2, device=DEV)
    for bad in (x.cpu(), x[:, :32], x.double(), x.unsqueeze(0)):
        with pytest.raises((ValueError, TypeError)):
            qg.moe_layer(bad, r, L.experts, 2)
        with pytest.raises((ValueError, TypeError)):
            qg.moe_experts(bad, ids, w, L.experts)
    for k in (0, 4, -1):
        with pytest.raises(ValueError):
            qg.moe_layer(x, r, L.experts, k)
        with pytest.raises(ValueError):
            qg.moe_route(x, r, k)
    for bad in (torch.zeros(4, 64, device=DEV), torch.zeros(3, 32, device=DEV), r.double(), r.cpu(), r.t().contiguous().t()):
        with pytest.raises(ValueError):
            qg.moe_layer(x, bad, L.experts, 2)
    with pytest.raises(ValueError):
        qg.moe_layer(x, r, L.experts, 2, scoring="tanh")
    with pytest.raises(ValueError):
        qg.moe_layer(x, r, L.experts, 2, bias=torch.zeros(4, device=DEV))
    with pytest.raises(ValueError):
        qg.moe_layer(x, r, L.experts, 2, y=torch.empty(2, 64, dtype=torch.float16, device=DEV))
    for i, ww in ((ids.long(), w), (ids, w.double()), (ids[:1], w[:1]), (ids.t(), w.t()), (ids[:, :0], w[:, :0]),
                  (torch.zeros(2, 33, dtype=torch.int32, device=DEV), torch.zeros(2, 33, device=DEV))):
        with pytest.raises(ValueError):
            qg.moe_experts(x, i, ww, L.experts)
    q, d = torch.zeros(2, 64, 32, dtype=torch.int8, device=DEV), torch.zeros(2, 64, 1, dtype=torch.float16, device=DEV)
    dq, dd = torch.zeros(2, 32, 64, dtype=torch.int8, device=DEV), torch.zeros(2, 32, 2, dtype=torch.float16, device=DEV)
    qg.QuantizedExperts((q, d), (q, d), (dq, dd))
    for bad in (((q, d), (q[:1], d[:1]), (dq, dd)), ((q, d), (q, d), (q, d)), ((q, d.float()), (q, d), (dq, dd)),
                ((q[:, :40], d[:, :40]), (q[:, :40], d[:, :40]), (dq, dd)), ((q.float(), d), (q, d), (dq, dd))):
        with pytest.raises(ValueError):
            qg.QuantizedExperts(*bad)
    with pytest.raises(ValueError):
        qg.QuantizedExperts((q, d), (q, d), (dq, dd), n_shared=3)
