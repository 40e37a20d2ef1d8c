"""The mixture-of-experts and 8-bit operators, case by case: inputs, plain forms, values in 64 bits.

``listed()`` and ``draw()`` give cases, ``prepare()`` what a program holds before the call,
``run()`` one pass: the library's own kernels where ``own`` is true, otherwise the same
operator in elementary torch operations in 32 bits.  ``exact()`` gives the outputs from the
definitions in 64 bits, ``work()`` the bytes and operations that a pass cannot do without.

Operators (W is [M, K], X is [N, K], as everywhere in this library):

* ``route``: router logits (64-bit sums, rounded to fp32 once), the k best experts of each
  token (ties to the lowest index) and their weights;
* ``layer``: router, SwiGLU experts in q8_0 / q4_0 and their weighted sum, for a few tokens;
* ``experts``: the same experts with the choice and the weights given (-1 selects nothing);
* ``linear``: activations rounded to int8 with one scale a token, times int8 weights with one
  scale a channel;
* ``matmul``: the same product with the activations' int8 values and scales given.
"""

import torch

own = False  # set by whoever imports this: the library's kernels instead of the plain forms

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
BLOCK = {"q8_0": 34, "q4_0": 18}  # bytes of 32 weights


def _route(name, n, e, k, hidden, x, w, scoring, bias, scale, normalize):
    return {"name": name, "op": "route", "n": n, "experts": e, "k": k, "hidden": hidden, "x": x, "w": w,
            "scoring": scoring, "bias": bias, "scale": scale, "normalize": normalize}


def _moe(name, op, n, e, shared, k, hidden, ffn, fmt, down, x, scoring, normalize=True):
    return {"name": name, "op": op, "n": n, "experts": e, "shared": shared, "k": k, "hidden": hidden, "ffn": ffn,
            "fmt": fmt, "down": down, "x": x, "scoring": scoring, "normalize": normalize}


def _int8(name, op, n, m, k, x, y, bias):
    return {"name": name, "op": op, "n": n, "m": m, "kdim": k, "x": x, "y": y, "bias": bias}


def listed():
    return [
        # one token of a decode step chooses among many small experts: pure latency
        _route("route 1 of 128", 1, 128, 8, 2048, "bf16", "f32", "softmax", False, 1.0, True),
        # a prompt's tokens, sigmoid scores with a balancing bias and a scale
        _route("route 512 of 256", 512, 256, 8, 4096, "bf16", "bf16", "sigmoid", True, 2.5, True),
        # one token, many small experts in 4 bits: a decode step at batch 1
        _moe("layer 1x128 q4_0", "layer", 1, 128, 0, 8, 2048, 768, "q4_0", "q4_0", "bf16", "softmax"),
        # one token, few large experts (the library's 4096 / 11008 layer): bandwidth
        _moe("layer 1x8 q8_0", "layer", 1, 8, 0, 2, 4096, 11008, "q8_0", "q8_0", "f32", "softmax"),
        # a handful of tokens, ragged sizes, mixed formats, shared experts, weights not normalised
        _moe("layer 7x60 mixed", "layer", 7, 60, 2, 4, 1440, 1056, "q4_0", "q8_0", "f16", "softmax", False),
        # a small decode batch, sigmoid scores, shared experts
        _moe("layer 16x64 q8_0", "layer", 16, 64, 2, 6, 4096, 1408, "q8_0", "q8_0", "bf16", "sigmoid"),
        # the smallest call with the choice given by the caller's own router
        _moe("experts 1x32 q8_0", "experts", 1, 32, 0, 4, 2048, 1024, "q8_0", "q8_0", "f32", "given"),
        # a full decode batch, nearly every expert chosen, some choices dropped (-1)
        _moe("experts 64x128 q4_0", "experts", 64, 128, 0, 8, 2048, 768, "q4_0", "q4_0", "bf16", "given"),
        # one token through a wide projection: streams the weights
        _int8("linear 1", "linear", 1, 11008, 4096, "bf16", "bf16", False),
        # a prompt through gate and up in one matrix: bound by the tensor cores
        _int8("linear 4096", "linear", 4096, 22016, 4096, "bf16", "bf16", False),
        # a decode batch through the down projection, fp32 out
        _int8("matmul 16", "matmul", 16, 4096, 11008, "f32", "f32", False),
        # a ragged batch, odd row counts, with a bias
        _int8("matmul 1000 ragged", "matmul", 1000, 5003, 2064, "f32", "f16", True),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["route", "layer", "layer", "experts", "linear", "matmul"])
    x = rng.choice(["f32", "bf16", "f16"])
    if op == "route":
        e = _log(rng, 4, 320)
        c = _route("", _log(rng, 1, 512), e, rng.randint(1, min(e, 12)), 8 * _log(rng, 32, 640), x,
                   rng.choice(["f32", "bf16", "f16"]), rng.choice(["softmax", "sigmoid"]), rng.random() < 0.5,
                   rng.choice([1.0, 2.5]), rng.random() < 0.7)
    elif op in ("layer", "experts"):
        e = _log(rng, 4, 128)
        hidden, ffn = 32 * _log(rng, 8, 160), 32 * _log(rng, 4, 344)
        e = max(2, min(e, int(6e8 / (3 * hidden * ffn))))
        n = _log(rng, 1, 64)
        k = rng.randint(1, min(e, 8))
        n = max(1, min(n, int(2.4e9 / (3 * hidden * ffn * k))))
        c = _moe("", op, n, e, rng.choice([0, 0, 1, 2]) if op == "layer" else 0, k, hidden, ffn,
                 rng.choice(["q8_0", "q4_0"]), rng.choice(["q8_0", "q4_0"]), x,
                 rng.choice(["softmax", "sigmoid"]) if op == "layer" else "given", rng.random() < 0.7)
    else:
        n, m, k = _log(rng, 1, 4096), _log(rng, 16, 22016), 16 * _log(rng, 4, 688)
        n = max(1, min(n, int(3.6e11 / (m * k))))
        c = _int8("", op, n, m, k, x, x if op == "linear" else rng.choice(["f32", "bf16", "f16"]), rng.random() < 0.5)
    del c["name"]
    return c


# ------------------------------------------------------------------ inputs

def _quantize_blocks(fmt, w):
    """fp32 [rows, K] -> ggml planes (q, d): blocks of 32 weights, one fp16 scale each."""
    b = w.view(w.shape[0], -1, 32)
    if fmt == "q8_0":
        d = b.abs().amax(-1) / 127
        q = (b / d.unsqueeze(-1)).round_().clamp_(-127, 127).to(torch.int8)
        return q.view(w.shape), d.half()
    top = b.gather(-1, b.abs().argmax(-1, keepdim=True))
    d = top.squeeze(-1) / -8
    q = (b / d.unsqueeze(-1) + 8.5).floor_().clamp_(0, 15).to(torch.uint8)
    return (q[..., :16] | (q[..., 16:] << 4)).view(w.shape[0], -1), d.half()


def _planes(fmt, e, rows, cols, g):
    w = torch.randn(e * rows, cols, generator=g, device="cuda").mul_(cols ** -0.5)
    q, d = _quantize_blocks(fmt, w)
    return q.view(e, rows, -1), d.view(e, rows, -1)


def _activations(n, k, dtype, g):
    """Rows as a norm leaves them: unit variance, and a few channels that stand out."""
    x = torch.randn(n, k, generator=g, device="cuda")
    x[:, torch.randint(0, k, (max(1, k // 256),), generator=g, device="cuda")] *= 8
    return x.to(DTYPES[dtype])


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    c = dict(case)
    s = {"case": c}
    if c["op"] in ("linear", "matmul"):
        w = torch.randn(c["m"], c["kdim"], generator=g, device="cuda").mul_(c["kdim"] ** -0.5)
        top = w.abs().amax(-1)
        s["ws"] = top / 127
        s["wq"] = (w / s["ws"][:, None]).round_().clamp_(-127, 127).to(torch.int8)
        s["bias"] = torch.randn(c["m"], generator=g, device="cuda") if c["bias"] else None
        x = _activations(c["n"], c["kdim"], c["x"], g)
        if c["op"] == "linear":
            s["x"] = x
        else:
            x = x.float()
            s["xs"] = x.abs().amax(-1) / 127
            s["xq"] = (x / s["xs"][:, None]).round_().clamp_(-127, 127).to(torch.int8)
        return s
    s["x"] = _activations(c["n"], c["hidden"], c["x"], g)
    e = c["experts"]
    if c["op"] != "experts":
        w = torch.randn(e, c["hidden"], generator=g, device="cuda").mul_(2 * c["hidden"] ** -0.5)
        s["router"] = w.to(DTYPES[c.get("w", "f32")])
        s["bias"] = torch.rand(e, generator=g, device="cuda").mul_(0.2) if c.get("bias") else None
    if c["op"] == "route":
        return s
    total = e + c["shared"]
    s["gate"] = _planes(c["fmt"], total, c["ffn"], c["hidden"], g)
    s["up"] = _planes(c["fmt"], total, c["ffn"], c["hidden"], g)
    s["down"] = _planes(c["down"], total, c["hidden"], c["ffn"], g)
    if c["op"] == "experts":
        order = torch.rand(c["n"], e, generator=g, device="cuda").argsort(-1)[:, :c["k"]]
        kept = torch.rand(c["n"], c["k"], generator=g, device="cuda") >= 0.03
        kept[:, 0] |= c["n"] == 1
        s["ids"] = torch.where(kept, order, torch.full_like(order, -1)).to(torch.int32)
        s["weights"] = torch.rand(c["n"], c["k"], generator=g, device="cuda").mul_(0.4)
    if own:
        import qgemv_roofline_b200 as qg
        s["moe"] = qg.QuantizedExperts(s["gate"], s["up"], s["down"], n_shared=c["shared"])
    return s


# ------------------------------------------------------------- plain forms

def _plain_route(x, router, k, scoring, bias, scale, normalize):
    logits = (x.double() @ router.double().T).float()
    if scoring == "softmax":
        p = torch.exp(logits - logits.amax(-1, keepdim=True))
        far = torch.exp(logits.double() - logits.amax(-1, keepdim=True).double())
        rank = logits if bias is None else far / far.sum(-1, keepdim=True) + bias.double()
    else:
        p = 1 / (1 + torch.exp(-logits))
        rank = logits if bias is None else 1 / (1 + torch.exp(-logits.double())) + bias.double()
    ids = torch.sort(rank, dim=-1, descending=True, stable=True)[1][:, :k]
    chosen = p.gather(1, ids)
    over = chosen.sum(-1, keepdim=True) if normalize else p.sum(-1, keepdim=True) if scoring == "softmax" else 1.0
    return ids.to(torch.int32), chosen / over * scale


def _dequant(fmt, planes):
    q, d = planes
    if fmt == "q4_0":
        b = q.view(*q.shape[:-1], -1, 16)
        q = torch.cat([b & 15, b >> 4], -1).float() - 8
    else:
        q = q.view(*q.shape[:-1], -1, 32).float()
    return (q * d.float().unsqueeze(-1)).view(*q.shape[:-2], -1)


def _plain_experts(s, ids, weights):
    """Each token through its experts. Few choices: their weights are gathered; many: every
    expert takes every token, and the weights of those not chosen are zero."""
    c = s["case"]
    x, total = s["x"].float(), c["experts"] + c["shared"]
    n, slots = ids.shape
    ids = ids.long()
    weights = torch.where(ids >= 0, weights, torch.zeros_like(weights))
    at = ids.clamp(min=0)
    if n * slots < total:
        gate = _dequant(c["fmt"], tuple(p[at] for p in s["gate"]))
        up = _dequant(c["fmt"], tuple(p[at] for p in s["up"]))
        a, b = (torch.matmul(w, x[:, None, :, None]).squeeze(-1) for w in (gate, up))
        h = a / (1 + torch.exp(-a)) * b * weights.unsqueeze(-1)
        down = _dequant(c["down"], tuple(p[at] for p in s["down"]))
        y = torch.matmul(down, h.unsqueeze(-1)).squeeze(-1).sum(1)
    else:
        dense = torch.zeros(n, total, device=x.device).scatter_add_(1, at, weights)
        a = torch.matmul(_dequant(c["fmt"], s["gate"]), x.T)  # [experts, ffn, n]
        b = torch.matmul(_dequant(c["fmt"], s["up"]), x.T)
        h = a / (1 + torch.exp(-a)) * b * dense.T.unsqueeze(1)
        y = torch.matmul(_dequant(c["down"], s["down"]), h).sum(0).T.contiguous()
    return y.to(s["x"].dtype)


def _with_shared(c, ids, weights):
    n, shared = ids.shape[0], c["shared"]
    more = torch.arange(c["experts"], c["experts"] + shared, device=ids.device, dtype=ids.dtype).expand(n, shared)
    return torch.cat([ids, more], 1), torch.cat([weights, torch.ones(n, shared, device=ids.device)], 1)


def _plain_quantize(x):
    x = x.float()
    s = x.abs().amax(-1) / 127
    return torch.where(s[:, None] > 0, x / s[:, None], torch.zeros_like(x)).round().clamp(-127, 127), s


def run(s):
    c = s["case"]
    op = c["op"]
    if op == "route":
        if own:
            import qgemv_roofline_b200 as qg
            ids, weights = qg.moe_route(s["x"], s["router"], c["k"], scoring=c["scoring"], bias=s["bias"],
                                        scale=c["scale"], normalize=c["normalize"])
        else:
            ids, weights = _plain_route(s["x"], s["router"], c["k"], c["scoring"], s["bias"], c["scale"], c["normalize"])
        return {"ids": ids, "weights": weights}
    if op == "layer":
        if own:
            import qgemv_roofline_b200 as qg
            return qg.moe_layer(s["x"], s["router"], s["moe"], c["k"], scoring=c["scoring"], normalize=c["normalize"])
        routed = _plain_route(s["x"], s["router"], c["k"], c["scoring"], None, 1.0, c["normalize"])
        return _plain_experts(s, *_with_shared(c, *routed))
    if op == "experts":
        if own:
            import qgemv_roofline_b200 as qg
            return qg.moe_experts(s["x"], s["ids"], s["weights"], s["moe"])
        return _plain_experts(s, s["ids"], s["weights"])
    if own:
        import qgemv_roofline_b200 as qg
        if op == "linear":
            return qg.int8_linear(s["x"], s["wq"], s["ws"], s["bias"], out_dtype=DTYPES[c["y"]])
        return qg.int8_matmul(s["xq"], s["xs"], s["wq"], s["ws"], s["bias"], out_dtype=DTYPES[c["y"]])
    xq, xs = _plain_quantize(s["x"]) if op == "linear" else (s["xq"].float(), s["xs"])
    y = torch.matmul(xq, s["wq"].float().T) * xs[:, None] * s["ws"]
    return (y if s["bias"] is None else y + s["bias"]).to(DTYPES[c["y"]])


# ------------------------------------------------------ from the definitions

def _exact_route(x, router, k, scoring, bias, scale, normalize):
    logits = torch.stack([(x.double() * w.double()).sum(-1) for w in router], 1).float().double()
    z = torch.logsumexp(logits, -1, keepdim=True)
    score = torch.exp(logits - z) if scoring == "softmax" else torch.sigmoid(logits)
    rank = (logits if bias is None else score + bias.double()).cpu().tolist()
    ids = [sorted(range(len(r)), key=lambda j: (-r[j], j))[:k] for r in rank]
    ids = torch.tensor(ids, device=x.device)
    w = score.gather(1, ids)
    return ids, (w / w.sum(-1, keepdim=True) if normalize else w) * scale


def _exact_weights(fmt, planes, e):
    q, d = planes[0][e], planes[1][e].double()
    if fmt == "q8_0":
        q = q.double()
    else:
        low, high = (q % 16).double() - 8, (q // 16).double() - 8
        q = torch.stack([low.view(*d.shape, 16), high.view(*d.shape, 16)], 2).flatten(1)
    return q * d.repeat_interleave(32, -1)


def exact(case, seed):
    c = dict(case)
    s = prepare(case, seed)
    op = c["op"]
    if op in ("linear", "matmul"):
        if op == "linear":
            x = s["x"].double()
            xs = (x.abs().amax(-1) / 127).float().double()  # the scale is an fp32 number
            xq = torch.round((x / xs.clamp(min=1e-300)[:, None]).float().double()).clamp(-127, 127)
        else:
            xq, xs = s["xq"].double(), s["xs"].double()
        y = torch.einsum("nk,mk->nm", xq, s["wq"].double()) * (xs[:, None] * s["ws"].double()[None, :])
        return y if s["bias"] is None else y + s["bias"].double()
    if op == "experts":
        ids, weights = s["ids"].long(), s["weights"].double()
    else:
        ids, weights = _exact_route(s["x"], s["router"], c["k"], c["scoring"], s["bias"], c.get("scale", 1.0), c["normalize"])
    if op == "route":
        return {"ids": ids.to(torch.int32), "weights": weights}
    x = s["x"].double()
    y = torch.zeros_like(x)
    for e in range(c["experts"] + c["shared"]):
        per = (weights * (ids == e)).sum(-1) if e < c["experts"] else torch.ones_like(x[:, 0])
        used = ((ids == e).any(-1) if e < c["experts"] else per > 0).nonzero()[:, 0]
        if len(used):
            gate = x[used] @ _exact_weights(c["fmt"], s["gate"], e).T
            up = x[used] @ _exact_weights(c["fmt"], s["up"], e).T
            h = gate * torch.sigmoid(gate) * up
            y[used] += per[used, None] * (h @ _exact_weights(c["down"], s["down"], e).T)
    return y


def work(case):
    c = case
    n = c["n"]
    if c["op"] in ("linear", "matmul"):
        m, k = c["m"], c["kdim"]
        x = n * k * (SIZE[c["x"]] if c["op"] == "linear" else 1) + (0 if c["op"] == "linear" else 4 * n)
        return {"bytes": m * k + 4 * m + x + n * m * SIZE[c["y"]] + (4 * m if c["bias"] else 0), "flops": 2 * n * m * k}
    e, k, hidden = c["experts"], c["k"], c["hidden"]
    x = n * hidden * SIZE[c["x"]]
    router = e * hidden * SIZE[c.get("w", "f32")]
    if c["op"] == "route":
        return {"bytes": x + router + (4 * e if c["bias"] else 0) + 8 * n * k, "flops": 2 * n * e * hidden}
    # distinct experts that n tokens choose, on average, and the shared ones
    active = e * (1 - (1 - k / e) ** n) + c["shared"]
    w = c["ffn"] * hidden / 32
    b = active * w * (2 * BLOCK[c["fmt"]] + BLOCK[c["down"]]) + 2 * x
    f = 2 * n * (k + c["shared"]) * 3 * c["ffn"] * hidden
    if c["op"] == "layer":
        return {"bytes": b + router, "flops": f + 2 * n * e * hidden}
    return {"bytes": b + 8 * n * k, "flops": f}
