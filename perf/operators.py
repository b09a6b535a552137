"""Cases of the 8-bit inference operators and of the filtered token choice.

One pass of the reverse process (``model.generate`` / ``model.sample``) with 8-bit projections is, per layer: residual
addition + RMSNorm with 8-bit rows out, the q/k/v product, attention, 8-bit rows of its output, the output product,
again addition + norm, the gate/up product, 8-bit rows of a * silu(g), the down product; then the head and the choice
of one token per masked position.  The cases below are those operators at the sizes of this repository's
configurations (768 wide, 8 layers, 1024 hidden, 30522 tokens; ~1B: 2048 / 5632 / 32000; 8B: 4096 / 12288 / 126464).

8-bit rows: e4m3 values with one power-of-two scale for each 128 consecutive columns of a row; weights carry one scale
for each block of 128 x 128.  With a = max |y| over the block, the scale is 2^ceil(log2(a / 448)), at least 2^-126 (2^0
where a is 0), and the value held is y / scale rounded to e4m3.
"""

import math

import torch

own = False

BLOCK = 128

LISTED = [
    # one sequence of sample()'s default length: launch latency
    {"name": "norm_32x768", "op": "norm", "T": 32, "d": 768, "stream": "bf16", "residual": True},
    # 8B width, 16k tokens, the fp32 residual stream with bf16 branches: bandwidth
    {"name": "norm_16384x4096_f32", "op": "norm", "T": 16384, "d": 4096, "stream": "f32", "residual": True},
    # a batch of 32 ragged prompts of the default model
    {"name": "norm_15001x768", "op": "norm", "T": 15001, "d": 768, "stream": "bf16", "residual": True},
    # attention output of a batch of the default model
    {"name": "quant_2048x768", "op": "quant", "T": 2048, "d": 768, "swiglu": False},
    # SwiGLU hidden of the ~1B shape, odd number of rows
    {"name": "swiglu_8191x5632", "op": "quant", "T": 8191, "d": 5632, "swiglu": True},
    # q/k/v projection for one sequence of 32: weights from memory, latency
    {"name": "linear_32x2304x768", "op": "linear", "M": 32, "N": 2304, "K": 768, "out": "bf16"},
    # q/k/v projection for 2048 tokens of the default model
    {"name": "linear_2048x2304x768", "op": "linear", "M": 2048, "N": 2304, "K": 768, "out": "bf16"},
    # vocabulary projection of the masked rows of a batch, fp32 logits, ragged in every direction
    {"name": "linear_777x30522x768_f32", "op": "linear", "M": 777, "N": 30522, "K": 768, "out": "f32"},
    # gate/up projection of the ~1B shape at 16k tokens: matrix rate
    {"name": "linear_16384x11264x2048", "op": "linear", "M": 16384, "N": 11264, "K": 2048, "out": "bf16"},
    # one step of sample() at its defaults: every position of one sequence, nucleus choice
    {"name": "sample_32x30522", "op": "sample", "T": 32, "V": 30522, "dtype": "bf16", "temperature": 1.0,
     "top_k": 0, "top_p": 0.9, "min_p": 0.0, "ids": True},
    # a batch early in the reverse process (flat rows), all filters
    {"name": "sample_4096x30522", "op": "sample", "T": 4096, "V": 30522, "dtype": "bf16", "temperature": 0.8,
     "top_k": 200, "top_p": 0.95, "min_p": 0.02, "ids": True},
    # the 8B vocabulary with fp32 logits
    {"name": "sample_1000x126464_f32", "op": "sample", "T": 1000, "V": 126464, "dtype": "f32", "temperature": 1.0,
     "top_k": 0, "top_p": 0.95, "min_p": 0.0, "ids": False},
]


def listed():
    return [dict(c) for c in LISTED]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "quant", "linear", "sample"])
    if op == "norm":
        return {"op": op, "T": _log(rng, 1, 16384), "d": _log(rng, 24, 4096), "stream": rng.choice(["bf16", "f32"]),
                "residual": rng.random() < 0.8}
    if op == "quant":
        return {"op": op, "T": _log(rng, 1, 8191), "d": _log(rng, 24, 5632), "swiglu": rng.random() < 0.6}
    if op == "linear":
        m, n, k = _log(rng, 1, 16384), _log(rng, 16, 11264), _log(rng, 32, 2048)
        return {"op": op, "M": m, "N": n, "K": k, "out": rng.choice(["bf16", "bf16", "f32"])}
    t = _log(rng, 1, 4096)
    v = _log(rng, 2, min(126464, (4096 * 30522) // t))
    return {"op": op, "T": t, "V": v, "dtype": rng.choice(["bf16", "f32"]),
            "temperature": round(rng.uniform(0.3, 1.5), 3), "top_k": rng.choice([0, 0, _log(rng, 1, 1000)]),
            "top_p": rng.choice([1.0, round(rng.uniform(0.3, 0.99), 3)]),
            "min_p": rng.choice([0.0, 0.0, round(rng.uniform(0.001, 0.2), 4)]), "ids": rng.random() < 0.5}


def work(case):
    op = case["op"]
    if op == "norm":
        n = case["T"] * case["d"]
        s = 4 if case["stream"] == "f32" else 2
        per = (2 + s + s + 1) if case["residual"] else (s + 1)
        return {"bytes": n * per + case["T"] * -(-case["d"] // BLOCK) + 4 * case["d"], "flops": 6 * n}
    if op == "quant":
        n = case["T"] * case["d"]
        return {"bytes": n * (5 if case["swiglu"] else 3) + case["T"] * -(-case["d"] // BLOCK),
                "flops": n * (8 if case["swiglu"] else 2)}
    if op == "linear":
        m, n, k = case["M"], case["N"], case["K"]
        return {"bytes": m * k + n * k + m * n * (4 if case["out"] == "f32" else 2) + 4 * n, "flops": 2 * m * n * k}
    # with ids about half of the positions are masked, and only their rows are wanted
    rows = case["T"] * (0.5 if case["ids"] else 1.0)
    return {"bytes": rows * case["V"] * (4 if case["dtype"] == "f32" else 2) + 20 * case["T"],
            "flops": 4 * rows * case["V"]}


# ------------------------------------------------------------------ inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _aligned(t, multiple):
    """The same matrix with a row stride that is a multiple of ``multiple`` elements, as the framework allocates it."""
    rows, cols = t.shape
    buf = torch.zeros(rows, -(-cols // multiple) * multiple, dtype=torch.uint8, device=t.device).view(t.dtype) \
        if t.element_size() == 1 else torch.zeros(rows, -(-cols // multiple) * multiple, dtype=t.dtype, device=t.device)
    out = buf[:, :cols]
    out.copy_(t)
    return out


def prepare(case, seed):
    g = _generator(seed)
    op = case["op"]
    if op == "norm":
        T, d = case["T"], case["d"]
        # the residual stream of a trained model: a few wide channels, rows of different size
        channels = torch.exp(0.5 * _randn(g, d))
        stream = 2.0 * _randn(g, T, d) * channels
        dt = torch.float32 if case["stream"] == "f32" else torch.bfloat16
        s = {"case": dict(case), "weight": 1.0 + 0.1 * _randn(g, d), "eps": 1e-12}
        if case["residual"]:
            s["x"] = (0.3 * _randn(g, T, d)).to(torch.bfloat16)
            s["residual"] = stream.to(dt)
        else:
            s["x"], s["residual"] = stream.to(dt), None
        return s
    if op == "quant":
        T, d = case["T"], case["d"]
        x = _randn(g, T, 2 * d if case["swiglu"] else d) * torch.exp(0.4 * _randn(g, T, 1))
        return {"case": dict(case), "x": x.to(torch.bfloat16)}
    if op == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        xq, xs = _rows8(_randn(g, M, K) * torch.exp(0.3 * _randn(g, K)))
        bound = math.sqrt(6.0 / (N + K))
        w = (torch.rand(N, K, generator=g, device="cuda") * 2 - 1) * bound
        nb, kb = -(-N // BLOCK), -(-K // BLOCK)
        wp = torch.nn.functional.pad(w, (0, kb * BLOCK - K, 0, nb * BLOCK - N))
        e = _exponent(wp.view(nb, BLOCK, kb, BLOCK).abs().amax(dim=(1, 3)))
        full = _power(e).repeat_interleave(BLOCK, 0).repeat_interleave(BLOCK, 1)[:N, :K]
        wq = (w / full).to(torch.float8_e4m3fn)
        return {"case": dict(case), "xq": _aligned(xq, 16), "xs": xs, "wq": _aligned(wq, 16), "ws": _code(e),
                "bias": 0.1 * _randn(g, N)}
    T, V = case["T"], case["V"]
    # rows between nearly flat (early steps) and peaked (late steps), stored with the head's padded row stride
    sharp = 0.7 + 2.5 * torch.rand(T, 1, generator=g, device="cuda")
    logits = _randn(g, T, V) * sharp
    hot = torch.randint(0, V, (T, 8), generator=g, device="cuda")
    logits.scatter_add_(1, hot, 10.0 * torch.rand(T, 8, generator=g, device="cuda"))
    logits = _aligned(logits.to(torch.float32 if case["dtype"] == "f32" else torch.bfloat16), 256)
    s = {"case": dict(case), "logits": logits, "u": torch.rand(T, generator=g, device="cuda"), "ids": None}
    s["mask_id"] = 103 if V > 103 else 0
    if case["ids"]:
        ids = torch.randint(0, V, (T,), generator=g, device="cuda")
        masked = torch.rand(T, generator=g, device="cuda") < 0.5
        s["ids"] = torch.where(masked, torch.full_like(ids, s["mask_id"]), ids)
    return s


# ------------------------------------------------------------------ plain forms
def _exponent(amax):
    """ceil(log2(amax / 448)), at least -126, and 0 for 0: with amax = m 2^e, 0.5 <= m < 1, it is e - 9 up to m = 7/8."""
    m, e = torch.frexp(amax)
    e = torch.clamp(e - 9 + (m > 0.875).to(e.dtype), min=-126)
    return torch.where(amax > 0, e, torch.zeros_like(e))


def _power(e):
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _code(e):
    return (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _rows8(y):
    rows, cols = y.shape
    nb = -(-cols // BLOCK)
    yb = torch.nn.functional.pad(y, (0, nb * BLOCK - cols)).view(rows, nb, BLOCK)
    e = _exponent(yb.abs().amax(-1))
    q = (yb / _power(e).unsqueeze(-1)).to(torch.float8_e4m3fn)
    return q.view(rows, nb * BLOCK)[:, :cols], _code(e)


def _plain_norm(s):
    h = s["x"].float() if s["residual"] is None else s["x"].float() + s["residual"].float()
    y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + s["eps"]) * s["weight"]
    q, scale = _rows8(y)
    return {"q": q, "scale": scale, "stream": s["x"] if s["residual"] is None else h.to(s["residual"].dtype)}


def _plain_quant(s):
    x = s["x"].float()
    if s["case"]["swiglu"]:
        a, g = x.chunk(2, dim=-1)
        x = a * g / (1.0 + torch.exp(-g))
    q, scale = _rows8(x)
    return {"q": q, "scale": scale}


def _widen(q, scale, rows):
    n, k = q.shape
    f = scale.to(torch.float32).repeat_interleave(rows, 0)[:n] if rows > 1 else scale.to(torch.float32)
    return q.to(torch.float32) * f.repeat_interleave(BLOCK, 1)[:, :k]


def _plain_linear(s):
    y = torch.matmul(_widen(s["xq"], s["xs"], 1), _widen(s["wq"], s["ws"], BLOCK).t()) + s["bias"]
    return y if s["case"]["out"] == "f32" else y.to(torch.bfloat16)


def _plain_sample(s):
    c = s["case"]
    z = s["logits"].double()
    rows, V = z.shape
    z, order = torch.sort(z, dim=-1, descending=True, stable=True)
    w = torch.exp((z - z[:, :1]) / c["temperature"])
    keep = torch.ones_like(w, dtype=torch.bool)
    if 0 < c["top_k"] < V:
        keep[:, c["top_k"]:] = False
    if c["top_p"] < 1.0:
        cum = torch.cumsum(torch.where(keep, w, 0.0), -1)
        keep[:, 1:] &= cum[:, :-1] < c["top_p"] * cum[:, -1:]
    if c["min_p"] > 0.0:
        keep &= w >= c["min_p"]
    by_index = torch.zeros_like(w).scatter_(1, order, torch.where(keep, w, 0.0))
    cum = torch.cumsum(by_index, -1)
    token = (cum <= s["u"].double().unsqueeze(1) * cum[:, -1:]).sum(-1).clamp(max=V - 1)
    return token if s["ids"] is None else torch.where(s["ids"] == s["mask_id"], token, s["ids"])


PLAIN = {"norm": _plain_norm, "quant": _plain_quant, "linear": _plain_linear, "sample": _plain_sample}


# ------------------------------------------------------------------ the framework's operators
def _own(s):
    from src import ops
    c = s["case"]
    if c["op"] == "norm":
        q, scale, stream = ops.rms_norm_fp8(s["x"], s["weight"], s["eps"], residual=s["residual"])
        return {"q": q, "scale": scale, "stream": stream}
    if c["op"] == "quant":
        q, scale = ops.quantize_fp8(s["x"], "swiglu" if c["swiglu"] else None)
        return {"q": q, "scale": scale}
    if c["op"] == "linear":
        return ops.fp8_matmul(s["xq"], s["xs"], s["wq"], s["ws"], bias=s["bias"],
                              out_dtype=torch.float32 if c["out"] == "f32" else torch.bfloat16)
    return ops.sample_tokens(s["logits"], s["u"], temperature=c["temperature"], top_k=c["top_k"], top_p=c["top_p"],
                             min_p=c["min_p"], ids=s["ids"], mask_token_id=s["mask_id"])


def run(state):
    return _own(state) if own else PLAIN[state["case"]["op"]](state)


# ------------------------------------------------------------------ definitions in 64 bits
def _exact_rows8(y):
    """(y / scale without the rounding to 8 bits, scale) of rows of float64."""
    rows, cols = y.shape
    nb = -(-cols // BLOCK)
    yb = torch.cat([y, y.new_zeros(rows, nb * BLOCK - cols)], 1).reshape(rows, nb, BLOCK)
    a = yb.abs().max(dim=-1).values
    e = torch.ceil(torch.log2(torch.where(a > 0, a, torch.full_like(a, 448.0)) / 448.0)).clamp(min=-126.0)
    scale = torch.pow(torch.full_like(e, 2.0), e)
    return (yb / scale.unsqueeze(-1)).reshape(rows, nb * BLOCK)[:, :cols], scale


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        h = s["x"].double()
        if s["residual"] is not None:
            h = h + s["residual"].double()
        y = s["weight"].double() * h / torch.sqrt((h * h).sum(-1, keepdim=True) / case["d"] + s["eps"])
        q, scale = _exact_rows8(y)
        return {"q": q, "scale": scale, "stream": h}
    if case["op"] == "quant":
        x = s["x"].double()
        if case["swiglu"]:
            x = x[:, :case["d"]] * x[:, case["d"]:] * torch.sigmoid(x[:, case["d"]:])
        q, scale = _exact_rows8(x)
        return {"q": q, "scale": scale}
    if case["op"] == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        row = torch.arange(N, device="cuda") // BLOCK
        col = torch.arange(K, device="cuda") // BLOCK
        a = s["xq"].double() * s["xs"].double()[:, col]
        b = s["wq"].double() * s["ws"].double()[row][:, col]
        return torch.addmm(s["bias"].double(), a, b.t().contiguous())
    return _exact_sample(s)


def _exact_sample(s):
    """The choice from its definition: ranks, the mass in front of each rank, then the distribution function."""
    c = s["case"]
    z = s["logits"].double()
    rows, V = z.shape
    rank_to_index = torch.argsort(-z, dim=-1, stable=True)
    rank = torch.empty_like(rank_to_index)
    rank.scatter_(1, rank_to_index, torch.arange(V, device=z.device).expand(rows, V))
    k = c["top_k"] if 0 < c["top_k"] < V else V
    p = torch.exp((z - z.max(-1, keepdim=True).values) / c["temperature"])
    p = torch.where(rank < k, p, torch.zeros_like(p))
    total = p.sum(-1, keepdim=True)
    ranked = p.gather(1, rank_to_index)
    before = (ranked.cumsum(-1) - ranked).gather(1, rank)
    kept = rank < k
    if c["top_p"] < 1.0:
        kept &= (rank == 0) | (before < c["top_p"] * total)
    if c["min_p"] > 0.0:
        kept &= p >= c["min_p"]
    p = torch.where(kept, p, torch.zeros_like(p))
    cdf = p.cumsum(-1)
    target = s["u"].double().unsqueeze(1) * cdf[:, -1:]
    token = torch.searchsorted(cdf, target, right=True).squeeze(1).clamp(max=V - 1)
    return token if s["ids"] is None else torch.where(s["ids"] == s["mask_id"], token, s["ids"])
