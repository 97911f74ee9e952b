"""The operators of a long-document encoder in 8 bits, as cases to be timed and compared.

Five kinds:

  quantize   a half-precision activation to e4m3 with one fp32 scale per row and block of 128 columns (`ops.quantize_fp8`)
  norm       residual + LayerNorm, the result in half precision and in e4m3 with its scales (`ops.add_layernorm_fp8`)
  linear     matrix product of e4m3 operands with a scale per block of 128, bias and optional residual (`ops.linear_fp8`)
  ffn        the feed-forward half of a layer as a program runs it: quantize, up-projection with GELU whose result stays in
             8 bits, down-projection with residual
  attention  sliding-window attention with first tokens that stay visible (`ops.window_attention`): whole documents, or a few
             query tokens against the keys and values kept so far

`own = False` computes them in plain torch operations in 32 bits, `own = True` through the framework's operators.
Block scales: x `[ceil(K / 128), rows]`, w `[ceil(N / 128), ceil(K / 128)]`, both fp32; a value stands for code * scale.
"""
import math

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
BLOCK = 128            # columns per scale
E4M3_MAX = 448.0
MIN_AMAX = 2.0 ** -40  # a block whose largest magnitude is below this is scaled as if it were this
EPS = 1e-12
D = 64                 # head dimension of every geometry here


def listed():
    return [
        # one token's hidden state on its way into an 8-bit projection: latency is everything
        {"name": "quantize_1x768_f16", "kind": "quantize", "M": 1, "K": 768, "dtype": "f16"},
        # the attention output of a batch of long documents, in front of the output projection
        {"name": "quantize_65536x1024_bf16", "kind": "quantize", "M": 65536, "K": 1024, "dtype": "bf16"},
        # the LayerNorm between two 8-bit projections: a short odd request, and a batch of documents
        {"name": "norm_333x1024_bf16", "kind": "norm", "M": 333, "K": 1024, "dtype": "bf16", "residual": False},
        {"name": "norm_32768x768_f16_res", "kind": "norm", "M": 32768, "K": 768, "dtype": "f16", "residual": True},
        # the QKV projection of a single token
        {"name": "linear_1x768x2304_f16", "kind": "linear", "M": 1, "K": 768, "N": 2304, "out": "f16", "residual": False},
        # an output projection for a few hundred tokens of ragged requests
        {"name": "linear_777x1024x1024_bf16_res", "kind": "linear", "M": 777, "K": 1024, "N": 1024, "out": "bf16", "residual": True},
        # a throughput batch through a wide projection, fp32 result at the graph's edge
        {"name": "linear_16384x1024x4096_f32", "kind": "linear", "M": 16384, "K": 1024, "N": 4096, "out": "f32", "residual": False},
        # the feed-forward half of a layer of the large geometry for a batch of long documents
        {"name": "ffn_32768x1024x4096_f16", "kind": "ffn", "M": 32768, "K": 1024, "N": 4096, "dtype": "f16"},
        # documents of up to 4096 tokens, ragged, a window of 256 to either side, the first token seen by all
        {"name": "attn_4x4096_w256_ragged_f16", "kind": "attention", "B": 4, "Sq": 4096, "Sk": 4096, "heads": 12, "kv_heads": 12,
         "left": 256, "right": 256, "sinks": 1, "lo": 1000, "dtype": "f16"},
        # one long text read left to right, grouped key / value heads, the first four tokens kept
        {"name": "attn_1x16384_causal1024_gqa_bf16", "kind": "attention", "B": 1, "Sq": 16384, "Sk": 16384, "heads": 16, "kv_heads": 4,
         "left": 1023, "right": 0, "sinks": 4, "lo": 16384, "dtype": "bf16"},
        # one new token against a short cache: the smallest call
        {"name": "attn_token_1x1000_w256_f16", "kind": "attention", "B": 1, "Sq": 1, "Sk": 1000, "heads": 12, "kv_heads": 12,
         "left": 255, "right": 0, "sinks": 4, "lo": 1000, "dtype": "f16"},
        # one new token for each of 32 requests against long ragged caches, a wide window
        {"name": "attn_token_32x16384_w8192_gqa_bf16", "kind": "attention", "B": 32, "Sq": 1, "Sk": 16384, "heads": 16, "kv_heads": 4,
         "left": 8191, "right": 0, "sinks": 16, "lo": 2000, "dtype": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case: kinds in turn of chance, sizes spread over the logarithm of their ranges, odd ones among them."""
    kind = rng.choice(["quantize", "norm", "linear", "linear", "ffn", "attention", "attention", "token"])
    half = rng.choice(["f16", "bf16"])
    if kind in ("quantize", "norm"):
        K = 16 * _log_int(rng, 4, 256)
        M = _log_int(rng, 1, max(1, min(131072, 65536 * 1024 // K)))
        c = {"kind": kind, "M": M, "K": K, "dtype": rng.choice([half, half, "f32"]) if kind == "quantize" else half}
        if kind == "norm":
            c["residual"] = rng.random() < 0.5
        return c
    if kind in ("linear", "ffn"):
        K = 16 * _log_int(rng, 4, 256)
        N = 16 * _log_int(rng, 4, 256)
        if rng.random() < 0.5:          # widths of whole blocks, as most models have them
            K, N = -(-K // 128) * 128, -(-N // 128) * 128
        M = _log_int(rng, 1, max(1, min(65536, (1 << 36) // (K * N))))
        if kind == "ffn":
            return {"kind": kind, "M": M, "K": K, "N": N, "dtype": half}
        return {"kind": kind, "M": M, "K": K, "N": N, "out": rng.choice([half, half, "f32"]), "residual": rng.random() < 0.5}
    heads, kv_heads = rng.choice([(12, 12), (16, 16), (16, 4), (12, 1), (16, 2)])
    sinks = rng.choice([0, 1, 4, 16, 64])
    if kind == "token":
        Sq = rng.choice([1, 1, 1, 1, 2, 5])
        Sk = _log_int(rng, 16, 32768)
        B = _log_int(rng, 1, max(1, min(64, (1 << 19) // Sk)))
        left = min(Sk, _log_int(rng, 1, 16384)) if rng.random() < 0.8 else -1
        right = 0
    else:
        Sq = Sk = _log_int(rng, 8, 8192)
        B = _log_int(rng, 1, max(1, min(64, (1 << 25) // (Sk * Sk))))
        left = _log_int(rng, 1, 2048)
        right = rng.choice([0, left, left, _log_int(rng, 1, 512)])
    lo = max(Sq if kind == "token" else 1, int(Sk * rng.uniform(0.1, 0.9))) if rng.random() < 0.5 else Sk
    return {"kind": "attention", "B": B, "Sq": Sq, "Sk": Sk, "heads": heads, "kv_heads": kv_heads, "left": left, "right": right,
            "sinks": sinks, "lo": lo, "dtype": half}


# ---------------------------------------------------------------------------------------------------- preparation
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _activation(g, M, K, dtype):
    """Rows of a hidden state: a few channels are several times as large as the rest, as they are in trained models."""
    channel = torch.exp(0.7 * torch.randn(K, device="cuda", generator=g))
    return (torch.randn((M, K), device="cuda", generator=g) * channel).to(dtype)


def _block_amax(x):
    """Largest magnitude of every row's blocks of 128 columns, `[rows, ceil(K / 128)]`."""
    pad = -x.shape[1] % BLOCK
    return torch.nn.functional.pad(x.abs(), (0, pad)).reshape(x.shape[0], -1, BLOCK).amax(-1)


def _spread(scale, K):
    """A `[rows, blocks]` array repeated over its blocks' columns, `[rows, K]`."""
    return scale.repeat_interleave(BLOCK, 1)[:, :K]


def _quantize(x):
    """fp32 `[rows, K]` -> (e4m3 codes, scales `[ceil(K / 128), rows]`)."""
    amax = _block_amax(x).clamp_min(MIN_AMAX)
    top = torch.full_like(amax, E4M3_MAX)      # tensor by tensor: a quotient with a Python number is a product with a reciprocal
    q = (x * _spread(top / amax, x.shape[1])).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    return q, (amax / top).t().contiguous()


def _weight(g, N, K):
    """An e4m3 weight `[N, K]` with a scale per 128 x 128 block."""
    w = torch.randn((N, K), device="cuda", generator=g) * 0.03
    nb, kb = -(-N // BLOCK), -(-K // BLOCK)
    full = torch.nn.functional.pad(w, (0, kb * BLOCK - K, 0, nb * BLOCK - N)).reshape(nb, BLOCK, kb, BLOCK)
    amax = full.abs().amax((1, 3)).clamp_min(MIN_AMAX)
    q = (full * (E4M3_MAX / amax)[:, None, :, None]).clamp(-E4M3_MAX, E4M3_MAX).reshape(nb * BLOCK, kb * BLOCK)[:N, :K]
    return q.to(torch.float8_e4m3fn).contiguous(), (amax / E4M3_MAX).contiguous()


def prepare(case, seed):
    g = _generator(seed)
    st = dict(case)
    kind = case["kind"]

    def normal(*shape):
        return torch.randn(shape, device="cuda", generator=g)

    if kind == "attention":
        dt, B, Sq, Sk = DTYPES[case["dtype"]], case["B"], case["Sq"], case["Sk"]
        H, Hkv = case["heads"] * D, case["kv_heads"] * D
        lengths = torch.randint(case["lo"], Sk + 1, (B,), device="cuda", generator=g, dtype=torch.int32)
        if Sq == Sk:                                   # a packed projection: Q | K | V side by side
            qkv = normal(B, Sq, H + 2 * Hkv).to(dt)
            st["q"], st["k"], st["v"] = qkv[..., :H], qkv[..., H:H + Hkv], qkv[..., H + Hkv:]
            st["q_start"] = None
        else:                                          # new tokens at the end of what the cache holds
            st["q"] = normal(B, Sq, H).to(dt)
            st["k"], st["v"] = normal(B, Sk, Hkv).to(dt), normal(B, Sk, Hkv).to(dt)
            st["q_start"] = lengths - Sq
        st["kv_len"] = lengths
        return st
    M, K = case["M"], case["K"]
    if kind in ("quantize", "norm", "ffn"):
        st["x"] = _activation(g, M, K, DTYPES[case["dtype"]])
    if kind == "norm":
        st["r"] = normal(M, K).to(DTYPES[case["dtype"]]) if case["residual"] else None
        st["gamma"], st["beta"] = 1.0 + 0.1 * normal(K), 0.1 * normal(K)
    if kind == "linear":
        N = case["N"]
        st["x8"], st["xs"] = _quantize(_activation(g, M, K, torch.float32))
        st["w8"], st["ws"] = _weight(g, N, K)
        st["bias"] = 0.1 * normal(N)
        out = DTYPES[case["out"]]
        st["r"] = normal(M, N).to(torch.float16 if out == torch.float32 else out) if case["residual"] else None
        st["out_dtype"] = out
    if kind == "ffn":
        N = case["N"]
        st["w1"], st["ws1"] = _weight(g, N, K)
        st["w2"], st["ws2"] = _weight(g, K, N)
        st["b1"], st["b2"] = 0.1 * normal(N), 0.1 * normal(K)
    return st


# ---------------------------------------------------------------------------------------------------- one pass
def _plain_linear(x8, xs, w8, ws, bias):
    x = x8.float() * _spread(xs.t(), x8.shape[1])
    w = w8.float() * _spread(ws, w8.shape[1]).repeat_interleave(BLOCK, 0)[:w8.shape[0]]
    return x @ w.t() + bias


def _plain_norm(x, gamma, beta):
    d = x - x.mean(-1, keepdim=True)
    return d * torch.rsqrt((d * d).mean(-1, keepdim=True) + EPS) * gamma + beta


def _visible(case, lengths, q_start):
    """`[B, Sq, Sk]`: which keys a query sees."""
    j = torch.arange(case["Sk"], device="cuda")
    pos = torch.arange(case["Sq"], device="cuda")[None, :] + (0 if q_start is None else q_start[:, None])
    seen = torch.ones((), dtype=torch.bool, device="cuda")
    if case["left"] >= 0:
        seen = seen & (j >= pos[..., None] - case["left"])
    if case["right"] >= 0:
        seen = seen & (j <= pos[..., None] + case["right"])
    return ((j < case["sinks"]) | seen) & (j < lengths[:, None, None])


def _plain_attention(st):
    B, Sq, Sk, heads, kv_heads = (st[n] for n in ("B", "Sq", "Sk", "heads", "kv_heads"))
    q = st["q"].float().reshape(B, Sq, kv_heads, heads // kv_heads, D).permute(0, 2, 3, 1, 4)
    k = st["k"].float().reshape(B, Sk, kv_heads, 1, D).permute(0, 2, 3, 1, 4)
    v = st["v"].float().reshape(B, Sk, kv_heads, 1, D).permute(0, 2, 3, 1, 4)
    hidden = ~_visible(st, st["kv_len"], st["q_start"])[:, None, None]
    s = (q @ k.transpose(-1, -2)).mul_(D ** -0.5).masked_fill_(hidden, -math.inf)
    s.sub_(s.amax(-1, keepdim=True).clamp_min(-1e30)).exp_()
    o = (s @ v) / s.sum(-1, keepdim=True).clamp_min(1e-30)
    return o.permute(0, 3, 1, 2, 4).reshape(B, Sq, heads * D).to(st["q"].dtype)


def run(st):
    kind = st["kind"]
    if own:
        from tnn_b200 import ops
        if kind == "quantize":
            q, s = ops.quantize_fp8(st["x"])
            return {"q": q, "scale": s}
        if kind == "norm":
            y, q, s = ops.add_layernorm_fp8(st["x"], st["gamma"], st["beta"], EPS, residual=st["r"])
            return {"y": y, "q": q, "scale": s}
        if kind == "linear":
            epi = ops.EPI_BIAS if st["r"] is None else ops.EPI_BIAS_RESIDUAL
            return ops.linear_fp8(st["x8"], st["xs"], st["w8"], st["ws"], st["bias"], residual=st["r"], epilogue=epi,
                                  out_dtype=st["out_dtype"])
        if kind == "ffn":
            q, s = ops.quantize_fp8(st["x"])
            q, s = ops.linear_fp8(q, s, st["w1"], st["ws1"], st["b1"], epilogue=ops.EPI_BIAS_GELU,
                                  out_dtype=torch.float8_e4m3fn)
            return ops.linear_fp8(q, s, st["w2"], st["ws2"], st["b2"], residual=st["x"], epilogue=ops.EPI_BIAS_RESIDUAL,
                                  out_dtype=st["x"].dtype)
        return ops.window_attention(st["q"], st["k"], st["v"], st["heads"], st["kv_heads"], window=(st["left"], st["right"]),
                                    sinks=st["sinks"], kv_len=st["kv_len"], q_start=st["q_start"])
    if kind == "quantize":
        q, s = _quantize(st["x"].float())
        return {"q": q, "scale": s}
    if kind == "norm":
        x = st["x"].float() if st["r"] is None else st["x"].float() + st["r"].float()
        y = _plain_norm(x, st["gamma"], st["beta"])
        q, s = _quantize(y)
        return {"y": y.to(st["x"].dtype), "q": q, "scale": s}
    if kind == "linear":
        y = _plain_linear(st["x8"], st["xs"], st["w8"], st["ws"], st["bias"])
        return (y if st["r"] is None else y + st["r"].float()).to(st["out_dtype"])
    if kind == "ffn":
        x = st["x"].float()
        q, s = _quantize(x)
        h = _plain_linear(q, s, st["w1"], st["ws1"], st["b1"])
        q, s = _quantize(0.5 * h * (1.0 + torch.erf(h * math.sqrt(0.5))))
        return (_plain_linear(q, s, st["w2"], st["ws2"], st["b2"]) + x).to(st["x"].dtype)
    return _plain_attention(st)


# ---------------------------------------------------------------------------------------------------- work
def _pairs(case, length):
    """(query, key) pairs of a sequence of `length` keys that see each other, over one head."""
    sinks, left, right = case["sinks"], case["left"], case["right"]
    first = 0 if case["Sq"] == case["Sk"] else length - case["Sq"]
    n = 0
    for i in range(case["Sq"]):
        pos = first + i
        lo = 0 if left < 0 else max(0, pos - left)
        hi = length if right < 0 else min(length, pos + right + 1)
        n += max(0, hi - lo) + max(0, min(sinks, length, lo if hi > lo else length))
    return n


def work(case):
    """Each input read once, each output written once; of a long cache only the keys and values that are visible."""
    kind = case["kind"]
    if kind == "attention":
        B, Sq, Sk = case["B"], case["Sq"], case["Sk"]
        length = (case["lo"] + Sk) // 2                    # the mean: lengths are uniform in [lo, Sk]
        pairs = B * _pairs(case, length)
        keys = length
        if Sq != Sk and case["left"] >= 0:
            keys = min(length, case["left"] + Sq + case["sinks"])
        n_bytes = 2 * B * (2 * Sq * case["heads"] * D + 2 * keys * case["kv_heads"] * D)
        return {"bytes": n_bytes, "flops": 4 * D * case["heads"] * pairs}
    M, K = case["M"], case["K"]
    size = {"f16": 2, "bf16": 2, "f32": 4}
    blocks = -(-K // BLOCK)
    if kind == "quantize":
        return {"bytes": M * K * (size[case["dtype"]] + 1) + 4 * M * blocks, "flops": 3 * M * K}
    if kind == "norm":
        per = 2 * (3 if case["residual"] else 2) + 1
        return {"bytes": M * K * per + 4 * M * blocks + 8 * K, "flops": 12 * M * K}
    N = case["N"]
    if kind == "linear":
        n_bytes = M * K + N * K + 4 * blocks * (M + -(-N // BLOCK)) + 4 * N + M * N * size[case["out"]]
        return {"bytes": n_bytes + (2 * M * N if case["residual"] else 0), "flops": 2 * M * N * K}
    # what enters and leaves the pair of projections; the 8-bit activation between them is its own product
    return {"bytes": 2 * N * K + 2 * 2 * M * K + 4 * (N + K), "flops": 4 * M * N * K}


# ---------------------------------------------------------------------------------------------------- 64-bit result
def _exact_e4m3(v):
    """Nearest e4m3 value (ties to even), as double."""
    e = torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -20))).clamp_min(-6.0)
    step = torch.exp2(e - 3.0)
    return (torch.round(v / step) * step).clamp(-E4M3_MAX, E4M3_MAX)


def _exact_quantize(x):
    """double `[rows, K]` -> (e4m3 values as double, scales `[ceil(K / 128), rows]`).  The quantizer is defined on 32-bit
    values: 448 / amax and its product with a value are rounded to 32 bits before the code is.  Half-precision values and
    amax have few bits, so the quotient lies on a tie between two codes far more often than by chance, and those two
    roundings, not the last bit of a computation, decide which."""
    q, s = torch.empty_like(x), []
    for k in range(0, x.shape[1], BLOCK):
        amax = x[:, k:k + BLOCK].abs().amax(1).clamp_min(MIN_AMAX)
        inverse = (E4M3_MAX / amax.float().double()).float()
        q[:, k:k + BLOCK] = _exact_e4m3((x[:, k:k + BLOCK].float() * inverse[:, None]).double())
        s.append(amax / E4M3_MAX)
    return q, torch.stack(s)


def _exact_linear(q, s, w8, ws, bias):
    y = bias.double()[None, :].repeat(q.shape[0], 1)
    for i, k in enumerate(range(0, q.shape[1], BLOCK)):
        w = w8[:, k:k + BLOCK].double() * ws[:, i].double().repeat_interleave(BLOCK)[:w8.shape[0], None]
        y += (q[:, k:k + BLOCK] * s[i].double()[:, None]) @ w.t()
    return y


def _exact_attention(st):
    B, Sq, heads, kv_heads = st["B"], st["Sq"], st["heads"], st["kv_heads"]
    out = torch.zeros((B, Sq, heads * D), dtype=torch.float64, device="cuda")
    for b in range(B):
        n = int(st["kv_len"][b])
        first = 0 if st["q_start"] is None else int(st["q_start"][b])
        for i0 in range(0, Sq, 1024):
            i1 = min(Sq, i0 + 1024)
            pos = torch.arange(first + i0, first + i1, device="cuda")[:, None]
            lo = 0 if st["left"] < 0 else max(0, min(n, first + i0 - st["left"]))
            hi = n if st["right"] < 0 else max(0, min(n, first + i1 + st["right"]))
            keys = torch.cat([torch.arange(min(st["sinks"], lo), device="cuda"), torch.arange(lo, hi, device="cuda")])
            if keys.numel() == 0:
                continue
            seen = torch.ones((i1 - i0, keys.numel()), dtype=torch.bool, device="cuda")
            if st["left"] >= 0:
                seen &= keys >= pos - st["left"]
            if st["right"] >= 0:
                seen &= keys <= pos + st["right"]
            seen |= keys < st["sinks"]
            for h in range(heads):
                kv = slice(h // (heads // kv_heads) * D, h // (heads // kv_heads) * D + D)
                s = st["q"][b, i0:i1, h * D:(h + 1) * D].double() @ st["k"][b, keys, kv].double().t() / math.sqrt(D)
                p = torch.where(seen, s, -math.inf).softmax(-1)
                p = torch.where(seen.any(-1, keepdim=True), p, 0.0)
                out[b, i0:i1, h * D:(h + 1) * D] = p @ st["v"][b, keys, kv].double()
    return out


def exact(case, seed):
    """`run`'s outputs in 64-bit floating point on the same inputs; 8-bit values are rounded where the operator is defined
    to round them (the operands of a product), nothing else is."""
    st = prepare(case, seed)
    kind = case["kind"]
    if kind == "attention":
        return _exact_attention(st)
    if kind == "linear":
        y = _exact_linear(st["x8"].double(), st["xs"], st["w8"], st["ws"], st["bias"])
        return y if st["r"] is None else y + st["r"].double()
    x = st["x"].double()
    if kind == "quantize":
        q, s = _exact_quantize(x)
        return {"q": q, "scale": s}
    if kind == "norm":
        x = x if st["r"] is None else x + st["r"].double()
        var, mean = torch.var_mean(x, -1, correction=0, keepdim=True)
        y = (x - mean) / torch.sqrt(var + EPS) * st["gamma"].double() + st["beta"].double()
        q, s = _exact_quantize(y)
        return {"y": y, "q": q, "scale": s}
    h = _exact_linear(*_exact_quantize(x), st["w1"], st["ws1"], st["b1"])
    h = 0.5 * h * (1.0 + torch.erf(h * math.sqrt(0.5)))
    return _exact_linear(*_exact_quantize(h), st["w2"], st["ws2"], st["b2"]) + x
