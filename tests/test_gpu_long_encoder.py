"""GPU: the encoder for long documents, 8-bit matrix weights and sliding-window attention together, as `Encoder` runs them."""
import math

import numpy as np
import pytest
import torch

from tnn_b200 import capi, ops
from tnn_b200.encoder import Encoder
from tnn_b200.model_synth import EncoderConfig, make_workload

pytestmark = pytest.mark.gpu

F8 = torch.float8_e4m3fn


@pytest.fixture(autouse=True)
def _status_clean(cuda_device):
    yield
    torch.cuda.synchronize()
    assert capi.device_status() == capi.OK


def _workload(layers, B, S, with_ffn=True, lo=30):
    cfg = EncoderConfig(layers, 256, 4, 512, with_ffn=with_ffn)
    return make_workload(cfg, B, S, seed=S + layers, length_range=(min(lo, S), S), randomize_affine=True, num_layers=layers)


def _inputs(wl, dev):
    return torch.from_numpy(wl.x).to(dev), torch.from_numpy(wl.mask_add).to(dev)


def exact(wl, window, sinks, dev):
    """The stack in 64 bits, nothing rounded."""
    t = lambda a: torch.from_numpy(np.asarray(a)).to(dev).double()   # noqa: E731
    x, S, heads, eps = t(wl.x), wl.x.shape[1], wl.cfg.heads, wl.cfg.ln_eps
    j = torch.arange(S, device=dev)
    seen = torch.ones(S, S, dtype=torch.bool, device=dev)
    if window is not None:
        if window[0] >= 0:
            seen &= j[None] >= j[:, None] - window[0]
        if window[1] >= 0:
            seen &= j[None] <= j[:, None] + window[1]
        seen |= j[None] < sinks
    seen = seen[None] & (t(wl.mask_add).reshape(-1, 1, S) > -5000)

    def norm(v, g, b):
        var, mean = torch.var_mean(v, -1, correction=0, keepdim=True)
        return (v - mean) / torch.sqrt(var + eps) * t(g) + t(b)

    for w in wl.weights:
        q, k, v = ((x @ t(m) + t(b)).reshape(*x.shape[:2], heads, 64).transpose(1, 2)
                   for m, b in ((w.wq, w.bq), (w.wk, w.bk), (w.wv, w.bv)))
        s = torch.where(seen[:, None], q @ k.transpose(-1, -2) / 8, -math.inf)
        p = torch.where(seen.any(-1)[:, None, :, None], s.softmax(-1), 0.0)
        x = norm((p @ v).transpose(1, 2).reshape(x.shape) @ t(w.wo) + t(w.bo) + x, w.ln1_g, w.ln1_b)
        if wl.cfg.with_ffn:
            h = x @ t(w.w1) + t(w.b1)
            x = norm(0.5 * h * (1 + torch.erf(h / math.sqrt(2))) @ t(w.w2) + t(w.b2) + x, w.ln2_g, w.ln2_b)
    return x


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("layers,B,S,window,sinks,ffn", [(1, 2, 200, (32, 32), 1, True), (2, 3, 333, (64, 0), 4, True), (1, 2, 130, None, 0, True),
                                                         (2, 2, 150, (16, 16), 0, False), (1, 1, 1, (4, 4), 1, True)])
def test_8_bit_stack_with_a_window(cuda_device, layers, B, S, window, sinks, ffn, dtype):
    """A code is off by at most 2^-4 of its value, evenly spread: 2^-4 / sqrt(3) = 3.6e-2 of the root mean square of an operand,
    5.1e-2 of a product of two.  Four products a layer (two without the feed-forward half) add at most that to a value that the
    residual and the LayerNorm keep at its size, as independent errors: 0.1 sqrt(layers).  bf16 adds 2^-8."""
    wl = _workload(layers, B, S, ffn)
    x, mask = _inputs(wl, cuda_device)
    enc = Encoder.from_workload(wl, dtype, cuda_device, fp8=True, window=window, sinks=sinks)
    got = enc.forward(x, mask)
    want = exact(wl, window, sinks, cuda_device)
    assert got.dtype == torch.float32 and got.shape == x.shape
    assert float((got.double() - want).norm() / want.norm()) <= 0.1 * math.sqrt(layers) + 2.0 ** -6
    assert torch.equal(got, enc.forward_ops(x, mask))


@pytest.mark.parametrize("window,sinks", [((40, 40), 2), ((-1, 0), 0), ((-1, -1), 0)])
def test_half_precision_stack_with_a_window(cuda_device, window, sinks):
    """fp16: the bounds of the full-attention stack (max-abs 2e-2 of values of size 1)."""
    wl = _workload(2, 3, 260)
    x, mask = _inputs(wl, cuda_device)
    got = Encoder.from_workload(wl, torch.float16, cuda_device, window=window, sinks=sinks).forward(x, mask)
    want = exact(wl, window, sinks, cuda_device)
    assert float((got.double() - want).abs().max()) <= 2e-2
    if window == (-1, -1):
        plain = Encoder.from_workload(wl, torch.float16, cuda_device).forward(x, mask)
        assert float((got - plain).abs().max()) <= 2e-2


def test_in_place_stack_and_its_operators(cuda_device):
    """forward_hidden on the caller's buffer is the sequence of operators, bit for bit."""
    wl = _workload(1, 2, 190)
    x, mask = _inputs(wl, cuda_device)
    m2 = mask.reshape(2, 190).contiguous()
    kv_len = ops.mask_to_kv_len(m2)
    enc = Encoder.from_workload(wl, torch.float16, cuda_device, fp8=True, window=(50, 20), sinks=3)
    L, eps = enc.layers[0], wl.cfg.ln_eps
    h = ops.convert(x, torch.float16)
    q = ops.linear_fp8(*ops.quantize_fp8(h), *L["w_qkv"], L["b_qkv"])
    c = ops.window_attention(q[..., :256], q[..., 256:512], q[..., 512:], 4, window=(50, 20), sinks=3, mask_add=m2, kv_len=kv_len)
    t = ops.linear_fp8(*ops.quantize_fp8(c), *L["w_o"], L["b_o"], residual=h, epilogue=ops.EPI_BIAS_RESIDUAL)
    a, a8, s = ops.add_layernorm_fp8(t, L["ln1_g"], L["ln1_b"], eps)
    f = ops.linear_fp8(a8, s, *L["w_ffn1"], L["b_ffn1"], epilogue=ops.EPI_BIAS_GELU, out_dtype=F8)
    t = ops.linear_fp8(*f, *L["w_ffn2"], L["b_ffn2"], residual=a, epilogue=ops.EPI_BIAS_RESIDUAL)
    want = ops.add_layernorm(t, L["ln2_g"], L["ln2_b"], eps)
    buf = h.clone()
    assert enc.forward_hidden(buf, m2, kv_len) is buf
    assert torch.equal(buf, want)


def test_padding_changes_nothing(cuda_device):
    """A sequence in a padded batch gives what it gives alone: row for row in 8 bits, to the rounding of half the tile's sums."""
    wl = _workload(2, 4, 300, lo=40)
    x, mask = _inputs(wl, cuda_device)
    enc = Encoder.from_workload(wl, torch.float16, cuda_device, fp8=True, window=(30, 30), sinks=1)
    got = enc.forward(x, mask)
    noisy = x.clone()
    for b, n in enumerate(wl.lengths):
        noisy[b, int(n):] = 3.0
    again = enc.forward(noisy, mask)
    for b, n in enumerate(wl.lengths):
        assert torch.equal(got[b, :int(n)], again[b, :int(n)])


def test_captured_stack(cuda_device):
    wl = _workload(2, 2, 150)
    x, mask = _inputs(wl, cuda_device)
    enc = Encoder.from_workload(wl, torch.float16, cuda_device, fp8=True, window=(20, 20), sinks=1)
    inputs = [x, x.flip(0).contiguous(), x * 0.5]
    want = [enc.forward(v, mask).clone() for v in inputs]
    static = x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = enc.forward(static, mask)
    for v, w in zip(inputs, want):
        static.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, w)


def test_refusals(cuda_device):
    wl = _workload(1, 1, 20)
    for kw in ({"fp8": True}, {"window": (4, 4)}):
        with pytest.raises(ValueError):
            Encoder.from_workload(wl, torch.float16, cuda_device, fold_layernorm=True, **kw)


def test_calls_at_once_on_several_streams_and_in_graphs(cuda_device):
    def randn(seed, *shape):
        return torch.randn(*shape, generator=torch.Generator(device="cpu").manual_seed(seed)).to(cuda_device)

    def attention(B, S, heads, kv_heads, window, sinks, Sq):
        q, k, v = (randn(i, B, n, h * 64).half() for i, n, h in ((1, Sq, heads), (2, S, kv_heads), (3, S, kv_heads)))
        start = torch.full((B,), S - Sq, dtype=torch.int32, device=cuda_device)
        return lambda: ops.window_attention(q, k, v, heads, kv_heads, window=window, sinks=sinks, q_start=start)

    def linear(M, N, K, out):
        x8, xs = ops.quantize_fp8(randn(4, M, K))
        w8, ws = ops.pack_weight_fp8(0.05 * randn(5, K, N))
        y = lambda: ops.linear_fp8(x8, xs, w8, ws, epilogue=ops.EPI_BIAS_GELU, out_dtype=out)   # noqa: E731
        return (lambda: y()[0].view(torch.uint8)) if out == F8 else y

    def norm(M, H):
        x, g, b = randn(6, M, H).half(), randn(7, H), randn(8, H)
        return lambda: ops.add_layernorm_fp8(x, g, b, 1e-5, residual=x)[0]

    jobs = [attention(3, 1500, 8, 2, (200, 0), 4, 1500), attention(40, 300, 4, 4, (20, 20), 1, 300), attention(7, 3000, 16, 4, (-1, 0), 0, 1),
            linear(2000, 1024, 1024, torch.float16), linear(5, 2304, 768, torch.float16), linear(100, 1024, 512, F8),
            linear(2000, 1024, 512, F8), norm(2000, 2096), norm(500, 768), norm(1000, 4096)]
    want = [job() for job in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    for _ in range(10):
        got = []
        for job, stream in zip(jobs, streams):
            with torch.cuda.stream(stream):
                got.append([job() for _ in range(3)])
        torch.cuda.synchronize()
        assert all(torch.equal(y, w) for ys, w in zip(got, want) for y in ys)
    graphs = []
    for job in jobs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, [job() for _ in range(3)]))
    for _ in range(10):
        for (graph, _), stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(y, w) for (_, ys), w in zip(graphs, want) for y in ys)
