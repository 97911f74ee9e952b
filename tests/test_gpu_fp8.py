"""GPU: block-scaled 8-bit operands: the quantizer, LayerNorm with an 8-bit result, the weight pre-pack and the GEMM, against
plain implementations in 64 bits (the quantizer, whose every rounding is defined, bit for bit)."""
import math

import pytest
import torch

from tnn_b200 import capi, ops

pytestmark = pytest.mark.gpu

F16, BF16, F32, F8 = torch.float16, torch.bfloat16, torch.float32, torch.float8_e4m3fn
U32 = 2.0 ** -24                       # half a step of fp32
HALF_STEP = {F16: 2.0 ** -11, BF16: 2.0 ** -8, F32: U32, F8: 2.0 ** -4}


@pytest.fixture(autouse=True)
def _status_clean(cuda_device):
    yield
    torch.cuda.synchronize()
    assert capi.device_status() == capi.OK


def _gen(seed):
    return torch.Generator(device="cpu").manual_seed(seed)


def _randn(dev, seed, *shape):
    return torch.randn(*shape, generator=_gen(seed)).to(dev)


def quantize_ref(x):
    """The definition in fp32 on the CPU, one rounding per operation: (codes, scales `[blocks, rows]`)."""
    x = x.detach().cpu().float()
    rows, K = x.shape
    pad = -K % 128
    b = torch.nn.functional.pad(x, (0, pad)).reshape(rows, -1, 128)
    bits = b.view(torch.int32) & 0x7FFFFFFF                  # magnitudes as integers: a NaN is the largest
    amax = bits.amax(-1).clamp_min(int(torch.tensor(2.0 ** -40).view(torch.int32))).view(torch.float32)
    top = torch.full_like(amax, 448.0)
    q = (b * (top / amax)[..., None]).clamp(-448.0, 448.0).to(F8)
    return q.reshape(rows, -1)[:, :K], (amax / top).t().contiguous()


def same_codes(got, want):
    """Equal codes; a NaN of either sign is a NaN."""
    g, w = got.cpu().float(), want.float()
    return torch.equal(g.isnan(), w.isnan()) and torch.equal(g.nan_to_num(nan=0.0), w.nan_to_num(nan=0.0))


def values(q, s):
    """What codes and scales stand for, fp64 `[rows, K]`."""
    return q.double() * s.t().repeat_interleave(128, 1)[:, :q.shape[1]].double()


# ---------------------------------------------------------------------------------------------------- quantizer
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("rows,K", [(1, 16), (1, 768), (3, 128), (7, 144), (33, 112), (130, 1040), (5, 4096), (1025, 272)])
def test_quantize_is_its_definition(cuda_device, rows, K, dtype):
    x = (_randn(cuda_device, rows + K, rows, K) * torch.exp(_randn(cuda_device, K, K))).to(dtype)
    q, s = ops.quantize_fp8(x)
    wq, ws = quantize_ref(x)
    assert torch.equal(s.cpu(), ws)
    assert same_codes(q, wq)


def test_quantize_zeros_tiny_huge_infinite_and_nan(cuda_device):
    x = torch.zeros(6, 256, dtype=F32, device=cuda_device)
    x[1, :128] = 1e-38                                       # below the least amax: scaled as if that were it
    x[2, 5], x[2, 130] = 3e38, -3e38
    x[3, 7] = math.inf
    x[4, 200] = math.nan
    x[5] = torch.linspace(-1, 1, 256)
    q, s = ops.quantize_fp8(x)
    wq, ws = quantize_ref(x)
    assert torch.equal(torch.isnan(s.cpu()), torch.isnan(ws)) and torch.equal(s.cpu().nan_to_num(), ws.nan_to_num())
    assert same_codes(q, wq)
    v = values(q, s)
    assert bool((v[0] == 0).all()) and not bool(torch.isfinite(v[3, :128]).any()) and bool(torch.isnan(v[4, 128:]).all())
    assert bool(torch.isfinite(v[3, 128:]).all()) and bool(torch.isfinite(v[4, :128]).all())   # other blocks are untouched


def test_quantize_strided_rows_and_given_outputs(cuda_device):
    base = _randn(cuda_device, 3, 40, 1024).to(F16)
    x = base[:, 256:256 + 400]
    out = torch.zeros(40, 512, dtype=torch.uint8, device=cuda_device).view(F8)
    scale = torch.full((4, 64), 7.0, device=cuda_device)
    q, s = ops.quantize_fp8(x, out=out[:, :400], out_scale=scale[:, 8:48])
    wq, ws = quantize_ref(x)
    assert same_codes(q, wq) and torch.equal(s.cpu(), ws)
    assert bool((out[:, 400:].view(torch.uint8) == 0).all())
    assert bool((scale[:, :8] == 7).all()) and bool((scale[:, 48:] == 7).all())
    assert bool(torch.equal(ops.quantize_fp8(x.reshape(8, 5, 400))[0].reshape(40, 400).view(torch.uint8), q.contiguous().view(torch.uint8)))
    e, es = ops.quantize_fp8(x[:0])
    assert e.shape == (0, 400) and es.shape == (4, 0)


@pytest.mark.parametrize("K,N", [(16, 8), (128, 128), (144, 200), (768, 264), (1040, 72)])
def test_pack_weight(cuda_device, K, N):
    w = _randn(cuda_device, K * N, K, N + 8)[:, :N] * 0.03
    q, s = ops.pack_weight_fp8(w)
    t = w.t().cpu()
    for n in range(0, N, 128):
        for k in range(0, K, 128):
            b = t[n:n + 128, k:k + 128]
            amax, top = b.abs().amax(), torch.tensor(448.0)
            assert float(s[n // 128, k // 128]) == float(amax / top)
            assert same_codes(q[n:n + 128, k:k + 128], (b * (top / amax)).clamp(-448, 448).to(F8))


# ---------------------------------------------------------------------------------------------------- LayerNorm
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("resid", [False, True])
@pytest.mark.parametrize("rows,H", [(1, 768), (9, 16), (333, 1024), (5, 272), (2, 4096), (1201, 144), (65, 2048), (700, 1552), (31, 784), (130, 1040), (67, 2064), (1500, 2096), (19, 3088),
                                    (7, 512), (4001, 528), (2999, 1280)])
def test_add_layernorm_fp8(cuda_device, rows, H, resid, dtype):
    x = _randn(cuda_device, rows + H, rows, H).to(dtype)
    r = _randn(cuda_device, rows + H + 1, rows, H).to(dtype) if resid else None
    g, b = 1 + 0.1 * _randn(cuda_device, 5, H), 0.1 * _randn(cuda_device, 6, H)
    y, q, s = ops.add_layernorm_fp8(x, g, b, 1e-12, residual=r)
    t = x.double() + (r.double() if resid else 0)
    var, mean = torch.var_mean(t, -1, correction=0, keepdim=True)
    want = (t - mean) / torch.sqrt(var + 1e-12) * g.double() + b.double()
    # fp32 error of a normalised value: the sum of H terms by a tree of 32 lanes over H / 32 terms (mean and variance), the
    # rest a handful of roundings of values of magnitude |want| + |b|, and of the inputs' sum relative to the deviation.
    size = want.abs() + b.double().abs() + (t.abs().amax(-1, keepdim=True) / torch.sqrt(var + 1e-12)) * g.double().abs()
    err32 = (H / 32 + 16) * U32 * size
    assert bool(((y.double() - want).abs() <= HALF_STEP[dtype] * want.abs() + 2.0 ** -24 + err32).all())
    amax = torch.nn.functional.pad(want.abs(), (0, -H % 128)).reshape(rows, -1, 128).amax(-1)
    worst = torch.nn.functional.pad(err32, (0, -H % 128)).reshape(rows, -1, 128).amax(-1)
    assert bool(((s.t().double() * 448 - amax).abs() <= worst + 4 * U32 * amax).all())
    step = s.t().double().repeat_interleave(128, 1)[:, :H]
    # half a step of e4m3, subnormal codes (below 2^-6) half of 2^-9; the scale's own error twice
    bound = 2.0 ** -4 * want.abs() + step * 2.0 ** -10 + err32 * 1.0625 + 8 * U32 * want.abs()
    assert bool(((values(q, s) - want).abs() <= bound).all())
    y2, q2, s2 = ops.add_layernorm_fp8(x, g, b, 1e-12, residual=r, half=False)
    assert y2 is None and torch.equal(q2.view(torch.uint8), q.view(torch.uint8)) and torch.equal(s2, s)


# ---------------------------------------------------------------------------------------------------- GEMM
def _operands(dev, M, N, K, seed=0):
    x8, xs = ops.quantize_fp8(_randn(dev, M + K + seed, M, K) * torch.exp(0.5 * _randn(dev, K, K)))
    w8, ws = ops.pack_weight_fp8((_randn(dev, N + 3 * K + seed, K, N) * 0.05).contiguous())
    return x8, xs, w8, ws


def _product(x8, xs, w8, ws):
    """(x . w^T, the same over magnitudes) in fp64."""
    x = values(x8, xs)
    w = w8.double() * ws.double().repeat_interleave(128, 0)[:w8.shape[0]].repeat_interleave(128, 1)[:, :w8.shape[1]]
    return x @ w.t(), x.abs() @ w.abs().t()


def _check(got, want, size, K, half_step, extra=0.0):
    """`size` = sum of the magnitudes that were added up.  Every one of the K additions may lose half a step of a partial sum
    (a whole one where the tensor core truncates), which is at most `size`; as random errors they add up to the root of that."""
    err = (got.double() - want).abs()
    assert bool((err <= half_step * want.abs() + (K + 8) * 2 * U32 * size + extra + 2.0 ** -25).all()), float(err.max())
    rms = float(err.norm() / want.norm())
    assert rms <= half_step + 2 * U32 * math.sqrt(K + 8) * float(size.norm() / want.norm()) + float(extra if isinstance(extra, float) else 0) * math.sqrt(want.numel()) / float(want.norm())


SHAPES = [(1, 8, 16), (1, 768, 768), (5, 200, 144), (17, 64, 4096), (64, 2304, 768), (128, 136, 272), (129, 264, 128), (200, 72, 1040),
          (257, 1000, 400), (300, 128, 2048), (777, 1024, 1024), (1025, 520, 656), (2500, 1280, 256)]


@pytest.mark.parametrize("out", [F16, BF16, F32])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_linear_fp8(cuda_device, M, N, K, out):
    x8, xs, w8, ws = _operands(cuda_device, M, N, K)
    bias = 0.1 * _randn(cuda_device, N, N)
    y = ops.linear_fp8(x8, xs, w8, ws, bias, out_dtype=out)
    want, size = _product(x8, xs, w8, ws)
    _check(y, want + bias.double(), size + bias.double().abs(), K, HALF_STEP[out])
    assert torch.equal(y, ops.linear_fp8(x8, xs, w8, ws, bias, out_dtype=out))


@pytest.mark.parametrize("epi", ["none", "bias", "gelu", "tanh", "residual"])
@pytest.mark.parametrize("M,N,K,block_n", [(m, n, k, bn) for m, n, k in ((41, 200, 400), (300, 392, 272), (513, 256, 128)) for bn in (64, 128, 256)] +
                         [(1, 8, 16, -1), (3, 200, 400, -1), (16, 1400, 2064, -1), (8, 264, 1040, -1), (9, 4000, 1168, -1), (5, 2600, 272, -1), (41, 264, 1040, -1), (17, 2600, 400, -1), (128, 264, 400, -1)])
def test_linear_fp8_epilogues_on_every_tile(cuda_device, M, N, K, epi, block_n):
    x8, xs, w8, ws = _operands(cuda_device, M, N, K, 5)
    bias = None if epi == "none" else 0.1 * _randn(cuda_device, N, N)
    want, size = _product(x8, xs, w8, ws)
    if bias is not None:
        want, size = want + bias.double(), size + bias.double().abs()
    for out in (F16, F32):
        res, extra = None, 0.0
        w = want
        if epi == "gelu":
            code, w = ops.EPI_BIAS_GELU, 0.5 * want * (1 + torch.erf(want / math.sqrt(2)))
            # the derivative of GELU and tanh is at most 1.13; the tail's fit is within 3.0e-6, its fp32 evaluation (8 steps and a
            # product of magnitude 0.5, ex2.approx 2^-22) within 1e-6 more
            extra = 4e-6 * w.abs() if out == F32 else 4e-6 + 2.0 ** -22 * w.abs()
        elif epi == "tanh":
            code, w = ops.EPI_BIAS_TANH, torch.tanh(want)
            extra = 4e-6 * w.abs() if out == F32 else 2.0 ** -10 * w.abs()
        elif epi == "residual":
            code, res = ops.EPI_BIAS_RESIDUAL, _randn(cuda_device, 9, M, N).to(BF16 if out == F32 else F16)
            w = want + res.double()
        else:
            code = ops.EPI_BIAS
        y = ops.linear_fp8(x8, xs, w8, ws, bias, residual=res, epilogue=code, out_dtype=out, block_n=block_n)
        err = (y.double() - w).abs()
        bound = HALF_STEP[out] * w.abs() + 1.13 * (K + 8) * 2 * U32 * (size + (0 if res is None else res.double().abs())) + extra + 2.0 ** -25
        assert bool((err <= bound).all()), float((err - bound).max())


@pytest.mark.parametrize("epi", ["bias", "gelu", "residual"])
@pytest.mark.parametrize("M,N,K,block_n", [(m, n, k, bn) for m, n, k in ((1, 16, 64), (41, 272, 400), (300, 1040, 256), (129, 128, 144))
                                           for bn in (0, 128, 256)] + [(2, 144, 1040, -1), (16, 1040, 400, -1), (7, 272, 2064, -1), (33, 272, 400, -1), (101, 272, 400, -1)])
def test_linear_fp8_with_an_8_bit_result(cuda_device, M, N, K, epi, block_n):
    x8, xs, w8, ws = _operands(cuda_device, M, N, K, 7)
    bias = 0.1 * _randn(cuda_device, N, N)
    want, size = _product(x8, xs, w8, ws)
    want, size, res, extra, code = want + bias.double(), size + bias.double().abs(), None, 0.0, ops.EPI_BIAS
    if epi == "gelu":
        code, want = ops.EPI_BIAS_GELU, 0.5 * want * (1 + torch.erf(want / math.sqrt(2)))
        extra = 4e-6 + 2.0 ** -22 * want.abs()
    if epi == "residual":
        code, res = ops.EPI_BIAS_RESIDUAL, _randn(cuda_device, 9, M, N).to(F16)
        want, size = want + res.double(), size + res.double().abs()
    q, s = ops.linear_fp8(x8, xs, w8, ws, bias, residual=res, epilogue=code, out_dtype=F8, block_n=block_n)
    assert q.shape == (M, N) and s.shape == (-(-N // 128), M)
    err32 = 1.13 * (K + 8) * 2 * U32 * size + extra
    pad = lambda t: torch.nn.functional.pad(t, (0, -N % 128)).reshape(M, -1, 128).amax(-1)   # noqa: E731
    assert bool(((s.t().double() * 448 - pad(want.abs())).abs() <= pad(err32 + 0 * want) + 4 * U32 * pad(want.abs()) + 2.0 ** -40).all())
    step = s.t().double().repeat_interleave(128, 1)[:, :N]
    bound = 2.0 ** -4 * want.abs() + step * 2.0 ** -10 + 1.07 * err32 + 8 * U32 * want.abs()
    assert bool(((values(q, s) - want).abs() <= bound).all())


def test_gelu_over_its_whole_range(cuda_device):
    """y = GELU(bias): every bias from -40 to 40 and far out, in half precision, and infinities and NaN as the formula gives them."""
    N = 4096
    x8, xs = ops.quantize_fp8(torch.zeros(1, 16, device=cuda_device))
    w8, ws = ops.pack_weight_fp8(torch.zeros(16, N, device=cuda_device))
    for lo, hi in ((-40, 40), (-6.5, 6.5), (-1, 1), (-60000, 60000)):
        bias = torch.linspace(lo, hi, N).to(cuda_device)
        y = ops.linear_fp8(x8, xs, w8, ws, bias, epilogue=ops.EPI_BIAS_GELU)[0].double()
        want = bias.double() * 0.5 * torch.erfc(-bias.double() / math.sqrt(2))
        assert bool(((y - want).abs() <= 4e-6 + HALF_STEP[F16] * want.abs() * (1 + 2.0 ** -10) + 2.0 ** -25).all())
    bias = torch.zeros(N, device=cuda_device)
    bias[0], bias[1] = math.nan, math.inf
    y = ops.linear_fp8(x8, xs, w8, ws, bias, epilogue=ops.EPI_BIAS_GELU)[0]
    assert bool(torch.isnan(y[0])) and bool(torch.isinf(y[1])) and bool((y[2:] == 0).all())


def test_linear_fp8_rows_do_not_depend_on_the_batch_or_the_tile(cuda_device):
    x8, xs, w8, ws = _operands(cuda_device, 700, 520, 656)
    bias = _randn(cuda_device, 1, 520)
    y = ops.linear_fp8(x8, xs, w8, ws, bias, out_dtype=F32)
    for rows in (slice(3, 134), slice(100, 400)):
        part = ops.linear_fp8(x8[rows], xs[:, rows].contiguous(), w8, ws, bias, out_dtype=F32)
        assert torch.equal(part, y[rows])
    for bn in (64, 128, 256):
        assert torch.equal(ops.linear_fp8(x8, xs, w8, ws, bias, out_dtype=F32, block_n=bn), y)
    few = ops.linear_fp8(x8[:128], xs[:, :128].contiguous(), w8, ws, bias, out_dtype=F32)       # a few rows: an order of its own
    for rows in (slice(0, 1), slice(5, 12), slice(3, 44)):
        part = ops.linear_fp8(x8[rows], xs[:, rows].contiguous(), w8, ws, bias, out_dtype=F32)
        assert torch.equal(part, few[rows])
    want, size = _product(x8, xs, w8, ws)
    _check(few, want[:128] + bias.double(), size[:128] + bias.double().abs(), 656, HALF_STEP[F32])


@pytest.mark.parametrize("out", [F16, F32, F8])
@pytest.mark.parametrize("epi", ["bias", "residual"])
@pytest.mark.parametrize("M,N,block_n", [(30000, 328, 256), (30000, 264, 256), (20000, 200, 128), (20000, 72, 64)])
def test_linear_fp8_many_tiles_per_cta_with_a_ragged_last_column(cuda_device, M, N, block_n, epi, out):
    """Tiles of unequal width follow one another on a CTA: an output strip is written again only when its store has read it."""
    if out == F8 and (block_n == 64 or N % 16):
        block_n, N = 128, N // 16 * 16
    x8, xs, w8, ws = _operands(cuda_device, M, N, 144, 11)
    bias = _randn(cuda_device, 1, N)
    res = _randn(cuda_device, 2, M, N).to(F16) if epi == "residual" else None
    code = ops.EPI_BIAS if res is None else ops.EPI_BIAS_RESIDUAL
    got = ops.linear_fp8(x8, xs, w8, ws, bias, residual=res, epilogue=code, out_dtype=out, block_n=block_n)
    for r in (slice(0, 200), slice(M // 2, M // 2 + 300), slice(M - 100, M)):      # one tile per CTA: no strip is used twice
        part = ops.linear_fp8(x8[r], xs[:, r].contiguous(), w8, ws, bias, residual=None if res is None else res[r], epilogue=code,
                              out_dtype=out, block_n=block_n)
        if out == F8:
            assert torch.equal(part[0].view(torch.uint8), got[0][r].view(torch.uint8)) and torch.equal(part[1], got[1][:, r])
        else:
            assert torch.equal(part, got[r])
    want, size = _product(x8, xs, w8, ws)
    want = want + bias.double() + (0 if res is None else res.double())
    y = values(*got) if out == F8 else got.double()
    step = 0 if out != F8 else got[1].t().double().repeat_interleave(128, 1)[:, :N] * 2.0 ** -10
    bound = HALF_STEP[out] * want.abs() * 1.01 + step + 1e-4 * (size + bias.double().abs() + (0 if res is None else res.double().abs()))
    assert bool(((y - want).abs() <= bound).all())


@pytest.mark.parametrize("out", [F16, F32, F8])
@pytest.mark.parametrize("M,N,block_n", [(1, 80, 0), (13, 272, -1), (41, 272, -1), (41, 272, 128), (300, 272, 256), (130, 144, 128)])
def test_linear_fp8_strides_and_what_lies_around_the_output(cuda_device, M, N, block_n, out):
    K = 272
    x8, xs, w8, ws = _operands(cuda_device, M, N, K, 3)
    bias = _randn(cuda_device, 1, N)
    wide = torch.zeros(M, K + 48, dtype=torch.uint8, device=cuda_device).view(F8)
    wide[:, :K].view(torch.uint8).copy_(x8.view(torch.uint8))
    scales = torch.full((xs.shape[0], M + 5), 9.0, device=cuda_device)
    scales[:, :M] = xs
    res = _randn(cuda_device, 2, M, N + 24).to(F16)[:, :N]
    code = ops.EPI_BIAS_RESIDUAL
    plain = ops.linear_fp8(x8, xs, w8, ws, bias, residual=res.contiguous(), epilogue=code, out_dtype=out, block_n=block_n)
    back = torch.full((M + 4, N + 32), 0, dtype=torch.uint8 if out == F8 else out, device=cuda_device)
    back.view(torch.uint8).fill_(0x5B)
    y = (back.view(F8) if out == F8 else back)[2:M + 2, :N]
    ys = torch.full((-(-N // 128), M + 3), 5.0, device=cuda_device)
    kw = {"out_scale": ys[:, :M]} if out == F8 else {}
    got = ops.linear_fp8(wide[:, :K], scales[:, :M], w8, ws, bias, residual=res, epilogue=code, out=y, block_n=block_n, **kw)
    if out == F8:
        assert torch.equal(got[1], plain[1]) and bool((ys[:, M:] == 5).all())
        got, plain = got[0], plain[0]
    assert torch.equal(got.contiguous().view(torch.uint8), plain.view(torch.uint8))
    bytes_ = back.view(torch.uint8)
    width = N * (1 if out == F8 else out.itemsize)
    assert bool((bytes_[:2] == 0x5B).all()) and bool((bytes_[-2:] == 0x5B).all()) and bool((bytes_[:, width:] == 0x5B).all())


def test_linear_fp8_a_nan_or_an_infinity_stays_in_its_row(cuda_device):
    M, N, K = 300, 264, 400
    x = _randn(cuda_device, 1, M, K)
    x[7, 3], x[200, 399] = math.nan, math.inf
    x8, xs = ops.quantize_fp8(x)
    w8, ws = ops.pack_weight_fp8(_randn(cuda_device, 2, K, N) * 0.05)
    y = ops.linear_fp8(x8, xs, w8, ws, out_dtype=F32)
    bad = ~torch.isfinite(y)
    assert bool(bad[7].all()) and bool(bad[200].all())
    bad[7] = bad[200] = False
    assert not bool(bad.any())


def test_feed_forward_in_a_captured_graph_and_on_another_stream(cuda_device):
    """quantize -> up-projection with GELU (8-bit result) -> down-projection with residual -> LayerNorm, as a layer runs it:
    eager, on a side stream and replayed from a CUDA graph on new inputs, bit for bit."""
    M, H, F = 333, 768, 1024
    w1, s1 = ops.pack_weight_fp8(_randn(cuda_device, 1, H, F) * 0.03)
    w2, s2 = ops.pack_weight_fp8(_randn(cuda_device, 2, F, H) * 0.03)
    b1, b2 = 0.1 * _randn(cuda_device, 3, F), 0.1 * _randn(cuda_device, 4, H)
    g, b = 1 + 0.1 * _randn(cuda_device, 5, H), 0.1 * _randn(cuda_device, 6, H)

    def layer(x):
        q, s = ops.quantize_fp8(x)
        q, s = ops.linear_fp8(q, s, w1, s1, b1, epilogue=ops.EPI_BIAS_GELU, out_dtype=F8)
        y = ops.linear_fp8(q, s, w2, s2, b2, residual=x, epilogue=ops.EPI_BIAS_RESIDUAL)
        return ops.add_layernorm_fp8(y, g, b, 1e-12)

    xs = [_randn(cuda_device, 10 + i, M, H).to(F16) for i in range(3)]
    want = [[t.clone().view(torch.uint8) for t in layer(x)] for x in xs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [t.view(torch.uint8) for t in layer(xs[1])]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, w) for a, w in zip(got, want[1]))
    static = xs[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = layer(static)
    for x, w in zip(xs, want):
        static.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o.view(torch.uint8), v) for o, v in zip(outs, w))


def test_rows_beyond_2_31_elements(cuda_device):
    M, K, tail = 1_100_000, 2048, 300
    x = torch.empty(M, K, dtype=BF16, device=cuda_device)
    x[-tail:] = _randn(cuda_device, 1, tail, K).to(BF16)
    near = x[-tail:].clone()
    codes, scales = ops.quantize_fp8(x)
    want, want_scales = ops.quantize_fp8(near)
    assert torch.equal(codes[-tail:].view(torch.uint8), want.view(torch.uint8)) and torch.equal(scales[:, -tail:], want_scales)
    w8, ws = ops.pack_weight_fp8(0.05 * _randn(cuda_device, 2, K, 64))
    assert torch.equal(ops.linear_fp8(codes, scales, w8, ws)[-tail:], ops.linear_fp8(want, want_scales, w8, ws))
    g, b = _randn(cuda_device, 3, K), _randn(cuda_device, 4, K)
    for far, here in zip(ops.add_layernorm_fp8(x, g, b, 1e-5, half=False)[1:], ops.add_layernorm_fp8(near, g, b, 1e-5, half=False)[1:]):
        far = far[-tail:] if far.dtype == F8 else far[:, -tail:]
        assert torch.equal(far.view(torch.uint8), here.view(torch.uint8)) if far.dtype == F8 else torch.equal(far, here)
