"""GPU: window attention at the ends of what its arguments may be (positions and windows of any size, layouts, who sees the first
tokens), against a plain implementation in 64 bits."""
import math

import pytest
import torch

from tnn_b200 import capi, ops

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
HALF_STEP = {F16: 2.0 ** -11, BF16: 2.0 ** -8}


@pytest.fixture(autouse=True)
def _status_clean(cuda_device):
    yield
    torch.cuda.synchronize()
    assert capi.device_status() == capi.OK


def _randn(dev, seed, *shape):
    return torch.randn(*shape, generator=torch.Generator(device="cpu").manual_seed(seed)).to(dev)


def visible(Sq, Sk, window, sinks, kv_len, q_start, dev):
    """`[B, Sq, Sk]` in 64-bit positions; kv_len and q_start are lists."""
    j = torch.arange(Sk, device=dev)
    pos = torch.arange(Sq, device=dev)[None, :, None] + torch.tensor(q_start, device=dev)[:, None, None]
    near = torch.ones(len(q_start), Sq, Sk, dtype=torch.bool, device=dev)
    if window[0] >= 0:
        near &= j >= pos - window[0]
    if window[1] >= 0:
        near &= j <= pos + window[1]
    return (near | (j < sinks)) & (j < torch.tensor(kv_len, device=dev)[:, None, None])


def reference(q, k, v, heads, kv_heads, seen):
    """(result, bound on an element's error), fp64 `[B, Sq, heads * 64]`."""
    B, Sq, Sk, dt = q.shape[0], q.shape[1], k.shape[1], q.dtype
    split = lambda t, n: t.double().reshape(B, t.shape[1], n, 64).transpose(1, 2)   # noqa: E731
    qq = split(q, heads)
    kk, vv = (split(t, kv_heads).repeat_interleave(heads // kv_heads, 1) for t in (k, v))
    s = torch.where(seen[:, None], qq @ kk.transpose(-1, -2) / 8, -math.inf)
    p = torch.where(seen.any(-1)[:, None, :, None], s.softmax(-1), 0.0)
    # a weight is rounded to the half type once; a score is a sum of 64 products in fp32 (a whole step each where the tensor core
    # truncates) and its error is the weight's relative one, in numerator and denominator; ex2.approx 2^-22; the weights' sum and
    # the output's are fp32 sums of Sk terms; weights below f16's range lose at most 2^-25 of the largest; the result is rounded
    score = 2 * 66 * 2.0 ** -23 / 8 * float((qq.abs() @ kk.abs().transpose(-1, -2)).amax()) + 2.0 ** -21
    tiny = Sk * 2.0 ** -25 * float(vv.abs().amax()) if dt == F16 else 0.0
    inside = (p @ vv.abs()) * (HALF_STEP[dt] * (1 + 2.0 ** -6) + score + (Sk + 64) * 2.0 ** -23) + tiny
    want = p @ vv
    bound = HALF_STEP[dt] * (want.abs() + inside) + inside + 2.0 ** -24
    merge = lambda t: t.transpose(1, 2).reshape(B, Sq, heads * 64)   # noqa: E731
    return merge(want), merge(bound)


def check(out, want, bound):
    err = (out.double() - want).abs()
    assert bool((err <= bound).all()), "largest excess %g" % float((err - bound).max())


# ---------------------------------------------------------------------------------------------------- positions and widths
@pytest.mark.parametrize("Sq", [1, 5, 150])
@pytest.mark.parametrize("sinks", [0, 3])
@pytest.mark.parametrize("window,starts", [
    ((2 ** 26, 0), [2 ** 27, 2 ** 26 + 30, 2 ** 26 - 10, 0]),                # the window begins beyond, at, before key 0
    ((0, 2 ** 26), [-2 ** 27, -2 ** 26 - 20, -2 ** 26 + 40, 250]),
    ((2 ** 27 - 25, 2 ** 27), [2 ** 27, -2 ** 27 - 7, 0, 2 ** 26]),
    ((2 ** 31 - 100, -1), [2 ** 31 - 1 - 150, -2 ** 31, 2 ** 31 - 1, 0]),    # the largest positions there are
    ((-1, 2 ** 31 - 50), [-2 ** 31, 2 ** 31 - 1, -2 ** 31 + 60, 0]),
    ((2 ** 31 + 2 ** 20, 2 ** 62), [2 ** 31 - 1, -2 ** 31, 0, 2 ** 26]),     # finite, and beyond every position
])
def test_positions_and_windows_of_any_size(cuda_device, window, starts, sinks, Sq):
    q = _randn(cuda_device, 1, 4, Sq, 256).to(F16)
    k, v = (_randn(cuda_device, i, 4, 260, 128).to(F16) for i in (2, 3))
    q_start = torch.tensor(starts, dtype=torch.int32, device=cuda_device)
    out = ops.window_attention(q, k, v, 4, 2, window=window, sinks=sinks, q_start=q_start)
    seen = visible(Sq, 260, window, sinks, [260] * 4, starts, cuda_device)
    check(out, *reference(q, k, v, 4, 2, seen))
    assert bool((out[~seen.any(-1)] == 0).all())


# ---------------------------------------------------------------------------------------------------- first tokens, read left to right
def causal(seen, q_start, right, dev):
    """`seen` without the keys beyond each query's position + right."""
    Sq, Sk = seen.shape[1:]
    pos = torch.arange(Sq, device=dev)[None, :, None] + torch.tensor(q_start, device=dev)[:, None, None]
    return seen & (torch.arange(Sk, device=dev) <= pos + right)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("left", [0, 20, 100, -1])
@pytest.mark.parametrize("sinks", [1, 4, 64])
def test_a_text_in_one_call_is_the_text_token_by_token(cuda_device, sinks, left, dtype):
    """One call over 200 tokens, pieces of them against the cache so far, and single tokens: every row sees the same keys, so each
    is within its bound of the one exact result."""
    n, heads, kv_heads = 200, 4, 2
    q = _randn(cuda_device, sinks, 1, n, heads * 64).to(dtype)
    k, v = (_randn(cuda_device, sinks + i, 1, n, kv_heads * 64).to(dtype) for i in (1, 2))
    seen = causal(visible(n, n, (left, 0), sinks, [n], [0], cuda_device), [0], 0, cuda_device)
    want, bound = reference(q, k, v, heads, kv_heads, seen)
    kw = {"window": (left, 0), "sinks": sinks, "causal_sinks": True}
    check(ops.window_attention(q, k, v, heads, kv_heads, **kw), want, bound)
    for step in (1, 7, 70):                                  # single tokens and seven in the form for a few, 70 in tiles
        for at in range(0, n, step):
            end = min(n, at + step)
            length = torch.tensor([end], dtype=torch.int32, device=cuda_device)
            start = torch.tensor([at], dtype=torch.int32, device=cuda_device)
            k2, v2 = k.clone(), v.clone()
            k2[:, end:], v2[:, end:] = math.nan, math.nan    # not there yet
            out = ops.window_attention(q[:, at:end], k2, v2, heads, kv_heads, kv_len=length, q_start=start, **kw)
            check(out, want[:, at:end], bound[:, at:end])


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("Sq", [1, 6, 25, 60, 300])   # 2, 12, 50 rows (two blocks) in the form for a few, the others in tiles
@pytest.mark.parametrize("window,sinks,starts", [
    ((5, 0), 64, [0, 30, 63, 64, 200]), ((40, 3), 50, [0, 44, 49, 52, 300]), ((-1, 0), 200, [0, 100, 199, 250, -20]), ((3, 0), 97, [90, 96, 97, 101, 500]),
    ((0, 0), 300, [-400, -2, 0, 299, 10 ** 6]), ((10, -1), 20, [0, 5, 600, -100, 19]), ((2 ** 27, 2 ** 26), 9, [-2 ** 26, -2 ** 26 + 4, 2 ** 26, 0, -2 ** 27])])
def test_causal_first_tokens_at_their_edges(cuda_device, window, sinks, starts, Sq, masked):
    Sk, lens = 600, [600, 599, 600, 70, 600]
    q = _randn(cuda_device, Sq, 5, Sq, 256).to(F16)
    k, v = (_randn(cuda_device, Sq + i, 5, Sk, 128).to(F16) for i in (1, 2))
    seen = visible(Sq, Sk, window, sinks, lens, starts, cuda_device)
    if window[1] >= 0:
        seen = causal(seen, starts, window[1], cuda_device)
    mask = None
    if masked:
        mask = torch.zeros(5, Sk, device=cuda_device)
        mask[:, 3::5] = -10000.0
        seen = seen & (mask > -5000)[:, None]
    out = ops.window_attention(q, k, v, 4, 2, window=window, sinks=sinks, mask_add=mask, causal_sinks=True,
                               kv_len=torch.tensor(lens, dtype=torch.int32, device=cuda_device),
                               q_start=torch.tensor(starts, dtype=torch.int32, device=cuda_device))
    check(out, *reference(q, k, v, 4, 2, seen))
    assert bool((out[~seen.any(-1)] == 0).all())


@pytest.mark.parametrize("Sq", [1, 200])
def test_keys_of_later_tokens_leave_the_first_row_alone(cuda_device, Sq):
    q, k, v = (_randn(cuda_device, i, 1, 200, 128).to(F16) for i in range(3))
    kw = {"window": (64, 0), "sinks": 4, "causal_sinks": True}
    first = ops.window_attention(q[:, :Sq], k, v, 2, **kw)[0, 0]
    k[:, 1:] = math.nan
    if Sq == 1:
        v[:, 1:] = math.nan                                  # (values that another query of the call sees have to be finite)
    else:
        v[:, 1:] = 60000.0
    assert torch.equal(ops.window_attention(q[:, :Sq], k, v, 2, **kw)[0, 0], first)
    want, bound = reference(q[:, :1], k[:, :1], v[:, :1], 2, 2, torch.ones(1, 1, 1, dtype=torch.bool, device=cuda_device))
    check(first[None, None], want, bound)


def test_encoder_with_causal_first_tokens(cuda_device):
    """A stack over a text and over a prefix of it agree on the prefix, bit for bit in tiles that do not depend on the length."""
    from tnn_b200.encoder import Encoder
    from tnn_b200.model_synth import EncoderConfig, make_workload
    wl = make_workload(EncoderConfig(2, 256, 4, 512), 1, 300, seed=3, length_range=(300, 300), num_layers=2)
    x = torch.from_numpy(wl.x).to(cuda_device)
    for fp8 in (True, False):
        enc = Encoder.from_workload(wl, F16, cuda_device, fp8=fp8, window=(40, 0), sinks=4, causal_sinks=True)
        whole = enc.forward(x)
        later = x.clone()
        later[:, 2:] += 1.0                                  # a change behind the first two tokens
        assert torch.equal(enc.forward(later)[:, :2], whole[:, :2])
        assert not torch.equal(enc.forward(later)[:, 2:4], whole[:, 2:4])


# ---------------------------------------------------------------------------------------------------- layouts
@pytest.mark.parametrize("B,Sq,Sk", [(3, 150, 150), (3, 1, 400), (5, 40, 333), (2, 6, 90)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_sequences_side_by_side(cuda_device, B, Sq, Sk, dtype):
    """`[S, B, width]` tensors, seen as `[B, S, width]`: the stride from one sequence to the next is the smaller one."""
    q = _randn(cuda_device, 1, Sq, B, 256).to(dtype)
    k, v = (_randn(cuda_device, i, Sk, B, 128).to(dtype) for i in (2, 3))
    starts, lens = [Sk - Sq - b for b in range(B)], [Sk - b for b in range(B)]
    kw = {"window": (64, 3), "sinks": 2, "q_start": torch.tensor(starts, dtype=torch.int32, device=cuda_device),
          "kv_len": torch.tensor(lens, dtype=torch.int32, device=cuda_device)}
    back = torch.full((Sq + 2, B, 272), 7.0, dtype=dtype, device=cuda_device)
    views = [t.transpose(0, 1) for t in (q, k, v)]
    got = ops.window_attention(*views, 4, 2, out=back[1:Sq + 1, :, :256].transpose(0, 1), **kw)
    check(got, *reference(*views, 4, 2, visible(Sq, Sk, (64, 3), 2, lens, starts, cuda_device)))
    assert torch.equal(got, ops.window_attention(*(t.contiguous() for t in views), 4, 2, **kw))
    assert bool((back[0] == 7).all()) and bool((back[-1] == 7).all()) and bool((back[..., 256:] == 7).all())


def test_an_output_whose_rows_overlap_is_refused(cuda_device):
    q = torch.zeros(2, 5, 128, dtype=F16, device=cuda_device)
    for strides in ((256, 128, 1), (64, 128, 1), (512, 128, 1), (128, 248, 1), (120, 256, 1)):
        out = torch.empty(5000, dtype=F16, device=cuda_device).as_strided((2, 5, 128), strides)
        with pytest.raises(capi.B200Error):
            ops.window_attention(q, q, q, 2, out=out)


@pytest.mark.parametrize("Sq", [1, 25, 130])
def test_causal_first_tokens_captured_and_on_two_streams(cuda_device, Sq):
    k, v = (_randn(cuda_device, i, 2, 500, 128).to(F16) for i in (1, 2))
    cases = [(_randn(cuda_device, 5 + i, 2, Sq, 256).to(F16), s) for i, s in enumerate(([0, 3], [300, 40], [2 ** 30, -50]))]
    start = lambda s: torch.tensor(s, dtype=torch.int32, device=cuda_device)   # noqa: E731

    def call(q, s):
        return ops.window_attention(q, k, v, 4, 2, window=(30, 0), sinks=70, q_start=s, causal_sinks=True)

    want = [call(q, start(s)) for q, s in cases]
    for (q, s), w in zip(cases, want):
        seen = causal(visible(Sq, 500, (30, 0), 70, [500, 500], s, cuda_device), s, 0, cuda_device)
        check(w, *reference(q, k, v, 4, 2, seen))
    q0, s0 = cases[0][0].clone(), start(cases[0][1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(q0, s0)
    side = torch.cuda.Stream()
    for (q, s), w in zip(cases, want):
        q0.copy_(q)
        s0.copy_(start(s))
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            eager = call(q0, s0)
        torch.cuda.synchronize()
        assert torch.equal(out, w) and torch.equal(eager, w)
