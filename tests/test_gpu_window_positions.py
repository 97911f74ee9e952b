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
