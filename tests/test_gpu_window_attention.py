"""GPU: sliding-window attention with first tokens that stay visible, against a plain implementation in 64 bits."""
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


def visible(B, Sq, Sk, window, sinks, kv_len, q_start, mask, dev):
    j = torch.arange(Sk, device=dev)
    pos = torch.arange(Sq, device=dev)[None, :, None] + (0 if q_start is None else q_start.long()[:, None, None])
    seen = torch.ones(B, Sq, Sk, dtype=torch.bool, device=dev)
    if window[0] >= 0:
        seen &= j >= pos - window[0]
    if window[1] >= 0:
        seen &= j <= pos + window[1]
    seen |= j < sinks
    if kv_len is not None:
        seen &= j < kv_len.long()[:, None, None]
    if mask is not None:
        seen &= (mask > -5000.0)[:, None, :]
    return seen


def reference(q, k, v, heads, kv_heads, window, sinks, mask=None, kv_len=None, q_start=None, scale=0.125):
    """(result, bound on an element's error beside the result's own rounding), fp64 `[B, Sq, heads * 64]`."""
    B, Sq, Sk, dt = q.shape[0], q.shape[1], k.shape[1], q.dtype
    seen = visible(B, Sq, Sk, window, sinks, kv_len, q_start, mask, q.device)
    used = seen.any(1)                                        # keys that no query of the sequence sees may hold anything
    split = lambda t, n: t.double().reshape(B, t.shape[1], n, 64).transpose(1, 2)   # noqa: E731
    qq = split(q, heads)
    kk = split(torch.where(used[..., None], k, 0), kv_heads).repeat_interleave(heads // kv_heads, 1)
    vv = split(torch.where(used[..., None], v, 0), kv_heads).repeat_interleave(heads // kv_heads, 1)
    s = qq @ kk.transpose(-1, -2) * scale
    if mask is not None:
        s = s + torch.where(mask > -5000.0, mask, 0).double()[:, None, None, :]
    s = torch.where(seen[:, None], s, -math.inf)
    p = torch.where(seen.any(-1)[:, None, :, None], s.softmax(-1), 0.0)
    size = p @ vv.abs()
    # weights are rounded to the half type once; a score is a sum of 64 products in fp32 (whole steps where the tensor core
    # truncates) and its error is the weight's relative one, in numerator and denominator; ex2.approx 2^-22; weights below
    # f16's range lose at most 2^-25 of the largest
    score = 2 * 66 * 2.0 ** -23 * abs(scale) * float((qq.abs() @ kk.abs().transpose(-1, -2)).amax()) + 2.0 ** -21
    if mask is not None:
        score += 4 * 2.0 ** -23 * float(torch.where(mask > -5000.0, mask, 0).abs().max())
    tiny = Sk * 2.0 ** -25 * float(vv.abs().amax()) if dt == F16 else 0.0
    bound = size * (HALF_STEP[dt] * (1 + 2.0 ** -6) + score + (Sk + 64) * 2.0 ** -23) + tiny
    merge = lambda t: t.transpose(1, 2).reshape(B, Sq, heads * 64)   # noqa: E731
    return merge(p @ vv), merge(bound), seen


def check(out, want, bound):
    err = (out.double() - want).abs()
    limit = HALF_STEP[out.dtype] * (want.abs() + bound) + bound + 2.0 ** -24
    assert bool((err <= limit).all()), "largest excess %g" % float((err - limit).max())


def run(dev, B, Sq, Sk, heads, kv_heads, window, sinks, dtype, lens=None, starts=None, mask=None, seed=0):
    q = _randn(dev, seed + 1, B, Sq, heads * 64).to(dtype)
    k = _randn(dev, seed + 2, B, Sk, kv_heads * 64).to(dtype)
    v = _randn(dev, seed + 3, B, Sk, kv_heads * 64).to(dtype)
    kv_len = None if lens is None else torch.tensor(lens, dtype=torch.int32, device=dev)
    q_start = None if starts is None else torch.tensor(starts, dtype=torch.int32, device=dev)
    out = ops.window_attention(q, k, v, heads, kv_heads, window=window, sinks=sinks, mask_add=mask, kv_len=kv_len, q_start=q_start)
    want, bound, seen = reference(q, k, v, heads, kv_heads, window, sinks, mask, kv_len, q_start)
    check(out, want, bound)
    empty = ~seen.any(-1)
    assert bool((out[empty] == 0).all())
    return q, k, v, kv_len, q_start, out


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("S,window,sinks", [
    (1, (0, 0), 0), (2, (1, 1), 0), (31, (3, 0), 1), (127, (16, 16), 4), (128, (128, 128), 0), (129, (0, 0), 0), (130, (-1, -1), 0),
    (200, (33, 0), 33), (256, (64, 64), 1), (257, (0, 5), 200), (384, (-1, 0), 0), (500, (0, -1), 7), (640, (127, 129), 128),
    (777, (200, 100), 300), (1000, (255, 0), 4), (1100, (5000, 5000), 3), (600, (0, 0), 600)])
def test_self_attention_windows(cuda_device, S, window, sinks, dtype):
    run(cuda_device, 2, S, S, 2, 2, window, sinks, dtype, seed=S)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("window,sinks", [((142, 142), 16), ((6, 6), 1), ((2, 2), 40), ((30, 3), 70), ((17, 0), 96), ((100, 60), 33), ((0, 31), 97), ((3, 0), 95)])
def test_first_tokens_behind_a_short_last_tile(cuda_device, window, sinks, masked, dtype):
    mask = None
    if masked:
        mask = torch.zeros(3, 700, device=cuda_device)
        mask[:, [1, 30, 31, 32, 69, 500]] = -10000.0
        mask[:, 0], mask[:, 2::7] = 1.5, -2.0
    q, k, v, kv_len, _, out = run(cuda_device, 3, 700, 700, 2, 1, window, sinks, dtype, lens=[700, 433, 20], mask=mask, seed=sinks)
    # at the end of a cache: places between the first tokens and the windows may hold anything
    starts = torch.tensor([500, 400, 300], dtype=torch.int32, device=cuda_device)
    clean = ops.window_attention(q[:, :150], k, v, 2, 1, window=window, sinks=sinks, q_start=starts, mask_add=mask)
    k, v = k.clone(), v.clone()
    k[:, sinks:300 - window[0]], v[:, sinks:300 - window[0]] = math.nan, math.inf
    assert torch.equal(ops.window_attention(q[:, :150], k, v, 2, 1, window=window, sinks=sinks, q_start=starts, mask_add=mask), clean)


@pytest.mark.parametrize("heads,kv_heads", [(4, 4), (4, 2), (4, 1), (6, 3)])
@pytest.mark.parametrize("window,sinks", [((100, 100), 2), ((50, 0), 0)])
def test_grouped_heads_and_ragged_lengths(cuda_device, heads, kv_heads, window, sinks):
    run(cuda_device, 5, 333, 333, heads, kv_heads, window, sinks, F16, lens=[333, 0, 1, 130, 257], seed=heads * 10 + kv_heads)


def test_lengths_out_of_range_are_clamped(cuda_device):
    a = run(cuda_device, 3, 200, 200, 2, 2, (64, 64), 1, F16, lens=[200, 0, 200])
    kv = torch.tensor([1000, -3, 200], dtype=torch.int32, device=cuda_device)
    b = ops.window_attention(a[0], a[1], a[2], 2, window=(64, 64), sinks=1, kv_len=kv)
    assert torch.equal(a[5], b)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("Sq,Sk,window,sinks,lens", [
    (1, 1, (0, 0), 0, [1, 1]), (1, 70, (-1, 0), 0, [70, 33]), (1, 1000, (255, 0), 4, [1000, 17]), (1, 3000, (1023, 0), 16, [2999, 1500]),
    (2, 600, (100, 0), 1, [600, 2]), (5, 500, (64, 0), 0, [500, 5]), (8, 300, (10, 10), 2, [300, 200]), (16, 1500, (700, 0), 64, [1500, 900]),
    (40, 900, (300, 0), 4, [900, 41]), (130, 700, (128, 0), 5, [700, 130]), (3, 400, (1, 0), 390, [400, 395])])
@pytest.mark.parametrize("heads,kv_heads", [(4, 4), (8, 2), (12, 1)])
def test_new_tokens_against_a_cache(cuda_device, Sq, Sk, window, sinks, lens, heads, kv_heads, dtype):
    run(cuda_device, 2, Sq, Sk, heads, kv_heads, window, sinks, dtype, lens=lens, starts=[n - Sq for n in lens], seed=Sq + Sk)


@pytest.mark.parametrize("Sq", [1, 4, 150])
def test_positions_before_the_first_and_beyond_the_last_key(cuda_device, Sq):
    """A window that lies wholly outside the keys leaves the first tokens, or, without them, nothing."""
    for sinks in (0, 3):
        run(cuda_device, 4, Sq, 260, 2, 2, (20, 5), sinks, F16, lens=[260, 260, 260, 100], starts=[-400, 255, 2000, 130], seed=sinks)


@pytest.mark.parametrize("Sq,Sk", [(300, 300), (1, 300), (3, 700)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_additive_mask_with_holes(cuda_device, Sq, Sk, dtype):
    g = torch.Generator(device="cpu").manual_seed(Sq + Sk)
    mask = torch.where(torch.rand(3, Sk, generator=g) < 0.3, -10000.0, 0.0)
    mask[1] += torch.randn(Sk, generator=g) * (mask[1] == 0)
    mask[2, : Sk // 2] = -math.inf
    mask[2, Sk // 2] = torch.finfo(torch.float32).min
    starts = None if Sq == Sk else [Sk - Sq] * 3
    run(cuda_device, 3, Sq, Sk, 4, 2, (90, 40), 8, dtype, lens=[Sk, Sk - 37, Sk], starts=starts, mask=mask.to(cuda_device))


@pytest.mark.parametrize("Sq", [1, 2, 200])
def test_every_key_dropped_gives_zeros(cuda_device, Sq):
    mask = torch.full((2, 200), -10000.0, device=cuda_device)
    out = run(cuda_device, 2, Sq, 200, 2, 1, (-1, -1), 4, F16, mask=mask)[5]
    assert bool((out == 0).all())


@pytest.mark.parametrize("Sq,Sk", [(300, 300), (1, 900), (6, 500)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_places_that_nobody_may_see_hold_nan_and_infinities(cuda_device, Sq, Sk, dtype):
    lens = [Sk - 113, Sk - 1, 40]
    starts = None if Sq == Sk else [n - Sq for n in lens]
    q, k, v, kv_len, q_start, out = run(cuda_device, 3, Sq, Sk, 4, 2, (150, 0), 5, dtype, lens=lens, starts=starts)
    for bad in (math.nan, math.inf, -math.inf):
        k2, v2 = k.clone(), v.clone()
        for b, n in enumerate(lens):
            k2[b, n:], v2[b, n:] = bad, bad
        got = ops.window_attention(q, k2, v2, 4, 2, window=(150, 0), sinks=5, kv_len=kv_len, q_start=q_start)
        assert torch.equal(got, out)
    # dropped by the mask, in the middle of what is visible
    mask = torch.zeros(3, Sk, device=cuda_device)
    mask[:, 20:37] = -10000.0
    mask[:, 3] = math.nan
    clean = ops.window_attention(q, k, v, 4, 2, window=(150, 0), sinks=5, kv_len=kv_len, q_start=q_start, mask_add=mask)
    k2, v2 = k.clone(), v.clone()
    k2[:, 20:37], v2[:, 20:37], v2[:, 3] = math.nan, math.inf, math.nan
    got = ops.window_attention(q, k2, v2, 4, 2, window=(150, 0), sinks=5, kv_len=kv_len, q_start=q_start, mask_add=mask)
    assert torch.equal(got, clean)


@pytest.mark.parametrize("Sq", [1, 7, 70, 200])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_cache_places_outside_every_window_hold_nan(cuda_device, Sq, dtype):
    """Places given up behind the window and not yet written in front of it, with no kv_len to say so."""
    starts = [611, 333, 0]
    q, k, v, _, q_start, out = run(cuda_device, 3, Sq, 1000, 4, 2, (100, 0), 3, dtype, starts=starts)
    k2, v2 = k.clone(), v.clone()
    for b, p in enumerate(starts):
        k2[b, 3:max(3, p - 100)], v2[b, 3:max(3, p - 100)] = math.nan, math.nan
        k2[b, max(3, p + Sq):], v2[b, max(3, p + Sq):] = math.inf, math.nan
    assert torch.equal(ops.window_attention(q, k2, v2, 4, 2, window=(100, 0), sinks=3, q_start=q_start), out)


@pytest.mark.parametrize("Sq", [1, 150])
def test_masks_of_the_lowest_value_with_no_threshold(cuda_device, Sq):
    q, k, v = (_randn(cuda_device, i, 3, n, 128).half() for i, n in enumerate((Sq, 300, 300)))
    lowest = torch.finfo(torch.float32).min
    mask = torch.zeros(3, 300, device=cuda_device)
    mask[0], mask[1, 100:] = lowest, lowest
    mask[2], mask[2, 7], mask[2, 9] = -math.inf, -2.0 ** 126, -2.0 ** 126     # the only keys left: equal masks, of any size
    out = ops.window_attention(q, k, v, 2, mask_add=mask, exclude_below=-math.inf)
    assert bool((out[0] == 0).all())
    drop = torch.zeros(3, 300, device=cuda_device)
    drop[1, 100:] = -10000.0
    drop[0], drop[2] = -10000.0, -10000.0
    want, bound, _ = reference(q, k, v, 2, 2, (-1, -1), 0, drop)
    check(out[1], want[1], bound[1])
    # scores vanish beside 2^126, so the two weigh the same
    mean = v[2, [7, 9]].double().mean(0)
    assert bool(((out[2].double() - mean).abs() <= HALF_STEP[F16] * mean.abs() + 2.0 ** -24).all())


@pytest.mark.parametrize("Sq,Sk", [(150, 150), (1, 600)])
def test_packed_views_strided_cache_and_what_lies_around_the_output(cuda_device, Sq, Sk):
    heads, kv_heads, B = 4, 2, 3
    H, Hk = heads * 64, kv_heads * 64
    cache = _randn(cuda_device, 1, B + 1, Sk + 9, 2 * Hk + 64).to(F16)
    k, v = cache[:B, 4:4 + Sk, :Hk], cache[:B, 4:4 + Sk, Hk:2 * Hk]
    q = _randn(cuda_device, 2, B, Sq, 3 * H).to(F16)[..., H:2 * H]
    back = torch.full((B, Sq + 2, H + 16), 7.0, dtype=F16, device=cuda_device)
    starts = torch.full((B,), Sk - Sq, dtype=torch.int32, device=cuda_device)
    got = ops.window_attention(q, k, v, heads, kv_heads, window=(100, 0), sinks=3, q_start=starts, out=back[:, 1:Sq + 1, :H])
    want = ops.window_attention(q.contiguous(), k.contiguous(), v.contiguous(), heads, kv_heads, window=(100, 0), sinks=3, q_start=starts)
    assert torch.equal(got, want)
    assert bool((back[:, 0] == 7).all()) and bool((back[:, -1] == 7).all()) and bool((back[..., H:] == 7).all())


def test_large_scores_move_the_running_maximum(cuda_device):
    """Scores that grow along the keys make every tile move the maximum; equal ones never do."""
    B, S = 1, 700
    q = torch.ones(B, S, 64, device=cuda_device).to(F16)
    v = _randn(cuda_device, 1, B, S, 64).to(F16)
    for step in (0.02, -0.02, 0.0):
        k = (torch.arange(S, device=cuda_device)[None, :, None] * step).expand(B, S, 64).to(F16).contiguous()
        for Sq in (S, 1):
            st = torch.tensor([S - Sq], dtype=torch.int32, device=cuda_device)
            out = ops.window_attention(q[:, :Sq], k, v, 1, window=(-1, -1), q_start=st)
            want, bound, _ = reference(q[:, :Sq].contiguous(), k, v, 1, 1, (-1, -1), 0, q_start=st)
            check(out, want, bound)


@pytest.mark.parametrize("scale", [1.0, 0.03, 0.0, -0.125])
def test_scales(cuda_device, scale):
    q, k, v = (_randn(cuda_device, i, 1, 300, 128).to(BF16) for i in range(3))
    for n in (300, 2):
        out = ops.window_attention(q[:, :n], k, v, 2, window=(100, 100), sinks=2, scale=scale)
        want, bound, _ = reference(q[:, :n], k, v, 2, 2, (100, 100), 2, scale=scale)
        check(out, want, bound)


def test_a_sequence_does_not_depend_on_its_batch(cuda_device):
    B, S, heads = 6, 400, 4
    q, k, v = (_randn(cuda_device, i, B, S, heads * 64).to(F16) for i in range(3))
    lens = torch.tensor([400, 10, 399, 256, 128, 1], dtype=torch.int32, device=cuda_device)
    for Sq in (S, 1):
        st = lens - Sq if Sq == 1 else None
        out = ops.window_attention(q[:, :Sq], k, v, heads, window=(90, 30), sinks=2, kv_len=lens, q_start=st)
        for b in range(B):
            one = ops.window_attention(q[b:b + 1, :Sq], k[b:b + 1], v[b:b + 1], heads, window=(90, 30), sinks=2, kv_len=lens[b:b + 1],
                                       q_start=None if st is None else st[b:b + 1])
            if Sq == S:
                assert torch.equal(one[0], out[b])
            else:                                             # the number of CTAs that share a sequence's keys may differ
                want, bound, _ = reference(q[b:b + 1, :1], k[b:b + 1], v[b:b + 1], heads, heads, (90, 30), 2, None, lens[b:b + 1], st[b:b + 1])
                check(one, want, bound)


def test_many_items_per_cta(cuda_device):
    """More items than resident CTAs, of unequal length, some without a key."""
    lens = [300, 0, 17, 128, 299, 1, 64, 0, 250, 33] * 4
    run(cuda_device, 40, 300, 300, 6, 2, (70, 20), 1, F16, lens=lens)


def test_captured_replayed_and_on_another_stream(cuda_device):
    B, heads = 2, 4
    k, v = (_randn(cuda_device, i, B, 700, heads * 64).to(F16) for i in (1, 2))
    for Sq in (1, 160):
        qs = [_randn(cuda_device, 5 + i, B, Sq, heads * 64).to(F16) for i in range(3)]
        lens = [torch.tensor(t, dtype=torch.int32, device=cuda_device) for t in ([700, 300], [161, 700], [200, 699])]

        def call(q, n):
            return ops.window_attention(q, k, v, heads, window=(200, 0), sinks=4, kv_len=n, q_start=n - Sq)

        want = [call(q, n).clone() for q, n in zip(qs, lens)]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = call(qs[1], lens[1])
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(got, want[1])
        q0, n0 = qs[0].clone(), lens[0].clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call(q0, n0)
        for q, n, w in zip(qs, lens, want):
            q0.copy_(q)
            n0.copy_(n)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, w)


def test_full_window_agrees_with_attention(cuda_device):
    """An unlimited window over full sequences is what `attention` computes."""
    B, S, heads = 2, 384, 4
    qkv = _randn(cuda_device, 3, B, S, 3 * heads * 64).to(F16)
    H = heads * 64
    a = ops.attention(qkv, heads)
    b = ops.window_attention(qkv[..., :H], qkv[..., H:2 * H], qkv[..., 2 * H:], heads)
    want, bound, _ = reference(qkv[..., :H], qkv[..., H:2 * H], qkv[..., 2 * H:], heads, heads, (-1, -1), 0)
    check(a, want, bound)
    check(b, want, bound)


def test_empty_calls(cuda_device):
    q = torch.zeros(2, 0, 64, dtype=F16, device=cuda_device)
    k = torch.zeros(2, 5, 64, dtype=F16, device=cuda_device)
    assert ops.window_attention(q, k, k, 1).shape == (2, 0, 64)
    assert ops.window_attention(k[:0], k[:0], k[:0], 1).shape == (0, 5, 64)


@pytest.mark.parametrize("Sq", [1, 100])
def test_places_beyond_2_31_elements_of_a_cache(cuda_device, Sq):
    Sk, first = 4_400_000, 4
    cache = torch.empty(2, Sk, 256, dtype=F16, device=cuda_device)            # 4.5 GB, keys and values side by side
    q_start = torch.tensor([Sk - Sq, Sk - Sq - 1000], dtype=torch.int32, device=cuda_device)
    q = _randn(cuda_device, 1, 2, Sq, 64).half()
    kv = []
    for b, p in enumerate(q_start.tolist()):
        places = torch.cat([torch.arange(first), torch.arange(p - 300, p + Sq)]).to(cuda_device)
        rows = _randn(cuda_device, 2 + b, len(places), 256).half()
        cache[b, places] = rows
        kv.append(rows)
    out = ops.window_attention(q, cache[..., :64], cache[..., 64:128], 1, window=(300, 0), sinks=first, kv_len=q_start + Sq, q_start=q_start)
    near = torch.stack(kv)                                                    # the same, with nothing in between
    starts = torch.full((2,), first + 300, dtype=torch.int32, device=cuda_device)
    want, bound, _ = reference(q, near[..., :64], near[..., 64:128], 1, 1, (300, 0), first, q_start=starts)
    check(out, want, bound)
