"""Host-side operator wrappers over the C ABI: one function per fused layer of the path.

Names and argument meaning follow the fused TNN layers (FusedLinear, FusedAttention, LayerNorm) that the graph pass
emits; tensors are torch CUDA tensors used as device buffers.  Every function launches through `extern "C"` entry
points of libtnn_b200.so on the current torch stream; nothing here computes with torch.
"""
import ctypes

import torch

from . import capi
from .capi import EPI_BIAS, EPI_BIAS_GELU, EPI_BIAS_RESIDUAL, EPI_BIAS_TANH  # noqa: F401


def _require_cuda(*ts):
    for t in ts:
        if t is not None and not t.is_cuda:
            raise ValueError("tnn_b200 operators take CUDA tensors only (there is no CPU path)")


def _rows(t, width, at_least=0):
    """`t` as rows of `width` elements: (tensor that holds them, number of rows, row stride).  A contiguous tensor, the
    usual one, needs no view of its own: making views costs more than filling a descriptor.  What does not divide into
    such rows is refused by `reshape`; so are fewer than `at_least` rows, which a kernel would reach beyond."""
    if t.is_contiguous() and width and t.numel() % width == 0:
        rows, ld = t.numel() // width, width
    else:
        t = t.reshape(-1, width)
        assert t.stride(1) == 1
        rows, ld = t.shape[0], t.stride(0)
    assert rows >= at_least, "fewer rows than the input has"
    return t, rows, ld


def pack_weight(w_kn, dtype=torch.float16, out=None):
    """fp32 `[K, N]` (TNN MatMul weight layout, y = x.W) -> `dtype` `[N, K]` on the device."""
    _require_cuda(w_kn)
    assert w_kn.dtype == torch.float32 and w_kn.dim() == 2 and w_kn.stride(1) == 1
    K, N = w_kn.shape
    if out is None:
        out = torch.empty((N, K), dtype=dtype, device=w_kn.device)
    assert out.shape[0] == N and out.shape[1] == K and out.stride(1) == 1
    rc = capi.lib().b200_pack_weight(w_kn.data_ptr(), K, N, w_kn.stride(0), out.data_ptr(), out.stride(0),
                                     capi.dtype_code(out.dtype), capi.stream_ptr())
    capi.check(rc, "b200_pack_weight")
    return out


def fold_layernorm_weight(w_kn, gamma, beta, bias=None, dtype=torch.float16, out=None):
    """For y = LayerNorm(x; gamma, beta).W + bias: returns (w_nk with gamma folded in, c1, c2), see include/tnn_b200.h."""
    _require_cuda(w_kn, gamma, beta, bias)
    K, N = w_kn.shape
    if out is None:
        out = torch.empty((N, K), dtype=dtype, device=w_kn.device)
    c1 = torch.empty((N,), dtype=torch.float32, device=w_kn.device)
    c2 = torch.empty((N,), dtype=torch.float32, device=w_kn.device)
    rc = capi.lib().b200_fold_layernorm_weight(w_kn.data_ptr(), K, N, w_kn.stride(0), gamma.data_ptr(),
                                               beta.data_ptr(), capi.ptr(bias), out.data_ptr(), out.stride(0),
                                               capi.dtype_code(out.dtype), c1.data_ptr(), c2.data_ptr(),
                                               capi.stream_ptr())
    capi.check(rc, "b200_fold_layernorm_weight")
    return out, c1, c2


def stats_buffer(rows, width, device):
    """Row-statistics buffer of a `[rows, width]` activation: `[ceil(width/32), rows, 2]` fp32."""
    return torch.empty(((width + 31) // 32, rows, 2), dtype=torch.float32, device=device)


def convert(src, dtype, out=None):
    _require_cuda(src)
    assert src.is_contiguous()
    if out is None:
        out = torch.empty(src.shape, dtype=dtype, device=src.device)
    assert out.is_contiguous() and out.numel() == src.numel()
    rc = capi.lib().b200_convert(src.data_ptr(), capi.dtype_code(src.dtype), out.data_ptr(),
                                 capi.dtype_code(out.dtype), src.numel(), capi.stream_ptr())
    capi.check(rc, "b200_convert")
    return out


def _linear_desc(x, w_nk, bias, residual, epilogue, out_dtype, out, block_n, out_stats=None, ln_in=None, res_ln=None,
                 ln_eps=1e-12):
    _require_cuda(x, w_nk, bias, residual, out)
    K = x.shape[-1]
    N = w_nk.shape[0]
    assert w_nk.shape[1] == K and w_nk.stride(1) == 1
    x2, M, ldx = _rows(x, K)
    if out is None:
        out = torch.empty(x.shape[:-1] + (N,), dtype=out_dtype or x.dtype, device=x.device)
    y2, _, ldy = _rows(out, N, M)
    d = capi.LinearDesc(x2.data_ptr(), w_nk.data_ptr(), capi.ptr(bias), None, y2.data_ptr(), M, N, K, ldx,
                        w_nk.stride(0), 0, ldy, capi.dtype_code(x.dtype), capi.dtype_code(out.dtype), epilogue, block_n)
    if residual is not None:
        assert residual.dtype == x.dtype
        r2, _, d.ldr = _rows(residual, N, M)
        d.residual = r2.data_ptr()
    # LayerNorm folding: ln_in = (stats of x, c1, c2); res_ln = (stats of residual, gamma, beta)
    d.ln_eps = float(ln_eps)
    if out_stats is not None:
        d.out_stats = out_stats.data_ptr()
    if ln_in is not None:
        d.ln_in_stats, d.ln_c1, d.ln_c2 = (t.data_ptr() for t in ln_in)
    if res_ln is not None:
        d.res_ln_stats, d.res_ln_gamma, d.res_ln_beta = (t.data_ptr() for t in res_ln)
    return d, out


def linear(x, w_nk, bias=None, residual=None, epilogue=EPI_BIAS, out_dtype=None, out=None, block_n=0,
           out_stats=None, ln_in=None, res_ln=None, ln_eps=1e-12):
    """y[M,N] = epilogue(x[M,K] . w_nk[N,K]^T + bias (+ residual)); x may be `[..., K]`."""
    d, out = _linear_desc(x, w_nk, bias, residual, epilogue, out_dtype, out, block_n, out_stats, ln_in, res_ln, ln_eps)
    rc = capi.lib().b200_linear_fwd(ctypes.byref(d), capi.stream_ptr())
    capi.check(rc, "b200_linear_fwd")
    return out


def mask_to_kv_len(mask_add, exclude_below=-5000.0, out=None):
    """mask_add fp32 `[B, S]` (or `[B,1,1,S]`) -> int32 `[B]`."""
    _require_cuda(mask_add)
    S = mask_add.shape[-1]
    m2 = mask_add.reshape(-1, S)
    assert m2.is_contiguous() and m2.dtype == torch.float32
    if out is None:
        out = torch.empty((m2.shape[0],), dtype=torch.int32, device=mask_add.device)
    rc = capi.lib().b200_mask_to_kv_len(m2.data_ptr(), m2.shape[0], S, exclude_below, out.data_ptr(),
                                        capi.stream_ptr())
    capi.check(rc, "b200_mask_to_kv_len")
    return out


def attention(qkv, heads, mask_add=None, kv_len=None, scale=None, exclude_below=-5000.0, out=None):
    """qkv `[B, S, 3*heads*64]` packed (Q | K | V along the last axis) -> context `[B, S, heads*64]`."""
    _require_cuda(qkv, mask_add, kv_len, out)
    B, S, W = qkv.shape
    H = heads * 64
    assert W == 3 * H and qkv.stride(2) == 1 and qkv.stride(0) == S * qkv.stride(1)
    if out is None:
        out = torch.empty((B, S, H), dtype=qkv.dtype, device=qkv.device)
    es = qkv.element_size()
    q = qkv.data_ptr()
    ld = qkv.stride(1)
    d = capi.AttentionDesc(q, q + H * es, q + 2 * H * es, None, None, out.data_ptr(), B, S, ld, ld, ld, out.stride(1), heads,
                           64, capi.dtype_code(qkv.dtype), 0.125 if scale is None else float(scale), float(exclude_below))
    if mask_add is not None:
        m2 = mask_add if mask_add.is_contiguous() and mask_add.numel() == B * S else mask_add.reshape(B, S)
        assert m2.is_contiguous() and m2.dtype == torch.float32
        d.mask_add = m2.data_ptr()
    if kv_len is not None:
        assert kv_len.dtype == torch.int32 and kv_len.numel() == B
        d.kv_len = kv_len.data_ptr()
    rc = capi.lib().b200_attention_fwd(ctypes.byref(d), capi.stream_ptr())
    capi.check(rc, "b200_attention_fwd")
    return out


def _layernorm_desc(x, gamma, beta, eps, residual, out_dtype, out):
    _require_cuda(x, gamma, beta, residual, out)
    H = x.shape[-1]
    assert gamma.dtype == torch.float32 and beta.dtype == torch.float32
    x2, rows, ldx = _rows(x, H)
    if out is None:
        out = torch.empty(x.shape, dtype=out_dtype or x.dtype, device=x.device)
    y2, _, ldy = _rows(out, H, rows)
    d = capi.LayerNormDesc(x2.data_ptr(), None, gamma.data_ptr(), beta.data_ptr(), y2.data_ptr(), rows, H, ldx, 0, ldy,
                           capi.dtype_code(x.dtype), capi.dtype_code(out.dtype), float(eps))
    if residual is not None:
        assert residual.dtype == x.dtype
        r2, _, d.ldr = _rows(residual, H, rows)
        d.residual = r2.data_ptr()
    return d, out


def add_layernorm(x, gamma, beta, eps, residual=None, out_dtype=None, out=None):
    d, out = _layernorm_desc(x, gamma, beta, eps, residual, out_dtype, out)
    rc = capi.lib().b200_add_layernorm_fwd(ctypes.byref(d), capi.stream_ptr())
    capi.check(rc, "b200_add_layernorm_fwd")
    return out


def embedding_layernorm(input_ids, segment_ids, word_emb, type_emb, pos_emb, gamma, beta, eps, out_dtype=torch.float16,
                        out=None):
    """`[B,S]` int32 ids (+ segment ids or None) -> LayerNorm(word + segment + position embeddings) `[B,S,H]`."""
    _require_cuda(input_ids, segment_ids, word_emb, type_emb, pos_emb, gamma, beta, out)
    B, S = input_ids.shape
    H = word_emb.shape[1]
    assert input_ids.dtype == torch.int32 and input_ids.is_contiguous()
    assert word_emb.stride(1) == 1 and pos_emb.dtype == word_emb.dtype and pos_emb.shape[0] >= S
    assert pos_emb.stride(0) == word_emb.stride(0)
    if out is None:
        out = torch.empty((B, S, H), dtype=out_dtype, device=input_ids.device)
    d = capi.EmbeddingDesc()
    d.input_ids, d.word_emb, d.pos_emb = input_ids.data_ptr(), word_emb.data_ptr(), pos_emb.data_ptr()
    if segment_ids is not None:
        assert segment_ids.dtype == torch.int32 and segment_ids.is_contiguous() and type_emb is not None
        assert type_emb.dtype == word_emb.dtype and type_emb.stride(0) == word_emb.stride(0)
        d.segment_ids, d.type_emb, d.type_vocab = segment_ids.data_ptr(), type_emb.data_ptr(), type_emb.shape[0]
    d.gamma, d.beta, d.out = gamma.data_ptr(), beta.data_ptr(), out.data_ptr()
    d.B, d.S, d.H, d.vocab = B, S, H, word_emb.shape[0]
    d.ld_table, d.ld_out = word_emb.stride(0), out.reshape(-1, H).stride(0)
    d.table_dtype, d.out_dtype, d.eps = capi.dtype_code(word_emb.dtype), capi.dtype_code(out.dtype), float(eps)
    rc = capi.lib().b200_embedding_layernorm_fwd(ctypes.byref(d), capi.stream_ptr())
    capi.check(rc, "b200_embedding_layernorm_fwd")
    return out


def mask_from_input_mask(input_mask, masked_value=-10000.0, exclude_below=-5000.0, out_mask=None, out_kv_len=None):
    """int32 0/1 `[B,S]` -> (additive fp32 mask `[B,S]`, int32 kv_len `[B]`), into the given buffers if any."""
    _require_cuda(input_mask, out_mask, out_kv_len)
    B, S = input_mask.shape
    assert input_mask.dtype == torch.int32 and input_mask.is_contiguous()
    mask_add = out_mask if out_mask is not None else torch.empty((B, S), dtype=torch.float32, device=input_mask.device)
    kv_len = out_kv_len if out_kv_len is not None else torch.empty((B,), dtype=torch.int32, device=input_mask.device)
    assert mask_add.dtype == torch.float32 and mask_add.is_contiguous() and mask_add.numel() == B * S
    assert kv_len.dtype == torch.int32 and kv_len.numel() == B
    rc = capi.lib().b200_mask_from_input_mask(input_mask.data_ptr(), B, S, masked_value, exclude_below,
                                              mask_add.data_ptr(), kv_len.data_ptr(), capi.stream_ptr())
    capi.check(rc, "b200_mask_from_input_mask")
    return mask_add, kv_len


def qa_head(x, weight, bias=None, out=None):
    """Span-extraction head: `x` `[..., H]` half precision, `weight` fp32 `[H, N]` (N <= 4), `bias` fp32 `[N]` or None
    -> fp32 `[N, M]` (M = tokens): row n is output n of every token (the graph's `unstack:n`)."""
    _require_cuda(x, weight, bias, out)
    H = x.shape[-1]
    x2 = x.reshape(-1, H)
    M, N = x2.shape[0], weight.shape[1]
    assert weight.dtype == torch.float32 and weight.is_contiguous() and weight.shape[0] == H and x2.stride(1) == 1
    if out is None:
        out = torch.empty((N, M), dtype=torch.float32, device=x.device)
    d = capi.QAHeadDesc()
    d.x, d.weight, d.out = x2.data_ptr(), weight.data_ptr(), out.data_ptr()
    if bias is not None:
        assert bias.dtype == torch.float32 and bias.numel() == N
        d.bias = bias.data_ptr()
    d.M, d.H, d.N = M, H, N
    d.ldx, d.ld_out, d.x_dtype = x2.stride(0), out.stride(0), capi.dtype_code(x.dtype)
    rc = capi.lib().b200_qa_head_fwd(ctypes.byref(d), capi.stream_ptr())
    capi.check(rc, "b200_qa_head_fwd")
    return out


# ---------------------------------------------------------------------------- 8-bit operands with block scales
FP8_BLOCK = 128   # consecutive values of a row that share a scale


def _call(name, desc, device):
    """Launch `name` on the current stream of the device the tensors are on, whichever device is current."""
    fn = getattr(capi.lib(), name)
    if device.index == torch.cuda.current_device():
        rc = fn(ctypes.byref(desc), capi.stream_ptr())
    else:
        with torch.cuda.device(device):
            rc = fn(ctypes.byref(desc), capi.stream_ptr())
    capi.check(rc, name)


def _check(ok, what):
    if not ok:
        raise ValueError(what)


def _same_device(x, *ts):
    _require_cuda(x, *ts)
    for t in ts:
        _check(t is None or t.device == x.device, "tensors on different devices")


def _vector(t, n, what):
    _check(t is None or (t.dtype == torch.float32 and t.numel() == n and t.is_contiguous()),
           "%s: fp32, %d contiguous values" % (what, n))


def _blocks(n):
    return -(-n // FP8_BLOCK)


def _scale_rows(scale, blocks, rows, what):
    """Row stride of a `[blocks, rows]` fp32 scale array."""
    _check(scale.dtype == torch.float32 and tuple(scale.shape) == (blocks, rows) and (rows <= 1 or scale.stride(1) == 1),
           "%s: fp32 [%d, %d] with contiguous rows" % (what, blocks, rows))
    ld = scale.stride(0) if blocks > 1 else rows
    _check(ld >= rows, "%s: overlapping rows" % what)
    return ld


def _codes(t, shape, what):
    _check(t.dtype == torch.float8_e4m3fn and tuple(t.shape) == tuple(shape), "%s: float8_e4m3fn %s" % (what, tuple(shape)))


def _out_rows(t, width, rows, what):
    """`t` as exactly `rows` rows of `width` contiguous elements that the kernel may write: (tensor, row stride).  A view is
    needed, never a copy: results written to a copy would be lost."""
    if t.is_contiguous():
        _check(t.numel() == rows * width, "%s: %d rows of %d" % (what, rows, width))
        return t, width
    try:
        t = t.view(-1, width)
    except RuntimeError:
        raise ValueError("%s: cannot be seen as rows of %d without a copy" % (what, width)) from None
    _check(t.shape[0] == rows and t.stride(1) == 1 and (rows <= 1 or t.stride(0) >= width), "%s: %d rows of %d" % (what, rows, width))
    return t, t.stride(0)


def quantize_fp8(x, out=None, out_scale=None):
    """x `[..., K]` (f16, bf16 or f32) -> (codes `[..., K]` float8_e4m3fn, scales fp32 `[ceil(K/128), rows]`).  A value
    stands for code * scale of its row and block of 128 columns (include/tnn_b200.h has the exact rounding)."""
    _same_device(x, out, out_scale)
    K = x.shape[-1]
    x2, rows, ldx = _rows(x, K)
    if out is None:
        out = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=x.device)
    _codes(out, x.shape, "out")
    q2, ldq = _out_rows(out, K, rows, "out")
    if out_scale is None:
        out_scale = torch.empty((_blocks(K), rows), dtype=torch.float32, device=x.device)
    d = capi.QuantizeFp8Desc(x2.data_ptr(), q2.data_ptr(), out_scale.data_ptr(), rows, K, ldx, ldq,
                             _scale_rows(out_scale, _blocks(K), rows, "out_scale"), capi.dtype_code(x.dtype))
    if rows:
        _call("b200_quantize_fp8", d, x.device)
    return out, out_scale


def pack_weight_fp8(w_kn, out=None, out_scale=None):
    """fp32 `[K, N]` (TNN MatMul weight layout, y = x.W) -> (codes `[N, K]` float8_e4m3fn, fp32 scales per 128 x 128 block
    `[ceil(N/128), ceil(K/128)]`) for `linear_fp8`."""
    _same_device(w_kn, out, out_scale)
    _check(w_kn.dtype == torch.float32 and w_kn.dim() == 2 and w_kn.stride(1) == 1, "w_kn: fp32 [K, N], contiguous columns")
    K, N = w_kn.shape
    if out is None:
        out = torch.empty((N, K), dtype=torch.float8_e4m3fn, device=w_kn.device)
    if out_scale is None:
        out_scale = torch.empty((_blocks(N), _blocks(K)), dtype=torch.float32, device=w_kn.device)
    _codes(out, (N, K), "out")
    _check(out.stride(1) == 1 and out.stride(0) >= K, "out: contiguous rows")
    _check(out_scale.dtype == torch.float32 and tuple(out_scale.shape) == (_blocks(N), _blocks(K)) and out_scale.is_contiguous(),
           "out_scale: contiguous fp32 [%d, %d]" % (_blocks(N), _blocks(K)))
    with torch.cuda.device(w_kn.device):
        rc = capi.lib().b200_pack_weight_fp8(w_kn.data_ptr(), K, N, w_kn.stride(0), out.data_ptr(), out.stride(0),
                                             out_scale.data_ptr(), capi.stream_ptr())
    capi.check(rc, "b200_pack_weight_fp8")
    return out, out_scale


def add_layernorm_fp8(x, gamma, beta, eps, residual=None, out=None, out8=None, out_scale=None, half=True):
    """(residual +) LayerNorm whose result leaves as `(y in x's dtype, codes, scales)`: `add_layernorm` and `quantize_fp8`
    of its fp32 result in one pass.  `half=False`: codes and scales only (y is None)."""
    _same_device(x, gamma, beta, residual, out, out8, out_scale)
    H = x.shape[-1]
    _vector(gamma, H, "gamma")
    _vector(beta, H, "beta")
    x2, rows, ldx = _rows(x, H)
    _check(out is None or half, "out is given but half=False")
    if out is None and half:
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if out8 is None:
        out8 = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=x.device)
    _codes(out8, x.shape, "out8")
    q2, ldq = _out_rows(out8, H, rows, "out8")
    if out_scale is None:
        out_scale = torch.empty((_blocks(H), rows), dtype=torch.float32, device=x.device)
    d = capi.LayerNormFp8Desc(x2.data_ptr(), None, gamma.data_ptr(), beta.data_ptr(), None, q2.data_ptr(), out_scale.data_ptr(),
                              rows, H, ldx, 0, 0, ldq, _scale_rows(out_scale, _blocks(H), rows, "out_scale"),
                              capi.dtype_code(x.dtype), float(eps))
    if out is not None:
        _check(out.dtype == x.dtype, "out: the dtype of x")
        y2, d.ldy = _out_rows(out, H, rows, "out")
        d.y = y2.data_ptr()
    if residual is not None:
        _check(residual.dtype == x.dtype, "residual: the dtype of x")
        r2, _, d.ldr = _rows(residual, H, rows)
        d.residual = r2.data_ptr()
    if rows:
        _call("b200_add_layernorm_fp8_fwd", d, x.device)
    return out, out8, out_scale


def linear_fp8(x8, x_scale, w8, w_scale, bias=None, residual=None, epilogue=EPI_BIAS, out_dtype=torch.float16, out=None,
               out_scale=None, block_n=0):
    """y = epilogue(x . w^T + bias (+ residual)) on block-scaled e4m3 operands: x8 `[..., K]` with x_scale
    `[ceil(K/128), rows]` (`quantize_fp8`), w8 `[N, K]` with w_scale (`pack_weight_fp8`).  `out_dtype` f16, bf16 or f32
    returns y `[..., N]`; float8_e4m3fn returns (codes, scales `[ceil(N/128), rows]`) for another `linear_fp8`."""
    _same_device(x8, x_scale, w8, w_scale, bias, residual, out, out_scale)
    K = x8.shape[-1]
    _check(x8.dtype == torch.float8_e4m3fn and w8.dtype == torch.float8_e4m3fn, "x8, w8: float8_e4m3fn")
    _check(w8.dim() == 2 and w8.shape[1] == K and w8.stride(1) == 1 and (w8.shape[0] <= 1 or w8.stride(0) >= K),
           "w8: [N, %d] with contiguous rows" % K)
    N = w8.shape[0]
    _check(w_scale.dtype == torch.float32 and tuple(w_scale.shape) == (_blocks(N), _blocks(K)) and w_scale.is_contiguous(),
           "w_scale: contiguous fp32 [%d, %d]" % (_blocks(N), _blocks(K)))
    _vector(bias, N, "bias")
    x2, M, ldx = _rows(x8, K)
    if out is not None:
        out_dtype = out.dtype
    else:
        out = torch.empty(x8.shape[:-1] + (N,), dtype=out_dtype, device=x8.device)
    f8 = out_dtype == torch.float8_e4m3fn
    y2, ldy = _out_rows(out, N, M, "out")
    d = capi.LinearFp8Desc(x2.data_ptr(), w8.data_ptr(), x_scale.data_ptr(), w_scale.data_ptr(), capi.ptr(bias), None,
                           y2.data_ptr(), None, M, N, K, ldx, w8.stride(0) if N > 1 else K, 0, ldy,
                           _scale_rows(x_scale, _blocks(K), M, "x_scale"), 0,
                           capi.E4M3 if f8 else capi.dtype_code(out_dtype), capi.F16, epilogue, block_n)
    if f8:
        if out_scale is None:
            out_scale = torch.empty((_blocks(N), M), dtype=torch.float32, device=x8.device)
        d.ld_y_scale = _scale_rows(out_scale, _blocks(N), M, "out_scale")
        d.y_scale = out_scale.data_ptr()
    if residual is not None:
        _check(epilogue == EPI_BIAS_RESIDUAL, "a residual needs epilogue=EPI_BIAS_RESIDUAL")
        _check(residual.dtype in (torch.float16, torch.bfloat16), "residual: f16 or bf16")
        r2, _, d.ldr = _rows(residual, N, M)
        d.residual, d.res_dtype = r2.data_ptr(), capi.dtype_code(residual.dtype)
    if M:
        _call("b200_linear_fp8_fwd", d, x8.device)
    return (out, out_scale) if f8 else out


# ---------------------------------------------------------------------------- sliding-window attention
def _heads_view(t, heads, what):
    """(row stride, batch stride) of a `[B, S, heads * 64]` tensor whose heads lie side by side."""
    _check(t.dim() == 3 and t.shape[2] == heads * 64 and t.stride(2) == 1, "%s: [B, S, %d], contiguous heads" % (what, heads * 64))
    ld = t.stride(1) if t.shape[1] > 1 else heads * 64
    return ld, (t.stride(0) if t.shape[0] > 1 else t.shape[1] * ld)


def _per_sequence(t, B, what):
    _check(t is None or (t.dtype == torch.int32 and t.numel() == B and t.is_contiguous()), "%s: int32 [%d]" % (what, B))


def window_attention(q, k, v, heads, kv_heads=None, window=(-1, -1), sinks=0, mask_add=None, kv_len=None, q_start=None,
                     scale=None, exclude_below=-5000.0, out=None):
    """Attention of q `[B, Sq, heads*64]` over k, v `[B, Sk, kv_heads*64]` (views of a packed QKV activation will do) ->
    `[B, Sq, heads*64]`.  A query at position p sees the keys j < kv_len with j < sinks or p - left <= j <= p + right,
    `window` = (left, right), negative = unlimited on that side.

    kv_len `[B]` int32: keys of each sequence (None: all Sk).  q_start `[B]` int32: position of each sequence's first query
    (None: 0); Sq new tokens at the end of a cache have q_start = kv_len - Sq.  mask_add fp32 `[B, Sk]`: additive key mask, a
    key at or below `exclude_below` is dropped.  A query that sees no key yields zeros; keys and values that no query may see
    (beyond kv_len, or dropped) may hold anything."""
    kv_heads = heads if kv_heads is None else kv_heads
    _same_device(q, k, v, mask_add, kv_len, q_start, out)
    _check(heads > 0 and kv_heads > 0 and heads % kv_heads == 0, "kv_heads divides heads")
    _check(q.dtype == k.dtype == v.dtype, "q, k, v: one dtype")
    _check(sinks >= 0, "sinks >= 0")
    ldq, q_batch = _heads_view(q, heads, "q")
    ldk, k_batch = _heads_view(k, kv_heads, "k")
    ldv, v_batch = _heads_view(v, kv_heads, "v")
    B, Sq, Sk = q.shape[0], q.shape[1], k.shape[1]
    _check(k.shape[:2] == v.shape[:2] and k.shape[0] == B, "k, v: [%d, Sk, ...]" % B)
    _per_sequence(kv_len, B, "kv_len")
    _per_sequence(q_start, B, "q_start")
    if out is None:
        out = torch.empty((B, Sq, heads * 64), dtype=q.dtype, device=q.device)
    _check(out.dtype == q.dtype and tuple(out.shape) == tuple(q.shape), "out: the dtype and shape of q")
    ldo, o_batch = _heads_view(out, heads, "out")
    m2 = None
    if mask_add is not None:
        _check(mask_add.dtype == torch.float32 and mask_add.numel() == B * Sk and mask_add.is_contiguous(),
               "mask_add: contiguous fp32 [%d, %d]" % (B, Sk))
        m2 = mask_add.data_ptr()
    d = capi.WindowAttentionDesc(q.data_ptr(), k.data_ptr(), v.data_ptr(), m2, capi.ptr(kv_len), capi.ptr(q_start), out.data_ptr(),
                                 B, Sq, Sk, ldq, ldk, ldv, ldo, q_batch, k_batch, v_batch, o_batch, window[0], window[1], sinks,
                                 heads, kv_heads, 64, capi.dtype_code(q.dtype), 0.125 if scale is None else float(scale),
                                 float(exclude_below))
    if B and Sq:
        _call("b200_window_attention_fwd", d, q.device)
    return out
