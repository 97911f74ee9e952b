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


def _rows(t, width, at_least=0, written=False):
    """`t` as rows of `width` elements: (tensor that holds them, number of rows, row stride).  A contiguous tensor, the
    usual one, needs no view of its own: making views costs more than filling a descriptor.  What does not divide into
    such rows is refused by `reshape`; so are fewer than `at_least` rows, which a kernel would reach beyond, and, where the
    kernel writes, what could only be copied: the results would be lost with the copy."""
    if t.is_contiguous() and width and t.numel() % width == 0:
        rows, ld = t.numel() // width, width
    else:
        given, t = t, t.reshape(-1, width)
        assert t.stride(1) == 1 and not (written and t.data_ptr() != given.data_ptr()), "out: rows that need no copy"
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
    y2, _, ldy = _rows(out, N, M, True)
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
    y2, _, ldy = _rows(out, H, rows, True)
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
_F8 = torch.float8_e4m3fn
_entry = {}       # entry points by name: looking one up in the library object costs more than in a dict


def _call(name, desc, index):
    """Launch `name` on the current stream of device `index`, the one the tensors are on, whichever device is current."""
    fn = _entry.get(name)
    if fn is None:
        fn = _entry[name] = getattr(capi.lib(), name)
    if index == torch.cuda.current_device():
        rc = fn(ctypes.byref(desc), capi.stream_ptr(index))
    else:
        with torch.cuda.device(index):
            rc = fn(ctypes.byref(desc), capi.stream_ptr(index))
    if rc != capi.OK:
        capi.check(rc, name)


def _device_index(x, *ts):
    """The one CUDA device of all these tensors."""
    index = x.get_device()
    for t in ts:
        if t is not None and t.get_device() != index:
            raise ValueError("tensors on different devices")
    if index < 0:
        _require_cuda(x)
    return index


def _new(rows, cols, dtype, device):
    """Uninitialised contiguous matrix (empty_strided costs 1.5 us of host time, empty 2.4)."""
    return torch.empty_strided((rows, cols), (cols, 1), dtype=dtype, device=device)


def _new_like(x, dtype):
    """Uninitialised contiguous tensor of x's shape."""
    if x.is_contiguous():
        return torch.empty_like(x, dtype=dtype)
    return torch.empty(x.shape, dtype=dtype, device=x.device)


def _vector(t, n, what):
    if t is not None and not (t.dtype == torch.float32 and t.numel() == n and t.is_contiguous()):
        raise ValueError("%s: fp32, %d contiguous values" % (what, n))


def _blocks(n):
    return -(-n // FP8_BLOCK)


def _scale_rows(scale, blocks, rows, what):
    """Row stride of a `[blocks, rows]` fp32 scale array."""
    if scale.dtype != torch.float32 or scale.shape != (blocks, rows):
        raise ValueError("%s: fp32 [%d, %d]" % (what, blocks, rows))
    if scale.is_contiguous():
        return rows
    if (rows > 1 and scale.stride(1) != 1) or (blocks > 1 and scale.stride(0) < rows):
        raise ValueError("%s: contiguous rows that do not overlap" % what)
    return scale.stride(0) if blocks > 1 else rows


def _codes(t, shape, what):
    if t.dtype != _F8 or t.shape != shape:
        raise ValueError("%s: float8_e4m3fn %s" % (what, tuple(shape)))


def _out_rows(t, width, rows, what):
    """`t` as exactly `rows` rows of `width` contiguous elements that the kernel may write: (address, row stride).  A view is
    needed, never a copy: results written to a copy would be lost."""
    if not t.is_contiguous():
        try:
            t = t.view(-1, width)
        except RuntimeError:
            raise ValueError("%s: cannot be seen as rows of %d without a copy" % (what, width)) from None
        if t.shape[0] != rows or t.stride(1) != 1 or (rows > 1 and t.stride(0) < width):
            raise ValueError("%s: %d rows of %d" % (what, rows, width))
        return t.data_ptr(), (t.stride(0) if rows > 1 else width)
    if t.numel() != rows * width:
        raise ValueError("%s: %d rows of %d" % (what, rows, width))
    return t.data_ptr(), width


def quantize_fp8(x, out=None, out_scale=None):
    """x `[..., K]` (f16, bf16 or f32) -> (codes `[..., K]` float8_e4m3fn, scales fp32 `[ceil(K/128), rows]`).  A value
    stands for code * scale of its row and block of 128 columns (include/tnn_b200.h has the exact rounding)."""
    index = _device_index(x, out, out_scale)
    K = x.shape[-1]
    blocks = _blocks(K)
    x2, rows, ldx = _rows(x, K)
    if out is None:
        out = _new_like(x, _F8)
        q, ldq = out.data_ptr(), K
    else:
        _codes(out, x.shape, "out")
        q, ldq = _out_rows(out, K, rows, "out")
    if out_scale is None:
        out_scale = _new(blocks, rows, torch.float32, x.device)
        lds = rows
    else:
        lds = _scale_rows(out_scale, blocks, rows, "out_scale")
    d = capi.QuantizeFp8Desc(x2.data_ptr(), q, out_scale.data_ptr(), rows, K, ldx, ldq, lds, capi.dtype_code(x.dtype))
    if rows:
        _call("b200_quantize_fp8", d, index)
    return out, out_scale


def pack_weight_fp8(w_kn, out=None, out_scale=None):
    """fp32 `[K, N]` (TNN MatMul weight layout, y = x.W) -> (codes `[N, K]` float8_e4m3fn, fp32 scales per 128 x 128 block
    `[ceil(N/128), ceil(K/128)]`) for `linear_fp8`."""
    index = _device_index(w_kn, out, out_scale)
    if w_kn.dtype != torch.float32 or w_kn.dim() != 2 or w_kn.stride(1) != 1:
        raise ValueError("w_kn: fp32 [K, N], contiguous columns")
    K, N = w_kn.shape
    if out is None:
        out = _new(N, K, _F8, w_kn.device)
    _codes(out, (N, K), "out")
    w, ldw = _out_rows(out, K, N, "out")
    if out_scale is None:
        out_scale = _new(_blocks(N), _blocks(K), torch.float32, w_kn.device)
    if out_scale.dtype != torch.float32 or out_scale.shape != (_blocks(N), _blocks(K)) or not out_scale.is_contiguous():
        raise ValueError("out_scale: contiguous fp32 [%d, %d]" % (_blocks(N), _blocks(K)))
    with torch.cuda.device(index):
        rc = capi.lib().b200_pack_weight_fp8(w_kn.data_ptr(), K, N, w_kn.stride(0) if K > 1 else N, w, ldw, out_scale.data_ptr(),
                                             capi.stream_ptr())
    capi.check(rc, "b200_pack_weight_fp8")
    return out, out_scale


def add_layernorm_fp8(x, gamma, beta, eps, residual=None, out=None, out8=None, out_scale=None, half=True):
    """(residual +) LayerNorm whose result leaves as `(y in x's dtype, codes, scales)`: `add_layernorm` and `quantize_fp8`
    of its fp32 result in one pass.  `half=False`: codes and scales only (y is None)."""
    index = _device_index(x, gamma, beta, residual, out, out8, out_scale)
    H = x.shape[-1]
    blocks = _blocks(H)
    _vector(gamma, H, "gamma")
    _vector(beta, H, "beta")
    x2, rows, ldx = _rows(x, H)
    y, ldy = None, 0
    if out is not None:
        if not half or out.dtype != x.dtype:
            raise ValueError("out: the dtype of x, and none with half=False")
        y, ldy = _out_rows(out, H, rows, "out")
    elif half:
        out = _new_like(x, x.dtype)
        y, ldy = out.data_ptr(), H
    if out8 is None:
        out8 = _new_like(x, _F8)
        q, ldq = out8.data_ptr(), H
    else:
        _codes(out8, x.shape, "out8")
        q, ldq = _out_rows(out8, H, rows, "out8")
    if out_scale is None:
        out_scale = _new(blocks, rows, torch.float32, x.device)
        lds = rows
    else:
        lds = _scale_rows(out_scale, blocks, rows, "out_scale")
    r, ldr = None, 0
    if residual is not None:
        if residual.dtype != x.dtype:
            raise ValueError("residual: the dtype of x")
        r2, _, ldr = _rows(residual, H, rows)
        r = r2.data_ptr()
    d = capi.LayerNormFp8Desc(x2.data_ptr(), r, gamma.data_ptr(), beta.data_ptr(), y, q, out_scale.data_ptr(), rows, H, ldx, ldr, ldy,
                              ldq, lds, capi.dtype_code(x.dtype), eps)
    if rows:
        _call("b200_add_layernorm_fp8_fwd", d, index)
    return out, out8, out_scale


def linear_fp8(x8, x_scale, w8, w_scale, bias=None, residual=None, epilogue=EPI_BIAS, out_dtype=torch.float16, out=None,
               out_scale=None, block_n=0):
    """y = epilogue(x . w^T + bias (+ residual)) on block-scaled e4m3 operands: x8 `[..., K]` with x_scale
    `[ceil(K/128), rows]` (`quantize_fp8`), w8 `[N, K]` with w_scale (`pack_weight_fp8`).  `out_dtype` f16, bf16 or f32
    returns y `[..., N]`; float8_e4m3fn returns (codes, scales `[ceil(N/128), rows]`) for another `linear_fp8`."""
    index = _device_index(x8, x_scale, w8, w_scale, bias, residual, out, out_scale)
    N, K = w8.shape
    if x8.dtype != _F8 or w8.dtype != _F8 or x8.shape[-1] != K:
        raise ValueError("x8 [..., K], w8 [N, K]: float8_e4m3fn")
    if w8.is_contiguous():
        ldw = K
    elif w8.stride(1) == 1 and (N <= 1 or w8.stride(0) >= K):
        ldw = w8.stride(0) if N > 1 else K
    else:
        raise ValueError("w8: [N, K] with contiguous rows")
    kb, nb = -(-K // FP8_BLOCK), -(-N // FP8_BLOCK)
    if w_scale.dtype != torch.float32 or w_scale.shape != (nb, kb) or not w_scale.is_contiguous():
        raise ValueError("w_scale: contiguous fp32 [%d, %d]" % (nb, kb))
    _vector(bias, N, "bias")
    x2, M, ldx = _rows(x8, K)
    ldxs = _scale_rows(x_scale, kb, M, "x_scale")
    if out is not None:
        out_dtype = out.dtype
        y, ldy = _out_rows(out, N, M, "out")
    else:
        out = (_new(M, N, out_dtype, x8.device) if x8.dim() == 2
               else torch.empty(x8.shape[:-1] + (N,), dtype=out_dtype, device=x8.device))
        y, ldy = out.data_ptr(), N
    f8 = out_dtype == _F8
    ys, ldys = None, 0
    if f8:
        if out_scale is None:
            out_scale = _new(nb, M, torch.float32, x8.device)
        ldys = _scale_rows(out_scale, nb, M, "out_scale")
        ys = out_scale.data_ptr()
    r, ldr, r_code = None, 0, capi.F16
    if residual is not None:
        if epilogue != EPI_BIAS_RESIDUAL or residual.dtype not in (torch.float16, torch.bfloat16):
            raise ValueError("residual: f16 or bf16, with epilogue=EPI_BIAS_RESIDUAL")
        r2, _, ldr = _rows(residual, N, M)
        r, r_code = r2.data_ptr(), capi.dtype_code(residual.dtype)
    d = capi.LinearFp8Desc(x2.data_ptr(), w8.data_ptr(), x_scale.data_ptr(), w_scale.data_ptr(), capi.ptr(bias), r, y, ys, M, N, K,
                           ldx, ldw, ldr, ldy, ldxs, ldys, capi.E4M3 if f8 else capi.dtype_code(out_dtype), r_code, epilogue, block_n)
    if M:
        _call("b200_linear_fp8_fwd", d, index)
    return (out, out_scale) if f8 else out


# ---------------------------------------------------------------------------- sliding-window attention
def _heads_view(t, S, W, what):
    """(row stride, batch stride) of a `[B, S, W]` tensor whose heads lie side by side (strides of single rows or sequences mean
    nothing)."""
    if t.is_contiguous():
        return W, S * W
    batch, ld, one = t.stride()
    if one != 1:
        raise ValueError("%s: contiguous heads" % what)
    if S <= 1:
        ld = W
    return ld, (batch if t.shape[0] > 1 else S * ld)


def _per_sequence(t, B, what):
    if t is not None and not (t.dtype == torch.int32 and t.numel() == B and t.is_contiguous()):
        raise ValueError("%s: int32 [%d]" % (what, B))


def window_attention(q, k, v, heads, kv_heads=None, window=(-1, -1), sinks=0, mask_add=None, kv_len=None, q_start=None,
                     scale=None, exclude_below=-5000.0, out=None, causal_sinks=False):
    """Attention of q `[B, Sq, heads*64]` over k, v `[B, Sk, kv_heads*64]` (views of a packed QKV activation will do) ->
    `[B, Sq, heads*64]`.  A query at position p sees the keys j < kv_len with j < sinks or p - left <= j <= p + right,
    `window` = (left, right), negative = unlimited on that side.  `causal_sinks`: j <= p + right for the first keys too; a text
    read left to right (right = 0) with more than one of them needs it, or its first queries see tokens behind themselves.

    kv_len `[B]` int32: keys of each sequence (None: all Sk).  q_start `[B]` int32: position of each sequence's first query
    (None: 0); Sq new tokens at the end of a cache have q_start = kv_len - Sq.  mask_add fp32 `[B, Sk]`: additive key mask, a
    key at or below `exclude_below` is dropped.  A query that sees no key yields zeros; keys and values that no query may see
    (outside every window, beyond kv_len, or dropped) may hold anything."""
    if kv_heads is None:
        kv_heads = heads
    index = _device_index(q, k, v, mask_add, kv_len, q_start, out)
    if heads <= 0 or kv_heads <= 0 or heads % kv_heads or sinks < 0:
        raise ValueError("kv_heads divides heads, sinks >= 0")
    dtype = q.dtype
    if k.dtype != dtype or v.dtype != dtype:
        raise ValueError("q, k, v: one dtype")
    W, Wk = heads * 64, kv_heads * 64
    if q.dim() != 3 or k.dim() != 3:
        raise ValueError("q [B, Sq, %d], k, v [B, Sk, %d]" % (W, Wk))
    B, Sq, Wq = q.shape
    Bk, Sk, W_k = k.shape
    if Wq != W or W_k != Wk or Bk != B or v.shape != k.shape:
        raise ValueError("q [B, Sq, %d], k, v [B, Sk, %d]" % (W, Wk))
    ldq, q_batch = _heads_view(q, Sq, W, "q")
    ldk, k_batch = _heads_view(k, Sk, Wk, "k")
    ldv, v_batch = _heads_view(v, Sk, Wk, "v")
    _per_sequence(kv_len, B, "kv_len")
    _per_sequence(q_start, B, "q_start")
    if out is None:
        out = torch.empty_strided((B, Sq, W), (Sq * W, W, 1), dtype=dtype, device=q.device)
        ldo, o_batch = W, Sq * W
    else:
        if out.dtype != dtype or out.shape != q.shape:
            raise ValueError("out: the dtype and shape of q")
        ldo, o_batch = _heads_view(out, Sq, W, "out")
    if mask_add is not None and not (mask_add.dtype == torch.float32 and mask_add.numel() == B * Sk and mask_add.is_contiguous()):
        raise ValueError("mask_add: contiguous fp32 [%d, %d]" % (B, Sk))
    d = capi.WindowAttentionDesc(q.data_ptr(), k.data_ptr(), v.data_ptr(), capi.ptr(mask_add), capi.ptr(kv_len), capi.ptr(q_start),
                                 out.data_ptr(), B, Sq, Sk, ldq, ldk, ldv, ldo, q_batch, k_batch, v_batch, o_batch, window[0],
                                 window[1], sinks, heads, kv_heads, 64, capi.dtype_code(dtype), 0.125 if scale is None else scale,
                                 exclude_below, 1 if causal_sinks else 0)
    if B and Sq:
        _call("b200_window_attention_fwd", d, index)
    return out
