"""CPU: what the 8-bit operators and window attention refuse, at the C ABI (no launch happens: the descriptors are refused
before a device is looked at) and in the operator wrappers."""
import ctypes
import glob
import os
import re

import pytest
import torch

from tnn_b200 import capi, ops

F8 = torch.float8_e4m3fn
CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tnn_b200", "csrc")


def _fill(d, **kw):
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def _linear(**kw):
    d = capi.LinearFp8Desc()
    _fill(d, x=256, w_nk=256, x_scale=256, w_scale=256, y=256, M=10, N=64, K=128, ldx=128, ldw=128, ldy=64, ld_x_scale=10, out_dtype=capi.F16)
    return capi.lib().b200_linear_fp8_fwd(ctypes.byref(_fill(d, **kw)), None)


@pytest.mark.parametrize("kw", [
    dict(x=None), dict(w_nk=None), dict(x_scale=None), dict(w_scale=None), dict(y=None), dict(M=-1), dict(N=0), dict(K=0), dict(K=120),
    dict(N=60), dict(ldx=120), dict(ldx=136), dict(ldw=64), dict(ldy=56), dict(ldy=68), dict(ld_x_scale=9), dict(x=264), dict(w_nk=264),
    dict(y=264), dict(bias=260), dict(out_dtype=4), dict(out_dtype=-1), dict(epilogue=4), dict(epilogue=capi.EPI_BIAS_RESIDUAL),
    dict(epilogue=capi.EPI_BIAS_RESIDUAL, residual=256, ldr=56), dict(epilogue=capi.EPI_BIAS_RESIDUAL, residual=256, ldr=64, res_dtype=capi.F32),
    dict(out_dtype=capi.E4M3), dict(out_dtype=capi.E4M3, y_scale=256, ld_y_scale=9), dict(out_dtype=capi.E4M3, y_scale=256, ld_y_scale=10, N=56),
    dict(block_n=192), dict(block_n=-64), dict(block_n=-1, M=129, ld_x_scale=129), dict(block_n=64, out_dtype=capi.E4M3, y_scale=256, ld_y_scale=10)])
def test_linear_fp8_refuses(kw):
    assert _linear(**kw) == capi.ERR_PARAM


def test_sizes_beyond_the_kernels():
    assert _linear(K=(1 << 24) + 16, ldx=1 << 25, ldw=1 << 25) == capi.ERR_UNSUPPORTED
    assert _linear(M=0, ld_x_scale=0) == capi.OK                    # nothing to do
    assert _window(head_dim=128) == capi.ERR_UNSUPPORTED
    assert _window(B=70000) == capi.ERR_UNSUPPORTED
    assert _window(Sk=(1 << 24) + 1) == capi.ERR_UNSUPPORTED
    assert _window(Sq=0) == capi.OK and _window(B=0) == capi.OK
    assert _norm(H=4112, ldx=4112, ldy=4112, ldq=4112) == capi.ERR_UNSUPPORTED


def _quantize(**kw):
    d = _fill(capi.QuantizeFp8Desc(), x=256, q=256, scale=256, rows=3, K=128, ldx=128, ldq=128, ld_scale=3, x_dtype=capi.F16)
    return capi.lib().b200_quantize_fp8(ctypes.byref(_fill(d, **kw)), None)


@pytest.mark.parametrize("kw", [dict(x=None), dict(q=None), dict(scale=None), dict(rows=-1), dict(K=0), dict(K=120), dict(ldx=124), dict(ldx=120),
                                dict(ldq=120), dict(ldq=136), dict(ld_scale=2), dict(x=264), dict(q=264), dict(x_dtype=capi.E4M3), dict(x_dtype=-1)])
def test_quantize_refuses(kw):
    assert _quantize(**kw) == capi.ERR_PARAM


def _norm(**kw):
    d = _fill(capi.LayerNormFp8Desc(), x=256, gamma=256, beta=256, y=256, q=256, scale=256, rows=3, H=128, ldx=128, ldy=128, ldq=128, ld_scale=3,
              dtype=capi.F16)
    return capi.lib().b200_add_layernorm_fp8_fwd(ctypes.byref(_fill(d, **kw)), None)


@pytest.mark.parametrize("kw", [dict(x=None), dict(gamma=None), dict(beta=None), dict(q=None), dict(scale=None), dict(rows=-1), dict(H=0), dict(H=136),
                                dict(ldx=120), dict(ldy=120), dict(ldq=136), dict(ld_scale=2), dict(residual=256), dict(residual=264, ldr=128),
                                dict(dtype=capi.F32), dict(gamma=260), dict(q=260)])
def test_add_layernorm_fp8_refuses(kw):
    assert _norm(**kw) == capi.ERR_PARAM


def _window(**kw):
    d = _fill(capi.WindowAttentionDesc(), q=256, k=256, v=256, out=256, B=2, Sq=5, Sk=7, ldq=256, ldk=128, ldv=128, ldo=256, q_batch=1280,
              k_batch=896, v_batch=896, o_batch=1280, left=3, right=0, heads=4, kv_heads=2, head_dim=64, dtype=capi.F16, scale=0.125)
    return capi.lib().b200_window_attention_fwd(ctypes.byref(_fill(d, **kw)), None)


@pytest.mark.parametrize("kw", [dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(B=-1), dict(Sq=-1), dict(Sk=0), dict(heads=0),
                                dict(kv_heads=0), dict(kv_heads=3), dict(sinks=-1), dict(dtype=capi.F32), dict(dtype=capi.E4M3), dict(ldq=248),
                                dict(ldq=260), dict(ldk=120), dict(ldv=100), dict(ldo=248), dict(q_batch=1284), dict(k_batch=0), dict(v_batch=-8),
                                dict(o_batch=1024), dict(q=264), dict(k=264), dict(v=264), dict(out=264), dict(mask_add=256, mask_exclude_below=float("nan"))])
def test_window_attention_refuses(kw):
    assert _window(**kw) == capi.ERR_PARAM


def test_null_descriptors_and_pack_weight():
    l = capi.lib()
    for f in (l.b200_quantize_fp8, l.b200_add_layernorm_fp8_fwd, l.b200_linear_fp8_fwd, l.b200_window_attention_fwd):
        assert f(None, None) == capi.ERR_PARAM
    good = [256, 128, 64, 64, 256, 128, 256, None]
    for i, v in ((0, None), (4, None), (6, None), (1, 0), (1, 120), (2, 0), (3, 63), (5, 112), (5, 136), (4, 264)):
        assert l.b200_pack_weight_fp8(*[v if k == i else a for k, a in enumerate(good)]) == capi.ERR_PARAM


# ---------------------------------------------------------------------------------------------------- wrappers
@pytest.fixture
def launches(monkeypatch):
    """CPU tensors go through the wrappers' checks; what would be launched is recorded."""
    seen = []
    monkeypatch.setattr(ops, "_require_cuda", lambda *ts: None)
    monkeypatch.setattr(ops, "_call", lambda name, desc, index: seen.append((name, desc)))
    return seen


def _f8(*shape):
    return torch.zeros(shape, dtype=torch.uint8).view(F8)


def _scales(*shape):
    return torch.ones(shape)


def test_wrappers_refuse_cpu_tensors():
    for call in (lambda: ops.quantize_fp8(torch.zeros(2, 16)), lambda: ops.pack_weight_fp8(torch.zeros(16, 8)),
                 lambda: ops.window_attention(*[torch.zeros(1, 2, 64, dtype=torch.float16)] * 3, 1)):
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("kw", [
    dict(x8=torch.zeros(5, 256)), dict(w8=torch.zeros(64, 256)), dict(w8=_f8(64, 128)), dict(xs=_scales(2, 4)), dict(xs=_scales(5, 2)),
    dict(xs=_scales(2, 5).double()), dict(xs=_scales(5, 2).t()), dict(ws=_scales(1, 1)), dict(ws=_scales(2, 2)), dict(bias=torch.zeros(32)),
    dict(bias=torch.zeros(64).half()), dict(out=torch.zeros(5, 32).half()), dict(out=torch.zeros(4, 64).half()), dict(out=torch.zeros(64, 5).half().t()),
    dict(out_dtype=F8, out_scale=_scales(1, 4)), dict(residual=torch.zeros(5, 64)), dict(residual=torch.zeros(5, 64).half(), epilogue=ops.EPI_BIAS),
    dict(out_dtype=torch.int8)])
def test_linear_fp8_wrapper_refuses(launches, kw):
    a = dict(x8=_f8(5, 256), xs=_scales(2, 5), w8=_f8(64, 256), ws=_scales(1, 2), epilogue=ops.EPI_BIAS_RESIDUAL)
    a.update(kw)
    with pytest.raises((ValueError, AssertionError)):
        ops.linear_fp8(a.pop("x8"), a.pop("xs"), a.pop("w8"), a.pop("ws"), a.pop("bias", None), **a)
    assert not launches


def test_linear_fp8_wrapper_descriptor(launches):
    out = torch.zeros(2, 3, 80).half()[..., :64]
    scales = _scales(2, 9)[:, 1:7]
    ops.linear_fp8(_f8(2, 3, 256), scales, _f8(64, 272)[:, :256], _scales(1, 2), out=out)
    name, d = launches[0]
    assert name == "b200_linear_fp8_fwd"
    assert (d.M, d.N, d.K, d.ldx, d.ldw, d.ldy, d.ld_x_scale, d.out_dtype) == (6, 64, 256, 256, 272, 80, 9, capi.F16)
    assert (d.y, d.x_scale) == (out.data_ptr(), scales.data_ptr())
    y, s = ops.linear_fp8(_f8(6, 256), _scales(2, 6), _f8(272, 256), _scales(3, 2), out_dtype=F8)
    assert y.dtype == F8 and tuple(s.shape) == (3, 6) and launches[1][1].out_dtype == capi.E4M3


@pytest.mark.parametrize("kw", [dict(out=_f8(4, 256)), dict(out=torch.zeros(5, 256)), dict(out=_f8(256, 5).t()), dict(out_scale=_scales(2, 4)),
                                dict(out_scale=_scales(5, 2).t()), dict(x=torch.zeros(5, 256).double()), dict(x=torch.zeros(5, 256, dtype=torch.int32))])
def test_quantize_wrapper_refuses(launches, kw):
    a = dict(x=torch.zeros(5, 256).half())
    a.update(kw)
    with pytest.raises((ValueError, AssertionError)):
        ops.quantize_fp8(a.pop("x"), **a)
    assert not launches


@pytest.mark.parametrize("kw", [dict(gamma=torch.ones(128)), dict(gamma=torch.ones(256).half()), dict(out=torch.zeros(5, 256)), dict(out8=_f8(5, 128)),
                                dict(residual=torch.zeros(5, 256)), dict(residual=torch.zeros(4, 256).half()), dict(out=torch.zeros(5, 256).half(), half=False)])
def test_add_layernorm_fp8_wrapper_refuses(launches, kw):
    a = dict(gamma=torch.ones(256), beta=torch.zeros(256))
    a.update(kw)
    with pytest.raises((ValueError, AssertionError)):
        ops.add_layernorm_fp8(torch.zeros(5, 256).half(), a.pop("gamma"), a.pop("beta"), 1e-12, **a)
    assert not launches


@pytest.mark.parametrize("kw", [
    dict(q=torch.zeros(2, 5, 192).half()), dict(q=torch.zeros(2, 5, 256)), dict(k=torch.zeros(2, 6, 128).half()), dict(k=torch.zeros(1, 7, 128).half()),
    dict(k=torch.zeros(2, 7, 128).bfloat16()), dict(q=torch.zeros(2, 256, 5).half().transpose(1, 2)), dict(kv_heads=3), dict(kv_heads=0), dict(sinks=-1),
    dict(kv_len=torch.zeros(2)), dict(kv_len=torch.zeros(3, dtype=torch.int32)), dict(q_start=torch.zeros(2, dtype=torch.int64)),
    dict(mask_add=torch.zeros(2, 8)), dict(mask_add=torch.zeros(2, 7).half()), dict(out=torch.zeros(2, 5, 256)), dict(out=torch.zeros(2, 4, 256).half())])
def test_window_attention_wrapper_refuses(launches, kw):
    a = dict(q=torch.zeros(2, 5, 256).half(), k=torch.zeros(2, 7, 128).half(), v=torch.zeros(2, 7, 128).half(), kv_heads=2)
    a.update(kw)
    with pytest.raises(ValueError):
        ops.window_attention(a.pop("q"), a.pop("k"), a.pop("v"), 4, **a)
    assert not launches


def test_window_attention_wrapper_descriptor(launches):
    qkv = torch.zeros(2, 9, 512).half()
    ops.window_attention(qkv[..., :256], qkv[..., 256:384], qkv[..., 384:], 4, 2, window=(3, -1), sinks=2)
    d = launches[0][1]
    assert (d.B, d.Sq, d.Sk, d.ldq, d.ldk, d.ldv, d.ldo) == (2, 9, 9, 512, 512, 512, 256)
    assert (d.q_batch, d.k_batch, d.v_batch, d.o_batch) == (9 * 512, 9 * 512, 9 * 512, 9 * 256)
    assert (d.left, d.right, d.sinks, d.heads, d.kv_heads, d.scale) == (3, -1, 2, 4, 2, 0.125)
    assert (d.q, d.k, d.v) == tuple(qkv.data_ptr() + 2 * o for o in (0, 256, 384))


# ---------------------------------------------------------------------------------------------------- sources
@pytest.mark.parametrize("name", sorted(os.path.basename(f) for f in glob.glob(os.path.join(CSRC, "*.cu"))))
def test_every_commit_of_an_8_bit_kernel_stands_with_its_ummas(name):
    """The rule of test_kernel_sources.py (a commit covers the UMMAs of the thread that executes it) for umma_f8_commit."""
    with open(os.path.join(CSRC, name)) as f:
        text = re.sub(r"//[^\n]*", "", f.read())
    for m in re.finditer(r"\bumma_f8_commit\(", text):
        depth, i = 0, m.start()
        while depth >= 0:
            i -= 1
            depth += {"}": 1, "{": -1}.get(text[i], 0)
        assert re.search(r"\bumma_f8_ss(_pair)?\(", text[i:m.start()]), text[max(0, m.start() - 120):m.end() + 40]
