"""Host-side mirror of the fused encoder: packed device weights + the launch sequence of one Forward.

`Encoder.from_workload` does what the fused layers' `Init` does in the TNN plug-in: upload the fp32 `[K,N]` MatMul
weights, pre-pack them to half-precision `[N,K]` (Q/K/V concatenated into one `[3H,H]` operand), keep biases and
LayerNorm parameters in fp32.  `forward` is `Instance::Forward` for the fused graph: fp32 activations in, the fused
region in fp16/bf16, fp32 out.  All compute goes through the C ABI (tnn_b200.capi); there is no torch math here.
"""
import ctypes

import numpy as np
import torch

from . import capi, ops


class Encoder:
    def __init__(self, cfg, dtype, device):
        self.cfg = cfg
        self.dtype = dtype
        self.device = device
        self.layers = []          # dicts of device tensors (kept alive here)
        self._c_layers = None
        self._ws = None
        self._ws_key = None
        self.fold = False
        self.fp8 = False          # matrix weights in block-scaled e4m3
        self.window = None        # (left, right): sliding-window attention
        self.sinks = 0
        self.causal_sinks = False

    @classmethod
    def from_workload(cls, wl, dtype=torch.float16, device="cuda", fold_layernorm=False, fp8=False, window=None, sinks=0,
                      causal_sinks=False):
        """`fold_layernorm`: prepare the weights for the five-launch form of a layer (both LayerNorms folded into
        the neighbouring GEMMs); only full encoder layers can be folded.  Off by default: at BERT's K = 768 the
        seven-launch layer with its own LayerNorm kernel is the faster one, and it is what the TNN plug-in runs.

        For long documents: `fp8` keeps the matrix weights in e4m3 with a scale per 128 x 128 block and runs the four GEMMs
        of a layer on 8-bit operands (activations between launches stay in `dtype`, the feed-forward's inner one in 8 bits).
        It halves the bytes of the weights; at hidden sizes of 768 and 1024 a layer takes 1.2 to 1.5 times as long as in half
        precision.  `window=(left, right)` lets every token see that many neighbours and the first `sinks` tokens only.  A sequence whose
        keys are all masked then yields an attention output of zeros.  `causal_sinks` (for `right` = 0): a token sees no first
        token behind itself.  With a window, padding costs less as `kv_len` alone (`forward_hidden`) than as a mask."""
        enc = cls(wl.cfg, dtype, torch.device(device))
        enc.fold = bool(fold_layernorm) and wl.cfg.with_ffn
        enc.fp8, enc.window, enc.sinks, enc.causal_sinks = bool(fp8), window, int(sinks), bool(causal_sinks)
        if enc.fold and (enc.fp8 or window is not None):
            raise ValueError("fold_layernorm is a form of the half-precision, full-attention layer")
        H, F = wl.cfg.hidden, wl.cfg.ffn

        def dev(a):
            return torch.from_numpy(np.ascontiguousarray(a, dtype=np.float32)).to(enc.device)

        prev = None
        for lw in wl.weights:
            L = {}
            if enc.fp8:
                enc.layers.append(cls._fp8_layer(lw, wl.cfg, dev))
                continue
            w_qkv = torch.empty((3 * H, H), dtype=dtype, device=enc.device)
            L["b_qkv"] = dev(np.concatenate([lw.bq, lw.bk, lw.bv]))
            if enc.fold and prev is not None:
                # LN2 of the previous layer is folded into this layer's QKV projection
                w_cat = dev(np.concatenate([lw.wq, lw.wk, lw.wv], axis=1))
                _, L["qkv_c1"], L["qkv_c2"] = ops.fold_layernorm_weight(w_cat, prev["ln2_g"], prev["ln2_b"],
                                                                        L["b_qkv"], dtype, out=w_qkv)
            else:
                for i, w in enumerate((lw.wq, lw.wk, lw.wv)):
                    ops.pack_weight(dev(w), dtype, out=w_qkv[i * H:(i + 1) * H])
            L["w_qkv"] = w_qkv
            L["w_o"] = ops.pack_weight(dev(lw.wo), dtype)
            L["b_o"] = dev(lw.bo)
            L["ln1_g"], L["ln1_b"] = dev(lw.ln1_g), dev(lw.ln1_b)
            if wl.cfg.with_ffn:
                L["b_ffn1"] = dev(lw.b1)
                if enc.fold:
                    L["w_ffn1"], L["ffn1_c1"], L["ffn1_c2"] = ops.fold_layernorm_weight(
                        dev(lw.w1), L["ln1_g"], L["ln1_b"], L["b_ffn1"], dtype)
                else:
                    L["w_ffn1"] = ops.pack_weight(dev(lw.w1), dtype)
                L["w_ffn2"] = ops.pack_weight(dev(lw.w2), dtype)
                L["b_ffn2"] = dev(lw.b2)
                L["ln2_g"], L["ln2_b"] = dev(lw.ln2_g), dev(lw.ln2_b)
            enc.layers.append(L)
            prev = L
        torch.cuda.synchronize(enc.device)
        return enc

    @staticmethod
    def _fp8_layer(lw, cfg, dev):
        L = {"b_qkv": dev(np.concatenate([lw.bq, lw.bk, lw.bv])), "b_o": dev(lw.bo), "ln1_g": dev(lw.ln1_g), "ln1_b": dev(lw.ln1_b)}
        L["w_qkv"] = ops.pack_weight_fp8(dev(np.concatenate([lw.wq, lw.wk, lw.wv], axis=1)))   # (codes, scales)
        L["w_o"] = ops.pack_weight_fp8(dev(lw.wo))
        if cfg.with_ffn:
            L["w_ffn1"], L["w_ffn2"] = ops.pack_weight_fp8(dev(lw.w1)), ops.pack_weight_fp8(dev(lw.w2))
            L["b_ffn1"], L["b_ffn2"] = dev(lw.b1), dev(lw.b2)
            L["ln2_g"], L["ln2_b"] = dev(lw.ln2_g), dev(lw.ln2_b)
        return L

    def _attention(self, qkv, m2, kv_len):
        cfg = self.cfg
        scale = 1.0 / float(np.sqrt(cfg.head_dim))
        if self.window is None:
            return ops.attention(qkv, cfg.heads, m2, kv_len, scale=scale)
        H = cfg.hidden
        return ops.window_attention(qkv[..., :H], qkv[..., H:2 * H], qkv[..., 2 * H:], cfg.heads, window=self.window,
                                    sinks=self.sinks, mask_add=m2, kv_len=kv_len, scale=scale, causal_sinks=self.causal_sinks)

    def _fp8_stack(self, h, m2, kv_len, out=None):
        """The layers on 8-bit operands: h `[B,S,H]` half precision -> the same; eight launches a layer and a quantizer in
        front of the first.  Every LayerNorm also writes the 8-bit operand of the GEMMs behind it."""
        cfg = self.cfg
        codes, scales = ops.quantize_fp8(h)
        last = self.layers[-1] if self.layers else None
        for L in self.layers:
            end = L is last
            qkv = ops.linear_fp8(codes, scales, *L["w_qkv"], L["b_qkv"], out_dtype=self.dtype)
            ctx = ops.quantize_fp8(self._attention(qkv, m2, kv_len))
            t = ops.linear_fp8(*ctx, *L["w_o"], L["b_o"], residual=h, epilogue=ops.EPI_BIAS_RESIDUAL, out_dtype=self.dtype)
            if end and not cfg.with_ffn:
                return ops.add_layernorm(t, L["ln1_g"], L["ln1_b"], cfg.ln_eps, out=out)
            h, codes, scales = ops.add_layernorm_fp8(t, L["ln1_g"], L["ln1_b"], cfg.ln_eps)
            if not cfg.with_ffn:
                continue
            f1 = ops.linear_fp8(codes, scales, *L["w_ffn1"], L["b_ffn1"], epilogue=ops.EPI_BIAS_GELU, out_dtype=torch.float8_e4m3fn)
            t = ops.linear_fp8(*f1, *L["w_ffn2"], L["b_ffn2"], residual=h, epilogue=ops.EPI_BIAS_RESIDUAL, out_dtype=self.dtype)
            if end:
                return ops.add_layernorm(t, L["ln2_g"], L["ln2_b"], cfg.ln_eps, out=out)
            h, codes, scales = ops.add_layernorm_fp8(t, L["ln2_g"], L["ln2_b"], cfg.ln_eps)
        return h

    # ------------------------------------------------------------------ layer-by-layer path (any config)
    def forward_ops(self, x_f32, mask_add=None, out_f32=True):
        """x_f32 `[B,S,H]` fp32 device tensor -> `[B,S,H]`; one launch per fused layer."""
        if self.fold:
            return self._forward_ops_folded(x_f32, mask_add, out_f32)
        B, S, H = x_f32.shape
        h = ops.convert(x_f32.contiguous(), self.dtype)
        m2 = kv_len = None
        if mask_add is not None:
            m2 = mask_add.reshape(B, S).contiguous()
            kv_len = ops.mask_to_kv_len(m2)
        h = self._fp8_stack(h, m2, kv_len) if self.fp8 else self._half_stack(h, m2, kv_len)
        return ops.convert(h, torch.float32) if out_f32 else h

    def _half_stack(self, h, m2, kv_len, out=None):
        cfg = self.cfg
        for L in self.layers:
            end = out if L is self.layers[-1] else None
            qkv = ops.linear(h, L["w_qkv"], L["b_qkv"])
            ctx = self._attention(qkv, m2, kv_len)
            t = ops.linear(ctx, L["w_o"], L["b_o"], residual=h, epilogue=ops.EPI_BIAS_RESIDUAL)
            a = ops.add_layernorm(t, L["ln1_g"], L["ln1_b"], cfg.ln_eps, out=None if cfg.with_ffn else end)
            if cfg.with_ffn:
                f1 = ops.linear(a, L["w_ffn1"], L["b_ffn1"], epilogue=ops.EPI_BIAS_GELU)
                t2 = ops.linear(f1, L["w_ffn2"], L["b_ffn2"], residual=a, epilogue=ops.EPI_BIAS_RESIDUAL)
                h = ops.add_layernorm(t2, L["ln2_g"], L["ln2_b"], cfg.ln_eps, out=end)
            else:
                h = a
        return h

    def _forward_ops_folded(self, x_f32, mask_add, out_f32):
        """The five-launch layer, one C-ABI call per launch (what b200_encoder_fwd does with fold_layernorm = 1)."""
        cfg = self.cfg
        B, S, H = x_f32.shape
        eps = cfg.ln_eps
        h0 = ops.convert(x_f32.contiguous(), self.dtype)
        m2 = kv_len = None
        if mask_add is not None:
            m2 = mask_add.reshape(B, S).contiguous()
            kv_len = ops.mask_to_kv_len(m2)
        st1 = ops.stats_buffer(B * S, H, x_f32.device)
        st2 = ops.stats_buffer(B * S, H, x_f32.device)
        t2 = None
        prev = None
        for L in self.layers:
            if prev is None:
                qkv = ops.linear(h0, L["w_qkv"], L["b_qkv"])
            else:
                qkv = ops.linear(t2, L["w_qkv"], None, ln_in=(st2, L["qkv_c1"], L["qkv_c2"]), ln_eps=eps)
            ctx = ops.attention(qkv, cfg.heads, m2, kv_len, scale=1.0 / float(np.sqrt(cfg.head_dim)))
            if prev is None:
                t1 = ops.linear(ctx, L["w_o"], L["b_o"], residual=h0, epilogue=ops.EPI_BIAS_RESIDUAL,
                                out_stats=st1, ln_eps=eps)
            else:
                t1 = ops.linear(ctx, L["w_o"], L["b_o"], residual=t2, epilogue=ops.EPI_BIAS_RESIDUAL,
                                out_stats=st1, res_ln=(st2, prev["ln2_g"], prev["ln2_b"]), ln_eps=eps)
            f1 = ops.linear(t1, L["w_ffn1"], None, epilogue=ops.EPI_BIAS_GELU,
                            ln_in=(st1, L["ffn1_c1"], L["ffn1_c2"]), ln_eps=eps)
            t2 = ops.linear(f1, L["w_ffn2"], L["b_ffn2"], residual=t1, epilogue=ops.EPI_BIAS_RESIDUAL,
                            out_stats=st2, res_ln=(st1, L["ln1_g"], L["ln1_b"]), ln_eps=eps)
            prev = L
        h = ops.add_layernorm(t2, prev["ln2_g"], prev["ln2_b"], eps)
        return ops.convert(h, torch.float32) if out_f32 else h

    # ------------------------------------------------------------------ single-call path (full encoder layers)
    def _layer_array(self):
        if self._c_layers is None:
            arr = (capi.EncoderLayerWeights * len(self.layers))()
            for i, L in enumerate(self.layers):
                c = arr[i]
                c.w_qkv, c.b_qkv = L["w_qkv"].data_ptr(), L["b_qkv"].data_ptr()
                c.w_o, c.b_o = L["w_o"].data_ptr(), L["b_o"].data_ptr()
                c.ln1_gamma, c.ln1_beta = L["ln1_g"].data_ptr(), L["ln1_b"].data_ptr()
                c.w_ffn1, c.b_ffn1 = L["w_ffn1"].data_ptr(), L["b_ffn1"].data_ptr()
                c.w_ffn2, c.b_ffn2 = L["w_ffn2"].data_ptr(), L["b_ffn2"].data_ptr()
                c.ln2_gamma, c.ln2_beta = L["ln2_g"].data_ptr(), L["ln2_b"].data_ptr()
                if self.fold:
                    c.ffn1_c1, c.ffn1_c2 = L["ffn1_c1"].data_ptr(), L["ffn1_c2"].data_ptr()
                    if "qkv_c1" in L:
                        c.qkv_c1, c.qkv_c2 = L["qkv_c1"].data_ptr(), L["qkv_c2"].data_ptr()
            self._c_layers = arr
        return self._c_layers

    def workspace(self, tokens):
        key = tokens
        if self._ws_key != key:
            n = capi.lib().b200_encoder_workspace_bytes(tokens, self.cfg.hidden, self.cfg.ffn,
                                                        capi.dtype_code(self.dtype))
            self._ws = torch.empty((n + 256,), dtype=torch.uint8, device=self.device)
            self._ws_key = key
        off = (-self._ws.data_ptr()) % 256
        return self._ws.data_ptr() + off

    def forward_hidden(self, hidden, mask2d=None, kv_len=None):
        """In-place stack over `hidden` `[B,S,H]` (fp16/bf16 device tensor) through b200_encoder_fwd (8-bit weights and
        windows: through the operators)."""
        if not self.cfg.with_ffn:
            raise ValueError("b200_encoder_fwd runs full encoder layers; use forward_ops for attention-only blocks")
        if hidden.dtype != self.dtype or not hidden.is_contiguous():   # it is written through its address, row behind row
            raise ValueError("hidden: contiguous %s" % self.dtype)
        if self.fp8 or self.window is not None:   # launch by launch; the last LayerNorm writes the result in place
            (self._fp8_stack if self.fp8 else self._half_stack)(hidden, mask2d, kv_len, out=hidden)
            return hidden
        B, S, H = hidden.shape
        d = capi.EncoderDesc(hidden.data_ptr(), capi.ptr(mask2d), capi.ptr(kv_len), self._layer_array(),
                             self.workspace(B * S), B, S, H, self.cfg.ffn, self.cfg.heads, len(self.layers),
                             capi.dtype_code(self.dtype), float(self.cfg.ln_eps), -5000.0, 1 if self.fold else 0)
        rc = capi.lib().b200_encoder_fwd(ctypes.byref(d), capi.stream_ptr())
        capi.check(rc, "b200_encoder_fwd")
        return hidden

    def forward(self, x_f32, mask_add=None):
        """fp32 `[B,S,H]` in -> fp32 `[B,S,H]` out (conversion kernels at both ends, as the fused TNN graph does)."""
        if not self.cfg.with_ffn:
            return self.forward_ops(x_f32, mask_add)
        B, S, H = x_f32.shape
        h = ops.convert(x_f32.contiguous(), self.dtype)
        m2 = kv = None
        if mask_add is not None:
            m2 = mask_add.reshape(B, S).contiguous()
            kv = ops.mask_to_kv_len(m2)
        self.forward_hidden(h, m2, kv)
        return ops.convert(h, torch.float32)
