"""CPU: the causal form of first tokens and the layouts of the output, in the descriptor and through the wrappers."""
import ctypes

import pytest
import torch

from tnn_b200 import capi, ops


@pytest.mark.parametrize("value,rc", [(0, capi.OK), (1, capi.OK), (2, capi.ERR_PARAM), (-1, capi.ERR_PARAM)])
def test_causal_sinks_is_0_or_1(value, rc):
    d = capi.WindowAttentionDesc()
    for k, v in dict(q=256, k=256, v=256, out=256, B=2, Sq=0, Sk=7, ldq=256, ldk=128, ldv=128, ldo=256, q_batch=1280, k_batch=896, v_batch=896,
                     o_batch=1280, left=3, right=0, heads=4, kv_heads=2, head_dim=64, dtype=capi.F16, scale=0.125, causal_sinks=value).items():
        setattr(d, k, v)
    assert capi.lib().b200_window_attention_fwd(ctypes.byref(d), None) == rc      # no queries: nothing is launched


@pytest.mark.parametrize("given,field", [({}, 0), ({"causal_sinks": False}, 0), ({"causal_sinks": True}, 1)])
def test_wrapper_passes_it_on(monkeypatch, given, field):
    seen = []
    monkeypatch.setattr(ops, "_require_cuda", lambda *ts: None)
    monkeypatch.setattr(ops, "_call", lambda name, desc, index: seen.append(desc))
    monkeypatch.setattr(ops, "_device_index", lambda *ts: 0)
    q = torch.zeros(1, 5, 128).half()
    ops.window_attention(q, q, q, 2, window=(3, 0), sinks=4, **given)
    assert seen[0].causal_sinks == field and seen[0].mask_exclude_below == -5000.0


@pytest.mark.parametrize("B,Sq,ldo,o_batch,fits", [
    (2, 5, 256, 1280, True), (2, 5, 256, 1272, False), (3, 5, 768, 256, True), (3, 5, 760, 256, False), (3, 5, 768, 264, False), (3, 5, 784, 264, True),
    (2, 1, 256, 256, True), (2, 1, 256, 248, False), (2, 2, 1 << 40, 256, True), (2, 1 << 24, 1 << 40, 256, True), (2, 5, 256, 0, False), (2, 5, 256, -1280, False)])
def test_rows_of_the_output_do_not_overlap(B, Sq, ldo, o_batch, fits):
    """Behind one another or interleaved; what fits goes on to the device, which is not there."""
    if torch.cuda.is_available() and fits:
        pytest.skip("the addresses are not real")
    d = capi.WindowAttentionDesc()
    for k, v in dict(q=256, k=256, v=256, out=256, B=B, Sq=Sq, Sk=7, ldq=256, ldk=256, ldv=256, ldo=ldo, q_batch=2048, k_batch=2048, v_batch=2048,
                     o_batch=o_batch, left=3, right=0, heads=4, kv_heads=4, head_dim=64, dtype=capi.F16, scale=0.125).items():
        setattr(d, k, v)
    assert (capi.lib().b200_window_attention_fwd(ctypes.byref(d), None) != capi.ERR_PARAM) == fits
