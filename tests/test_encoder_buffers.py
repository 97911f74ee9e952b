"""CPU: which buffers the in-place stack takes (no launch happens: they are refused first)."""
import pytest
import torch

from tnn_b200.encoder import Encoder
from tnn_b200.model_synth import EncoderConfig


@pytest.mark.parametrize("fp8,window", [(False, None), (True, None), (False, (4, 4)), (True, (4, 4))])
@pytest.mark.parametrize("hidden", [
    torch.zeros(2, 9, 256).half()[:, :5],                    # a copy of it would take the result
    torch.zeros(2, 5, 512).half()[..., :256], torch.zeros(5, 2, 256).half().transpose(0, 1), torch.zeros(2, 5, 256), torch.zeros(2, 5, 256).bfloat16()])
def test_forward_hidden_refuses_what_it_cannot_write_in_place(monkeypatch, hidden, fp8, window):
    enc = Encoder(EncoderConfig(1, 256, 4, 512), torch.float16, torch.device("cpu"))
    enc.fp8, enc.window = fp8, window

    def stack(h, mask, kv_len, out=None):
        raise AssertionError("ran")

    monkeypatch.setattr(enc, "_fp8_stack", stack)
    monkeypatch.setattr(enc, "_half_stack", stack)
    monkeypatch.setattr(enc, "_layer_array", stack)
    with pytest.raises(ValueError):
        enc.forward_hidden(hidden)
