"""CPU: an output that the operators could only write into a copy is refused; views that need none are taken."""
import pytest
import torch

from tnn_b200 import ops


@pytest.fixture(autouse=True)
def _cpu(monkeypatch):
    monkeypatch.setattr(ops, "_require_cuda", lambda *ts: None)   # the descriptors only


def _linear(out):
    return ops._linear_desc(torch.zeros(2, 5, 128).half(), torch.zeros(64, 128).half(), None, None, ops.EPI_BIAS, None, out, 0)[0]


def _layernorm(out):
    return ops._layernorm_desc(torch.zeros(2, 5, 64).half(), torch.ones(64), torch.zeros(64), 1e-5, None, None, out)[0]


@pytest.mark.parametrize("desc", [_linear, _layernorm])
def test_an_output_that_needs_a_copy_is_refused(desc):
    for out in (torch.zeros(2, 9, 64).half()[:, :5], torch.zeros(5, 2, 64).half().transpose(0, 1), torch.zeros(2, 64, 5).half().transpose(1, 2)):
        with pytest.raises(AssertionError):
            desc(out)


@pytest.mark.parametrize("desc", [_linear, _layernorm])
def test_rows_at_a_stride_are_written_in_place(desc):
    for out, ld in ((torch.zeros(2, 5, 64).half(), 64), (torch.zeros(2, 5, 96).half()[..., 32:], 96), (torch.zeros(10, 64).half(), 64),
                    (torch.zeros(12, 80).half()[1:11, :64], 80)):
        d = desc(out)
        assert d.y == out.data_ptr() and d.ldy == ld
