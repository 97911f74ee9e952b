"""CPU: orders between the generic and the async proxy and between a kernel's end and its copies that no run can be relied on to
show."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tnn_b200", "csrc")


def _source(name):
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"//[^\n]*", "", f.read())


def _body(text, head):
    """The body of the function whose definition begins with `head`."""
    i = text.index("{", text.index(head))
    depth, j = 1, i
    while depth:
        j += 1
        depth += {"{": 1, "}": -1}.get(text[j], 0)
    return text[i:j + 1]


def test_the_answer_of_a_take_over_is_read_before_the_next_request_may_overwrite_it():
    text = _source("window_attention.cu")
    body = _body(text, "int taken_over(")
    read, fence = body.index("ld.shared.b128"), body.index("fence_async_proxy_shared()")
    assert read < fence < body.index("return ok")
    # every request's answer goes through it: the slot is not read anywhere else, and asked for by the thread that reads it
    assert len(re.findall(r"\btaken_over\(", text)) == 2 and len(re.findall(r"\btake_over\(", text)) == 2
    assert text.count("clusterlaunchcontrol.try_cancel") == 1 and text.count("OFF_TAKEN") == 4


@pytest.mark.parametrize("name,kernel", [("window_attention.cu", "window_attention_kernel("), ("linear_fp8.cu", "linear_fp8_kernel(")])
def test_a_cta_that_gave_up_leaves_nothing_in_flight(name, kernel):
    """Any role may have a load, a UMMA or a request of its own on its way when another one gives up, so the wait for them stands
    behind the CTA's last barrier, where every role has stopped, and before TMEM goes back."""
    body = _body(_source(name), kernel)
    end = body[body.rindex("__syncthreads()"):]
    assert re.search(r"if \(warp == 1\) \{\s*if \(\*abort_flag != 0\) let_copies_land\(\);\s*tcgen05_fence_after\(\);\s*tmem_dealloc\(", end)
    assert not re.search(r"\b(tma_load|umma|take_over|tma_store_[23]d)", end)
