"""CPU: orders between the generic and the async proxy and between a kernel's end and its copies that no run can be relied on to
show."""
import os
import re

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
