"""What the expert kernels (csrc/moe.cu) do before their own dependency wait, by
reading the source.  They are launched while the kernel before them still runs:
until `pdl_wait()` a kernel may set up its barriers and clear its shared memory,
but it may read nothing that another grid writes (the choices, the digits), nor
start a bounded wait, which would count the other kernel's time."""

import os
import re

import pytest

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                      "qgemv_roofline_b200", "csrc", "moe.cu")


def body(kernel):
    """The text between a kernel's outer braces, without comments."""
    with open(SOURCE) as f:
        text = re.sub(r"//[^\n]*", "", f.read())
    at = text.index("{", re.search(rf"\b{kernel}\(MoeArgs", text).end())
    depth = 0
    for i in range(at, len(text)):
        depth += {"{": 1, "}": -1}.get(text[i], 0)
        if depth == 0:
            return text[at:i]
    raise AssertionError(f"{kernel} does not end")


@pytest.mark.parametrize("kernel", ["k_moe_up", "k_moe_down"])
@pytest.mark.parametrize("use", ["build_table", ".put(", "mbar_wait(", ".entry(", "a.ids", "a.weights", "a.hdig", "a.xdig"])
def test_nothing_global_and_no_bounded_wait_before_the_dependency_wait(kernel, use):
    text = body(kernel)
    assert text.count("pdl_wait();") == 1
    assert use not in text[:text.index("pdl_wait();")]


@pytest.mark.parametrize("kernel", ["k_moe_up", "k_moe_down"])
def test_every_thread_takes_the_dependency_wait(kernel):
    text = body(kernel)
    before = text[:text.index("pdl_wait();")]
    assert before.count("{") - before.count("}") == 1  # the kernel's own brace: in no branch
