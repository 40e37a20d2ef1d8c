"""The bounded waits of the expert and int8 kernels, by reading the source: where a
warp waits, it goes on or gives up as one (`warp_wait`, a vote); the wait of a
single thread (`mbar_wait`) is left to the producer thread of the experts."""

import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "qgemv_roofline_b200", "csrc")


def code(name):
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"//[^\n]*", "", f.read())


@pytest.mark.parametrize("name", ["moe.cu", "int8.cu"])
def test_a_warp_gives_up_as_one(name):
    text = code(name)
    vote = re.search(r"bool warp_wait\([^{]*\{\s*return __all_sync\(0xffffffffu, mbar_wait\([^;]*\)\);\s*\}", text)
    assert vote
    rest = text[:vote.start()] + text[vote.end():]
    single = [m.start() for m in re.finditer(r"(?<!bool )\bmbar_wait\(", rest)]
    if name == "moe.cu":
        feed = re.search(r"struct Feed \{.*?\n\};", rest, re.S)  # one thread's
        single = [i for i in single if not feed.start() < i < feed.end()]
        assert len(re.findall(r"\bfeed\.put\(", rest)) == len(re.findall(r"Feed<FMT> feed\{", rest)) == 2
        for m in re.finditer(r"Feed<FMT> feed\{", rest):
            assert rest[:m.start()].rstrip().endswith("if (lane == 0) {")
    assert not single, [rest[i:i + 60] for i in single]
    assert len(re.findall(r"(?<!bool )\bwarp_wait\(", rest)) >= 4


def test_the_q4_converters_give_up_as_one():
    """gemv_tc.cu: the converter warps' waits, whose loop holds a __syncwarp."""
    text = code("gemv_tc.cu")
    part = text[text.index("(i / C::SAD) - 1) & 1)"):]
    assert re.match(r"[^;]*;\s*ok = __all_sync\(0xffffffffu, ok\);\s*if \(!ok\) break;", part)
