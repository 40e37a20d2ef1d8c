"""The numbers that the CPU restatement of the experts' ring (test_moe_ring_protocol.py)
works with are the kernels' (csrc/moe.cu).  It checks the protocol; the kernels' own
code is checked on the GPU."""

import os
import re

import test_moe_ring_protocol as ring

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                      "qgemv_roofline_b200", "csrc", "moe.cu")


def test_the_ring_has_the_kernels_numbers():
    with open(SOURCE) as f:
        text = f.read()
    value = lambda name: int(re.search(rf"constexpr int {name} = (\d+);", text).group(1))
    assert (value("MOE_S"), value("MOE_KS"), value("MOE_RT")) == (ring.STAGES, ring.SPLITS, ring.TILES)
    assert value("MOE_S") % value("MOE_KS") == 0  # a stage serves one split
