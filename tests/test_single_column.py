"""Matrices of one column, whose last stride means nothing (torch calls them contiguous
whatever it is)."""

import types

import pytest
import torch

import qgemv_roofline_b200 as qg
from qgemv_roofline_b200 import moe

STRIDES = [(1, 0), (1, 1), (1, 5), (7, 3)]


@pytest.mark.parametrize("strides", STRIDES)
def test_a_router_of_one_column(strides):
    router = torch.zeros(64).as_strided((6, 1), strides)
    r = moe._router(router, 2, "softmax", None, 1.0, True, types.SimpleNamespace(index=-1))
    assert (r.n_experts, r.ldw) == (6, strides[0])


def test_rows_still_need_a_unit_stride():
    router = torch.zeros(64).as_strided((6, 2), (2, 3))
    with pytest.raises(ValueError, match="unit last stride"):
        moe._router(router, 2, "softmax", None, 1.0, True, types.SimpleNamespace(index=-1))


@pytest.mark.gpu
@pytest.mark.parametrize("strides", STRIDES)
def test_single_columns(strides):
    router = torch.arange(64, device="cuda").float().as_strided((6, 1), strides)
    x = torch.tensor([[1.0], [-1.0]], device="cuda").as_strided((2, 1), (1, strides[1]))
    got, want = qg.moe_route(x, router, 3), qg.moe_route(x.clone(), router.clone(memory_format=torch.contiguous_format), 3)
    assert got[0].tolist() == want[0].tolist() == [[5, 4, 3], [0, 1, 2]] and torch.equal(got[1], want[1])
    q = torch.full((64,), 9, dtype=torch.int8, device="cuda")
    view = q.as_strided((2, 1), (strides[0] + 1, strides[1]))
    _, s = qg.quantize_int8(x, q=view)
    assert view.tolist() == [[127], [-127]] and s.tolist() == pytest.approx([1 / 127] * 2) and q.tolist().count(9) == 62
