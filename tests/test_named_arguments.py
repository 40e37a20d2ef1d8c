"""Every argument of the operators by its documented name (no GPU needed: a CPU
tensor is refused by the check of the first argument, after the names)."""

import inspect

import pytest
import torch

import qgemv_roofline_b200 as qg


@pytest.mark.parametrize("fn", [qg.moe_route, qg.moe_experts, qg.moe_layer, qg.quantize_int8, qg.int8_matmul,
                                qg.int8_linear])
def test_all_arguments_by_name(fn):
    names = list(inspect.signature(fn).parameters)
    kwargs = {n: torch.zeros(2, 32) if i == 0 else None for i, n in enumerate(names)}
    with pytest.raises(ValueError, match=f"{names[0]} must be a CUDA tensor"):
        fn(**kwargs)
    with pytest.raises(ValueError, match="CUDA tensor"):
        fn(torch.zeros(2, 32), **{n: None for n in names[1:]})
    with pytest.raises(TypeError):
        fn(**{n: None for n in names[1:]})


@pytest.mark.gpu
def test_named_arguments_give_the_same():
    x, w = (torch.randn(n, 64, device="cuda") for n in (3, 40))
    (xq, xs), (wq, ws) = qg.quantize_int8(x=x), qg.quantize_int8(x=w)
    y = qg.int8_matmul(xq=xq, xs=xs, wq=wq, ws=ws, bias=None, out_dtype=torch.float16)
    assert torch.equal(y, qg.int8_matmul(xq, xs, wq, ws, out_dtype=torch.float16))
    assert torch.equal(qg.int8_linear(x=x, wq=wq, ws=ws), qg.int8_linear(x, wq, ws))
    ids, weights = qg.moe_route(x=x, router=w, top_k=2)
    assert torch.equal(ids, qg.moe_route(x, w, 2)[0])
