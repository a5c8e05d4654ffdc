"""Calls of the model operators that are allowed and easily forgotten: empty batches, operands that come back moved, graphs that hold half a step."""

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("weight", [1.0, 0.5, 0.0])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_a_loss_of_no_rows_with_targets(dtype, weight, reduction):
    from tandem_amd import ops

    x, idx, t = torch.empty(0, 50, device=DEV, dtype=dtype), torch.empty(0, 4, device=DEV, dtype=torch.int64), torch.empty(0, 4, device=DEV)
    how = dict(targets=torch.empty(0, device=DEV, dtype=torch.int64), weight=weight, reduction=reduction, temperature=2.0)
    loss, grad = ops.distill_loss_and_grad(x, idx, t, **how)
    alone = ops.distill_loss(x, idx, t, **how)
    leaf = x.clone().requires_grad_()
    trained = ops.distill_loss(leaf, idx, t, **how)
    trained.sum().backward()
    for got in (loss, alone, trained):
        assert got.shape == ((0,) if reduction == "none" else ()) and (got == 0).all()
    assert grad.shape == leaf.grad.shape == (0, 50)
