"""Corners of the training operators that keep no large tensor, on the GPU."""
import math

import pytest
import torch

from mvs_amd import ops

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def randn(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("upstream", [float("inf"), float("nan"), 0.0])
@pytest.mark.parametrize("n,C", [(1, 40), (20, 40), (300, 40), (1, 200), (3, 200), (20, 200), (300, 200), (700, 136)])
def test_linear_cross_entropy_without_a_kept_row_has_no_gradient(n, C, upstream, dtype):
    """... whatever comes from above: a loss divided by the number of rows kept hands down 1 / 0."""
    x, w = randn(n, C, seed=1).to(dtype).requires_grad_(), randn(150, C, seed=2).to(dtype).requires_grad_()
    t = torch.full((n,), -100, device="cuda")
    for reduction in ("sum", "mean", "none"):
        loss = ops.linear_cross_entropy(x, w, t, reduction=reduction)
        gx, gw = torch.autograd.grad(loss, (x, w), torch.full_like(loss, upstream))
        assert (gx == 0).all() and (gw == 0).all(), reduction
        assert math.isnan(float(loss.detach())) if reduction == "mean" else (loss == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("C", [40, 200, 1024, 2056])
def test_linear_cross_entropy_of_a_single_ignored_row_whatever_the_table_holds(C, bad, dtype):
    x, w = randn(1, C, seed=1).to(dtype), randn(150, C, seed=2).to(dtype)
    w[7], w[149, 3] = bad, bad
    x, w = x.requires_grad_(), w.requires_grad_()
    loss = ops.linear_cross_entropy(x, w, torch.tensor([-100], device="cuda"), reduction="sum")
    gx, gw = torch.autograd.grad(loss, (x, w))
    assert float(loss.detach()) == 0 and (gx == 0).all() and (gw == 0).all()
