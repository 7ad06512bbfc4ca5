"""Rows to 8-bit integers and back carry no derivative: one of the rows, or of the scales, is refused
and not dropped, on the CPU, through the package and through the dispatcher."""

import pytest
import torch
from torch.autograd import forward_ad


def _calls(ns):
    q, s = torch.ones(4, 32, dtype=torch.int8), torch.ones(4)
    for dtype in (torch.bfloat16, torch.float32):
        yield torch.ones(4, 32, dtype=dtype), lambda x: ns.int8_quantize(x)[1]
        yield s, lambda t, dtype=dtype: ns.int8_dequantize(q, t, dtype)


def _dual(f, x):
    with forward_ad.dual_level():
        f(forward_ad.make_dual(x, torch.ones_like(x)))


@pytest.mark.parametrize("derive", [
    lambda f, x: f(x.clone().requires_grad_(True)), _dual, lambda f, x: torch.func.jvp(f, (x,), (torch.ones_like(x),)),
    lambda f, x: torch.func.grad(lambda t: f(t).float().sum())(x)])
def test_derivatives(derive):
    from torchtitan_amd import _lib, ops

    for ns in (ops, torch.ops.moe_mi355x_int8):
        for x, f in _calls(ns):
            with pytest.raises(RuntimeError, match="no gradients"):
                derive(f, x)
            with torch.no_grad(), pytest.raises(_lib.MoEKernelError, match="GPU"):  # nothing to lose
                f(x.clone().requires_grad_(True))
            with forward_ad.dual_level(), pytest.raises(_lib.MoEKernelError, match="GPU"):
                f(x)
