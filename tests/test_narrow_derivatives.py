"""Derivatives that the MXFP4 and 8-bit-activation operators do not have are refused, not dropped, on
the CPU: reverse and forward mode and torch.func's transforms, through the package's functions
and through the dispatcher."""

import pytest
import torch
from torch.autograd import forward_ad

X = torch.ones(4, 64, dtype=torch.bfloat16)


def _serving():
    from torchtitan_amd import ops

    q, s, c = torch.zeros(2, 64, 32, dtype=torch.uint8), torch.zeros(2, 64, 2, dtype=torch.uint8), torch.tensor([2, 2])
    q1, s1 = torch.zeros(2, 128, 32, dtype=torch.uint8), torch.zeros(2, 128, 2, dtype=torch.uint8)
    b1, b2 = torch.ones(2, 128, dtype=torch.bfloat16), torch.ones(2, 64, dtype=torch.bfloat16)
    for ns in (ops, torch.ops.moe_mi355x_mx):
        yield X, lambda x, f=ns.grouped_swiglu_mxfp4: f(x, q, s, q, s, q, s, c)
        oss = ns.grouped_swiglu_oss_mxfp4
        yield X, lambda x, f=oss: f(x, q1, s1, b1, q, s, b2, c, 7.0)
        yield b1, lambda b, f=oss: f(X, q1, s1, b, q, s, b2, c, 7.0)
        yield b2, lambda b, f=oss: f(X, q1, s1, b1, q, s, b, c, 7.0)


def _reverse(f, x):
    f(x.clone().requires_grad_(True))


def _dual(f, x):
    with forward_ad.dual_level():
        f(forward_ad.make_dual(x, torch.ones_like(x)))


def _jvp(f, x):
    torch.func.jvp(f, (x,), (torch.ones_like(x),))


def _grad(f, x):
    torch.func.grad(lambda t: f(t).float().sum())(x)


@pytest.mark.parametrize("derive", [_reverse, _dual, _jvp, _grad])
def test_serving(derive):
    from torchtitan_amd import _lib

    for x, f in _serving():
        with pytest.raises(RuntimeError, match="no gradients"):
            derive(f, x)
        for plain in (x, x.clone().requires_grad_(True)):  # nothing to lose: on to the kernel, which wants a GPU
            with torch.no_grad(), pytest.raises(_lib.MoEKernelError, match="GPU"):
                f(plain)


def test_dual_levels_without_tangents():
    """Inside a dual level, on tensors without a tangent, there is nothing to refuse."""
    from torchtitan_amd import _lib

    for x, f in _serving():
        with forward_ad.dual_level(), pytest.raises(_lib.MoEKernelError, match="GPU"):
            f(x)


def test_training(monkeypatch):
    from torchtitan_amd import ops

    monkeypatch.setattr(ops, "require_gpu", lambda *t: None)
    w, c = torch.ones(2, 64, 64, dtype=torch.bfloat16), torch.tensor([2, 2])
    args = [X, w, w, w]
    for op in (ops.grouped_swiglu_ckpt8, ops.grouped_swiglu_mxfp4_train):
        for i in range(4):
            with pytest.raises(RuntimeError, match="forward mode"):
                _dual(lambda t: op(*args[:i], t, *args[i + 1:], c), args[i])
