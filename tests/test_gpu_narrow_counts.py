"""Counts that do not fit the rows, in the operators of MXFP4 and 8-bit activations: as the rows there are."""

import pytest
import torch

from tests.conftest import banner

pytestmark = pytest.mark.gpu


def _run(op, x, dy, ws, counts):
    leaves = [t.detach().requires_grad_(True) for t in (x, *ws)]
    y = op(*leaves, counts)[0]
    return [y.detach(), *torch.autograd.grad(y, leaves, dy)]


def _inputs(dev, rows, e, d, h):
    gen = torch.Generator(device=dev).manual_seed(rows)
    mk = lambda *s, std=1.0: (torch.randn(*s, generator=gen, device=dev) * std).bfloat16()  # noqa: E731
    return mk(rows, d), mk(rows, d), [mk(e, h, d, std=0.1), mk(e, d, h, std=0.1), mk(e, h, d, std=0.1)]


@pytest.mark.parametrize("four", [False, True], ids=["bf16", "mxfp4"])
def test_steps(dev, four):
    """Counts past the rows, negative ones, ones past 32 bits."""
    banner(f"counts that do not fit, {'mxfp4' if four else 'bf16'}")
    from torchtitan_amd import ops

    op = ops.grouped_swiglu_mxfp4_train if four else ops.grouped_swiglu_ckpt8
    x, dy, ws = _inputs(dev, 300, 4, 128, 64)
    for counts, as_if in (([100, -7, 150, 2 ** 40], [100, 0, 150, 50]), ([2 ** 62, 2 ** 62, 5, 1], [300, 0, 0, 0]),
                          ([-1, 400, 400, 0], [0, 300, 0, 0]), ([-5, -5, 20, -(2 ** 50)], [0, 0, 20, 0])):
        got, want = (_run(op, x, dy, ws, torch.tensor(c, device=dev)) for c in (counts, as_if))
        for a, b in zip(got, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("four", [False, True], ids=["bf16", "mxfp4"])
def test_sums_past_32_bits(dev, four):
    """1024 counts of all of two million rows add up past 2^31: the first expert has them all."""
    banner(f"counts whose sum passes 2^31, {'mxfp4' if four else 'bf16'}")
    from torchtitan_amd import ops

    op = ops.grouped_swiglu_mxfp4_train if four else ops.grouped_swiglu_ckpt8
    rows, e = 2 ** 21 + 37, 1024
    x, dy, ws = _inputs(dev, rows, e, 64, 64)
    counts = torch.full((e,), rows, device=dev)
    one = torch.zeros_like(counts)
    one[0] = rows
    got, want = (_run(op, x, dy, ws, c) for c in (counts, one))
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    packed = [t for w in ws for t in ops.mxfp4_quantize(w)]
    assert torch.equal(ops.grouped_swiglu_mxfp4(x, *packed, counts), ops.grouped_swiglu_mxfp4(x, *packed, one))
