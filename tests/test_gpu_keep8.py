"""The experts' training steps whose activations are kept in 8 bits (bf16 experts) or in 8 and 4
bits (MXFP4 experts), on the GPU, against 64 bits."""

import pytest
import torch

from tests import narrow_util as N
from tests.conftest import banner

pytestmark = pytest.mark.gpu

# the whole of a gradient: dgu, the halves of dx and the result are each rounded to bf16 once
# (2^-8 at most), two of them together at most here
NORM = 2 * 2.0 ** -8

STEPS = [
    ("one row", [0, 1, 0], 0, 64, 64),
    ("few rows", [3, 0, 5, 1], 2, 128, 192),
    ("ragged", [130, 0, 17, 260], 7, 320, 128),
    ("wide", [64, 200], 0, 576, 832),
    ("no rows for anyone", [0, 0], 3, 64, 128),
    ("no rows", [0, 0], 0, 64, 128),
]


def _inputs(counts, spare, d, h, seed, dev):
    gen = torch.Generator().manual_seed(seed)
    e, rows = len(counts), sum(counts) + spare
    mk = lambda *s, std=1.0: (torch.randn(*s, generator=gen) * std).bfloat16()  # noqa: E731
    x, dy = mk(rows, d), mk(rows, d)
    w1, w2, w3 = mk(e, h, d, std=0.1), mk(e, d, h, std=0.1), mk(e, h, d, std=0.1)
    return torch.tensor(counts), x, dy, w1, w2, w3


def _step(op, dev, counts, x, dy, *w, needs=(True,) * 4):
    leaves = [t.to(dev).requires_grad_(n) for t, n in zip((x, *w), needs)]
    y = op(*leaves, counts.to(dev))[0]
    got = torch.autograd.grad(y, [t for t in leaves if t.requires_grad], dy.to(dev))
    return [y.detach(), *got]


@pytest.mark.parametrize("four", [False, True], ids=["bf16", "mxfp4"])
@pytest.mark.parametrize("case", STEPS, ids=[c[0] for c in STEPS])
def test_step(dev, four, case):
    name, counts, spare, d, h = case
    banner(f"kept in 8 bits, {'mxfp4' if four else 'bf16'} {name}")
    from torchtitan_amd import ops

    op = ops.grouped_swiglu_mxfp4_train if four else ops.grouped_swiglu_ckpt8
    counts, x, dy, w1, w2, w3 = _inputs(counts, spare, d, h, d + h, dev)
    got = _step(op, dev, counts, x, dy, w1, w2, w3)
    want = N.gradients(x, w1, w2, w3, dy, counts, four)
    for what, g, (v, tol) in zip(("y", "dx", "dw1", "dw2", "dw3"), got, want):
        N.within(g, v, tol, f"{name} {what}", NORM)
    n = int(counts.sum())
    assert not got[0][n:].any() and not got[1][n:].any()
    for e, c in enumerate(counts.tolist()):
        if c == 0:
            assert not any(g[e].any() for g in got[2:])


def test_forward_alone(dev):
    """Without a backward to keep for: the same y, nothing kept, and a backward refuses."""
    banner("kept in 8 bits, forward alone")
    from torchtitan_amd import ops

    for counts, d, h in (([5, 0, 300, 40], 320, 192), ([700, 513], 512, 576)):
        c, x, dy, w1, w2, w3 = _inputs(counts, 3, d, h, 3, dev)
        args = [t.to(dev) for t in (x, w1, w2, w3, c)]
        y, kept = ops.grouped_swiglu_ckpt8(*args, False)
        assert torch.equal(y, ops.grouped_swiglu_ckpt8(*args)[0]) and kept.numel() == 0
    y = ops.grouped_swiglu_ckpt8(args[0].requires_grad_(True), *args[1:], False)[0]
    with pytest.raises(RuntimeError, match="nothing was kept"):
        y.float().sum().backward()


def test_backwards_of_given_tensors(dev):
    """The backward operators called directly: tensors in any strides, and refusals."""
    banner("kept in 8 bits, backward operators")
    from torchtitan_amd import ops

    c, x, dy, w1, w2, w3 = (t.to(dev) for t in _inputs([5, 0, 70], 0, 128, 192, 6, dev))

    def strided(t):
        wide = t.new_zeros(*t.shape[:-1], 2 * t.shape[-1])
        wide[..., 1::2] = t
        return wide[..., 1::2]

    eight = ops.grouped_swiglu_ckpt8(x, w1, w2, w3, c)[1]
    four = ops.grouped_swiglu_mxfp4_train(x, w1, w2, w3, c)[1]
    for bwd, args, kept, rest in ((ops.grouped_swiglu_ckpt8_backward, (dy, w1, w2, w3, c), eight, ()),
                                  (ops.grouped_swiglu_mxfp4_train_backward, (dy, c), four, (192,))):
        want = bwd(*args, kept, *rest)
        for a, b in zip(want, bwd(*map(strided, args), strided(kept), *rest)):
            assert torch.equal(a, b)
        for bad in (kept[:-1], kept.view(2, -1), kept[:0], kept.cpu()):
            with pytest.raises((ValueError, RuntimeError)):
                bwd(*args, bad, *rest)
        with pytest.raises(TypeError):
            bwd(*args, kept.view(torch.int8), *rest)
        with pytest.raises(TypeError):
            bwd(dy.float(), *args[1:], kept, *rest)
        with pytest.raises(ValueError):
            bwd(dy[:, :64], *args[1:], kept, *rest)
    for h in (128, 96, 256):
        with pytest.raises(ValueError):
            ops.grouped_swiglu_mxfp4_train_backward(dy, c, four, h)


def test_kept_values(dev):
    """What is kept is MXFP8 of x, and of g and u as 64 bits give them (a step off at a border)."""
    banner("kept in 8 bits, kept values")
    from torchtitan_amd import ops

    c, x, dy, w1, w2, w3 = _inputs([9, 0, 70], 0, 128, 96 * 2, 4, dev)
    x[3, 40], x[20, 5] = float("inf"), float("nan")
    x[5, :32], x[6, 32:64] = 0.0, 2.0 ** -130
    kept = ops.grouped_swiglu_ckpt8(*(t.to(dev) for t in (x, w1, w2, w3, c)))[1].cpu()
    offsets, size = ops._ckpt8_layout(79, 128, 192)
    assert kept.numel() == size
    x8, xs, g8, gs, u8, us = (kept[at:at + 79 * n].view(79, n) for at, n in zip(offsets, (128, 4, 192, 6, 192, 6)))

    def value(q, s):
        sc = torch.where(s == 255, torch.nan, torch.exp2(s.double() - 127))
        return q.view(torch.float8_e4m3fn).double() * sc.repeat_interleave(32, 1)

    want = N.q8(x)
    got = value(x8, xs)
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got[~want.isnan()], want[~want.isnan()])
    fine = [i for i in range(x.shape[0]) if i not in (3, 20)]
    for w, q, s in ((w1, g8, gs), (w3, u8, us)):
        got = value(q, s)
        for e, (a, b) in enumerate(N.segments(c, x.shape[0])):
            at = [i for i in range(a, b) if i in fine]
            if not at:
                continue
            v = x[at].double() @ w[e].double().t()
            off = N.spread(N.q8, v, N.sum_off(x[at].double(), w[e].double()))
            assert ((got[at] - N.q8(v)).abs() <= off).all()
        assert got[3].isnan().all() and got[20].isnan().all()


def test_gradients_are_differences(dev):
    """Where the kept values are exact (x of e4m3 values, gate and up rows that pick one of them), the
    gradients are the forward's: dx and the weights' against central differences in 64 bits."""
    banner("kept in 8 bits, differences")
    from torchtitan_amd import ops

    gen = torch.Generator().manual_seed(9)
    d = h = 64
    rows, counts = 6, torch.tensor([4, 2])
    x = (torch.randint(-8, 9, (rows, d), generator=gen) / 4).bfloat16()
    pick = lambda: torch.stack([torch.eye(d)[torch.randperm(d, generator=gen)[:h]] for _ in range(2)]).bfloat16()  # noqa: E731
    w1, w3 = pick(), pick()
    w2 = (torch.randn(2, d, h, generator=gen) * 0.1).bfloat16()
    dy = torch.randn(rows, d, generator=gen).bfloat16()
    got = _step(ops.grouped_swiglu_ckpt8, dev, counts, x, dy, w1, w2, w3)

    def loss(x, w1, w2, w3):
        total = 0.0
        for e, (a, b) in enumerate(N.segments(counts, rows)):
            hh = N.silu(x[a:b] @ w1[e].t()) * (x[a:b] @ w3[e].t())
            total = total + (hh @ w2[e].t() * dy[a:b].double()).sum()
        return total

    args = [t.double() for t in (x, w1, w2, w3)]
    want = N.gradients(x, w1, w2, w3, dy, counts, False)
    step = 2.0 ** -10  # central differences are off by step^2 / 6 times a third derivative of order 1 to 10
    for i, (g, (_v, tol)) in enumerate(zip(got[1:], want[1:])):
        flat = args[i].flatten()
        for j in torch.randperm(flat.numel(), generator=gen)[:40].tolist():
            ends = []
            for s in (step, -step):
                moved = [a.clone() for a in args]
                moved[i].view(-1)[j] += s
                ends.append(loss(*moved))
            diff = float((ends[0] - ends[1]) / (2 * step))
            assert abs(diff - float(g.flatten()[j])) <= float(tol.flatten()[j]) + 1e-4


@pytest.mark.parametrize("four", [False, True], ids=["bf16", "mxfp4"])
def test_gradients_asked_for(dev, four):
    """Each subset of the inputs alone gets the gradients that all together get."""
    banner("kept in 8 bits, subsets")
    from torchtitan_amd import ops

    op = ops.grouped_swiglu_mxfp4_train if four else ops.grouped_swiglu_ckpt8
    c, x, dy, w1, w2, w3 = _inputs([20, 0, 33], 4, 128, 64, 5, dev)
    want = _step(op, dev, c, x, dy, w1, w2, w3)[1:]
    for needs in ((True, False, False, False), (False, True, False, False), (False, False, True, False),
                  (False, False, False, True), (True, False, True, False), (False, True, True, True)):
        got = _step(op, dev, c, x, dy, w1, w2, w3, needs=needs)[1:]
        for g, v in zip(got, [v for v, n in zip(want, needs) if n]):
            assert torch.equal(g, v)


def test_mxfp4_step_serves(dev):
    """The training step's y is the packed weights' y, bit for bit where both take the same kernel."""
    banner("mxfp4 step against packed weights")
    from torchtitan_amd import ops

    c, x, dy, w1, w2, w3 = _inputs([400, 0, 333], 5, 320, 192, 6, dev)
    args = [t.to(dev) for t in (x, w1, w2, w3)]
    y = ops.grouped_swiglu_mxfp4_train(*args, c.to(dev))[0]
    packed = [t for w in args[1:] for t in ops.mxfp4_quantize(w)]
    assert torch.equal(y, ops.grouped_swiglu_mxfp4(args[0], *packed, c.to(dev)))


@pytest.mark.parametrize("four", [False, True], ids=["bf16", "mxfp4"])
def test_step_in_a_graph(dev, four):
    """Forward and backward captured; replays over two inputs with eager steps between them."""
    banner("kept in 8 bits, graph")
    from torchtitan_amd import ops

    op = ops.grouped_swiglu_mxfp4_train if four else ops.grouped_swiglu_ckpt8
    c, x, dy, *w = _inputs([40, 0, 100], 3, 128, 192, 7, dev)
    c, dy = c.to(dev), dy.to(dev)
    xs = [x.to(dev), (x * 0.5).to(dev)]
    leaves = [t.to(dev).requires_grad_(True) for t in w]

    def step(xx):
        xx = xx.detach().requires_grad_(True)
        y = op(xx, *leaves, c)[0]
        return [y.detach(), *torch.autograd.grad(y, [xx, *leaves], dy)]

    want = [step(xx) for xx in xs]
    fixed = xs[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(fixed)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(fixed)
    for turn in range(5):
        fixed.copy_(xs[turn % 2])
        g.replay()
        eager = step(xs[1 - turn % 2])
        torch.cuda.synchronize()
        for a, b in zip(out, want[turn % 2]):
            assert torch.equal(a, b)
        for a, b in zip(eager, want[1 - turn % 2]):
            assert torch.equal(a, b)
