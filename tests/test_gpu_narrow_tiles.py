"""The MXFP4 and 8-bit-activation operators at the shapes where a launch takes each of its tiles, and
where a workgroup works through many of them, against 64 bits on the device:

* training steps on every tile of the bf16 products (which tile a shape takes on 256 CUs is
  asserted, without a GPU), and the same rows bit for bit on each;
* the kernel for few rows with several units a workgroup: scales that come a unit ahead, rows
  that change between units, both numbers of row blocks, odd and even numbers of scale blocks;
* the kernel for many rows with several tiles a workgroup, more than its list holds among them,
  scales copied by dwords and by pairs, whole and partial stages.

Bounds element by element count the roundings; the norm's are the files' of the small shapes."""

import pytest
import torch

from tests import narrow_util as N
from tests.conftest import banner
from tests.test_gpu_gemm_tiles import CASES, CUS, DX384, DX512, FWD, LOW, SAME_ROWS, TALL, TWO, tile
from tests.test_gpu_keep8 import NORM
from tests.test_gpu_mxfp4 import Y_NORM

gpu = pytest.mark.gpu

# of the training steps: the forward's tiles are the bf16 SwiGLU's, dx has the gpt-oss kernels'
STEP_TILES = {"gate_up": {FWD, TALL}, "down": {FWD, TALL}, "dgu": {FWD, TWO, LOW}, "dx": {FWD, TWO, DX384, DX512, TALL}}


def step_tile(mode, e, d, h, rows):
    return tile(mode, mode == "dx", e, d, h, rows)


def test_steps_take_every_tile():
    for runs in ([(e, d, h, rows) for e, d, h, rows, *_ in CASES.values()],
                 [(e, d, h, rows) for (d, h), some in SAME_ROWS.items() for e, rows in some]):
        taken = {m: {step_tile(m, *run) for run in runs} for m in STEP_TILES}
        assert taken == STEP_TILES


@pytest.fixture
def on_device(dev, monkeypatch):
    """narrow_util's 64-bit formulas on the device."""
    monkeypatch.setattr(N, "E2M1", N.E2M1.to(dev))
    with torch.device(dev):
        yield dev


def _within(got, want, tol, what, norm):
    off = (got.detach().double() - want).abs()
    bad = ~(off <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} elements off, worst {off[bad].max():.3g}"
    size = want.norm()
    assert off.norm() <= norm * size, f"{what}: {off.norm() / size:.3g} of its size off"


def _step(op, x, dy, ws, counts):
    leaves = [t.detach().requires_grad_(True) for t in (x, *ws)]
    y, kept = op(*leaves, counts)
    return [y.detach(), *torch.autograd.grad(y, leaves, dy), kept]


# the products' shapes, and one whose MXFP4 forward has several tiles a workgroup with scales in dwords
STEPS = {**{n: c[:5] for n, c in CASES.items()}, "dword_scales": (32, 1024, 1024, 12000, 14)}


@gpu
@pytest.mark.parametrize("four", [False, True], ids=["bf16", "mxfp4"])
@pytest.mark.parametrize("name", list(STEPS))
def test_steps(on_device, name, four):
    banner(f"training step tiles {name} {'mxfp4' if four else 'bf16'}")
    from torchtitan_amd import ops

    e, d, h, rows, seed = STEPS[name]
    gen = torch.Generator().manual_seed(seed)
    load = torch.rand(e, generator=gen, device="cpu") ** 2
    load[e // 2] = 0  # an empty expert
    spare = seed % 3
    counts = torch.bincount(torch.multinomial(load, rows - spare if rows > spare else rows, replacement=True, generator=gen),
                            minlength=e)
    gd = torch.Generator(device=on_device).manual_seed(seed)
    rnd = lambda *s, std=1.0: (torch.randn(*s, generator=gd) * std).bfloat16()  # noqa: E731
    x, dy = rnd(rows, d), rnd(rows, d)
    ws = [rnd(e, h, d, std=d ** -0.5), rnd(e, d, h, std=h ** -0.5), rnd(e, h, d, std=d ** -0.5)]
    op = ops.grouped_swiglu_mxfp4_train if four else ops.grouped_swiglu_ckpt8
    got = _step(op, x, dy, ws, counts.to(on_device))
    again = _step(op, x, dy, ws, counts.to(on_device))
    for a, b in zip(got[:5], again[:5]):
        assert torch.equal(a, b)
    n = int(counts.sum())
    assert not got[0][n:].any() and not got[1][n:].any() and not any(g[e // 2].any() for g in got[2:5])
    for what, g, (v, tol) in zip(("y", "dx", "dw1", "dw2", "dw3"), got, N.gradients(x, *ws, dy, counts, four)):
        _within(g, v, tol, f"{name} {what}", NORM)


@gpu
@pytest.mark.parametrize("d,h", list(SAME_ROWS))
def test_steps_give_the_same_bits(on_device, d, h):
    """The first and the last expert with the same 100 and 150 rows and weights among more and fewer
    others, so that each launch takes another tile: the same y, gradients and kept bytes."""
    assert torch.cuda.get_device_properties(on_device).multi_processor_count == CUS
    banner(f"8-bit activations, same bits {d} / {h}")
    from torchtitan_amd import ops

    gd = torch.Generator(device=on_device).manual_seed(22)
    rnd = lambda *s, std=1.0: (torch.randn(*s, generator=gd) * std).bfloat16()  # noqa: E731
    n0, n1 = 100, 150
    shapes = [(h, d), (d, h), (h, d)]
    fixed_x, fixed_dy, fixed_w = rnd(n0 + n1, d), rnd(n0 + n1, d), [rnd(2, *s, std=s[1] ** -0.5) for s in shapes]
    first = None
    for e, rows in SAME_ROWS[d, h]:
        gen = torch.Generator().manual_seed(rows)
        rest = rows - n0 - n1 if e > 2 else 0
        mid = torch.bincount(torch.randint(max(e - 2, 1), (rest,), generator=gen, device="cpu"), minlength=e - 2) if e > 2 else []
        counts = torch.tensor([n0, *mid, n1])
        pad = rows - n0 - n1 - rest  # two experts: rows past the counts
        x, dy = (torch.cat([f[:n0], rnd(rest, d), f[n0:], rnd(pad, d)]) for f in (fixed_x, fixed_dy))
        ws = [torch.cat([f[:1], rnd(e - 2, *s, std=s[1] ** -0.5), f[1:]]) for f, s in zip(fixed_w, shapes)]
        y, dx, dw1, dw2, dw3, kept = _step(ops.grouped_swiglu_ckpt8, x, dy, ws, counts)
        offsets, _ = ops._ckpt8_layout(rows, d, h)
        parts = [kept[at:at + rows * c].view(rows, c) for at, c in zip(offsets, (d, d // 32, h, h // 32, h, h // 32))]
        own = [torch.cat([t[:n0], t[n0 + rest:n0 + rest + n1]]) for t in (y, dx, *parts)]
        own += [torch.stack([t[0], t[-1]]) for t in (dw1, dw2, dw3)]
        if first is None:
            first = own
        for i, (a, b) in enumerate(zip(first, own)):
            assert torch.equal(a, b), (e, rows, i)


# ---------------------------------------------------------------------------
# packed weights
# ---------------------------------------------------------------------------
WORKGROUPS = 2 * CUS  # of the kernel for few rows


def _few(e, seed, most=33):
    """Rows per expert: none to `most`, 12 at most on the average."""
    gen = torch.Generator().manual_seed(seed)
    n = torch.randint(0, most + 1, (e,), generator=gen)
    n[torch.randperm(e, generator=gen)[:e // 4]] = 0
    n[0], n[-1] = most, 1
    while int(n.sum()) > 12 * e:
        n = n * 3 // 4
        n[0] = most
    return n.tolist()


FEW = {  # counts, rows past them, D, H, rows of a unit
    "even blocks": (_few(64, 1), 3, 1024, 1024, 32),
    "odd blocks": (_few(72, 2), 0, 1184, 1056, 32),
    "a row each": ([1] * 100, 0, 640, 512, 32),
    "partial stages": (_few(48, 3, 60), 1, 1408, 1312, 32),
    "long contraction": (_few(32, 4), 2, 7168, 1312, 16),
    "long odd contraction": (_few(24, 5), 0, 6944, 1408, 16),
}
MANY = {  # counts, rows past them, D, H, tiles that a workgroup has at least
    "whole stages": ([900, 0, 1030] * 16, 5, 1024, 512, 3),
    "partial stages, dwords": ([1000, 700] * 20, 0, 1152, 640, 3),
    "pairs": ([513, 1, 800, 0] * 16, 2, 704, 832, 3),
    "odd blocks": ([300, 500, 1000] * 12, 1, 864, 672, 2),
    "past the list, pairs": ([21, 22, 19, 24] * 256, 7, 64, 2240, 65),
    "past the list, dwords": ([21, 0, 41, 24] * 256, 0, 128, 2816, 65),
}


def _cdiv(a, b):
    return -(-a // b)


def test_units_and_tiles():
    """The cases above have several units or tiles a workgroup in both products, or past the list in
    the first, and their rows per expert take the kernel that they are there for."""
    for name, (counts, spare, d, h, rows) in FEW.items():
        blocks = sum(_cdiv(n, rows) for n in counts)
        assert min(blocks * (h // 32), blocks * _cdiv(d, 64)) > WORKGROUPS, name
        assert sum(counts) + spare <= (20 if rows == 32 else 12) * min(len(counts), sum(counts) + spare), name
    for name, (counts, spare, d, h, tiles) in MANY.items():
        blocks = sum(_cdiv(n, 256) for n in counts)
        assert blocks * _cdiv(h, 128) > (tiles - 1) * CUS, name
        assert tiles > 64 or blocks * _cdiv(d, 256) > CUS, name
        assert sum(counts) > 20 * len(counts) and sum(counts) * _cdiv(max(2 * h, d), 256) > 1536, name


def _random_packed(gd, e, n, k):
    """Codes and scales of every kind: values of a size around k^-0.5."""
    q = torch.randint(0, 256, (e, n, k // 2), generator=gd, dtype=torch.uint8)
    mid = 127 - round(torch.log2(torch.tensor(2.93 * k ** 0.5, device="cpu")).item())
    return q, torch.randint(mid - 2, mid + 3, (e, n, k // 32), generator=gd, dtype=torch.uint8)


def _check_serving(dev, act, name, counts, spare, d, h, sample):
    from torchtitan_amd import ops

    e, rows = len(counts), sum(counts) + spare
    counts = torch.tensor(counts)
    gd = torch.Generator(device=dev).manual_seed(d + h + e)
    x = torch.randn(rows, d, generator=gd).bfloat16()
    glu = 2 if act == "oss" else 1
    w1, w2 = _random_packed(gd, e, glu * h, d), _random_packed(gd, e, d, h)
    if act == "silu":
        w3 = _random_packed(gd, e, h, d)
        run = lambda: ops.grouped_swiglu_mxfp4(x, *w1, *w2, *w3, counts)  # noqa: E731
    else:
        b1, b2 = torch.randn(e, 2 * h, generator=gd).bfloat16(), torch.randn(e, d, generator=gd).bfloat16()
        run = lambda: ops.grouped_swiglu_oss_mxfp4(x, *w1, b1, *w2, b2, counts, 1.5)  # noqa: E731
    got = run()
    assert torch.equal(run(), got) and not got[int(counts.sum()):].any()
    starts = (counts.cumsum(0) - counts).tolist()
    used = [i for i in range(e) if counts[i]]
    used = sorted({*used[:sample // 2], *used[-(sample // 2):], *used[::max(1, len(used) // sample)]})
    at = torch.cat([torch.arange(starts[i], starts[i] + int(counts[i])) for i in used])
    vals = lambda w: N.unpack4(w[0][used], w[1][used])  # noqa: E731
    xq = N.q4(x[at])
    if act == "silu":
        want, tol = N.experts4(xq, vals(w1), vals(w2), vals(w3), counts[used])
    else:
        v = vals(w1)
        want, tol = N.experts4(xq, v[:, 0::2], vals(w2), v[:, 1::2], counts[used], "oss", 1.5, b1[used].double(), b2[used].double())
    _within(got[at], want, tol, name, Y_NORM)


@gpu
@pytest.mark.parametrize("act", ["silu", "oss"])
@pytest.mark.parametrize("name", list(FEW))
def test_several_units(on_device, act, name):
    banner(f"mxfp4 experts, several units: {name} {act}")
    counts, spare, d, h, _ = FEW[name]
    _check_serving(on_device, act, name, counts, spare, d, h, len(counts))


@gpu
@pytest.mark.parametrize("act", ["silu", "oss"])
@pytest.mark.parametrize("name", list(MANY))
def test_several_tiles(on_device, act, name):
    banner(f"mxfp4 experts, several tiles: {name} {act}")
    counts, spare, d, h, _ = MANY[name]
    _check_serving(on_device, act, name, counts, spare, d, h, 60)
