"""8-bit integers on as many experts as are taken, and workgroups that go through more tiles than their
list holds. A sum of codes here is below 2^24, so that products in fp32 give it exactly in any
order, and what follows it is done step by step: the kernels' bits, not only values near them."""

import pytest
import torch

from tests import int8_util as I
from tests import narrow_util as N
from tests.conftest import banner
from tests.test_gpu_mxfp4 import Y_NORM

gpu = pytest.mark.gpu

BF = torch.bfloat16
CUS = 256
TILE = [(256, 256, 1), (128, 256, 1)]  # rows, columns, workgroups a CU


def _tile(*args):
    from torchtitan_amd import _lib

    return _lib.lib().moe_int8_tile(*args, CUS)


def _codes(gen, *shape):
    return torch.randint(-127, 128, shape, generator=gen, dtype=torch.int8, device=gen.device), torch.rand(
        *shape[:-1], generator=gen, device=gen.device) * 0.01 + 0.001


def _product(x, qw, sw):
    """The bits of x [M, K] by a weight in codes: the sum, then its row's scale, then its column's, each rounded."""
    from torchtitan_amd import ops

    assert x.shape[1] * 127 * 127 < 2 ** 24
    q, s = ops.int8_quantize(x)
    return ((q.float() @ qw.float().t()) * s.unsqueeze(-1) * sw).to(x.dtype)


def _counts(e, rows, gen, spare=0):
    load = torch.rand(e, generator=gen) ** 2
    load[e // 2] = load[1] = load[e - 2] = 0
    return torch.bincount(torch.multinomial(load, rows - spare, replacement=True, generator=gen), minlength=e)


# (experts, rows, contraction, columns, tile): both kernels, in whose scans a wave's lanes hold up to
# 4 or up to 16 experts each
GROUPED = [(256, 500, 144, 264, 4), (257, 600, 144, 264, 4), (300, 600, 272, 72, 4), (1024, 700, 256, 512, 4), (1024, 2000, 144, 264, 4),
           (256, 131072, 256, 256, 1), (257, 131072, 256, 256, 1), (300, 131072, 256, 512, 1), (1024, 131072, 256, 256, 1),
           (1024, 131072, 128, 256, 2)]


def test_the_kernels_that_they_take():
    for e, rows, k, n, tile in GROUPED:
        assert _tile(rows, e, k, n) == tile, (e, rows)
    for (e, rows, k, n), tile in MANY.items():
        bm, bn, per_cu = TILE[tile]
        assert _tile(rows, e, k, n) == tile and rows // bm * (n // bn) > 64 * CUS * per_cu


@gpu
@pytest.mark.parametrize("e,rows,k,n,tile", GROUPED)
def test_grouped_linear(dev, e, rows, k, n, tile):
    banner(f"grouped_linear_int8 {e} experts, {rows} rows, {n} x {k}")
    from torchtitan_amd import ops

    gen, gd = torch.Generator().manual_seed(e + rows), torch.Generator(device=dev).manual_seed(e + rows)
    qw, sw = _codes(gd, e, n, k)
    x = torch.randn(rows, k, generator=gd, device=dev).to(BF)
    some = _counts(e, rows, gen, 3)
    # each count all rows there are, so that the sums stop at them; all rows the last expert's
    all_first, last = torch.full((e,), rows), torch.zeros(e, dtype=torch.int64)
    last[e - 1] = rows
    for counts in (some, all_first, last):
        got = ops.grouped_linear_int8(x, qw, sw, counts.to(dev))
        want = torch.zeros_like(got)
        for i, a, b in I.segments(counts, rows):
            want[a:b] = _product(x[a:b], qw[i], sw[i])
        assert torch.equal(got, want), (got != want).nonzero()[0].tolist()


@gpu
@pytest.mark.parametrize("e,rows", [(257, 300), (300, 700), (1024, 1500), (257, 40000), (1024, 70000)])
def test_experts(dev, e, rows):
    """Each expert's rows come out as through a layer of it alone; some as 64 bits give them."""
    banner(f"grouped_swiglu_int8 {e} experts, {rows} rows")
    from torchtitan_amd import ops

    gen, gd = torch.Generator().manual_seed(e), torch.Generator(device=dev).manual_seed(e)
    d, h = 208, 144
    w = [t for s in ((e, h, d), (e, d, h), (e, h, d)) for t in _codes(gd, *s)]
    m1, b1, b2 = _codes(gd, e, 2 * h, d), torch.randn(e, 2 * h, generator=gd, device=dev), torch.randn(e, d, generator=gd, device=dev)
    x = torch.randn(rows, d, generator=gd, device=dev).to(BF)
    counts = _counts(e, rows, gen, 2)
    got = ops.grouped_swiglu_int8(x, *w, counts.to(dev))
    oss = ops.grouped_swiglu_oss_int8(x, *m1, b1, *w[2:4], b2, counts.to(dev), 7.0)
    tested = 0
    for i, a, b in I.segments(counts, rows):
        assert torch.equal(ops.swiglu_ffn_int8(x[a:b], *(t[i] for t in w)), got[a:b]), f"expert {i}"
        part = [t[i:i + 1] for t in (*m1, b1, *w[2:4], b2)]
        assert torch.equal(ops.grouped_swiglu_oss_int8(x[a:b], *part, torch.tensor([b - a], device=dev), 7.0), oss[a:b]), f"expert {i}"
        if tested < 6 or i > e - 6:
            tested += 1
            n, one = min(b - a, 5), [t[i:i + 1].cpu() for t in w]
            own, (p, bp1, bp2) = torch.tensor([n]), ([t[i:i + 1].cpu() for t in m1], b1[i:i + 1].cpu(), b2[i:i + 1].cpu())
            I.within(got[a:a + n], *I.experts(x[a:a + n].cpu(), one[:2], one[2:4], one[4:], own), f"expert {i}")
            I.within(oss[a:a + n], *I.oss(x[a:a + n].cpu(), p, bp1, one[2:4], bp2, own, 7.0), f"expert {i}, gpt-oss's")
    end = int(counts.sum())
    assert end < rows and not got[end:].any() and not oss[end:].any()


# (experts, rows, contraction, columns): tile, with more than 64 tiles a workgroup
MANY = {(1, 70000, 384, 16384): 0, (300, 66000, 128, 16640): 1}


@gpu
@pytest.mark.parametrize("e,rows,k,n", list(MANY))
def test_more_tiles_than_a_list_holds(dev, e, rows, k, n):
    banner(f"int8 products, more than 64 tiles a workgroup: {e} experts, {rows} rows, {n} x {k}")
    from torchtitan_amd import ops

    gen, gd = torch.Generator().manual_seed(7), torch.Generator(device=dev).manual_seed(7)
    qw, sw = _codes(gd, e, n, k)
    x = torch.randn(rows, k, generator=gd, device=dev).to(BF)
    counts = torch.tensor([rows]) if e == 1 else _counts(e, rows, gen, 1)
    got = ops.linear_int8(x, qw[0], sw[0]) if e == 1 else ops.grouped_linear_int8(x, qw, sw, counts.to(dev))
    for i, a, b in I.segments(counts, rows):
        for at in range(a, b, 8192):
            to = min(at + 8192, b)
            assert torch.equal(got[at:to], _product(x[at:to], qw[i], sw[i])), f"expert {i}, rows from {at}"
    assert not got[int(counts.sum()):].any()


@gpu
@pytest.mark.parametrize("e,rows", [(257, 300), (300, 900), (1024, 1500)])
def test_mxfp4_experts(dev, e, rows):
    """MXFP4's kernel for few rows takes its segments from the same scan."""
    banner(f"grouped_swiglu_mxfp4 {e} experts, {rows} rows")
    from torchtitan_amd import ops

    gen, gd = torch.Generator().manual_seed(e), torch.Generator(device=dev).manual_seed(e)
    d, h = 128, 96
    w = [ops.mxfp4_quantize(torch.randn(*s, generator=gd, device=dev) * 0.1) for s in ((e, h, d), (e, d, h), (e, h, d))]
    vals = [N.unpack4(*(t.cpu() for t in q)) for q in w]
    x = torch.randn(rows, d, generator=gd, device=dev).to(BF)
    for counts in (_counts(e, rows, gen, 2), torch.full((e,), rows)):
        got = ops.grouped_swiglu_mxfp4(x, *(t for q in w for t in q), counts.to(dev))
        want, tol = N.experts4(N.q4(x.cpu()), *vals, counts)
        N.within(got, want, tol, f"{e} experts", Y_NORM)
        assert not got[min(int(counts.sum()), rows):].any()
