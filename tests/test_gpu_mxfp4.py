"""MXFP4 quantization and the experts on packed weights, on the GPU, against 64 bits."""

import pytest
import torch

from tests import narrow_util as N
from tests.conftest import banner

pytestmark = pytest.mark.gpu

# y is one rounding to bf16 (2^-8 at most, 2^-8 / sqrt(3) in the mean square) of a value whose
# h can have moved by a step where it lies at a rounding's border
Y_NORM = 2.0 ** -8


def _blocks(gen, rows, cols, spread=2.0):
    x = torch.randn(rows, cols, generator=gen)
    return x * torch.exp(spread * torch.randn(rows, cols // 32, generator=gen)).repeat_interleave(32, 1)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", [(1, 32), (3, 96), (5, 7, 64), (257, 1472), (1030, 2880)])
def test_quantize_bits(dev, dtype, shape):
    banner(f"mxfp4_quantize {shape} {dtype}")
    from torchtitan_amd import ops

    gen = torch.Generator().manual_seed(1)
    x = _blocks(gen, torch.Size(shape).numel() // shape[-1], shape[-1]).to(dtype).view(shape)
    q, s = ops.mxfp4_quantize(x.to(dev))
    wq, ws = N.pack4(x)
    assert torch.equal(s.cpu(), ws) and torch.equal(q.cpu(), wq)
    back = ops.mxfp4_dequantize(q, s, dtype)
    assert back.dtype == dtype and torch.equal(back.cpu().double(), N.q4(x))


def test_quantize_every_rounding(dev):
    """Every fp32 value from 1/8 to 6 (below 1/4 all round to zero), both signs, in blocks whose
    scale is 1."""
    banner("mxfp4_quantize every rounding")
    from torchtitan_amd import ops

    top = torch.tensor(6.0).view(torch.int32).item()
    mid = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=dev)
    up = torch.tensor([0, 1, 0, 1, 0, 1, 0], dtype=torch.bool, device=dev)
    for start in range(0x3E000000, top + 1, 31 << 20):
        bits = torch.arange(start, min(start + (31 << 20), top + 1), dtype=torch.int32, device=dev)
        v = bits.view(torch.float32)
        pad = (-v.numel()) % 31
        v = torch.cat([v, v.new_zeros(pad)]).view(-1, 31)
        for sign in (1.0, -1.0):
            x = torch.cat([v * sign, v.new_full((v.shape[0], 1), 6.0)], 1)
            q, s = ops.mxfp4_quantize(x)
            assert bool((s == 127).all())
            code = torch.stack([q & 15, q >> 4], -1).flatten(-2)[:, :31]
            want = torch.zeros_like(code)
            for m, tie_up in zip(mid, up):
                want += torch.where(tie_up, v >= m, v > m)
            assert torch.equal(code & 7, want)
            assert bool(((code >> 3) == (1 if sign < 0 else 0)).logical_or(v == 0).all())


def test_quantize_odd_blocks(dev):
    """Zeros, signed zeros, borders of the scale, subnormals, the largest values, infinities and
    NaN; a block's neighbours keep theirs."""
    banner("mxfp4_quantize odd blocks")
    from torchtitan_amd import ops

    x = torch.randn(16, 96, generator=torch.Generator().manual_seed(2))
    x[0, :32] = 0.0
    x[0, 32:64] = -0.0
    x[1, :32] = torch.linspace(-6, 6, 32)
    x[1, 32:64] = torch.linspace(-6.0000005, 6, 32)  # past 6: the next scale
    x[2, :32] *= 2.0 ** -127
    x[2, 32:64] *= 2.0 ** -146
    x[3, :32] = torch.finfo(torch.float32).max
    x[3, 32:64] = torch.linspace(-3.4e38, 3.4e38, 32)
    x[4, 5], x[4, 40], x[5, 70] = float("inf"), float("-inf"), float("nan")
    x[6, :32], x[6, 3] = float("nan"), 1.0
    x[7, :32] = 2.0 ** -126
    for dtype in (torch.float32, torch.bfloat16):
        xd = x.to(dtype)
        q, s = ops.mxfp4_quantize(xd.to(dev))
        wq, ws = N.pack4(xd)
        fine = (ws != 255).repeat_interleave(16, 1)
        assert torch.equal(s.cpu(), ws)
        assert torch.equal(q.cpu()[fine], wq[fine])
        back = ops.mxfp4_dequantize(q, s, dtype).cpu().double()
        want = N.q4(xd)
        assert torch.equal(back.isnan(), want.isnan())
        assert torch.equal(back[~want.isnan()], want[~want.isnan()].to(dtype).double())


def test_dequantize_every_code(dev):
    """All bytes under all scales: values past the type's range become infinities, below it they
    are rounded as the type rounds."""
    banner("mxfp4_dequantize every code")
    from torchtitan_amd import ops

    q = torch.arange(256, dtype=torch.uint8).view(16, 16).repeat(256, 1)
    s = torch.arange(256, dtype=torch.uint8).repeat_interleave(16).view(-1, 1)
    for dtype in (torch.float32, torch.bfloat16):
        got = ops.mxfp4_dequantize(q.to(dev), s.to(dev), dtype).cpu()
        want = N.unpack4(q, s).to(dtype)
        assert torch.equal(got.isnan(), want.isnan())
        assert torch.equal(got[~want.isnan()], want[~want.isnan()])


def test_quantize_views(dev):
    """Strided and misaligned inputs, inputs of no rows, and rows whose offsets pass 2^31 elements."""
    banner("mxfp4_quantize views")
    from torchtitan_amd import ops

    x = _blocks(torch.Generator().manual_seed(3), 64, 128).bfloat16().to(dev)
    for v in (x.t(), x[1::2], x[:, 32:96], x.flatten()[1:-63].view(-1, 32 * 8 // 8)[:7], x.view(4, 16, 128).transpose(0, 1)):
        q, s = ops.mxfp4_quantize(v)
        wq, ws = N.pack4(v.cpu())
        assert torch.equal(q.cpu(), wq) and torch.equal(s.cpu(), ws)
        assert torch.equal(ops.mxfp4_dequantize(q, s).cpu().double(), N.q4(v.cpu()))
    q, s = ops.mxfp4_quantize(x[:0])
    assert q.shape == (0, 64) and s.shape == (0, 4) and ops.mxfp4_dequantize(q, s).shape == (0, 128)
    q, s = ops.mxfp4_quantize(x)
    got = ops.mxfp4_dequantize(q.t().contiguous().t(), s.t().contiguous().t())
    assert torch.equal(got.cpu().double(), N.q4(x.cpu()))
    big = torch.zeros(2 ** 31 // 4096 + 3, 4096, dtype=torch.bfloat16, device=dev)
    big[-1] = torch.arange(4096, device=dev) % 7
    q, s = ops.mxfp4_quantize(big)
    wq, ws = N.pack4(big[-1:].cpu())
    assert torch.equal(q[-1:].cpu(), wq) and torch.equal(s[-1:].cpu(), ws)
    assert not q[:-1].any()
    assert torch.equal(ops.mxfp4_dequantize(q, s)[-1:].cpu().double(), N.q4(big[-1:].cpu()))


# rows per expert: single tokens, empty experts, odd numbers, more than one tile; spare rows
# belong to no expert. Dims: whole and partial 256-k stages, odd numbers of blocks, one block
SERVE = [
    ("one row", [0, 0, 1, 0], 0, 64, 32),
    ("one row each", [1, 1, 1], 2, 96, 160),
    ("few rows", [3, 0, 8, 1], 0, 256, 128),
    ("17 rows", [17, 0, 2], 5, 288, 96),
    ("40 rows", [40, 33, 0, 64], 1, 544, 320),
    ("blocks past the row tile", [70, 100, 65, 3], 0, 320, 416),
    ("many rows", [300, 0, 77, 513], 9, 256, 256),
    ("many rows, odd dims", [1000, 130, 0, 300], 3, 416, 352),
    ("one expert", [700], 0, 96, 96),
    ("few rows, a long contraction", [3, 0, 1], 1, 7168, 64),
    ("two blocks of rows", [20, 33, 16, 0, 17, 32], 3, 2880, 96),
    ("17 rows, a long contraction", [17, 2, 0], 1, 4640, 4640),
    ("few rows, rows past the LDS", [2, 1], 0, 16384, 32),
    ("many experts", [0, 2, 0, 0, 17, 1] * 170 + [3, 0, 0, 9], 2, 64, 32),
    ("many experts, many rows", [0, 40, 0, 0, 300, 1] * 20, 2, 64, 96),
    ("many rows, partial stages", [240, 200, 0, 380], 1, 544, 320),
    ("past the row tile, odd blocks", [270, 300, 765, 3], 0, 320, 416),
    ("one expert, one stage", [2100], 0, 96, 96),
    ("small work, many rows", [510, 0, 255], 3, 288, 160),
    ("no rows for anyone", [0, 0, 0], 6, 64, 64),
]


def _packed(gen, e, n, k, std):
    w = torch.randn(e, n, k, generator=gen) * std * torch.exp(torch.randn(e, n, k // 32, generator=gen)).repeat_interleave(32, -1)
    return N.pack4(w)


@pytest.mark.parametrize("act", ["silu", "oss"])
@pytest.mark.parametrize("case", SERVE, ids=[c[0] for c in SERVE])
def test_serve(dev, act, case):
    name, counts, spare, d, h = case
    banner(f"mxfp4 experts {act} {name}")
    from torchtitan_amd import ops

    gen = torch.Generator().manual_seed(len(name) + d)
    e, rows = len(counts), sum(counts) + spare
    counts = torch.tensor(counts)
    x = torch.randn(rows, d, generator=gen).bfloat16()
    glu = 2 if act == "oss" else 1
    w1, w2 = _packed(gen, e, glu * h, d, 0.1), _packed(gen, e, d, h, 0.1)
    dv = lambda *ts: [t.to(dev) for t in ts]  # noqa: E731
    if act == "silu":
        w3 = _packed(gen, e, h, d, 0.1)
        got = ops.grouped_swiglu_mxfp4(*dv(x, *w1, *w2, *w3, counts))
        want, tol = N.experts4(N.q4(x), N.unpack4(*w1), N.unpack4(*w2), N.unpack4(*w3), counts)
    else:
        b1, b2 = torch.randn(e, 2 * h, generator=gen).bfloat16(), torch.randn(e, d, generator=gen).bfloat16()
        got = ops.grouped_swiglu_oss_mxfp4(*dv(x, *w1, b1, *w2, b2, counts), 1.5)
        v = N.unpack4(*w1)
        want, tol = N.experts4(N.q4(x), v[:, 0::2], N.unpack4(*w2), v[:, 1::2], counts, "oss", 1.5, b1.double(), b2.double())
    N.within(got, want, tol, name, Y_NORM)
    n = int(counts.sum())
    assert not got[n:].any()


@pytest.mark.parametrize("rows", [40, 2000])
def test_serve_odd_counts(dev, rows):
    """Counts that sum past the rows, negative counts, int32 counts: as the rows there are."""
    banner("mxfp4 experts odd counts")
    from torchtitan_amd import ops

    gen = torch.Generator().manual_seed(4)
    e, d, h = 5, 128, 96
    x = torch.randn(rows, d, generator=gen).bfloat16()
    w1, w2, w3 = _packed(gen, e, h, d, 0.1), _packed(gen, e, d, h, 0.1), _packed(gen, e, h, d, 0.1)
    vals = [N.unpack4(*w) for w in (w1, w2, w3)]
    for counts in ([10, -3, 20, 2 ** 40, 7], [2 ** 62, 2 ** 62, 5, 1, 1], [0, 0, 0, 0, rows]):
        c = torch.tensor(counts)
        got = ops.grouped_swiglu_mxfp4(*(t.to(dev) for t in (x, *w1, *w2, *w3, c)))
        want, tol = N.experts4(N.q4(x), *vals, c)
        N.within(got, want, tol, str(counts), Y_NORM)
    c = torch.tensor([10, 0, 20, 3, 7], dtype=torch.int32)
    a = ops.grouped_swiglu_mxfp4(*(t.to(dev) for t in (x, *w1, *w2, *w3, c)))
    b = ops.grouped_swiglu_mxfp4(*(t.to(dev) for t in (x, *w1, *w2, *w3, c.long())))
    assert torch.equal(a, b)
    empty = ops.grouped_swiglu_mxfp4(*(t.to(dev) for t in (x[:0], *w1, *w2, *w3, c)))
    assert empty.shape == (0, d)


@pytest.mark.parametrize("rows", [12, 600, 1800])
def test_serve_not_finite(dev, rows):
    """A row with an infinity or NaN spoils itself, an expert with a NaN scale its own rows;
    every other row keeps its bits."""
    banner(f"mxfp4 experts not finite {rows}")
    from torchtitan_amd import ops

    gen = torch.Generator().manual_seed(5)
    e, d, h = 3, 288, 160
    counts = torch.tensor([rows // 3] * 3)
    x = torch.randn(rows, d, generator=gen).bfloat16()
    w = [*_packed(gen, e, h, d, 0.1), *_packed(gen, e, d, h, 0.1), *_packed(gen, e, h, d, 0.1)]
    run = lambda xx, ww: ops.grouped_swiglu_mxfp4(*(t.to(dev) for t in (xx, *ww, counts)))  # noqa: E731
    want = run(x, w)
    bad = x.clone()
    bad[1, 3], bad[rows - 1, 287] = float("inf"), float("nan")
    got = run(bad, w)
    keep = torch.ones(rows, dtype=torch.bool)
    keep[1] = keep[rows - 1] = False
    assert got[1].isnan().all() and got[rows - 1].isnan().all()
    assert torch.equal(got[keep], want[keep])
    spoiled = [t.clone() for t in w]
    spoiled[1][1, 0, 0] = 255
    got = run(x, spoiled)
    a, b = rows // 3, 2 * (rows // 3)
    assert torch.equal(got[:a], want[:a]) and torch.equal(got[b:], want[b:]) and got[a:b].isnan().all()


@pytest.mark.parametrize("times", [1, 70])
def test_serve_views_and_alignment(dev, times):
    banner("mxfp4 experts views")
    from torchtitan_amd import ops

    gen = torch.Generator().manual_seed(6)
    e, d, h, rows = 4, 96, 64, 30 * times
    counts = torch.tensor([8, 2, 0, 20]).to(dev) * times
    x = torch.randn(rows, d, generator=gen).bfloat16().to(dev)
    w = [t.to(dev) for t in (*_packed(gen, e, h, d, 0.1), *_packed(gen, e, d, h, 0.1), *_packed(gen, e, h, d, 0.1))]
    want = ops.grouped_swiglu_mxfp4(x, *w, counts)

    def shifted(t):  # the same values one element off an aligned address
        flat = torch.zeros(t.numel() + 1, dtype=t.dtype, device=dev)
        flat[1:] = t.flatten()
        return flat[1:].view(t.shape)

    def strided(t):
        wide = torch.zeros(*t.shape[:-1], 2 * t.shape[-1], dtype=t.dtype, device=dev)
        wide[..., 1::2] = t
        return wide[..., 1::2]

    for f in (shifted, strided):
        assert torch.equal(ops.grouped_swiglu_mxfp4(f(x), *(f(t) for t in w), f(counts)), want)


def test_serve_streams_and_graph(dev):
    """Calls on two streams at once, and two captured graphs replayed in turn with eager calls
    between, each against the eager result."""
    banner("mxfp4 experts streams and graph")
    from torchtitan_amd import ops

    gen = torch.Generator().manual_seed(7)
    e, d, h = 8, 512, 256
    w = [t.to(dev) for t in (*_packed(gen, e, h, d, 0.1), *_packed(gen, e, d, h, 0.1), *_packed(gen, e, h, d, 0.1))]
    xs, cs = [], []
    for n in (24, 1200):
        pick = torch.randint(0, e, (n,), generator=gen)
        xs.append([torch.randn(n, d, generator=gen).bfloat16().to(dev) for _ in range(3)])
        cs.append(torch.bincount(pick, minlength=e).to(dev))
    want = [[ops.grouped_swiglu_mxfp4(x, *w, c) for x in xx] for xx, c in zip(xs, cs)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        got = []
        for s, xx, c in zip(streams, xs, cs):
            with torch.cuda.stream(s):
                got.append(ops.grouped_swiglu_mxfp4(xx[0], *w, c))
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0][0]) and torch.equal(got[1], want[1][0])
    graphs = []
    for xx, c in zip(xs, cs):
        fixed, g = xx[0].clone(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = ops.grouped_swiglu_mxfp4(fixed, *w, c)
        graphs.append((g, fixed, out))
    for turn in range(6):
        k = turn % 2
        g, fixed, out = graphs[k]
        fixed.copy_(xs[k][turn % 3])
        g.replay()
        eager = ops.grouped_swiglu_mxfp4(xs[1 - k][turn % 3], *w, cs[1 - k])
        torch.cuda.synchronize()
        assert torch.equal(out, want[k][turn % 3]) and torch.equal(eager, want[1 - k][turn % 3])


def test_serve_takes_no_gradients(dev):
    banner("mxfp4 experts no gradients")
    from torchtitan_amd import ops

    gen = torch.Generator().manual_seed(8)
    w = [t.to(dev) for t in (*_packed(gen, 2, 32, 64, 0.1), *_packed(gen, 2, 64, 32, 0.1), *_packed(gen, 2, 32, 64, 0.1))]
    x, c = torch.randn(4, 64).bfloat16().to(dev).requires_grad_(True), torch.tensor([2, 2], device=dev)
    with pytest.raises(RuntimeError, match="no gradients"):
        ops.grouped_swiglu_mxfp4(x, *w, c)
    with torch.no_grad():
        assert torch.equal(ops.grouped_swiglu_mxfp4(x, *w, c), ops.grouped_swiglu_mxfp4(x.detach(), *w, c))
    q, s = ops.mxfp4_quantize(x)  # codes have no gradients to lose
    assert not q.requires_grad and torch.equal(q, ops.mxfp4_quantize(x.detach())[0])
    b1, b2 = torch.zeros(2, 64, device=dev, requires_grad=True), torch.zeros(2, 64, device=dev)
    m1 = [t.to(dev) for t in _packed(gen, 2, 64, 64, 0.1)]
    with pytest.raises(RuntimeError, match="no gradients"):
        ops.grouped_swiglu_oss_mxfp4(x.detach(), *m1, b1, *w[2:4], b2, c, 7.0)
