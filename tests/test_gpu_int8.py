"""8-bit integers on the GPU against 64 bits: rows to codes and back, dense and grouped products,
the shared expert and the experts on packed weights."""

import pytest
import torch

from tests import int8_util as I
from tests.conftest import banner

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


# ---------------------------------------------------------------------------
# quantization
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("shape", [(1, 1), (3, 7), (2, 8), (5, 7, 64), (257, 1472), (4, 4096), (3, 4104), (2, 20480), (130, 2880),
                                   (2, 4097)])
def test_quantize_bits(dev, dtype, shape):
    banner(f"int8_quantize {shape} {dtype}")
    from torchtitan_amd import ops

    gen = torch.Generator().manual_seed(1)
    x = I.rows(gen, torch.Size(shape).numel() // shape[-1], shape[-1], dtype).view(shape)
    q, s = ops.int8_quantize(x.to(dev))
    wq, ws = I.pack(x)
    assert q.dtype == torch.int8 and s.shape == shape[:-1]
    assert torch.equal(s.cpu(), ws) and torch.equal(q.cpu(), wq)
    back = ops.int8_dequantize(q, s, dtype)
    assert back.dtype == dtype and torch.equal(back.cpu(), (wq.float() * ws.unsqueeze(-1)).to(dtype))


def test_quantize_borders(dev):
    """Halves of the largest (ties and what lies next to them), every bf16 below the largest."""
    banner("int8_quantize borders")
    from torchtitan_amd import ops

    bits = torch.arange(0, 0x4000, dtype=torch.int32).to(torch.int16).view(BF)  # 0 .. 2
    for top in (2.0, 127.0, 254.0, 1.9921875, 3.0, 1.0078125):
        x = torch.cat([bits[bits <= top], torch.tensor([top], dtype=BF)])
        x = torch.stack([x, -x])
        for v in (x, x.float() * 1.0000001):
            q, s = ops.int8_quantize(v.to(dev))
            wq, ws = I.pack(v)
            assert torch.equal(q.cpu(), wq) and torch.equal(s.cpu(), ws), top
    n = torch.arange(-127, 127).float() + 0.5  # exact ties, r = 1
    x = torch.cat([n, torch.tensor([127.0])]).unsqueeze(0)
    q, s = ops.int8_quantize(x.to(dev))
    assert s.item() == 1.0 and torch.equal(q.cpu()[0, :-1].float(), n.round())


def test_quantize_odd_rows(dev):
    """Zeros, the smallest numbers, the largest, infinities and NaN; a row's neighbours keep theirs."""
    banner("int8_quantize odd rows")
    from torchtitan_amd import ops

    for cols in (40, 41, 4200):
        x = torch.randn(9, cols, generator=torch.Generator().manual_seed(2))
        x[0] = 0.0
        x[1] = -0.0
        x[2] = 2.0 ** -149
        x[3] *= 2.0 ** -125
        x[4] *= 1e38 / x[4].abs().max()
        x[5, 3] = float("inf")
        x[6, -1] = float("nan")
        x[7, 0] = -float("inf")
        q, s = ops.int8_quantize(x.to(dev))
        wq, ws = I.pack(x)
        assert torch.equal(q.cpu(), wq)
        assert torch.equal(s.cpu().view(torch.int32)[:5], ws.view(torch.int32)[:5]) and s[8].item() == ws[8].item()
        assert s[5:8].isnan().all() and not q[5:8].any()
        assert ops.int8_dequantize(q, s)[5:8].isnan().all()


def test_quantize_views(dev):
    """Rows of a wider matrix, transposed, one element off, none at all."""
    banner("int8_quantize views")
    from torchtitan_amd import ops

    gen = torch.Generator().manual_seed(3)
    wide = torch.randn(33, 320, generator=gen).bfloat16().to(dev)
    for x in (wide[:, 64:192], wide[:, 1:129], wide[:, :131], wide.t(), wide[::2, ::2], wide[:1, 5:], wide[:0], wide.view(3, 11, 320)[:, :, 8:80],
              wide[:1].expand(4, 320)):
        q, s = ops.int8_quantize(x)
        wq, ws = I.pack(x.cpu())
        assert torch.equal(q.cpu(), wq) and torch.equal(s.cpu(), ws)
        assert torch.equal(ops.int8_dequantize(q, s, F32).cpu(), wq.float() * ws.unsqueeze(-1))


# ---------------------------------------------------------------------------
# products
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("k,n", [(16, 1), (48, 7), (128, 64), (144, 33), (272, 1001), (2304, 200), (7168, 48), (10240, 24)])
def test_linear(dev, k, n, dtype):
    from torchtitan_amd import ops

    gen = torch.Generator().manual_seed(4)
    w = I.weight(gen, n, k)
    bias = torch.randn(n, generator=gen)
    for m in (1, 2, 3, 5, 16, 17, 33, 100, 257, 300):
        banner(f"linear_int8 {m} x {n} x {k} {dtype}")
        x = I.rows(gen, m, k, dtype)
        for b in (None, bias.to(dtype)):
            got = ops.linear_int8(x.to(dev), *(t.to(dev) for t in w), None if b is None else b.to(dev))
            assert got.dtype == dtype
            I.within(got, *I.linear(x, *w, b, dtype), f"{m} rows")


def test_linear_extremes(dev):
    """The longest contraction at the codes' largest products, whose sums pass 2^31 - 2^25; a code of
    -128, which int8_quantize does not give."""
    banner("linear_int8 extremes")
    from torchtitan_amd import ops

    k = 131072
    x = torch.full((2, k), -3.0)
    x[1, ::2] = 3.0
    qw = torch.full((3, k), -128, dtype=torch.int8)
    qw[1, ::2], qw[2] = 127, 127
    sw = torch.tensor([0.5, 0.25, 1e-3])
    for m in (1, 150):
        xx = x.repeat(m, 1)
        got = ops.linear_int8(xx.to(dev), qw.to(dev), sw.to(dev))
        I.within(got, *I.linear(xx, qw, sw, None, F32), "extremes")


@pytest.mark.parametrize("dtype", [BF, F32])
def test_linear_of_rows_at_the_end_of_the_range(dev, dtype):
    """Rows that hold the type's lowest value, by weights that bring the result back into its range, as
    well as rows and weights at the small end: no product of a sum with one scale alone may overflow
    or lose bits."""
    banner(f"linear_int8 range {dtype}")
    from torchtitan_amd import ops

    gen = torch.Generator().manual_seed(8)
    k, n = 208, 72
    for r in (1, 3, 150, 700):
        x = I.rows(gen, r, k, dtype)
        x[0, 5] = torch.finfo(dtype).min
        if r > 1:
            x[1] *= 2.0 ** -80
            x[2] *= 2.0 ** 105
        for power in (-30, 0, 10):
            w = I.weight(gen, n, k, std=2.0 ** power)
            bias = torch.randn(n, generator=gen).to(dtype)
            y, tol = I.linear(x, *w, bias, dtype)
            got = ops.linear_int8(x.to(dev), *(t.to(dev) for t in w), bias.to(dev))
            inside = (y.abs() + tol < torch.finfo(dtype).max).all(-1)
            assert inside[1:].all() and (bool(inside[0]) or power >= 0), "range"
            I.within(got[inside.to(dev)], y[inside], tol[inside], f"{r} rows, weights of 2^{power}")


def test_layers_of_rows_at_the_end_of_the_range(dev):
    banner("layers range")
    from torchtitan_amd import ops

    gen = torch.Generator().manual_seed(9)
    e, d, h = 3, 144, 80
    for per in (1, 3, 200):
        counts = torch.full((e,), per)
        x = I.rows(gen, e * per, d, BF)
        x[::2, 7] = torch.finfo(BF).min
        x[::2] *= 2.0 ** -10
        w1, w3 = (I.weight(gen, e, h, d, std=2.0 ** -100) for _ in range(2))
        w2 = I.weight(gen, e, d, h)
        got = ops.grouped_swiglu_int8(x.to(dev), *(t.to(dev) for w in (w1, w2, w3) for t in w), counts.to(dev))
        I.within(got, *I.experts(x, w1, w2, w3, counts), f"{per} rows an expert")


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("e,k,n", [(1, 64, 24), (5, 208, 40), (8, 2304, 136), (40, 320, 260), (3, 96, 1001)])
def test_grouped_linear(dev, e, k, n, dtype):
    from torchtitan_amd import ops

    gen = torch.Generator().manual_seed(5)
    w = I.weight(gen, e, n, k)
    bias = torch.randn(e, n, generator=gen).to(dtype)
    for per in (0.3, 2, 20, 90):
        counts = torch.poisson(torch.full((e,), float(per)) * torch.rand(e, generator=gen) * 2, generator=gen).long()
        counts[e // 2] = 0 if e > 1 else counts[0]
        for spare in (0, 3):
            r = int(counts.sum()) + spare
            banner(f"grouped_linear_int8 {counts.tolist()[:8]} + {spare} x {n} x {k} {dtype}")
            x = I.rows(gen, r, k, dtype)
            for b in (None, bias):
                got = ops.grouped_linear_int8(x.to(dev), *(t.to(dev) for t in w), counts.to(dev), None if b is None else b.to(dev))
                f = lambda i, xe: I.linear(xe, w[0][i], w[1][i], None if b is None else b[i], dtype)  # noqa: E731, B023
                I.within(got, *I.grouped(x, n, counts, f, dtype), f"{per} a row")


def test_counts_past_the_rows(dev):
    """Negative counts are none, those past the rows there are end at them; any integer type."""
    banner("int8 counts")
    from torchtitan_amd import ops

    gen = torch.Generator().manual_seed(6)
    e, k, n = 5, 96, 80
    w = I.weight(gen, e, n, k)
    wd = [t.to(dev) for t in w]
    for r in (40, 700):
        x = I.rows(gen, r, k)
        for counts in ([10, -3, 20, 2 ** 40, 7], [2 ** 62, 2 ** 62, 5, 1, 1], [0, 0, 0, 0, r], [0] * 5):
            c = torch.tensor(counts)
            got = ops.grouped_linear_int8(x.to(dev), *wd, c.to(dev))
            I.within(got, *I.grouped(x, n, c, lambda i, xe: I.linear(xe, w[0][i], w[1][i], None, BF), BF), str(counts))
        c = torch.tensor([10, 0, 20, 3, 5], dtype=torch.int32).to(dev)
        assert torch.equal(ops.grouped_linear_int8(x.to(dev), *wd, c), ops.grouped_linear_int8(x.to(dev), *wd, c.long()))


# ---------------------------------------------------------------------------
# layers
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("d,h", [(16, 16), (64, 48), (304, 144), (2304, 1024)])
def test_feed_forward(dev, d, h):
    from torchtitan_amd import ops

    gen = torch.Generator().manual_seed(7)
    w1, w2, w3 = I.weight(gen, h, d), I.weight(gen, d, h), I.weight(gen, h, d)
    wd = [t.to(dev) for t in (*w1, *w2, *w3)]
    for m in (1, 4, 7, 40, 300):
        banner(f"swiglu_ffn_int8 {m} x {d} x {h}")
        x = I.rows(gen, m, d)
        got = ops.swiglu_ffn_int8(x.to(dev), *wd)
        hid = I.hidden(x, w1, w3, None, 0.0)
        I.within(got, *I.second(*hid, *w2, None, BF), f"{m} rows")
    x = I.rows(gen, 6, d).view(2, 3, d).to(dev)
    assert torch.equal(ops.swiglu_ffn_int8(x, *wd), ops.swiglu_ffn_int8(x.view(6, d), *wd).view(2, 3, d))


@pytest.mark.parametrize("act", ["silu", "oss"])
@pytest.mark.parametrize("e,d,h", [(1, 32, 16), (6, 144, 208), (4, 2880, 720), (40, 272, 320)])
def test_experts(dev, act, e, d, h):
    from torchtitan_amd import ops

    gen = torch.Generator().manual_seed(8)
    w1 = I.weight(gen, e, h if act == "silu" else 2 * h, d)
    w2, w3 = I.weight(gen, e, d, h), I.weight(gen, e, h, d)
    for per in (0.3, 3, 25, 100):
        counts = torch.poisson(torch.full((e,), float(per)) * torch.rand(e, generator=gen) * 2, generator=gen).long()
        counts[e // 2] = 1 if e == 1 else 0
        r = int(counts.sum()) + 2
        banner(f"int8 experts {act} {e} of {d} / {h}, {r} rows")
        x = I.rows(gen, r, d)
        xd, cd = x.to(dev), counts.to(dev)
        if act == "silu":
            got = ops.grouped_swiglu_int8(xd, *(t.to(dev) for t in (*w1, *w2, *w3)), cd)
            I.within(got, *I.experts(x, w1, w2, w3, counts), f"{per} a row")
        else:
            for dt in (BF, F32):
                b1, b2 = torch.randn(e, 2 * h, generator=gen).to(dt), torch.randn(e, d, generator=gen).to(dt)
                got = ops.grouped_swiglu_oss_int8(xd, *(t.to(dev) for t in (*w1, b1, *w2, b2)), cd, 1.5)
                I.within(got, *I.oss(x, w1, b1, w2, b2, counts, 1.5), f"{per} a row")
