"""The block-scaled formats and the experts on them in 64 bits, in plain torch on the CPU,
with the bounds that a kernel's outputs are held to."""

from __future__ import annotations

import torch

E2M1 = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
BF16_HALF = 2.0 ** -8  # half a step of bf16, relative
F32_HALF = 2.0 ** -24


def _scale(amax: torch.Tensor, most: float) -> torch.Tensor:
    """2^k, the least k in [-127, 127] with amax <= most 2^k (amax 0: 2^-127)."""
    return torch.exp2(torch.ceil(torch.log2(amax / most)).clamp(-127, 127))


def _round4(a: torch.Tensor) -> torch.Tensor:
    """Codes 0..7 of |a| <= 6, ties to the even code."""
    mid = (E2M1[1:] + E2M1[:-1]) / 2
    lo, hi = torch.bucketize(a, mid), torch.bucketize(a, mid, right=True)
    return torch.where(lo % 2 == 0, lo, hi)


def _round8(a: torch.Tensor) -> torch.Tensor:
    unit = torch.exp2(torch.floor(torch.log2(a.abs().clamp(min=2.0 ** -6))) - 3)
    return (a / unit).round() * unit


def q4(v: torch.Tensor, scale_of: torch.Tensor | None = None) -> torch.Tensor:
    """MXFP4's values of v [.., K] (64 bits); scale_of: the values that set the scales."""
    b = v.double().unflatten(-1, (-1, 32))
    t = b if scale_of is None else scale_of.double().unflatten(-1, (-1, 32))
    top = t.abs().amax(-1, keepdim=True)
    s = _scale(top, 6.0)
    out = torch.copysign(E2M1[_round4((b / s).abs().clamp(max=6.0))], b) * s
    return torch.where(top.isfinite(), out, torch.nan).flatten(-2)


def q8(v: torch.Tensor, scale_of: torch.Tensor | None = None) -> torch.Tensor:
    b = v.double().unflatten(-1, (-1, 32))
    t = b if scale_of is None else scale_of.double().unflatten(-1, (-1, 32))
    top = t.abs().amax(-1, keepdim=True)
    s = _scale(top, 448.0)
    out = _round8((b / s).clamp(-448.0, 448.0)) * s
    return torch.where(top.isfinite(), out, torch.nan).flatten(-2)


def pack4(v: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """The bytes and scale bytes of MXFP4."""
    b = v.double().unflatten(-1, (-1, 32))
    top = b.abs().amax(-1, keepdim=True)
    s = _scale(top, 6.0)
    code = _round4((b / s).abs()) | (torch.signbit(b).long() << 3)
    code = torch.where(top.isfinite(), code, 0).to(torch.uint8).flatten(-2)
    byte = torch.where(top.isfinite(), torch.log2(s) + 127, 255).to(torch.uint8).squeeze(-1)
    return code[..., 0::2] | (code[..., 1::2] << 4), byte


def unpack4(q: torch.Tensor, s: torch.Tensor) -> torch.Tensor:
    both = torch.cat([E2M1, -E2M1])
    v = torch.stack([both[(q & 15).long()], both[(q >> 4).long()]], -1).flatten(-2)
    sc = torch.where(s == 255, torch.nan, torch.exp2(s.double() - 127))
    return v * sc.repeat_interleave(32, dim=-1)


def spread(quant, v: torch.Tensor, off: torch.Tensor) -> torch.Tensor:
    """How far apart quant's results can be for values within `off` of v: the range over the
    values and the scales moved either way."""
    ends = (v - off, v, v + off)
    # the largest and the smallest magnitudes that can set a block's scale
    sizes = (torch.copysign((v.abs() - off).clamp(min=0), v), torch.copysign(v.abs() + off, v))
    got = torch.stack([quant(e, s) for e in ends for s in sizes])
    return got.amax(0) - got.amin(0)


def silu(g: torch.Tensor) -> torch.Tensor:
    return g * torch.sigmoid(g)


def segments(counts: torch.Tensor, rows: int) -> list[tuple[int, int]]:
    """Rows [a, b) of each expert, clamped to the rows there are; negative counts are none."""
    out, at = [], 0
    for c in counts.tolist():
        n = min(max(c, 0), rows - at)
        out.append((at, at + n))
        at += n
    return out


def sum_off(a: torch.Tensor, b: torch.Tensor) -> torch.Tensor:
    """The most that a sum over K products a @ b.T in 32 bits, in any order, is off."""
    return a.shape[-1] * F32_HALF * (a.abs() @ b.abs().t())


def activation(act: str, g: torch.Tensor, u: torch.Tensor, limit: float) -> torch.Tensor:
    if act == "silu":
        return silu(g) * u
    g, u = g.clamp(max=limit), u.clamp(-limit, limit)
    return g * torch.sigmoid(1.702 * g) * (u + 1)


def activation_off(act: str, g, u, dg, du, limit: float) -> torch.Tensor:
    """What errors dg, du (and a few fp32 roundings) can do to the activation: silu' and the
    gpt-oss gate's slope stay within 1.13, the gate's size is at most |g|."""
    if act == "oss":
        g, u = g.clamp(max=limit), u.clamp(-limit, limit) + 1
    return 1.13 * dg * (u.abs() + du) + (g.abs() + dg) * du + 64 * F32_HALF * (g * u).abs()


def experts4(xq, w1q, w2q, w3q, counts, act="silu", limit=7.0, b1=None, b2=None):
    """(y, its bound) of the experts on quantized operands: g, u and y within the sums' error,
    h's quantization moved where g and u can move it, y rounded to bf16 once."""
    rows = xq.shape[0]
    y = torch.zeros(rows, w2q.shape[1], dtype=torch.float64)
    tol = torch.zeros_like(y)
    for e, (a, b) in enumerate(segments(counts, rows)):
        if a == b:
            continue
        x = xq[a:b]
        g, u = x @ w1q[e].t(), x @ w3q[e].t()
        dg, du = sum_off(x, w1q[e]), sum_off(x, w3q[e])
        if b1 is not None:
            g, u = g + b1[e, 0::2], u + b1[e, 1::2]
            dg, du = dg + F32_HALF * g.abs(), du + F32_HALF * u.abs()
        h = activation(act, g, u, limit)
        off = spread(q4, h, activation_off(act, g, u, dg, du, limit))
        hq = q4(h)
        ye = hq @ w2q[e].t() + (b2[e] if b2 is not None else 0)
        te = sum_off(hq, w2q[e]) + off @ w2q[e].abs().t()
        y[a:b], tol[a:b] = ye, te + BF16_HALF * (ye.abs() + te)
    return y, tol


def gradients(x, w1, w2, w3, dy, counts, four: bool):
    """[(value, bound)] of y, dx, dw1, dw2, dw3 of the experts that keep g and u in MXFP8, on bf16
    operands (four False: dw with the kept x and h) or on MXFP4 ones."""
    rows, h_dim = x.shape[0], w1.shape[1]
    xf = q4(x) if four else x.double()
    w1, w2, w3 = ((q4(w) if four else w.double()) for w in (w1, w2, w3))
    kept_x = xf if four else q8(x)
    dy = dy.double()
    y = torch.zeros(rows, x.shape[1], dtype=torch.float64)
    out = [y, y.clone(), *(torch.zeros_like(w) for w in (w1, w2, w3))]
    tol = [torch.zeros_like(t) for t in out]

    def put(i, at, value, bound):
        out[i][at], tol[i][at] = value, bound + BF16_HALF * (value.abs() + bound)

    for e, (a, b) in enumerate(segments(counts, rows)):
        if a == b:
            continue
        at = slice(a, b)
        xe, de = xf[at], dy[at]
        g, u = xe @ w1[e].t(), xe @ w3[e].t()
        og, ou = sum_off(xe, w1[e]), sum_off(xe, w3[e])
        h = silu(g) * u
        if four:
            oh = spread(q4, h, activation_off("silu", g, u, og, ou, 0.0))
            h = q4(h)
        else:  # h rounded to bf16
            oh = activation_off("silu", g, u, og, ou, 0.0)
            oh = oh + BF16_HALF * (h.abs() + oh)
        put(0, at, h @ w2[e].t(), sum_off(h, w2[e]) + oh @ w2[e].abs().t())
        kg, ku = q8(g), q8(u)
        og, ou = spread(q8, g, og), spread(q8, u, ou)
        s = torch.sigmoid(kg)
        dh = de @ w2[e]
        odh = sum_off(de, w2[e].t())
        du = dh * kg * s
        slope = s * (1 + kg * (1 - s))
        dg = dh * ku * slope
        # silu' is within 1.13 and its own slope within 0.5; one rounding to bf16 after a few in fp32
        odu = odh * (kg * s).abs() + (dh.abs() + odh) * 1.13 * og
        odg = odh * (ku * slope).abs() + (dh.abs() + odh) * (1.13 * ou + 0.5 * og * (ku.abs() + ou))
        odu, odg = (o + (BF16_HALF + 64 * F32_HALF) * (v.abs() + o) + 64 * F32_HALF * dh.abs() * w
                    for o, v, w in ((odu, du, 0 * ku.abs()), (odg, dg, ku.abs())))
        both, w13 = torch.cat([dg, du], 1), torch.cat([w1[e], w3[e]])
        put(1, at, both @ w13, sum_off(both, w13.t()) + torch.cat([odg, odu], 1) @ w13.abs())
        kx = kept_x[at]
        kh, okh = (h, oh) if four else (kg * s * ku, 1.13 * og * (ku.abs() + ou) + (kg * s).abs() * ou)
        if not four:
            okh = okh + (BF16_HALF + 64 * F32_HALF) * (kh.abs() + okh)
        put(2, e, dg.t() @ kx, sum_off(dg.t(), kx.t()) + odg.t() @ kx.abs())
        put(3, e, de.t() @ kh, sum_off(de.t(), kh.t()) + de.abs().t() @ okh)
        put(4, e, du.t() @ kx, sum_off(du.t(), kx.t()) + odu.t() @ kx.abs())
    return list(zip(out, tol))


def within(got: torch.Tensor, want: torch.Tensor, tol: torch.Tensor, what: str, norm: float) -> None:
    """Every element within its bound, and the whole within `norm` of its size: the bounds
    take every rounding at its worst, which together they are not."""
    got = got.detach().double().cpu()
    off = (got - want).abs()
    bad = ~(off <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} elements off, worst {off[bad].max():.3g} for {tol[bad][off[bad].argmax()]:.3g}"
    size = want.norm()
    if size:
        assert off.norm() <= norm * size, f"{what}: {off.norm() / size:.3g} of its size off"
