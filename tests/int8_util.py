"""8-bit integers with a scale per row, and the products on them, in 64 bits in plain torch, with
the bounds that a kernel's outputs are held to."""

from __future__ import annotations

import torch

LEAST = 127.0 * 2.0 ** -126
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}  # half a step, relative
U = 2.0 ** -24  # one rounding to fp32


def multiplier(v: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """r and s [.., 1] of v's rows as 32-bit numbers (64 bits round to them correctly: a quotient of
    24 by 7 bits is never so near the middle of two of them without being it), r = 0 and s = NaN
    where a row is not finite."""
    top = v.abs().amax(-1, keepdim=True).double()
    a = top.float().clamp(min=LEAST).double()
    ok = top.isfinite()
    return torch.where(ok, (127.0 / a).float().double(), 0.0), torch.where(ok, (a / 127.0).float().double(), torch.nan)


def pack(v: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes (int8) and scales (fp32) of bf16 or fp32 rows."""
    r, s = multiplier(v)
    q = torch.where(r == 0, 0.0, torch.nan_to_num(v.double() * r).round())
    return q.to(torch.int8), s.squeeze(-1).float()


def values(q: torch.Tensor, s: torch.Tensor) -> torch.Tensor:
    return q.double() * s.double().unsqueeze(-1)


def linear(x: torch.Tensor, qw: torch.Tensor, sw: torch.Tensor, bias: torch.Tensor | None, dtype: torch.dtype):
    """(y, bound) of rows x [M, K] by a weight [N, K]. The sums of codes are exact; float(sum), its two
    scales and the bias are four roundings to fp32, then one to dtype."""
    q, s = pack(x)
    p = q.double() @ qw.double().T * s.double().unsqueeze(-1) * sw.double()
    y = p if bias is None else p + bias.double()
    tol = 3.01 * U * p.abs() + 1.01 * U * y.abs()
    return y, tol + HALF[dtype] * (y.abs() + tol) + 2.0 ** -140


def hidden(x, w1, w3, b, limit):
    """(h, its bound) of act(g, u): w1, w3 packed, b = (bias of g, of u) or None."""
    q, s = pack(x)
    def part(w, bias):
        p = q.double() @ w[0].double().T * s.double().unsqueeze(-1) * w[1].double()
        y = p if bias is None else p + bias.double()
        return y, 3.01 * U * p.abs() + (0 if bias is None else 1.01 * U * y.abs())
    g, dg = part(w1, b and b[0])
    u, du = part(w3, b and b[1])
    if b is not None:
        g, u = g.clamp(max=limit), u.clamp(-limit, limit) + 1
        du = du + 1.01 * U * u.abs()
        z = 1.702 * g
        dz = 1.702 * dg + 1.5 * U * z.abs()  # 1.702 in fp32, and the product
    else:
        z, dz = g, dg
    sig = 1 / (1 + torch.exp(-z))
    # the exponential, the sum and the reciprocal: each within 2 units of half a last place, and the
    # exponent's remainder: under 8 U together; past 2^100 the exponent is not corrected
    rel = 8 * U + torch.where(z < -60, z.abs() * U, 0.0)
    dsig = sig * (rel + dz * (1 - sig))
    h = g * sig * u
    dh = (dg * sig + g.abs() * dsig) * u.abs() + (g * sig).abs() * du + 2.02 * U * h.abs()
    return h, 1.01 * dh + 2.0 ** -120


def second(h, dh, qw, sw, bias, dtype):
    """(y, bound) of h's rows, quantized from values that dh bounds, by a packed weight: a code moves
    by one where h r lies nearer the middle of two than its own uncertainty, and the row's
    multiplier and scale move with its largest."""
    top, at = h.abs().max(-1, keepdim=True)
    r, s = multiplier(h)
    most = torch.maximum((dh.gather(-1, at) / top.clamp(min=LEAST)), ((h.abs() + dh).amax(-1, keepdim=True) / top.clamp(min=LEAST) - 1))
    drift = most + 2.02 * U  # of r and of s, relative
    t = h * r
    q = t.round()
    room = 0.5 - (t - q).abs()
    moved = (room <= dh * r + t.abs() * drift).double()
    w = qw.double() * sw.double().unsqueeze(-1)
    p = q @ w.T * s
    y = p if bias is None else p + bias.double()
    off = moved @ w.abs().T * s + drift * (q.abs() @ w.abs().T * s)
    tol = off + 3.01 * U * p.abs() + 1.01 * U * y.abs()
    return y, tol + HALF[dtype] * (y.abs() + tol) + 2.0 ** -120


def segments(counts, rows):
    """(expert, first row, end) of the experts with rows, clamped to the rows there are."""
    at = 0
    for e, c in enumerate(counts.tolist()):
        end = min(at + max(c, 0), rows)
        if end > at:
            yield e, at, end
        at = end


def grouped(x, n, counts, f, dtype):
    """(y, bound) [R, n] with f(expert, rows of x) -> (y, bound); zeros behind the last expert's."""
    y = torch.zeros(x.shape[0], n, dtype=torch.float64)
    tol = torch.zeros_like(y)
    for e, a, b in segments(counts, x.shape[0]):
        y[a:b], tol[a:b] = f(e, x[a:b])
    return y, tol


def experts(x, w1, w2, w3, counts):
    """The SwiGLU experts on packed weights ((q, s) each, [E, ..])."""
    def one(e, xe):
        h, dh = hidden(xe, [t[e] for t in w1], [t[e] for t in w3], None, 0.0)
        return second(h, dh, w2[0][e], w2[1][e], None, x.dtype)
    return grouped(x, w2[0].shape[1], counts, one, x.dtype)


def oss(x, m1, b1, m2, b2, counts, limit):
    def one(e, xe):
        g, u = [t[e, 0::2] for t in m1], [t[e, 1::2] for t in m1]
        h, dh = hidden(xe, g, u, (b1[e, 0::2], b1[e, 1::2]), limit)
        return second(h, dh, m2[0][e], m2[1][e], b2[e], x.dtype)
    return grouped(x, m2[0].shape[1], counts, one, x.dtype)


def within(got: torch.Tensor, want: torch.Tensor, tol: torch.Tensor, what: str) -> None:
    g = got.detach().cpu().double()
    assert g.shape == want.shape, f"{what}: {tuple(g.shape)} for {tuple(want.shape)}"
    nan = want.isnan()
    assert torch.equal(g.isnan(), nan), f"{what}: NaN where there is none, or none where there is"
    over = ((g - want).abs() > tol) & ~nan
    if over.any():
        i = over.nonzero()[0].tolist()
        raise AssertionError(f"{what}: {int(over.sum())} of {over.numel()} outside, first at {i}: {g[tuple(i)].item()!r} for "
                             f"{want[tuple(i)].item()!r} +- {tol[tuple(i)].item()!r}")


def weight(gen, *shape, std=0.1) -> tuple[torch.Tensor, torch.Tensor]:
    return pack(torch.randn(*shape, generator=gen) * std)


def rows(gen, n, cols, dtype=torch.bfloat16) -> torch.Tensor:
    return (torch.randn(n, cols, generator=gen) * torch.exp(torch.randn(1, cols, generator=gen))).to(dtype)
