"""Inference on 8-bit integers that is timed: rows to 8 bits with a scale for each, dense
and expert-grouped products with scales for each token and each output channel, and the
SwiGLU layers made of them.

Every case is a plain dict; ``kind`` names the operator:

* ``quantize``: a matrix to 8-bit integers with a scale for each row, and the values they
  stand for, in the matrix's type.
* ``linear``: a dense product of rows, quantized on the way, with a packed weight; with or
  without a bias.
* ``grouped``: the same with one weight per expert, on rows sorted by expert.
* ``ffn``: a shared expert, w2(silu(w1 x) w3 x), on packed weights.
* ``experts``: the same per expert (``act`` "silu"), or gpt-oss's biased and clamped experts
  ("oss"), on rows sorted by expert; the activation is quantized between the products.

Rows past the last expert's belong to no token and come out as zeros. With the 32-bit numbers

    a = max(max |v|, 127 * 2^-126), r = 127 / a, s = a / 127

of a row v, its codes are q = v r rounded once to the nearest integer, ties to even, and stand
for q s. A product of a row and a weight row (out channel) n is

    y_n = s s_n (q . q_n) + b_n

with a sum of integers, and the activation between two products, silu(g) u or gpt-oss's, is
quantized from 32 bits; the layers that have one take and return bf16.

Sizes are those of the layers that this repository's benchmark and tests name (dims
256/512, 2304/1024, 7168/2048, 2880/2880) and generic ones between them.
"""

from __future__ import annotations

import math

import torch

DEV = "cuda"
own = False
LIMIT = 7.0  # gpt-oss's clamp
ALPHA = 1.702
TINY = 127.0 * 2.0 ** -126


def listed() -> list[dict]:
    return [
        # The activations of one generation step of 64 sequences: a launch's latency.
        dict(name="quantize_step", kind="quantize", rows=64, cols=2304, dtype="bf16"),
        # The routed rows of 4 x 4096 tokens, top 8.
        dict(name="quantize_batch", kind="quantize", rows=131072, cols=2304, dtype="bf16"),
        # One token through a projection of a wide layer.
        dict(name="linear_token", kind="linear", rows=1, dim=7168, out=2048, bias=False, dtype="bf16"),
        # A prompt of an odd number of tokens in fp32, biased, to a width off every tile.
        dict(name="linear_prompt_fp32", kind="linear", rows=1003, dim=2880, out=1001, bias=True, dtype="fp32"),
        # 4 x 4096 tokens through a projection of a wide layer.
        dict(name="linear_batch", kind="linear", rows=16384, dim=7168, out=7168, bias=False, dtype="bf16"),
        # One generation step of 64 sequences through one biased projection of 32 experts, top 4.
        dict(name="grouped_step", kind="grouped", tokens=64, top_k=4, dim=2880, out=2880, experts=32, skew=0.3, spare=0,
             bias=True, dtype="bf16"),
        # 4 x 4096 tokens through one projection of the benchmark's layer, a few rows behind.
        dict(name="grouped_batch", kind="grouped", tokens=16384, top_k=8, dim=2304, out=1024, experts=256, skew=0.3,
             spare=77, bias=False, dtype="bf16"),
        # The shared expert of the benchmark's layer: one token, and 4 x 4096.
        dict(name="ffn_token", kind="ffn", rows=1, dim=2304, hidden=1024, dtype="bf16"),
        dict(name="ffn_batch", kind="ffn", rows=16384, dim=2304, hidden=1024, dtype="bf16"),
        # One token of one sequence through a 256-expert layer, top 8: eight experts' weights.
        dict(name="experts_token", kind="experts", act="silu", tokens=1, top_k=8, dim=2304, hidden=1024, experts=256,
             skew=0.0, spare=0, dtype="bf16"),
        # Prefill of a padded batch of prompts through gpt-oss-20b's experts, an odd number of tokens.
        dict(name="experts_prompts_gptoss", kind="experts", act="oss", tokens=4097, top_k=4, dim=2880, hidden=2880,
             experts=32, skew=0.3, spare=108, dtype="bf16"),
        # The benchmark's layer: 4 x 4096 tokens at once.
        dict(name="experts_batch", kind="experts", act="silu", tokens=16384, top_k=8, dim=2304, hidden=1024, experts=256,
             skew=0.3, spare=0, dtype="bf16"),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    kind = rng.choice(["quantize", "linear", "linear", "grouped", "ffn", "experts", "experts"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
    if kind == "quantize":
        cols = _log_int(rng, 100, 8000)
        return dict(kind=kind, rows=_log_int(rng, 1, 150_000_000 // cols), cols=cols, dtype=dtype)
    dim = 16 * _log_int(rng, 16, 448)
    if kind == "linear":
        return dict(kind=kind, rows=_log_int(rng, 1, 16384), dim=dim, out=_log_int(rng, 100, 7000),
                    bias=rng.random() < 0.4, dtype=dtype)
    if kind == "ffn":
        return dict(kind=kind, rows=_log_int(rng, 1, 16384), dim=dim, hidden=16 * _log_int(rng, 16, 128), dtype="bf16")
    dim = 16 * _log_int(rng, 16, 180)
    top_k = rng.choice([1, 2, 4, 6, 8])
    tail = dict(tokens=_log_int(rng, 1, 49152 // top_k), top_k=top_k, dim=dim, skew=rng.choice([0.0, 0.3, 0.7, 1.0]),
                spare=rng.choice([0, 0, _log_int(rng, 1, 300)]), dtype="bf16" if kind == "experts" else dtype)
    if kind == "grouped":
        return dict(kind=kind, out=_log_int(rng, 100, 2880), experts=rng.choice([8, 32, 48, 64, 128]),
                    bias=rng.random() < 0.4, **tail)
    act = rng.choice(["silu", "silu", "oss"])
    return dict(kind=kind, act=act, hidden=16 * _log_int(rng, 16, 128),
                experts=rng.choice([8, 32, 48, 64, 128]) if act == "silu" else 32, **tail)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _normal(gen, *shape, std=1.0, dtype=torch.bfloat16) -> torch.Tensor:
    t = torch.randn(*shape, generator=gen, device=DEV, dtype=torch.float32)
    return (t * std).to(dtype)


def _activations(gen, rows: int, cols: int, dtype) -> torch.Tensor:
    """Rows with channels of unlike size, as activations have them."""
    x = torch.randn(rows, cols, generator=gen, device=DEV)
    return (x * torch.exp(0.5 * torch.randn(1, cols, generator=gen, device=DEV))).to(dtype)


def _packed_normal(gen, *shape, std: float) -> tuple[torch.Tensor, torch.Tensor]:
    """A weight of a normal distribution, its rows' codes and scales."""
    q = torch.empty(shape, dtype=torch.int8, device=DEV)
    s = torch.empty(shape[:-1], dtype=torch.float32, device=DEV)
    for i in range(shape[0]) if len(shape) == 3 else [slice(None)]:
        v, scale = _codes(torch.randn(shape[-2:], generator=gen, device=DEV) * std)
        q[i], s[i] = v.to(torch.int8), scale
    return q, s


def _counts(case: dict, seed: int) -> torch.Tensor:
    """Rows per expert: every token takes its top_k experts, distinct, by random scores
    on top of each expert's own load."""
    gen = torch.Generator().manual_seed(seed + 17)
    e = case["experts"]
    load = case["skew"] * torch.randn(e, generator=gen, dtype=torch.float64)
    score = load - torch.log(-torch.log(torch.rand(case["tokens"], e, generator=gen, dtype=torch.float64)))
    return torch.bincount(score.topk(case["top_k"], dim=1).indices.reshape(-1), minlength=e)


def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device=DEV).manual_seed(seed)
    kind = case["kind"]
    dt = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
    st: dict = {"kind": kind, "bias": None}
    if kind == "quantize":
        st["x"] = _activations(gen, case["rows"], case["cols"], dt)
        return st
    d = case["dim"]
    if kind == "linear":
        st["x"] = _activations(gen, case["rows"], d, dt)
        st["w"] = _packed_normal(gen, case["out"], d, std=0.02)
        if case["bias"]:
            st["bias"] = _normal(gen, case["out"], std=0.5, dtype=dt)
        return st
    if kind == "ffn":
        h = case["hidden"]
        st["x"] = _activations(gen, case["rows"], d, dt)
        st["w"] = [*_packed_normal(gen, h, d, std=0.02), *_packed_normal(gen, d, h, std=0.02),
                   *_packed_normal(gen, h, d, std=0.02)]
        return st
    e = case["experts"]
    counts = _counts(case, seed)
    st["counts"] = counts.to(DEV)
    st["x"] = _activations(gen, int(counts.sum()) + case["spare"], d, dt)
    # the plain forms' plan: rows in a batch of one block of rows per expert with rows
    used = torch.nonzero(counts).flatten()
    n = counts[used]
    cap = max(int(n.max()), 1)
    owner = torch.repeat_interleave(torch.arange(used.numel()), n)
    start = torch.cumsum(n, 0) - n
    st["cap"], st["slot"] = cap, (owner * cap + torch.arange(owner.numel()) - start[owner]).to(DEV)
    st["used"] = used.to(DEV)
    if kind == "grouped":
        st["w"] = _packed_normal(gen, e, case["out"], d, std=0.02)
        if case["bias"]:
            st["bias"] = _normal(gen, e, case["out"], std=0.5, dtype=dt)
        return st
    h, st["act"] = case["hidden"], case["act"]
    if case["act"] == "silu":
        st["w"] = [*_packed_normal(gen, e, h, d, std=0.02), *_packed_normal(gen, e, d, h, std=0.02),
                   *_packed_normal(gen, e, h, d, std=0.02)]
    else:  # gate and up rows alternate
        st["w"] = [*_packed_normal(gen, e, 2 * h, d, std=0.02), _normal(gen, e, 2 * h, std=0.5),
                   *_packed_normal(gen, e, d, h, std=0.02), _normal(gen, e, d, std=0.5)]
    return st


# ---------------------------------------------------------------------------
# plain forms, in 32 bits
# ---------------------------------------------------------------------------
def _codes(v: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """The codes of rows [.., K] as fp32 numbers, and their scales [..]. A code is rounded from
    the whole product v r (48 bits), which 64 bits hold; the quotients are taken in 64 bits, since
    torch divides by and into a constant with a rounded reciprocal."""
    a = v.abs().amax(-1).float().clamp(min=TINY).double()
    r, s = (127.0 / a).float(), (a / 127.0).float()
    return torch.round(v.double() * r.double().unsqueeze(-1)).float(), s


def _spread(a: torch.Tensor, st: dict, e: int) -> torch.Tensor:
    """Rows [R, K] in one block of cap rows per expert, [E, cap, K], the rest zeros."""
    n = st["slot"].shape[0]
    return a.new_zeros(e * st["cap"], a.shape[1]).index_copy_(0, st["slot"], a[:n]).view(e, st["cap"], -1)


def _gather(b: torch.Tensor, st: dict, rows: int) -> torch.Tensor:
    """The rows of _spread's layout back in order; those past the last expert's are zeros."""
    n = st["slot"].shape[0]
    out = b.new_zeros(rows, b.shape[-1])
    out[:n] = b.reshape(-1, b.shape[-1])[st["slot"]]
    return out


def _product(x: torch.Tensor, qw: torch.Tensor, sw: torch.Tensor, bias) -> torch.Tensor:
    """Rows [E, M, K] in fp32, quantized, by packed weights [E, N, K]."""
    q, s = _codes(x)
    y = torch.bmm(q, qw.float().transpose(1, 2).contiguous()) * s.unsqueeze(-1) * sw.unsqueeze(1)
    return y if bias is None else y + bias.float().unsqueeze(1)


def _plain(st: dict):
    x, kind = st["x"], st["kind"]
    if kind == "quantize":
        q, s = _codes(x)
        return [(q * s.unsqueeze(-1)).to(x.dtype), s]
    if kind == "linear":
        bias = st["bias"]
        y = _product(x.float().unsqueeze(0), *(t.unsqueeze(0) for t in st["w"]), None if bias is None else bias.unsqueeze(0))
        return y[0].to(x.dtype)
    if kind == "ffn":
        w = [t.unsqueeze(0) for t in st["w"]]
        x32 = x.float().unsqueeze(0)
        g, u = _product(x32, w[0], w[1], None), _product(x32, w[4], w[5], None)
        return _product(g * torch.sigmoid(g) * u, w[2], w[3], None)[0].to(x.dtype)
    used = st["used"]
    xb = _spread(x.float(), st, used.numel())
    w = [t[used] for t in st["w"]]
    if kind == "grouped":
        y = _product(xb, *w, None if st["bias"] is None else st["bias"][used])
    elif st["act"] == "silu":
        g, u = _product(xb, w[0], w[1], None), _product(xb, w[4], w[5], None)
        y = _product(g * torch.sigmoid(g) * u, w[2], w[3], None)
    else:
        h1 = _product(xb, w[0], w[1], w[2])
        g, u = h1[..., 0::2].clamp(max=LIMIT), h1[..., 1::2].clamp(-LIMIT, LIMIT)
        y = _product(g * torch.sigmoid(ALPHA * g) * (u + 1), w[3], w[4], w[5])
    return _gather(y, st, x.shape[0]).to(x.dtype)


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(st: dict):
    if not own:
        return _plain(st)
    from torchtitan_amd import ops

    x, kind = st["x"], st["kind"]
    if kind == "quantize":
        q, s = ops.int8_quantize(x)
        return [ops.int8_dequantize(q, s, x.dtype), s]
    if kind == "linear":
        return ops.linear_int8(x, *st["w"], st["bias"])
    if kind == "grouped":
        return ops.grouped_linear_int8(x, *st["w"], st["counts"], st["bias"])
    if kind == "ffn":
        return ops.swiglu_ffn_int8(x, *st["w"])
    if st["act"] == "silu":
        return ops.grouped_swiglu_int8(x, *st["w"], st["counts"])
    return ops.grouped_swiglu_oss_int8(x, *st["w"], st["counts"], LIMIT)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case: dict) -> dict:
    el = 2.0 if case["dtype"] == "bf16" else 4.0
    if case["kind"] == "quantize":  # x in, its codes and scales out, and the values out again
        n = case["rows"] * case["cols"]
        return {"bytes": n * (2 * el + 1) + 4.0 * case["rows"], "flops": 0.0}
    d = case["dim"]
    if case["kind"] == "linear":
        m, n = case["rows"], case["out"]
        return {"bytes": el * m * (d + n) + n * (d + 4.0), "flops": 2.0 * m * n * d}
    if case["kind"] == "ffn":
        m, h = case["rows"], case["hidden"]
        return {"bytes": 2 * el * m * d + 3.0 * d * h, "flops": 6.0 * m * d * h}
    e, t = case["experts"], case["tokens"]
    rows = t * case["top_k"]
    used = e * (1.0 - (1.0 - case["top_k"] / e) ** t)  # experts that get a row
    if case["kind"] == "grouped":
        n = case["out"]
        return {"bytes": used * n * (d + 4.0) + el * rows * (d + n), "flops": 2.0 * rows * n * d}
    h = case["hidden"]
    return {"bytes": used * 3.0 * d * h + 2 * el * rows * d, "flops": 6.0 * rows * d * h}


# ---------------------------------------------------------------------------
# the same in 64 bits, an expert at a time
# ---------------------------------------------------------------------------
def _near(v: torch.Tensor) -> torch.Tensor:
    """The values that the 8-bit codes of v's rows stand for: multiplier and scale are 32-bit
    numbers by definition, the rest is exact."""
    top = v.abs().max(dim=1, keepdim=True).values.float().clamp(min=TINY).double()
    return torch.round(v * (127 / top).float().double()) * (top / 127).float().double()


def _values(q: torch.Tensor, s: torch.Tensor) -> torch.Tensor:
    return q.double() * s.double().unsqueeze(-1)


def _silu(g: torch.Tensor) -> torch.Tensor:
    return g / (1 + torch.exp(-g))


def exact(case: dict, seed: int):
    st = prepare(case, seed)
    kind, x, w = st["kind"], st["x"].double(), st.get("w")
    if kind == "quantize":
        return [_near(x), x.abs().amax(dim=1).clamp(min=TINY) / 127]
    if kind == "linear":
        y = _near(x) @ _values(*w).t()
        return y if st["bias"] is None else y + st["bias"].double()
    if kind == "ffn":
        xq = _near(x)
        return _near(_silu(xq @ _values(*w[0:2]).t()) * (xq @ _values(*w[4:6]).t())) @ _values(*w[2:4]).t()
    y = torch.zeros(x.shape[0], case["out"] if kind == "grouped" else case["dim"], dtype=torch.float64, device=DEV)
    r = 0
    for e, c in enumerate(st["counts"].tolist()):
        if c == 0:
            continue
        xe = _near(x[r:r + c])
        if kind == "grouped":
            ye = xe @ _values(w[0][e], w[1][e]).t()
            y[r:r + c] = ye if st["bias"] is None else ye + st["bias"][e].double()
        elif case["act"] == "silu":
            w1, w2, w3 = (_values(w[i][e], w[i + 1][e]) for i in (0, 2, 4))
            y[r:r + c] = _near(_silu(xe @ w1.t()) * (xe @ w3.t())) @ w2.t()
        else:
            h1 = xe @ _values(w[0][e], w[1][e]).t() + w[2][e].double()
            g, u = h1[:, 0::2].clamp(max=LIMIT), h1[:, 1::2].clamp(-LIMIT, LIMIT)
            h = _near(_silu(ALPHA * g) / ALPHA * (u + 1))
            y[r:r + c] = h @ _values(w[3][e], w[4][e]).t() + w[5][e].double()
        r += c
    return y
