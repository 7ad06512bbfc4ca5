"""8-bit integers as they are used: layers converted and asked for prompts and tokens, every kernel and
tile against each other, streams, graphs, views, rows that are not finite."""

from types import SimpleNamespace

import pytest
import torch

from tests import int8_util as I
from tests.conftest import banner

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
DIMS = SimpleNamespace(pp_enabled=False, cp_enabled=False, ep_enabled=False)


def _moe(dev, oss=False, d=256, h=192, hs=320, e=8, k=2, seed=0):
    from torchtitan_amd import FeedForward, GroupedExperts, Linear, MoE, TokenChoiceTopKRouter
    from torchtitan_amd.gpt_oss import GptOssMoE

    lin = lambda i, o: Linear.Config(in_features=i, out_features=o)  # noqa: E731
    moe = (GptOssMoE if oss else MoE).Config(
        num_experts=e, experts=GroupedExperts.Config(dim=d, hidden_dim=h, num_experts=e), score_before_experts=False,
        shared_experts=FeedForward.Config(w1=lin(d, hs), w2=lin(hs, d), w3=lin(d, hs)),
        router=TokenChoiceTopKRouter.Config(num_experts=e, gate=lin(d, e), top_k=k, score_func="sigmoid", route_norm=True)).build()
    gen = torch.Generator().manual_seed(seed)
    with torch.no_grad():
        for p in moe.parameters():
            p.copy_(torch.randn(p.shape, generator=gen) * 0.05)
    moe = moe.to(dev, BF)
    moe.expert_bias.data = moe.expert_bias.data.float()
    moe.tokens_per_expert.data = moe.tokens_per_expert.data.float()
    return moe


def _convert(moe):
    from torchtitan_amd.quantization import Int8WeightConverter

    model = torch.nn.ModuleDict({"moe": moe})
    return Int8WeightConverter.Config(fqns=["moe."]).build(parallel_dims=DIMS, model_compile_enabled=False).convert(model)


@pytest.mark.parametrize("oss", [False, True])
def test_a_layer_serves(dev, oss):
    """A MoE layer on 8-bit integers: the same routing as in bf16, the experts' rows and the shared
    expert's as 64 bits give them; its tokens one at a time are its prompt's bits."""
    banner(f"int8 layer oss={oss}")
    from torchtitan_amd import ops

    moe = _moe(dev, oss)
    x = torch.randn(3, 70, 256, generator=torch.Generator().manual_seed(1)).to(dev, BF)
    with torch.no_grad():
        plain = moe(x)
        assert _convert(moe) == ["moe.experts", "moe.shared_experts"]
        moe.eval()
        got = moe(x)
        # the layer against the one in bf16: the error of 8-bit operands, 2^-8 of a row's largest each
        assert (got - plain).float().norm() < 0.05 * plain.float().norm()
        flat = x.view(-1, 256)
        scores, idx, _ = moe.router(flat, moe.expert_bias)
        layout = moe.reorderer(scores, idx)
        rows = ops.permute(flat, layout.slot_pos, layout.tok_pos, None)
        counts, ex, ff = layout[2], moe.experts, moe.shared_experts
        y, shared = ex(rows, counts), ff(x)
        cpu = lambda mod, name: tuple(t.cpu() for t in mod.packed(name))  # noqa: E731
        if oss:
            want = I.oss(rows.cpu(), cpu(ex, "mlp1_weight"), ex.mlp1_bias.cpu(), cpu(ex, "mlp2_weight"), ex.mlp2_bias.cpu(),
                         counts.cpu(), ex.swiglu_limit)
        else:
            want = I.experts(rows.cpu(), cpu(ex, "w1"), cpu(ex, "w2"), cpu(ex, "w3"), counts.cpu())
        I.within(y, *want, "experts")
        hid = I.hidden(flat.cpu(), cpu(ff, "w1"), cpu(ff, "w3"), None, 0.0)
        I.within(shared.view(-1, 256), *I.second(*hid, *cpu(ff, "w2"), None, BF), "shared expert")
        for at in (0, 33, 69):
            one = moe(x[1:2, at:at + 1])
            assert torch.equal(one, got[1:2, at:at + 1]), f"token {at}"
    with pytest.raises(RuntimeError, match="no gradients"):
        moe(x.clone().requires_grad_(True))


def test_a_linear_serves(dev):
    banner("int8 linear module")
    from torchtitan_amd import Linear
    from torchtitan_amd.int8 import Int8Linear

    gen = torch.Generator().manual_seed(2)
    lin = Linear.Config(in_features=272, out_features=101, bias=True).build().to(dev)
    q = Int8Linear.from_linear(lin)
    for dt in (BF, F32):
        x = I.rows(gen, 30, 272, dt).view(2, 15, 272)
        got = q(x.to(dev))
        want = I.linear(x.view(30, 272), *(t.cpu() for t in q.packed("weight")), q.bias.cpu(), dt)
        I.within(got.view(30, 101), *want, str(dt))
    w = q.dequantize("weight", F32).cpu()
    assert torch.equal(w, q.weight_codes.cpu().float() * q.weight_scales.cpu().unsqueeze(-1))


# (rows, experts, contraction, columns): one for each kernel
TILES = [(4096, 1, 2304, 2304), (2048, 1, 2304, 2304), (1024, 1, 2304, 2304), (300, 1, 2304, 2304), (16, 1, 2304, 2304),
         (8200, 32, 1536, 2048), (5000, 32, 1536, 2048), (3000, 3, 272, 1001), (200, 32, 1536, 264)]


def test_tiles_are_all_taken():
    from torchtitan_amd import _lib

    got = {_lib.lib().moe_int8_tile(r, e, k, n, 256) for r, e, k, n in TILES}
    assert got == {0, 1, 2, 3, 4}


@pytest.mark.parametrize("r,e,k,n", TILES)
def test_every_tile(dev, r, e, k, n):
    """Each kernel and tile against 64 bits (on the GPU, whose exact sums of codes these sizes need), and a
    row's bits are the same whichever of them computes it."""
    banner(f"int8 tiles {r} rows, {e} of {n} x {k}")
    from torchtitan_amd import ops

    gen = torch.Generator().manual_seed(3)
    qw = torch.randint(-127, 128, (e, n, k), generator=gen, dtype=torch.int8).to(dev)
    sw = (torch.rand(e, n, generator=gen) * 0.01).to(dev)
    pick = torch.randint(0, e, (r,), generator=gen)
    counts = torch.bincount(pick, minlength=e)
    x = I.rows(gen, r, k).to(dev)
    if e == 1:
        got = ops.linear_int8(x, qw[0], sw[0])
    else:
        got = ops.grouped_linear_int8(x, qw, sw, counts.to(dev))
    xq, xs = ops.int8_quantize(x)
    at = 0
    for i, c in enumerate(counts.tolist()):
        p = (xq[at:at + c].double() @ qw[i].double().T) * xs[at:at + c].double().unsqueeze(-1) * sw[i].double()
        tol = 3.01 * I.U * p.abs()
        assert bool(((got[at:at + c].double() - p).abs() <= tol + I.HALF[BF] * (p.abs() + tol)).all()), f"expert {i}"
        if c:
            some = ops.linear_int8(x[at:at + min(c, 9)], qw[i], sw[i])
            assert torch.equal(some, got[at:at + min(c, 9)])
        at += c


@pytest.mark.parametrize("r,tile", [(6000, 0), (3000, 1), (1500, 2), (300, 3)])
def test_layers_on_every_tile(dev, r, tile):
    """The layers' products on each tile: an expert's first and last rows as they come out alone, the first
    ones as 64 bits give them. Biases in both types, linear's too."""
    banner(f"int8 layers on tile {tile}")
    from torchtitan_amd import _lib, ops

    gen = torch.Generator().manual_seed(11)
    e, d, h = 4, 1536, 720
    assert _lib.lib().moe_int8_tile(r, e, d, 2 * h, 256) == tile
    counts = torch.tensor([r // 4 + 5, 0, r // 2 - 20, r // 4 + 9])
    x = I.rows(gen, r, d)
    w1, w2, w3, m1 = (I.weight(gen, e, *s) for s in ((h, d), (d, h), (h, d), (2 * h, d)))
    b1, b2 = torch.randn(e, 2 * h, generator=gen), torch.randn(e, d, generator=gen)
    on = lambda *ts: [t.to(dev) for t in ts]  # noqa: E731
    xd, cd = x.to(dev), counts.to(dev)
    forms = [(ops.grouped_swiglu_int8, on(*w1, *w2, *w3), (), lambda i, t: I.experts(t, *([q[i:i + 1] for q in w] for w in (w1, w2, w3)),
                                                                                     torch.tensor([len(t)])))]
    for dt in (BF, F32):
        a1, a2 = b1.to(dt), b2.to(dt)
        forms += [(ops.grouped_swiglu_oss_int8, on(*m1, a1, *w2, a2), (7.0,),
                   lambda i, t, a1=a1, a2=a2: I.oss(t, [q[i:i + 1] for q in m1], a1[i:i + 1], [q[i:i + 1] for q in w2], a2[i:i + 1],
                                                    torch.tensor([len(t)]), 7.0)),
                  (lambda x, qw, sw, b, c: ops.grouped_linear_int8(x, qw, sw, c, b), on(*m1, a1), (),
                   lambda i, t, a1=a1: I.linear(t, m1[0][i], m1[1][i], a1[i], BF))]
    for f, weights, rest, want in forms:
        got = f(xd, *weights, cd, *rest)
        for i, a, b in I.segments(counts, r):
            part = [t[i:i + 1] for t in weights]
            n = min(7, b - a)
            for at in (a, b - n):
                alone = f(xd[at:at + n], *part, torch.tensor([n], device=dev), *rest)
                assert torch.equal(alone, got[at:at + n]), f"expert {i}, rows from {at}"
            I.within(got[a:a + n], *want(i, x[a:a + n]), f"expert {i}")
        assert not got[int(counts.sum()):].any()


def test_two_threads(dev):
    """Calls from two threads at once, each on a stream of its own."""
    banner("int8 threads")
    from concurrent.futures import ThreadPoolExecutor

    from torchtitan_amd import ops

    gen = torch.Generator().manual_seed(12)
    w = [t.to(dev) for s in ((8, 256, 512), (8, 512, 256), (8, 256, 512)) for t in I.weight(gen, *s)]
    xs = [I.rows(gen, n, 512).to(dev) for n in (16, 1600)]
    cs = [torch.full((8,), len(x) // 8, device=dev) for x in xs]
    want = [ops.grouped_swiglu_int8(x, *w, c) for x, c in zip(xs, cs)]
    torch.cuda.synchronize()

    def work(i):
        s = torch.cuda.Stream()
        with torch.no_grad(), torch.cuda.stream(s):
            got = [ops.grouped_swiglu_int8(xs[(i + k) % 2], *w, cs[(i + k) % 2]) for k in range(8)]
        s.synchronize()
        return all(torch.equal(g, want[(i + k) % 2]) for k, g in enumerate(got))

    with ThreadPoolExecutor(2) as pool:
        assert all(pool.map(work, range(4)))


def test_operands_on_other_devices_are_refused(dev):
    from torchtitan_amd import ops

    gen = torch.Generator().manual_seed(13)
    w = [t.to(dev) for s in ((2, 64, 96), (2, 96, 64), (2, 64, 96)) for t in I.weight(gen, *s)]
    x, c = I.rows(gen, 8, 96), torch.tensor([4, 4])
    for call in (lambda: ops.grouped_swiglu_int8(x.to(dev), *w, c), lambda: ops.grouped_swiglu_int8(x, *w, c.to(dev)),
                 lambda: ops.grouped_linear_int8(x.to(dev), w[0].cpu(), w[1], c.to(dev)), lambda: ops.linear_int8(x.to(dev), w[0][0], w[1][0].cpu()),
                 lambda: ops.linear_int8(x.to(dev), w[0][0], w[1][0], torch.zeros(64)), lambda: ops.int8_quantize(x)):
        with pytest.raises((RuntimeError, ValueError, NotImplementedError)):
            call()


def test_many_units_a_workgroup(dev):
    """Few rows on so many wide experts that a workgroup goes through several units and experts."""
    banner("int8 many units")
    from torchtitan_amd import _lib, ops

    gen = torch.Generator().manual_seed(4)
    e, k, n = 96, 512, 2064
    assert _lib.lib().moe_int8_tile(400, e, k, n, 256) == 4
    qw = torch.randint(-127, 128, (e, n, k), generator=gen, dtype=torch.int8)
    sw = torch.rand(e, n, generator=gen) * 0.01
    counts = torch.randint(0, 5, (e,), generator=gen)
    counts[7], counts[50] = 40, 17
    x = I.rows(gen, int(counts.sum()) + 1, k)
    got = ops.grouped_linear_int8(*(t.to(dev) for t in (x, qw, sw, counts)))
    f = lambda i, xe: I.linear(xe, qw[i], sw[i], None, BF)  # noqa: E731
    I.within(got, *I.grouped(x, n, counts, f, BF), "many units")


@pytest.mark.parametrize("r", [12, 900])
def test_not_finite(dev, r):
    """A row with an infinity or NaN spoils itself, a weight row with a NaN scale its column; all else
    keeps its bits."""
    banner(f"int8 not finite {r}")
    from torchtitan_amd import ops

    gen = torch.Generator().manual_seed(5)
    w1, w2, w3 = (I.weight(gen, 3, *s) for s in ((144, 272), (272, 144), (144, 272)))
    w = [t.to(dev) for t in (*w1, *w2, *w3)]
    counts = torch.tensor([r // 3] * 3, device=dev)
    x = I.rows(gen, r, 272).to(dev)
    want, y = ops.grouped_swiglu_int8(x, *w, counts), ops.grouped_linear_int8(x, w[0], w[1], counts)
    bad = x.clone()
    bad[1, 3], bad[r - 1, 271] = float("inf"), float("nan")
    keep = torch.ones(r, dtype=torch.bool)
    keep[1] = keep[r - 1] = False
    for f, ref in ((lambda t: ops.grouped_swiglu_int8(t, *w, counts), want), (lambda t: ops.grouped_linear_int8(t, w[0], w[1], counts), y)):
        got = f(bad)
        assert got[1].isnan().all() and got[r - 1].isnan().all() and torch.equal(got[keep], ref[keep])
    s1 = w[1].clone()
    s1[1, 5] = float("nan")
    got = ops.grouped_linear_int8(x, w[0], s1, counts)
    a, b = r // 3, 2 * (r // 3)
    assert got[a:b, 5].isnan().all()
    got[a:b, 5] = y[a:b, 5]
    assert torch.equal(got, y)
    zeros = ops.linear_int8(torch.zeros(r, 272, device=dev, dtype=BF), w[0][0], w[1][0], torch.ones(144, device=dev))
    assert torch.equal(zeros, torch.ones_like(zeros))  # rows of zeros have a scale


@pytest.mark.parametrize("times", [1, 60])
def test_views_and_alignment(dev, times):
    banner("int8 views")
    from torchtitan_amd import ops

    gen = torch.Generator().manual_seed(6)
    counts = torch.tensor([8, 2, 0, 20]).to(dev) * times
    x = I.rows(gen, 30 * times, 96).to(dev)
    w = [t.to(dev) for s in ((4, 64, 96), (4, 96, 64), (4, 64, 96)) for t in I.weight(gen, *s)]
    bias = torch.randn(4, 64, generator=gen).to(dev)

    def shifted(t):  # the same values one element off an aligned address
        flat = torch.zeros(t.numel() + 1, dtype=t.dtype, device=dev)
        flat[1:] = t.flatten()
        return flat[1:].view(t.shape)

    def strided(t):
        wide = torch.zeros(*t.shape[:-1], 2 * t.shape[-1], dtype=t.dtype, device=dev)
        wide[..., 1::2] = t
        return wide[..., 1::2]

    calls = [(ops.grouped_swiglu_int8, (x, *w, counts)), (ops.grouped_linear_int8, (x, w[0], w[1], counts, bias)),
             (ops.linear_int8, (x.view(3, -1, 96), w[0][0], w[1][0], bias[0])), (ops.linear_int8, (x.float(), w[0][1], w[1][1])),
             (ops.swiglu_ffn_int8, (x.view(5, -1, 96), *(t[2] for t in w)))]
    for op, args in calls:
        want = op(*args)
        for f in (shifted, strided):
            assert torch.equal(op(*(f(t) for t in args)), want), op
        assert torch.equal(op(args[0].transpose(0, 1).contiguous().transpose(0, 1), *args[1:]), want)


def test_empty(dev):
    banner("int8 no rows")
    from torchtitan_amd import ops

    gen = torch.Generator().manual_seed(7)
    w = [t.to(dev) for s in ((2, 64, 96), (2, 96, 64), (2, 64, 96)) for t in I.weight(gen, *s)]
    none, c = torch.zeros(0, 96, dtype=BF, device=dev), torch.zeros(2, dtype=torch.int64, device=dev)
    assert ops.linear_int8(none, w[0][0], w[1][0]).shape == (0, 64) and ops.linear_int8(none.view(3, 0, 96), w[0][0], w[1][0]).shape == (3, 0, 64)
    assert ops.grouped_linear_int8(none, w[0], w[1], c).shape == (0, 64)
    assert ops.swiglu_ffn_int8(none, *(t[0] for t in w)).shape == (0, 96) and ops.grouped_swiglu_int8(none, *w, c).shape == (0, 96)
    some = ops.grouped_swiglu_int8(torch.ones(7, 96, dtype=BF, device=dev), *w, c)  # rows, but no expert's
    assert some.shape == (7, 96) and not some.any()


def test_streams_and_graphs(dev):
    """Calls on two streams at once, and captured graphs replayed in turn with eager calls between, each
    against the eager result."""
    banner("int8 streams and graphs")
    from torchtitan_amd import ops

    gen = torch.Generator().manual_seed(8)
    e, d, h = 8, 512, 256
    w = [t.to(dev) for s in ((e, h, d), (e, d, h), (e, h, d)) for t in I.weight(gen, *s)]
    one = [t[0].contiguous() for t in w]
    jobs = []  # (a call of its rows, three inputs)
    for n in (24, 1200):
        c = torch.bincount(torch.randint(0, e, (n,), generator=gen), minlength=e).to(dev)
        xs = [I.rows(gen, n, d).to(dev) for _ in range(3)]
        jobs += [(lambda x, c=c: ops.grouped_swiglu_int8(x, *w, c), xs), (lambda x: ops.swiglu_ffn_int8(x, *one), xs),
                 (lambda x, c=c: ops.grouped_linear_int8(x, w[0], w[1], c), xs), (lambda x: torch.stack([t.float().sum() for t in ops.int8_quantize(x)]), xs)]
    want = [[f(x) for x in xs] for f, xs in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    for _ in range(4):
        got = []
        for s, (f, xs) in zip(streams, jobs):
            with torch.cuda.stream(s):
                got.append(f(xs[0]))
        torch.cuda.synchronize()
        assert all(torch.equal(g, ref[0]) for g, ref in zip(got, want))
    graphs = []
    for f, xs in jobs[:3] + jobs[4:7]:  # (without the sum of the test's own)
        fixed, g = xs[0].clone(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = f(fixed)
        graphs.append((g, fixed, out))
    refs, eager = want[:3] + want[4:7], jobs[:3] + jobs[4:7]
    for turn in range(18):
        k = turn % 6
        g, fixed, out = graphs[k]
        fixed.copy_(eager[k][1][turn % 3])
        g.replay()
        other = eager[5 - k][0](eager[5 - k][1][turn % 3])
        torch.cuda.synchronize()
        assert torch.equal(out, refs[k][turn % 3]) and torch.equal(other, refs[5 - k][turn % 3]), turn


def _op_cases(dev):
    from torchtitan_amd import ops

    gen = torch.Generator().manual_seed(9)
    ns = torch.ops.moe_mi355x_int8
    x, c = I.rows(gen, 40, 96).to(dev), torch.tensor([20, 0, 18], device=dev)
    w = [t.to(dev) for s in ((3, 64, 96), (3, 96, 64), (3, 64, 96), (3, 128, 96)) for t in I.weight(gen, *s)]
    b1, b2 = torch.randn(3, 128, generator=gen).to(dev), torch.randn(3, 96, generator=gen).to(dev)
    one = [t[0].contiguous() for t in w]
    return {"int8_quantize": (ns.int8_quantize, (x,)), "int8_dequantize": (ns.int8_dequantize, (*one[:2], F32)),
            "linear_int8": (ns.linear_int8, (x, *one[:2], b1[0, :64].contiguous())),
            "grouped_linear_int8": (ns.grouped_linear_int8, (x, *w[:2], c)),
            "swiglu_ffn_int8": (ns.swiglu_ffn_int8, (x, *one[:6])),
            "grouped_swiglu_int8": (ns.grouped_swiglu_int8, (x, *w[:6], c)),
            "grouped_swiglu_oss_int8": (ns.grouped_swiglu_oss_int8, (x, *w[6:8], b1, *w[2:4], b2, c, 7.0))}


OP_NAMES = ["int8_quantize", "int8_dequantize", "linear_int8", "grouped_linear_int8", "swiglu_ffn_int8", "grouped_swiglu_int8",
            "grouped_swiglu_oss_int8"]


def test_opcheck_covers_every_op():
    import torchtitan_amd.ops  # noqa: F401

    ns = torch.ops.moe_mi355x_int8
    registered = {n for n in dir(ns) if isinstance(getattr(ns, n, None), torch._ops.OpOverloadPacket)}
    assert registered <= set(OP_NAMES), registered - set(OP_NAMES)


@pytest.mark.parametrize("name", OP_NAMES)
def test_opcheck(dev, name):
    banner(f"opcheck {name}")
    op, args = _op_cases(dev)[name]
    torch.library.opcheck(op, args)


def test_compiled(dev):
    """A compiled function calls the operators whole."""
    banner("int8 compiled")
    from torchtitan_amd import ops

    gen = torch.Generator().manual_seed(10)
    w = [t.to(dev) for s in ((64, 96), (96, 64), (64, 96)) for t in I.weight(gen, *s)]
    x = I.rows(gen, 33, 96).to(dev)
    f = lambda t: ops.linear_int8(ops.swiglu_ffn_int8(t, *w) + t, *w[:2])  # noqa: E731
    with torch.no_grad():
        assert torch.equal(torch.compile(f, fullgraph=True, backend="aot_eager")(x), f(x))
