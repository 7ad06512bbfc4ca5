"""MoE layers on the MXFP4 and 8-bit-activation experts: trained with 8-bit activations, packed to
4 bits, and asked for prompts and single tokens; gpt-oss layers from a packed checkpoint."""

from types import SimpleNamespace

import pytest
import torch

from tests import narrow_util as N
from tests.conftest import banner

pytestmark = pytest.mark.gpu

DIMS = SimpleNamespace(pp_enabled=False, cp_enabled=False, ep_enabled=False)


def _build(conv, model):
    return conv.build(parallel_dims=DIMS, model_compile_enabled=False).convert(model)


def _layer(dev, d=256, h=192, e=8, k=2, seed=0, before=True, oss=False):
    from torchtitan_amd import GroupedExperts, Linear, MoE, TokenChoiceTopKRouter
    from torchtitan_amd.gpt_oss import GptOssMoE

    cls = GptOssMoE if oss else MoE
    moe = cls.Config(
        num_experts=e, experts=GroupedExperts.Config(dim=d, hidden_dim=h, num_experts=e),
        router=TokenChoiceTopKRouter.Config(num_experts=e, gate=Linear.Config(in_features=d, out_features=e), top_k=k,
                                            score_func="sigmoid", route_norm=True),
        score_before_experts=before).build()
    gen = torch.Generator().manual_seed(seed)
    with torch.no_grad():
        for p in moe.parameters():
            p.copy_(torch.randn(p.shape, generator=gen) * 0.05)
    moe = moe.to(dev, torch.bfloat16)
    moe.expert_bias.data = moe.expert_bias.data.float()
    moe.tokens_per_expert.data = moe.tokens_per_expert.data.float()
    return moe


def _routed(moe, x):
    """The routed rows the experts see, and what the layer makes of rows y."""
    from torchtitan_amd import ops

    flat = x.reshape(-1, x.shape[-1])
    with torch.no_grad():
        scores, idx, _ = moe.router(flat, moe.expert_bias)
        layout = moe.reorderer(scores, idx)
        s = layout[0]
        rows = ops.permute(flat, layout.slot_pos, layout.tok_pos, s if moe.score_before_experts else None)
        join = lambda y: ops.combine(None, y, layout.slot_pos, layout.tok_pos,  # noqa: E731
                                     None if moe.score_before_experts else s).view_as(x)
    return rows, layout[2], join


def test_train_pack_and_serve(dev):
    """A step of optimization with 8-bit activations, whose gradients are near the bf16 layer's; then
    the weights packed, a prompt, and its last tokens one at a time: the same routing, the
    experts' rows as 64 bits give them."""
    banner("layer: train, pack, serve")
    from torchtitan_amd.quantization import MXFP4WeightConverter, MXFP8ActivationCheckpointConverter

    gen = torch.Generator().manual_seed(1)
    x = torch.randn(2, 200, 256, generator=gen).bfloat16().to(dev)
    dy = torch.randn(2, 200, 256, generator=gen).bfloat16().to(dev)
    plain, kept = _layer(dev), _layer(dev)
    model = torch.nn.ModuleDict({"moe": kept})
    assert _build(MXFP8ActivationCheckpointConverter.Config(fqns=["experts"]), model) == ["moe.experts"]
    grads = []
    for moe in (plain, kept):
        xx = x.clone().requires_grad_(True)
        moe(xx).backward(dy)
        grads.append([xx.grad, *(p.grad for p in moe.parameters())])
    for a, b in zip(*grads):
        # e4m3 is off by 2^-4 of a value at most, and a product of three such factors by three
        # times that; the mean square over many terms is a third of the worst
        assert (a.float() - b.float()).norm() <= 3 * 2.0 ** -4 / 3 * a.float().norm()
    torch.optim.SGD(kept.parameters(), lr=0.1).step()
    weights = {n: p.detach().clone() for n, p in kept.experts.named_parameters()}
    assert _build(MXFP4WeightConverter.Config(fqns=["moe"]), model) == ["moe.experts"]
    assert not list(kept.experts.parameters())
    vals = [N.q4(weights[n].cpu()) for n in ("w1", "w2", "w3")]

    def check(x):
        with torch.no_grad():
            y = kept(x)
        rows, counts, join = _routed(kept, x)
        got = kept.experts(rows, counts)
        assert torch.equal(join(got), y)
        want, tol = N.experts4(N.q4(rows.cpu()), *vals, counts.cpu())
        N.within(got, want, tol, f"{x.shape[1]} tokens", 2.0 ** -8)

    check(x)
    for t in range(3):
        check(x[:1, 197 + t:198 + t])


def test_mxfp4_training_layer(dev):
    """The MXFP4 recipe through a layer: gradients of every parameter, near the bf16 layer's."""
    banner("layer: mxfp4 training")
    from torchtitan_amd.quantization import MXFP4Converter

    gen = torch.Generator().manual_seed(2)
    x = torch.randn(1, 333, 256, generator=gen).bfloat16().to(dev)
    dy = torch.randn(1, 333, 256, generator=gen).bfloat16().to(dev)
    for before in (True, False):
        plain, four = _layer(dev, before=before), _layer(dev, before=before)
        model = torch.nn.ModuleDict({"moe": four})
        assert _build(MXFP4Converter.Config(fqns=["experts"]), model) == ["moe.experts"]
        res = []
        for moe in (plain, four):
            xx = x.clone().requires_grad_(True)
            y = moe(xx)
            y.backward(dy)
            res.append([y.detach(), xx.grad, *(p.grad for p in moe.parameters())])
        for a, b in zip(*res):
            # e2m1 is off by a third of a value at most (1 between 0.5 and 1.5 steps apart), in the
            # mean square about an eighth; three such factors
            assert torch.isfinite(b.float()).all()
            assert (a.float() - b.float()).norm() <= 3 ** 0.5 / 3 * a.float().norm()
        with torch.no_grad():
            y = four(x)
        assert (y.float() - res[1][0].float()).norm() <= 2.0 ** -8 * y.float().norm()


def test_gpt_oss_layer(dev):
    """gpt-oss experts packed from a bf16 layer, and the same from a checkpoint's blocks."""
    banner("layer: gpt-oss packed")
    from torchtitan_amd.mxfp4 import MXFP4GptOssGroupedExperts
    from torchtitan_amd.quantization import MXFP4WeightConverter

    moe = _layer(dev, d=320, h=160, e=4, oss=True, before=False)
    with torch.no_grad():
        moe.experts.mlp1_weight.mul_(4)
    old = {n: p.detach().clone() for n, p in moe.experts.named_parameters()}
    model = torch.nn.ModuleDict({"moe": moe})
    assert _build(MXFP4WeightConverter.Config(fqns=["moe"]), model) == ["moe.experts"]
    v = N.q4(old["mlp1_weight"].cpu())
    loaded = MXFP4GptOssGroupedExperts.Config(dim=320, hidden_dim=160, num_experts=4).build().to(dev)
    at = "model.layers.0.mlp.experts."
    hf = {}
    for key, name in (("gate_up_proj", "mlp1"), ("down_proj", "mlp2")):
        q, s = N.pack4(old[name + "_weight"].cpu())
        hf |= {f"{at}{key}_blocks": q.unflatten(-1, (-1, 16)), f"{at}{key}_scales": s, f"{at}{key}_bias": old[name + "_bias"].cpu()}
    loaded.load_hf(hf, 0)
    for n in (1, 5, 300):
        x = torch.randn(1, n, 320, generator=torch.Generator().manual_seed(n)).bfloat16().to(dev)
        with torch.no_grad():
            y = moe(x)
        rows, counts, join = _routed(moe, x)
        got = moe.experts(rows, counts)
        assert torch.equal(join(got), y) and torch.equal(loaded(rows, counts), got)
        want, tol = N.experts4(N.q4(rows.cpu()), v[:, 0::2], N.q4(old["mlp2_weight"].cpu()), v[:, 1::2], counts.cpu(), "oss", 7.0,
                               old["mlp1_bias"].cpu().double(), old["mlp2_bias"].cpu().double())
        N.within(got, want, tol, f"{n} tokens", 2.0 ** -8)


def test_kept_bytes(dev):
    """What a training step holds between forward and backward: (D + 2H) 33/32 bytes a routed row
    (besides the weights, which the model holds)."""
    banner("layer: kept bytes")
    from torchtitan_amd import ops

    r, e, d, h = 4096, 4, 256, 192
    gen = torch.Generator().manual_seed(3)
    mk = lambda *s: (torch.randn(*s, generator=gen) * 0.1).bfloat16().to(dev).requires_grad_(True)  # noqa: E731
    x, w1, w2, w3 = mk(r, d), mk(e, h, d), mk(e, d, h), mk(e, h, d)
    counts = torch.tensor([1024] * 4, device=dev)
    held = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: held.append(t) or t, lambda t: t):
        ops.grouped_swiglu_ckpt8(x, w1, w2, w3, counts)
    own = {t.data_ptr() for t in (w1, w2, w3, counts)}
    assert sum(t.numel() * t.element_size() for t in held if t.data_ptr() not in own) == r * (d + 2 * h) * 33 // 32


def test_fake_tensors(dev):
    """The ops inside a compiled graph's tracing (fake tensors) give the eager shapes and types."""
    banner("layer: fake tensors")
    from torch._subclasses.fake_tensor import FakeTensorMode

    from torchtitan_amd import ops

    gen = torch.Generator().manual_seed(4)
    mk = lambda *s: torch.randn(*s, generator=gen).bfloat16().to(dev)  # noqa: E731
    x, w1, w2, w3, c = mk(40, 320), mk(2, 192, 320), mk(2, 320, 192), mk(2, 192, 320), torch.tensor([30, 8], device=dev)
    packed = [t for w in (w1, w2, w3) for t in ops.mxfp4_quantize(w)]
    dy = mk(40, 320)

    def calls(x, w1, w2, w3, c, dy, packed):
        out = [ops.mxfp4_quantize(x), ops.mxfp4_dequantize(packed[0], packed[1], torch.float32),
               ops.grouped_swiglu_mxfp4(x, *packed, c), ops.grouped_swiglu_ckpt8(x, w1, w2, w3, c, False)]
        kept = ops.grouped_swiglu_ckpt8(x, w1, w2, w3, c)
        four = ops.grouped_swiglu_mxfp4_train(x, w1, w2, w3, c)
        out += [kept, four, ops.grouped_swiglu_ckpt8_backward(dy, w1, w2, w3, c, kept[1], True, False, True),
                ops.grouped_swiglu_mxfp4_train_backward(dy, c, four[1], 192, False, True, False)]
        return [t for o in out for t in (o if isinstance(o, (tuple, list)) else (o,))]

    eager = calls(x, w1, w2, w3, c, dy, packed)
    with FakeTensorMode() as mode:
        fake = calls(*(mode.from_tensor(t) for t in (x, w1, w2, w3, c, dy)), [mode.from_tensor(t) for t in packed])
    for a, b in zip(eager, fake):
        assert a.shape == b.shape and a.dtype == b.dtype and a.device == b.device and a.stride() == b.stride()


def test_steps_on_two_streams(dev):
    """Two layers' steps on two streams at once give the bits of each alone."""
    banner("layer: two streams")
    from torchtitan_amd import ops

    def inputs(seed):
        gen = torch.Generator().manual_seed(seed)
        mk = lambda *s: (torch.randn(*s, generator=gen) * 0.1).bfloat16().to(dev)  # noqa: E731
        return mk(3000, 320), mk(4, 192, 320), mk(4, 320, 192), mk(4, 192, 320), torch.tensor([900, 0, 1500, 600], device=dev), mk(3000, 320)

    def step(op, x, w1, w2, w3, c, dy):
        leaves = [t.detach().requires_grad_(True) for t in (x, w1, w2, w3)]
        y = op(*leaves, c)[0]
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    jobs = [(ops.grouped_swiglu_ckpt8, inputs(1)), (ops.grouped_swiglu_mxfp4_train, inputs(2))]
    want = [step(op, *args) for op, args in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    for _ in range(4):
        got = []
        for s, (op, args) in zip(streams, jobs):
            with torch.cuda.stream(s):
                got.append(step(op, *args))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(p, q) for p, q in zip(a, b))


# ---------------------------------------------------------------------------
# opcheck: schema, fake kernel, autograd registration, AOT dispatch with dynamic shapes
# ---------------------------------------------------------------------------
def _op_cases(dev):
    from torchtitan_amd import ops

    gen = torch.Generator().manual_seed(5)
    r, e, d, h = 128, 4, 128, 192  # what is kept of these has no padding, whose bytes are not defined

    def bf(*shape, grad=False, scale=1.0):
        return (torch.randn(*shape, generator=gen) * scale).bfloat16().to(dev).requires_grad_(grad)

    mx = torch.ops.moe_mi355x_mx
    counts = torch.tensor([60, 0, 40, 28], device=dev)  # every row has an expert: what is kept of others is not defined
    x, w1, w2, w3 = bf(r, d), bf(e, h, d, scale=0.05), bf(e, d, h, scale=0.05), bf(e, h, d, scale=0.05)
    leaves = [t.clone().requires_grad_(True) for t in (x, w1, w2, w3)]
    packed = [t for w in (w1, w2, w3) for t in ops.mxfp4_quantize(w)]
    m1 = ops.mxfp4_quantize(bf(e, 2 * h, d, scale=0.05))
    kept = ops.grouped_swiglu_ckpt8(x, w1, w2, w3, counts)[1]
    four = ops.grouped_swiglu_mxfp4_train(x, w1, w2, w3, counts)[1]
    return {
        "mxfp4_quantize": (mx.mxfp4_quantize, (x,)),
        "mxfp4_dequantize": (mx.mxfp4_dequantize, (*packed[:2], torch.float32)),
        "grouped_swiglu_mxfp4": (mx.grouped_swiglu_mxfp4, (x, *packed, counts)),
        "grouped_swiglu_oss_mxfp4": (mx.grouped_swiglu_oss_mxfp4, (x, *m1, bf(e, 2 * h), *packed[2:4], bf(e, d), counts, 7.0)),
        "grouped_swiglu_ckpt8": (ops.grouped_swiglu_ckpt8, (*leaves, counts)),
        "grouped_swiglu_ckpt8_backward": (ops.grouped_swiglu_ckpt8_backward, (bf(r, d), w1, w2, w3, counts, kept)),
        "grouped_swiglu_mxfp4_train": (ops.grouped_swiglu_mxfp4_train, (*leaves, counts)),
        "grouped_swiglu_mxfp4_train_backward": (ops.grouped_swiglu_mxfp4_train_backward, (bf(r, d), counts, four, h)),
    }


OP_NAMES = ["mxfp4_quantize", "mxfp4_dequantize", "grouped_swiglu_mxfp4", "grouped_swiglu_oss_mxfp4",
            "grouped_swiglu_ckpt8", "grouped_swiglu_ckpt8_backward", "grouped_swiglu_mxfp4_train",
            "grouped_swiglu_mxfp4_train_backward"]


def test_opcheck_covers_every_op():
    import torchtitan_amd  # noqa: F401

    ns = torch.ops.moe_mi355x_mx
    registered = {n for n in dir(ns) if isinstance(getattr(ns, n, None), torch._ops.OpOverloadPacket)}
    assert registered <= set(OP_NAMES), registered - set(OP_NAMES)


@pytest.mark.parametrize("name", OP_NAMES)
def test_opcheck(dev, name):
    banner(f"opcheck {name}")
    op, args = _op_cases(dev)[name]
    torch.library.opcheck(op, args)
