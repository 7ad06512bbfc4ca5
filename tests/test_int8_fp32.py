"""Modules on 8-bit integers in place of ones that computed in fp32: rows in fp32 keep it. On the CPU the
products are the 64-bit oracle's, rounded once."""

import pytest
import torch

from tests import int8_util as I
from tests.conftest import banner

BF, F32 = torch.bfloat16, torch.float32


def _ffn(d, h):
    from torchtitan_amd import FeedForward, Linear

    lin = lambda i, o: Linear.Config(in_features=i, out_features=o)  # noqa: E731
    return _filled(FeedForward.Config(w1=lin(d, h), w2=lin(h, d), w3=lin(d, h)).build())


def _experts(e, d, h, grouped):
    from torchtitan_amd import GroupedExperts

    return _filled(GroupedExperts.Config(dim=d, hidden_dim=h, num_experts=e, use_grouped_mm=grouped).build())


def _filled(mod):
    gen = torch.Generator().manual_seed(21)
    with torch.no_grad():
        for p in mod.parameters():
            p.copy_(torch.randn(p.shape, generator=gen) * 0.1)
    return mod


def _packed(mod, *names):
    return [tuple(t.cpu() for t in mod.packed(n)) for n in names]


def _check_feed_forward(mod, x):
    w1, w2, w3 = _packed(mod, "w1", "w2", "w3")
    got = mod(x)
    rows = x.cpu().view(-1, x.shape[-1])
    assert got.dtype == F32 and got.shape == x.shape
    I.within(got.view(rows.shape), *I.second(*I.hidden(rows, w1, w3, None, 0.0), *w2, None, F32), "feed-forward")


def _check_experts(mod, x, counts):
    got = mod(x, counts)
    assert got.dtype == F32
    I.within(got, *I.experts(x.cpu(), *_packed(mod, "w1", "w2", "w3"), counts.cpu()), "experts")
    assert not got[int(counts.sum()):].any()


@pytest.fixture
def products(monkeypatch):
    from torchtitan_amd import ops

    def linear(x, qw, sw, bias=None):
        return I.linear(x.view(-1, x.shape[-1]), qw, sw, bias, x.dtype)[0].to(x.dtype).view(*x.shape[:-1], -1)

    def grouped(x, qw, sw, counts, bias=None):
        f = lambda e, t: I.linear(t, qw[e], sw[e], None, t.dtype)  # noqa: E731
        return I.grouped(x, qw.shape[1], counts, f, x.dtype)[0].to(x.dtype)

    monkeypatch.setattr(ops, "int8_quantize", I.pack)
    monkeypatch.setattr(ops, "linear_int8", linear)
    monkeypatch.setattr(ops, "grouped_linear_int8", grouped)
    # the layers' operators, which take bf16
    monkeypatch.setattr(ops, "swiglu_ffn_int8", lambda x, *w: x * 2)
    monkeypatch.setattr(ops, "grouped_swiglu_int8", lambda x, *w: x * 2)
    return ops


def test_feed_forward(products):
    from torchtitan_amd.int8 import Int8FeedForward

    mod = Int8FeedForward.from_feed_forward(_ffn(64, 48))
    x = I.rows(torch.Generator().manual_seed(1), 6, 64, F32).view(2, 3, 64)
    _check_feed_forward(mod, x)
    assert torch.equal(mod(x.bfloat16()), x.bfloat16() * 2)


def test_experts(products):
    from torchtitan_amd.int8 import Int8GroupedExperts

    counts = torch.tensor([3, 0, 5])
    x = I.rows(torch.Generator().manual_seed(2), 10, 64, F32)
    _check_experts(Int8GroupedExperts.from_experts(_experts(3, 64, 48, False)), x, counts)
    for grouped in (False, True):  # rows in bf16, and the grouped path, which rounds to it
        mod = Int8GroupedExperts.from_experts(_experts(3, 64, 48, grouped))
        t = x if grouped else x.bfloat16()
        assert mod(t, counts).dtype == t.dtype and torch.equal(mod(t, counts), (t.bfloat16() * 2).type_as(t))


@pytest.mark.gpu
@pytest.mark.parametrize("d,h", [(64, 48), (304, 144), (2304, 1024)])
def test_feed_forward_on_the_gpu(dev, d, h):
    from torchtitan_amd.int8 import Int8FeedForward

    mod = Int8FeedForward.from_feed_forward(_ffn(d, h).to(dev))
    gen = torch.Generator().manual_seed(3)
    for m in (1, 5, 300):
        banner(f"int8 feed-forward in fp32 {m} x {d} / {h}")
        x = I.rows(gen, m, d, F32).to(dev)
        with torch.no_grad():
            _check_feed_forward(mod, x.view(1, m, d))
            assert torch.equal(mod(x[m // 2:m // 2 + 1]), mod(x)[m // 2:m // 2 + 1])  # alone as in its batch


@pytest.mark.gpu
def test_experts_on_the_gpu(dev):
    """Experts of the for-loop path in fp32, few rows and many; a layer of them."""
    from torchtitan_amd.int8 import Int8GroupedExperts

    mod = Int8GroupedExperts.from_experts(_experts(6, 144, 208, False).to(dev))
    gen = torch.Generator().manual_seed(4)
    for per in (1, 8, 200):
        banner(f"int8 for-loop experts in fp32, {per} rows each")
        counts = torch.tensor([per, 0, 2 * per, per + 1, 3, per])
        x = I.rows(gen, int(counts.sum()) + 2, 144, F32)
        with torch.no_grad():
            _check_experts(mod, x.to(dev), counts.to(dev))


@pytest.mark.gpu
def test_a_layer_in_fp32(dev):
    """A MoE layer in fp32, for-loop experts and a shared one, before and after its conversion: an operand of a
    product is off by about amax / (127 sqrt 12), under 1 % of a row's size, four of them one behind another."""
    banner("int8 layer in fp32")
    from types import SimpleNamespace

    from torchtitan_amd import FeedForward, GroupedExperts, Linear, MoE, TokenChoiceTopKRouter
    from torchtitan_amd.quantization import Int8WeightConverter

    lin = lambda i, o: Linear.Config(in_features=i, out_features=o)  # noqa: E731
    moe = _filled(MoE.Config(
        num_experts=4, experts=GroupedExperts.Config(dim=256, hidden_dim=192, num_experts=4, use_grouped_mm=False),
        shared_experts=FeedForward.Config(w1=lin(256, 320), w2=lin(320, 256), w3=lin(256, 320)), score_before_experts=False,
        router=TokenChoiceTopKRouter.Config(num_experts=4, gate=lin(256, 4), top_k=2, score_func="sigmoid")).build()).to(dev)
    x = torch.randn(2, 50, 256, generator=torch.Generator().manual_seed(5)).to(dev)
    dims = SimpleNamespace(pp_enabled=False, cp_enabled=False, ep_enabled=False)
    with torch.no_grad():
        plain = moe(x)
        model = torch.nn.ModuleDict({"moe": moe})
        Int8WeightConverter.Config(fqns=["moe."]).build(parallel_dims=dims, model_compile_enabled=False).convert(model)
        got = moe(x)
    assert got.dtype == F32 and not torch.equal(got, got.bfloat16().float())
    assert (got - plain).norm() < 0.05 * plain.norm()
