"""Modules on 8-bit integers and their converter, on the CPU (rows are packed by the 64-bit oracle here)."""

from types import SimpleNamespace

import pytest
import torch

from tests import int8_util as I

DIMS = SimpleNamespace(pp_enabled=False, cp_enabled=False, ep_enabled=False)


@pytest.fixture
def convert(monkeypatch):
    from torchtitan_amd import ops
    from torchtitan_amd.quantization import Int8WeightConverter

    monkeypatch.setattr(ops, "int8_quantize", I.pack)
    monkeypatch.setattr("torchtitan_amd.quantization.has_gfx950", lambda: True)
    return lambda model, *fqns: Int8WeightConverter.Config(fqns=list(fqns)).build(
        parallel_dims=DIMS, model_compile_enabled=False).convert(model)


def _lin(i, o, bias=False):
    from torchtitan_amd import Linear

    return Linear.Config(in_features=i, out_features=o, bias=bias)


def _ffn(d=64, h=48, bias=False):
    from torchtitan_amd import FeedForward

    return FeedForward.Config(w1=_lin(d, h, bias), w2=_lin(h, d), w3=_lin(d, h))


def _experts(cls=None):
    from torchtitan_amd import GroupedExperts

    return (cls or GroupedExperts).Config(dim=64, hidden_dim=48, num_experts=2).build()


def _moe():
    from torchtitan_amd import GroupedExperts, MoE, TokenChoiceTopKRouter

    moe = MoE.Config(num_experts=2, experts=GroupedExperts.Config(dim=64, hidden_dim=48, num_experts=2), shared_experts=_ffn(),
                     router=TokenChoiceTopKRouter.Config(num_experts=2, gate=_lin(64, 2), top_k=1)).build()
    for p in moe.parameters():
        torch.nn.init.normal_(p)
    return moe


def test_a_layer_is_converted(convert):
    from torchtitan_amd import Linear
    from torchtitan_amd import int8 as M

    model = torch.nn.ModuleDict({"layer": torch.nn.ModuleDict({"moe": _moe(), "out": _lin(64, 80, True).build()}), "rest": _experts()})
    weights = {n: p.detach().clone() for n, p in model.named_parameters()}
    assert convert(model, "layer") == ["layer.moe.experts", "layer.moe.shared_experts", "layer.out"]
    moe, out = model["layer"]["moe"], model["layer"]["out"]
    assert type(moe.experts) is M.Int8GroupedExperts and type(moe.shared_experts) is M.Int8FeedForward
    assert type(out) is M.Int8Linear and type(moe.router.gate) is Linear and type(model["rest"]).__name__ == "GroupedExperts"
    for mod, at, name in ((moe.experts, "layer.moe.experts.w2", "w2"), (moe.shared_experts, "layer.moe.shared_experts.w1.weight", "w1"),
                          (out, "layer.out.weight", "weight")):
        q, s = I.pack(weights[at])
        assert torch.equal(mod.packed(name)[0], q) and torch.equal(mod.packed(name)[1], s)
    assert torch.equal(out.bias, weights["layer.out.bias"])
    assert {n for n, _ in model["layer"].named_parameters()} == {"moe.router.gate.weight"}
    assert {n for n in moe.experts.state_dict()} == {f"w{i}_{k}" for i in (1, 2, 3) for k in ("codes", "scales")}
    assert convert(model, "layer") == []  # converted already
    # a checkpoint of it goes into an empty one; a cast of the model leaves the scales in 32 bits
    other = M.Int8GroupedExperts.Config(dim=64, hidden_dim=48, num_experts=2).build()
    other.load_state_dict(moe.experts.state_dict())
    model.to(torch.bfloat16).half()
    for name in ("w1", "w2", "w3"):
        (q, s), (oq, os) = moe.experts.packed(name), other.packed(name)
        assert q.dtype == torch.int8 and s.dtype == torch.float32 and torch.equal(q, oq) and torch.equal(s, os)
    assert model["rest"].w1.dtype == torch.float16


def test_gpt_oss_experts(convert):
    from torchtitan_amd.gpt_oss import GptOssGroupedExperts
    from torchtitan_amd.int8 import Int8GptOssGroupedExperts

    experts = GptOssGroupedExperts.Config(dim=64, hidden_dim=48, num_experts=2, swiglu_limit=5.0).build()
    for p in experts.parameters():
        torch.nn.init.normal_(p)
    model = torch.nn.ModuleDict({"e": experts})
    assert convert(model, "e") == ["e"]
    got = model["e"]
    assert type(got) is Int8GptOssGroupedExperts and got.swiglu_limit == 5.0 and not list(got.parameters())
    assert torch.equal(got.mlp1_weight_codes, I.pack(experts.mlp1_weight)[0]) and got.mlp1_weight_scales.shape == (2, 96)
    assert torch.equal(got.mlp2_bias, experts.mlp2_bias.bfloat16())


def test_shared_modules_are_converted_once(convert):
    lin = _lin(64, 32).build()
    model = torch.nn.ModuleDict({"a": lin, "b": lin})
    assert convert(model, "a", "b") == ["a", "b"] and model["a"] is model["b"]
    ffn = _ffn().build()
    model = torch.nn.ModuleDict({"a": ffn})
    assert convert(model, "a.w1") == ["a.w1"]  # a projection of one alone
    assert type(model["a"].w1).__name__ == "Int8Linear" and type(model["a"].w2).__name__ == "Linear"


def test_what_cannot_be_converted_is_refused(convert):
    from torchtitan_amd import FeedForward, GroupedExperts, Linear
    from torchtitan_amd.quantization import MXFP4Converter

    class Scaled(GroupedExperts):
        pass

    class Other(Linear):
        pass

    hooked, part, marked = _experts(), _ffn().build(), _experts()
    hooked.register_forward_hook(lambda *a: None)
    part.w3.register_forward_pre_hook(lambda *a: None)
    marked.mxfp4 = True
    inner = _ffn().build()
    inner.w2 = Other(_lin(48, 64))
    for bad in (Scaled(GroupedExperts.Config(dim=64, hidden_dim=48, num_experts=2)), hooked, part, inner, marked, _ffn(bias=True).build()):
        model = torch.nn.ModuleDict({"a": _experts(), "b": bad})
        with pytest.raises(ValueError, match="b"):
            convert(model, "a", "b")
        assert type(model["a"]) is GroupedExperts  # nothing is replaced half way
    with pytest.raises(ValueError, match="multiples of 16"):
        convert(torch.nn.ModuleDict({"a": _lin(72, 64).build()}), "a")
    model = torch.nn.ModuleDict({"a": _experts()})
    convert(model, "a")
    conv = MXFP4Converter.Config(fqns=["a"]).build(parallel_dims=DIMS, model_compile_enabled=False)
    with pytest.raises(ValueError, match="cannot be converted to mxfp4"):
        conv.convert(model)
    with pytest.raises(ValueError, match="does not fit"):
        model["a"].pack("w1", torch.zeros(2, 32, 64))
    assert isinstance(part, FeedForward) and type(part.w1) is Linear


def test_sizes_and_types_are_checked_before_anything_is_replaced(convert):
    from torchtitan_amd import GroupedExperts

    for bad in (_lin(72, 64).build(), _ffn(h=40).build(), GroupedExperts.Config(dim=24, hidden_dim=48, num_experts=2).build(),
                _lin(64, 8).build().half(), _lin(64, 8).build().double()):
        model = torch.nn.ModuleDict({"a": _experts(), "b": bad})
        with pytest.raises((ValueError, TypeError), match="^b"):
            convert(model, "a", "b")
        assert type(model["a"]) is GroupedExperts and model["b"] is bad


def test_converter_needs_the_hardware(monkeypatch):
    from torchtitan_amd import quantization as Q

    monkeypatch.setattr(Q, "has_gfx950", lambda: False)
    with pytest.raises(ValueError, match="gfx950"):
        Q.Int8WeightConverter.Config(fqns=["a"]).build(parallel_dims=DIMS, model_compile_enabled=False)


def test_the_kernel_a_product_takes():
    """The tile goes by rows, experts and sizes; each is taken somewhere."""
    import os

    from torchtitan_amd import _lib

    if not os.path.exists(_lib.library_path()):
        from torchtitan_amd import build

        build.build()
    tile = _lib.lib().moe_int8_tile
    for args, want in (((1, 1, 2304, 2304), 4), ((96, 1, 2304, 1024), 4), ((300, 1, 2304, 2304), 3), ((8, 1, 7168, 7168), 3), ((4, 1, 7168, 7168), 4), ((1, 1, 16384, 2304), 3),
                       ((8, 256, 2304, 2048), 4), ((1024, 1, 2304, 2304), 2), ((2048, 1, 2304, 2304), 1), ((4096, 1, 2304, 2304), 0),
                       ((16384, 1, 7168, 7168), 0), ((8200, 32, 7168, 2048), 1)):
        assert tile(*args, 256) == want, args
    assert tile(-1, 1, 64, 64, 256) == -1 and tile(4, 1, 72, 64, 256) == -2 and tile(4, 1, 64, 64, 0) == -1
