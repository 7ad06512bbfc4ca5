"""The converters to packed weights, on the CPU: a model is converted whole or not at all."""

from types import SimpleNamespace

import pytest
import torch

from tests import int8_util as I

DIMS = SimpleNamespace(pp_enabled=False, cp_enabled=False, ep_enabled=False)


@pytest.fixture
def converters(monkeypatch):
    """By name, a function (model, *fqns) of the packed form's converter, and the rows it quantized."""
    from torchtitan_amd import ops
    from torchtitan_amd import quantization as Q

    monkeypatch.setattr("torchtitan_amd.quantization.has_gfx950", lambda: True)
    monkeypatch.setattr(ops, "int8_quantize", I.pack)
    monkeypatch.setattr(ops, "mxfp4_quantize", lambda w: (torch.zeros(*w.shape[:-1], w.shape[-1] // 2, dtype=torch.uint8),
                                                          torch.zeros(*w.shape[:-1], w.shape[-1] // 32, dtype=torch.uint8)))
    return {name: lambda model, *fqns, cls=getattr(Q, name): cls.Config(fqns=list(fqns)).build(
        parallel_dims=DIMS, model_compile_enabled=False).convert(model) for name in ("Int8WeightConverter", "MXFP4WeightConverter")}


def _experts(d=64, h=32, e=2):
    from torchtitan_amd import GroupedExperts

    return GroupedExperts.Config(dim=d, hidden_dim=h, num_experts=e).build()


def _lin(i, o, bias=False):
    from torchtitan_amd import Linear

    return Linear.Config(in_features=i, out_features=o, bias=bias)


@pytest.mark.parametrize("name,op", [("Int8WeightConverter", "int8_quantize"), ("MXFP4WeightConverter", "mxfp4_quantize")])
def test_a_later_module_that_cannot_be_packed(converters, monkeypatch, name, op):
    """Whatever packing a module raises (weights off the GPU, no memory left), those before it stay as they were."""
    from torchtitan_amd import ops

    pack, calls = getattr(ops, op), []

    def fails_at_the_fifth(w):
        calls.append(w)
        if len(calls) == 5:
            raise RuntimeError("no memory left")
        return pack(w)

    monkeypatch.setattr(ops, op, fails_at_the_fifth)
    model = torch.nn.ModuleDict({k: _experts() for k in "abc"})
    before = dict(model.named_parameters())
    with pytest.raises(RuntimeError, match="no memory"):
        converters[name](model, "a", "b", "c")
    after = dict(model.named_parameters())
    assert list(after) == list(before) and all(after[k] is before[k] for k in before)
    assert {type(m).__name__ for m in model.values()} == {"GroupedExperts"}
    monkeypatch.setattr(ops, op, pack)
    assert converters[name](model, "a", "b", "c") == ["a", "b", "c"] and not list(model.parameters())


def test_modules_that_could_not_run(converters):
    """More experts or output channels than the operators take, and feed-forwards whose widths a layer does not
    have, are refused by the converter, not by the first call."""
    from torchtitan_amd import FeedForward, GroupedExperts
    from torchtitan_amd.gpt_oss import GptOssGroupedExperts

    ffn = lambda w1, w2, w3: FeedForward.Config(w1=_lin(*w1), w2=_lin(*w2), w3=_lin(*w3)).build()  # noqa: E731
    meta = lambda make: torch.nn.Module.to(make, "meta")  # noqa: E731
    with torch.device("meta"):
        wide = _lin(16, 2 ** 22 + 1).build()
    oss = GptOssGroupedExperts.Config(dim=16, hidden_dim=16, num_experts=1025).build()
    for bad, what in ((_experts(16, 16, 1025), "experts"), (meta(oss), "experts"), (wide, "output channels"),
                      (_lin(16, 0).build(), "output channels"), (ffn((64, 32), (32, 48), (64, 32)), "w2"),
                      (ffn((64, 32), (32, 64), (64, 48)), "w3"), (ffn((64, 32), (32, 64), (48, 32)), "w3")):
        model = torch.nn.ModuleDict({"a": _experts(), "b": bad})
        with pytest.raises(ValueError, match=f"^b: .*{what}"):
            converters["Int8WeightConverter"](model, "a", "b")
        assert type(model["a"]) is GroupedExperts and model["b"] is bad
    model = torch.nn.ModuleDict({"a": _experts(16, 16, 1024)})
    assert converters["Int8WeightConverter"](model, "a") == ["a"]


@pytest.mark.parametrize("first", ["ffn", "proj"])
def test_a_projection_that_a_feed_forward_shares(converters, first):
    """It is replaced under its own name too, whichever name comes first."""
    from torchtitan_amd import FeedForward

    ffn = FeedForward.Config(w1=_lin(64, 32), w2=_lin(32, 64), w3=_lin(64, 32)).build()
    parts = {"ffn": ffn, "proj": ffn.w3}
    weight = ffn.w3.weight
    model = torch.nn.ModuleDict({k: parts[k] for k in sorted(parts, key=lambda k: k != first)})
    assert sorted(converters["Int8WeightConverter"](model, "ffn", "proj")) == ["ffn", "proj"]
    assert type(model["ffn"]).__name__ == "Int8FeedForward" and type(model["proj"]).__name__ == "Int8Linear"
    for mod, name in ((model["ffn"], "w3"), (model["proj"], "weight")):
        assert torch.equal(mod.packed(name)[0], I.pack(weight)[0])


@pytest.fixture
def mesh():
    """Two devices of which this process is the first (nothing is sent)."""
    import torch.distributed as dist
    from torch.distributed.device_mesh import init_device_mesh
    from torch.testing._internal.distributed.fake_pg import FakeStore

    dist.init_process_group("fake", store=FakeStore(), rank=0, world_size=2)
    try:
        yield init_device_mesh("cpu", (2,), mesh_dim_names=("tp",))
    finally:
        dist.destroy_process_group()


@pytest.mark.parametrize("dim", [0, 1])
def test_projections_sharded_over_devices(converters, mesh, dim):
    """Half of a weight is not taken for the whole; one that every device holds is."""
    from torch.distributed.tensor import DTensor, Replicate, Shard

    from torchtitan_amd import FeedForward, Linear

    def place(lin, placement):
        lin.weight = torch.nn.Parameter(DTensor.from_local(lin.weight.detach(), mesh, [placement], run_check=False))
        return lin

    def half():
        lin = place(_lin(32 if dim else 64, 32 if dim == 0 else 64).build(), Shard(dim))
        lin.in_features, lin.out_features = 64, 64
        return lin

    ffn = FeedForward.Config(w1=_lin(64, 64), w2=_lin(64, 64), w3=_lin(64, 64)).build()
    ffn.w3 = half()
    for bad in (half(), ffn):
        model = torch.nn.ModuleDict({"a": _experts(), "b": bad})
        with pytest.raises(ValueError, match="does not fit"):
            converters["Int8WeightConverter"](model, "a", "b")
        assert model["b"] is bad and isinstance(bad, (Linear, FeedForward)) and list(model["a"].parameters())
    lin = place(_lin(64, 32).build(), Replicate())
    model = torch.nn.ModuleDict({"b": lin})
    assert converters["Int8WeightConverter"](model, "b") == ["b"]
    assert torch.equal(model["b"].weight_codes, I.pack(lin.weight.to_local())[0])
