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
