"""How GroupedExperts choose their products, on the CPU: modules and models that were there before a
recipe was, and models of which a converter matches nothing or a module twice."""

from types import SimpleNamespace

import pytest
import torch

DIMS = SimpleNamespace(pp_enabled=False, cp_enabled=False, ep_enabled=False)


def _experts():
    from torchtitan_amd import GroupedExperts

    return GroupedExperts.Config(dim=64, hidden_dim=64, num_experts=2).build()


def test_modules_of_before(monkeypatch):
    """A whole module that was pickled before the 4-bit and 8-bit-activation recipes came has not their
    attributes: it runs as it did, and can be converted."""
    from torchtitan_amd import moe
    from torchtitan_amd import quantization as Q

    monkeypatch.setattr(moe, "_run_experts_grouped_mm", lambda w1, w2, w3, x, n: "bf16")
    monkeypatch.setattr(moe, "_run_experts_grouped_mm_mxfp8", lambda w1, w2, w3, x, n: "mxfp8")
    monkeypatch.setattr(moe, "_run_experts_grouped_mm_mxfp4", lambda w1, w2, w3, x, n: "mxfp4")
    for attr in ("mxfp8", "mxfp4"):
        m = _experts()
        for new in ("mxfp4", "ckpt8"):
            m.__dict__.pop(new, None)
        assert m(torch.zeros(4, 64), torch.tensor([2, 2])) == "bf16"
        model = torch.nn.ModuleDict({"experts": m})
        assert Q._mark_experts(model, ["experts"], attr) == ["experts"]
        assert m(torch.zeros(4, 64), torch.tensor([2, 2])) == attr


@pytest.fixture
def converter(monkeypatch):
    """The converters by name, built as on the hardware; the packing on the CPU."""
    from tests import narrow_util as N
    from torchtitan_amd import ops
    from torchtitan_amd import quantization as Q

    monkeypatch.setattr(Q, "has_gfx950", lambda: True)
    monkeypatch.setattr(ops, "mxfp4_quantize", N.pack4)

    def build(name, *fqns):
        conv = getattr(Q, name).Config(fqns=list(fqns))
        return conv.build(parallel_dims=DIMS, model_compile_enabled=False)
    return build


def test_shared_experts_are_packed_under_each_name(converter):
    """Experts that two layers share: one packed module in both places, under whichever name asked for."""
    from torchtitan_amd.mxfp4 import MXFP4GroupedExperts

    for fqns in (("a", "b"), ("b",)):
        m = _experts()
        torch.nn.init.normal_(m.w1), torch.nn.init.normal_(m.w2), torch.nn.init.normal_(m.w3)
        model = torch.nn.ModuleDict({n: torch.nn.ModuleDict({"experts": m}) for n in "ab"})
        assert converter("MXFP4WeightConverter", *fqns).convert(model) == [f"{n}.experts" for n in fqns]
        assert type(model["b"]["experts"]) is MXFP4GroupedExperts
        assert (model["a"]["experts"] is model["b"]["experts"]) == (len(fqns) == 2)
        assert len(list(model["a"].parameters())) == (0 if len(fqns) == 2 else 3)


def test_shared_experts_are_marked_once():
    from torchtitan_amd import quantization as Q

    for fqns, names in ((["a", "b"], ["a.experts"]), (["b"], ["b.experts"])):
        m = _experts()
        model = torch.nn.ModuleDict({n: torch.nn.ModuleDict({"experts": m}) for n in "ab"})
        assert Q._mark_experts(model, fqns, "ckpt8") == names and m.ckpt8


def _gptoss():
    from torchtitan_amd.gpt_oss import GptOssGroupedExperts

    return GptOssGroupedExperts.Config(dim=64, hidden_dim=64, num_experts=2).build()


def _packed():
    from torchtitan_amd.mxfp4 import MXFP4GroupedExperts

    return MXFP4GroupedExperts.Config(dim=64, hidden_dim=64, num_experts=2).build()


@pytest.mark.parametrize("name", ["MXFP4Converter", "MXFP8ActivationCheckpointConverter"])
@pytest.mark.parametrize("make", [_gptoss, _packed])
def test_experts_without_a_training_form_are_refused(converter, name, make):
    """gpt-oss's experts and packed ones have no such recipe: a match raises, and marks no others."""
    model = torch.nn.ModuleDict({"experts": _experts(), "later": torch.nn.ModuleDict({"experts": make()})})
    with pytest.raises(ValueError, match="later.experts"):
        converter(name, "experts").convert(model)
    assert not model["experts"].mxfp4 and not model["experts"].ckpt8
    model = torch.nn.ModuleDict({"experts": _experts(), "rest": make()})  # not matched: not refused
    assert converter(name, "experts").convert(model) == ["experts"]


def test_experts_that_cannot_be_packed_are_refused(converter):
    """A subclass may compute something else, a hook sees calls of the module it is on: neither goes
    with the module that is replaced."""
    from torchtitan_amd import GroupedExperts

    class Scaled(GroupedExperts):
        def forward(self, x, num_tokens_per_expert):
            return 2 * super().forward(x, num_tokens_per_expert)

    hooked = _experts()
    hooked.register_forward_pre_hook(lambda mod, args: None)
    for bad in (Scaled(GroupedExperts.Config(dim=64, hidden_dim=64, num_experts=2)), hooked):
        model = torch.nn.ModuleDict({"a": torch.nn.ModuleDict({"experts": _experts()}),
                                     "b": torch.nn.ModuleDict({"experts": bad})})
        with pytest.raises(ValueError, match="b.experts"):
            converter("MXFP4WeightConverter", "experts").convert(model)
        assert type(model["a"]["experts"]) is GroupedExperts  # nothing is replaced half way
    model = torch.nn.ModuleDict({"a": _packed()})
    assert converter("MXFP4WeightConverter", "a").convert(model) == []  # packed already


def test_a_checkpoint_goes_in_whole():
    """load_hf of a checkpoint with something missing or of another shape leaves every weight as it was."""
    from torchtitan_amd.mxfp4 import MXFP4GptOssGroupedExperts

    m = MXFP4GptOssGroupedExperts.Config(dim=64, hidden_dim=64, num_experts=2).build()
    at = "model.layers.0.mlp.experts."
    hf = {}
    for key, rows in (("gate_up_proj", 128), ("down_proj", 64)):
        hf |= {f"{at}{key}_blocks": torch.zeros(2, rows, 2, 16, dtype=torch.uint8),
               f"{at}{key}_scales": torch.zeros(2, rows, 2, dtype=torch.uint8), f"{at}{key}_bias": torch.zeros(2, rows)}
    m.load_hf(hf, 0)
    other = {k: v + 1 for k, v in hf.items()}
    for key in other:
        for bad in ({k: v for k, v in other.items() if k != key}, {**other, key: other[key][:1]}):
            with pytest.raises((KeyError, ValueError)):
                m.load_hf(bad, 0)
            assert not any(t.any() for t in m.state_dict().values()), key
    m.load_hf(other, 0)
    assert all((t == 1).all() for t in m.state_dict().values())
