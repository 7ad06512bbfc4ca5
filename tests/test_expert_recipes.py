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
