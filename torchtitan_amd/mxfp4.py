"""Experts whose weights are held packed in MXFP4, for inference.

``MXFP4GroupedExperts`` stands in for ``GroupedExperts``, ``MXFP4GptOssGroupedExperts`` for
``GptOssGroupedExperts`` (same ``forward(x, num_tokens_per_expert)``, so a MoE layer holds either);
``quantization.MXFP4WeightConverter`` swaps them into a model. The weights are buffers in the
layout of gpt-oss's own checkpoints: ``*_blocks`` [.., K / 2], two e2m1 codes per byte along the
contraction, the first in the low half, and ``*_scales`` [.., K / 32], e8m0. x and the activation
between the products are quantized in the kernels (``ops.grouped_swiglu_mxfp4``); few rows per
expert, as in generation, take a kernel that reads the weights once.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from . import ops
from .configurable import Module
from .gpt_oss import GptOssGroupedExperts
from .moe import GroupedExperts, _local

__all__ = ["MXFP4GptOssGroupedExperts", "MXFP4GroupedExperts"]


class _Packed(Module):
    weights: tuple[str, ...]

    def _buffer(self, name: str, *shape: int) -> None:
        """An empty packed matrix [.., K]: name_blocks and name_scales."""
        if shape[-1] % ops.MX_BLOCK:
            raise ValueError(f"MXFP4 weights take contractions in whole blocks of {ops.MX_BLOCK}, got {shape[-1]}")
        self.register_buffer(name + "_blocks", torch.empty(*shape[:-1], shape[-1] // 2, dtype=torch.uint8))
        self.register_buffer(name + "_scales", torch.empty(*shape[:-1], shape[-1] // ops.MX_BLOCK, dtype=torch.uint8))

    def packed(self, name: str) -> tuple[torch.Tensor, torch.Tensor]:
        return getattr(self, name + "_blocks"), getattr(self, name + "_scales")

    @torch.no_grad()
    def pack(self, name: str, weight: torch.Tensor) -> None:
        """Takes a weight in bf16 or fp32, on the GPU."""
        q, s = ops.mxfp4_quantize(_local(weight).detach())
        if q.shape != self.packed(name)[0].shape:
            raise ValueError(f"{name} of {list(weight.shape)} does not fit {list(self.packed(name)[0].shape)} bytes")
        setattr(self, name + "_blocks", q)
        setattr(self, name + "_scales", s)

    def dequantize(self, name: str, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        """The values of a packed weight."""
        return ops.mxfp4_dequantize(*self.packed(name), dtype)

    @classmethod
    def _like(cls, experts: Module, config: Module.Config) -> "_Packed":
        """An instance of this config with experts' weights packed."""
        with torch.device("meta"):
            out = config.build()
        for name in cls.weights:
            out.pack(name, getattr(experts, name))
        return out.train(experts.training)


class MXFP4GroupedExperts(_Packed):
    weights = ("w1", "w2", "w3")

    @dataclass(kw_only=True, slots=True)
    class Config(GroupedExperts.Config):
        pass

    def __init__(self, config: Config):
        super().__init__()
        d, h, e = config.dim, config.hidden_dim, config.num_experts
        self.num_experts = e
        self._buffer("w1", e, h, d)
        self._buffer("w2", e, d, h)
        self._buffer("w3", e, h, d)

    @classmethod
    def from_experts(cls, experts: GroupedExperts) -> "MXFP4GroupedExperts":
        e, h, d = _local(experts.w1).shape
        return cls._like(experts, cls.Config(dim=d, hidden_dim=h, num_experts=e))

    def forward(self, x: torch.Tensor, num_tokens_per_expert: torch.Tensor) -> torch.Tensor:
        y = ops.grouped_swiglu_mxfp4(x.bfloat16(), *self.packed("w1"), *self.packed("w2"), *self.packed("w3"),
                                     num_tokens_per_expert)
        return y.type_as(x)


class MXFP4GptOssGroupedExperts(_Packed):
    weights = ("mlp1_weight", "mlp2_weight")

    @dataclass(kw_only=True, slots=True)
    class Config(GptOssGroupedExperts.Config):
        pass

    def __init__(self, config: Config):
        super().__init__()
        d, h, e = config.dim, config.hidden_dim, config.num_experts
        self.num_experts = e
        self.swiglu_limit = config.swiglu_limit
        self._buffer("mlp1_weight", e, 2 * h, d)
        self._buffer("mlp2_weight", e, d, h)
        self.register_buffer("mlp1_bias", torch.empty(e, 2 * h, dtype=torch.bfloat16))
        self.register_buffer("mlp2_bias", torch.empty(e, d, dtype=torch.bfloat16))

    @classmethod
    def from_experts(cls, experts: GptOssGroupedExperts) -> "MXFP4GptOssGroupedExperts":
        e, d, h = _local(experts.mlp2_weight).shape
        out = cls._like(experts, cls.Config(dim=d, hidden_dim=h, num_experts=e, swiglu_limit=experts.swiglu_limit))
        for name in ("mlp1_bias", "mlp2_bias"):
            setattr(out, name, _local(getattr(experts, name)).detach().to(torch.bfloat16))
        return out

    def load_hf(self, hf: dict[str, torch.Tensor], layer: int) -> None:
        """Takes layer `layer`'s experts from a gpt-oss checkpoint as it is, its weights packed
        (model.layers.L.mlp.experts.{gate_up,down}_proj_{blocks,scales,bias}): blocks [.., K / 32, 16],
        scales [.., K / 32]. All of it or, where something is missing or does not fit, nothing."""
        taken = {}
        for name, key in (("mlp1", "gate_up_proj"), ("mlp2", "down_proj")):
            at = f"model.layers.{layer}.mlp.experts.{key}_"
            for own, t in ((f"{name}_weight_blocks", hf[at + "blocks"].flatten(-2)),
                           (f"{name}_weight_scales", hf[at + "scales"]),
                           (f"{name}_bias", hf[at + "bias"])):
                like = getattr(self, own)
                if t.shape != like.shape or (like.dtype == torch.uint8 and t.dtype != torch.uint8):
                    raise ValueError(f"{at[:-1]} for {own}: expected {like.dtype} {list(like.shape)}, got {t.dtype} "
                                     f"{list(t.shape)}")
                taken[own] = t
        for own, t in taken.items():
            like = getattr(self, own)
            setattr(self, own, t.to(like.device, torch.uint8 if like.dtype == torch.uint8 else torch.bfloat16).contiguous())

    def forward(self, x: torch.Tensor, num_tokens_per_expert: torch.Tensor) -> torch.Tensor:
        y = ops.grouped_swiglu_oss_mxfp4(x.bfloat16(), *self.packed("mlp1_weight"), self.mlp1_bias,
                                         *self.packed("mlp2_weight"), self.mlp2_bias, num_tokens_per_expert,
                                         float(self.swiglu_limit))
        return y.type_as(x)
