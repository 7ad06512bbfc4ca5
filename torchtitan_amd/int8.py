"""Layers whose weights are held in 8-bit integers with a scale for each output channel, for inference.

``Int8Linear`` stands in for ``Linear``, ``Int8FeedForward`` for ``FeedForward`` (the shared expert),
``Int8GroupedExperts`` for ``GroupedExperts`` and ``Int8GptOssGroupedExperts`` for
``GptOssGroupedExperts``, each with the forward signature of what it replaces;
``quantization.Int8WeightConverter`` swaps them into a model. A weight is two buffers: ``*_codes``
[.., N, K] int8 and ``*_scales`` [.., N] fp32 (``ops.int8_quantize`` of the weight's rows). Activations
are quantized to 8 bits by rows in the kernels, x and what lies between two products alike.

What computed in fp32 before does so still: a feed-forward, and experts of the for-loop path, give
rows in fp32 to two products each and their activation to a third, all in fp32. Experts of the
grouped path round such rows to bf16, as the ones that they stand for do, and gpt-oss's experts their
biases too.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch
import torch.nn.functional as F

from . import ops
from .configurable import Module
from .feed_forward import FeedForward
from .gpt_oss import GptOssGroupedExperts
from .linear import Linear
from .moe import GroupedExperts, _local

__all__ = ["Int8FeedForward", "Int8GptOssGroupedExperts", "Int8GroupedExperts", "Int8Linear"]


class _Packed(Module):
    def _buffer(self, name: str, *shape: int) -> None:
        """An empty matrix [.., N, K] in codes: name_codes and name_scales."""
        if shape[-1] % ops.INT8_MULTIPLE:
            raise ValueError(f"8-bit weights take contractions that are multiples of {ops.INT8_MULTIPLE}, got {shape[-1]}")
        self.register_buffer(name + "_codes", torch.empty(*shape, dtype=torch.int8))
        self.register_buffer(name + "_scales", torch.empty(*shape[:-1], dtype=torch.float32))

    def packed(self, name: str) -> tuple[torch.Tensor, torch.Tensor]:
        return getattr(self, name + "_codes"), getattr(self, name + "_scales")

    @torch.no_grad()
    def pack(self, name: str, weight: torch.Tensor) -> None:
        """Takes a weight in bf16 or fp32, on the GPU, whole."""
        weight = _local(weight).detach()
        if weight.shape != self.packed(name)[0].shape:
            raise ValueError(f"{name} of {list(weight.shape)} does not fit {list(self.packed(name)[0].shape)} codes")
        q, s = ops.int8_quantize(weight)
        setattr(self, name + "_codes", q)
        setattr(self, name + "_scales", s)

    def dequantize(self, name: str, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        """The values of a packed weight."""
        return ops.int8_dequantize(*self.packed(name), dtype)

    def _apply(self, fn, recurse=True):
        """As every module's, but the codes' scales stay fp32, whatever the model is cast to."""
        scales = {name: t for name, t in self._buffers.items() if name.endswith("_scales")}
        super()._apply(fn, recurse)
        for name, t in scales.items():
            if self._buffers[name].dtype != torch.float32:
                self._buffers[name] = t.to(self._buffers[name].device)
        return self


def _empty(config: Module.Config) -> Module:
    with torch.device("meta"):
        return config.build()


class Int8Linear(_Packed):
    @dataclass(kw_only=True, slots=True)
    class Config(Linear.Config):
        pass

    def __init__(self, config: Config):
        super().__init__()
        self.in_features, self.out_features = config.in_features, config.out_features
        self._buffer("weight", config.out_features, config.in_features)
        self.register_buffer("bias", torch.empty(config.out_features, dtype=torch.float32) if config.bias else None)

    @classmethod
    def from_linear(cls, linear: torch.nn.Linear) -> "Int8Linear":
        out = _empty(cls.Config(in_features=linear.in_features, out_features=linear.out_features, bias=linear.bias is not None))
        out.pack("weight", linear.weight)
        if linear.bias is not None:
            out.bias = _local(linear.bias).detach().float()
        return out.train(linear.training)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return ops.linear_int8(x, *self.packed("weight"), self.bias)


class Int8FeedForward(_Packed):
    @dataclass(kw_only=True, slots=True)
    class Config(FeedForward.Config):
        pass

    def __init__(self, config: Config):
        super().__init__()
        for name in ("w1", "w2", "w3"):
            lin = getattr(config, name)
            if lin.bias:
                raise ValueError(f"{type(self).__name__} has no biases, {name} has one")
            self._buffer(name, lin.out_features, lin.in_features)

    @classmethod
    def from_feed_forward(cls, ffn: FeedForward) -> "Int8FeedForward":
        lins = {name: getattr(ffn, name) for name in ("w1", "w2", "w3")}
        out = _empty(cls.Config(**{name: Linear.Config(in_features=lin.in_features, out_features=lin.out_features,
                                                       bias=lin.bias is not None) for name, lin in lins.items()}))
        for name, lin in lins.items():
            out.pack(name, lin.weight)
        return out.train(ffn.training)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if x.dtype == torch.float32:
            h = F.silu(ops.linear_int8(x, *self.packed("w1"))) * ops.linear_int8(x, *self.packed("w3"))
            return ops.linear_int8(h, *self.packed("w2"))
        y = ops.swiglu_ffn_int8(x.bfloat16(), *self.packed("w1"), *self.packed("w2"), *self.packed("w3"))
        return y.type_as(x)


class Int8GroupedExperts(_Packed):
    use_grouped_mm = True  # (of the class, for whole modules saved without it)

    @dataclass(kw_only=True, slots=True)
    class Config(GroupedExperts.Config):
        pass

    def __init__(self, config: Config):
        super().__init__()
        d, h, e = config.dim, config.hidden_dim, config.num_experts
        self.num_experts = e
        self.use_grouped_mm = config.use_grouped_mm
        self._buffer("w1", e, h, d)
        self._buffer("w2", e, d, h)
        self._buffer("w3", e, h, d)

    @classmethod
    def from_experts(cls, experts: GroupedExperts) -> "Int8GroupedExperts":
        e, h, d = _local(experts.w1).shape
        out = _empty(cls.Config(dim=d, hidden_dim=h, num_experts=e, use_grouped_mm=experts.use_grouped_mm))
        for name in ("w1", "w2", "w3"):
            out.pack(name, _local(getattr(experts, name)))
        return out.train(experts.training)

    def forward(self, x: torch.Tensor, num_tokens_per_expert: torch.Tensor) -> torch.Tensor:
        if x.dtype == torch.float32 and not self.use_grouped_mm:
            g, u = (ops.grouped_linear_int8(x, *self.packed(name), num_tokens_per_expert) for name in ("w1", "w3"))
            return ops.grouped_linear_int8(F.silu(g) * u, *self.packed("w2"), num_tokens_per_expert)
        y = ops.grouped_swiglu_int8(x.bfloat16(), *self.packed("w1"), *self.packed("w2"), *self.packed("w3"),
                                    num_tokens_per_expert)
        return y.type_as(x)


class Int8GptOssGroupedExperts(_Packed):
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
    def from_experts(cls, experts: GptOssGroupedExperts) -> "Int8GptOssGroupedExperts":
        e, d, h = _local(experts.mlp2_weight).shape
        out = _empty(cls.Config(dim=d, hidden_dim=h, num_experts=e, swiglu_limit=experts.swiglu_limit))
        for name in ("mlp1_weight", "mlp2_weight"):
            out.pack(name, _local(getattr(experts, name)))
        for name in ("mlp1_bias", "mlp2_bias"):
            setattr(out, name, _local(getattr(experts, name)).detach().to(torch.bfloat16))
        return out.train(experts.training)

    def forward(self, x: torch.Tensor, num_tokens_per_expert: torch.Tensor) -> torch.Tensor:
        y = ops.grouped_swiglu_oss_int8(x.bfloat16(), *self.packed("mlp1_weight"), self.mlp1_bias,
                                        *self.packed("mlp2_weight"), self.mlp2_bias, num_tokens_per_expert,
                                        float(self.swiglu_limit))
        return y.type_as(x)
