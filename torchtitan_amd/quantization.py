"""fp8 and MXFP8 for the MoE experts, with the interface of the reference's converters.

Mirrors ``Float8GroupedMMConverter`` (torchtitan/components/quantization/float8.py:220-300),
``MXFP8Converter`` (quantization/mx.py:25-134) and ``PAD_MULTIPLE_MAP`` /
``find_pad_multiple`` (quantization/__init__.py:34-57):
``<Converter>.Config(fqns=[...]).build(...).convert(model)`` switches every
``GroupedExperts`` whose fully qualified name contains one of ``fqns`` to the
MI355X quantized grouped GEMMs: fp8 e4m3 with dynamic rowwise scales, or
MXFP8 (e4m3 elements, one e8m0 scale per 32 along the contraction, RCEIL);
fp32 accumulation, bf16 outputs. Parameters stay bf16/fp32 master weights and
the state_dict is unchanged; quantization happens inside each forward and
backward.

Four more, with the same interface and without a counterpart in the reference:
``MXFP4Converter`` (training with MXFP4 products, gradients straight through),
``MXFP8ActivationCheckpointConverter`` (bf16 products, activations kept for the
backward in MXFP8), ``MXFP4WeightConverter`` (inference: the experts are
replaced by ones that hold their weights packed in 4 bits, ``mxfp4.py``) and
``Int8WeightConverter`` (inference: experts, shared experts and projections are
replaced by ones on 8-bit integers, ``int8.py``).
"""

from __future__ import annotations

import logging
from collections.abc import Callable
from dataclasses import dataclass, field

import torch
from torch import nn

from . import ops
from .configurable import Configurable
from .feed_forward import FeedForward
from .gpt_oss import GptOssGroupedExperts
from .int8 import Int8FeedForward, Int8GptOssGroupedExperts, Int8GroupedExperts, Int8Linear
from .linear import Linear
from .moe import GroupedExperts, TokenChoiceTopKRouter, _local
from .mxfp4 import MXFP4GptOssGroupedExperts, MXFP4GroupedExperts

__all__ = ["Float8GroupedMMConverter", "Int8WeightConverter", "MXFP4Converter", "MXFP4WeightConverter", "MXFP8ActivationCheckpointConverter",
           "MXFP8Converter", "PAD_MULTIPLE_MAP", "find_pad_multiple"]

logger = logging.getLogger(__name__)


def has_gfx950() -> bool:
    """True when the current GPU is an MI355X-class CDNA4 part (gfx950), whose
    fp8 e4m3 and block-scaled MFMAs these kernels use. The reference's converters
    check for CUDA SM89 / SM100 instead (torchtitan/tools/utils.py:20-33)."""
    if not torch.cuda.is_available():
        return False
    arch = getattr(torch.cuda.get_device_properties(torch.cuda.current_device()), "gcnArchName", "")
    return arch.split(":")[0] == "gfx950"

# token-group alignment of quantized grouped GEMMs (fp8: 16 one-byte elements;
# MXFP8: one 32-element scaling block)
PAD_MULTIPLE_MAP: dict[str, int] = {"float8": 16, "mxfp8": 32}


class Float8GroupedMMConverter(Configurable):
    @dataclass(kw_only=True, slots=True)
    class Config(Configurable.Config):
        fqns: list[str] | str = field(default_factory=list)

    def __init__(self, config: Config, *, parallel_dims, model_compile_enabled: bool):
        """Checks as float8.py:238-256 does: the hardware first, then the MoE
        training prototype's limits (no pipeline or context parallelism)."""
        self.fqns = _split_fqns(config.fqns)
        if not has_gfx950():
            raise ValueError("Float8 MoE training only supported on gfx950 (MI355X).")
        if not model_compile_enabled:
            logger.info("float8 MoE: the grouped GEMMs are hand-written kernels; compile is not needed for speed")
        assert not parallel_dims.pp_enabled, (
            "Float8 MoE training prototype does not yet support pipeline parallelism"
        )
        assert not parallel_dims.cp_enabled, (
            "Float8 MoE training prototype does not yet support context parallelism"
        )
        self.enabled = True

    def convert(self, model: nn.Module) -> list[str]:
        """Switches the matching GroupedExperts to fp8; returns their names."""
        return _mark_experts(model, self.fqns, "float8")

    def post_optimizer_hook(self, model) -> None:
        pass


def _split_fqns(fqns: list[str] | str) -> list[str]:
    return [f for f in fqns.split(",") if f] if isinstance(fqns, str) else list(fqns)


# how GroupedExperts multiply; the last two take no other beside them
_RECIPES = ("float8", "mxfp8", "mxfp4", "ckpt8")
_ALONE = ("mxfp4", "ckpt8")


def _mark_experts(model: nn.Module, fqns: list[str], attr: str) -> list[str]:
    matching = {}  # a module that several names share: under the first that matches
    for name, mod in model.named_modules(remove_duplicate=False):
        if isinstance(mod, GroupedExperts) and any(f in name for f in fqns):
            matching.setdefault(mod, name)
    for mod, name in matching.items():
        others = [r for r in _RECIPES if r != attr and getattr(mod, r)]
        if others and (attr in _ALONE or any(r in _ALONE for r in others)):
            raise ValueError(f"{name} is already converted to {others[0]}: {attr} experts are a recipe of their own")
    for mod in matching:
        setattr(mod, attr, True)
    return list(matching.values())


def _replace(model: nn.Module, matching: list[tuple[str, nn.Module]], make: Callable) -> list[str]:
    """Puts make(module) in the place of each of the (name, module), one for a module that several names
    share; returns the names. All are made before the first is put in place, so that one that cannot be
    (its weights are not on the GPU, the memory is spent) leaves the model as it was."""
    made = {}
    for _name, mod in matching:
        if mod not in made:
            made[mod] = make(mod)
    for name, mod in matching:
        parent, _, child = name.rpartition(".")
        setattr(model.get_submodule(parent), child, made[mod])
    return [name for name, _mod in matching]


class MXFP8Converter(Configurable):
    """MXFP8 grouped GEMMs for the matching experts (torchao's
    MXFP8TrainingOpConfig.from_recipe(MXFP8TrainingRecipe(recipe_name)) in the
    reference, mx.py:85-128). The kernels take ragged token groups, so no
    padding of the routed rows is needed without expert parallelism either."""

    RECIPES = ("mxfp8_rceil",)

    @dataclass(kw_only=True, slots=True)
    class Config(Configurable.Config):
        recipe_name: str = "mxfp8_rceil"
        fqns: list[str] | str = field(default_factory=list)

    def __init__(self, config: Config, *, parallel_dims, model_compile_enabled: bool):
        """Checks as mx.py:51-80 does: the hardware (block-scaled MFMA, gfx950
        here, SM100 there), then the recipe. Ragged token groups need no
        padding in these kernels, with or without expert parallelism."""
        self.enabled = False
        assert has_gfx950(), "MXFP8 is only supported on gfx950 (MI355X)"
        if config.recipe_name not in self.RECIPES:
            raise ValueError(f"unknown MXFP8 recipe {config.recipe_name!r}; options: {list(self.RECIPES)}")
        if not model_compile_enabled:
            logger.info("MXFP8 MoE: the grouped GEMMs are hand-written kernels; compile is not needed for speed")
        self.recipe_name = config.recipe_name
        self.fqns = _split_fqns(config.fqns)
        self.pad_token_groups_for_grouped_mm = not parallel_dims.ep_enabled
        self.config = config
        self.enabled = True

    def convert(self, model: nn.Module) -> list[str]:
        """Switches the matching GroupedExperts to MXFP8; returns their names."""
        if not self.enabled:
            return []
        return _mark_experts(model, self.fqns, "mxfp8")

    def post_optimizer_hook(self, model) -> None:
        pass


_PACKED = {GroupedExperts: MXFP4GroupedExperts, GptOssGroupedExperts: MXFP4GptOssGroupedExperts}
_INT8 = {GroupedExperts: Int8GroupedExperts.from_experts, GptOssGroupedExperts: Int8GptOssGroupedExperts.from_experts,
         FeedForward: Int8FeedForward.from_feed_forward, Linear: Int8Linear.from_linear}


class _ExpertsConverter(Configurable):
    """Marks the matching GroupedExperts; needs the hardware's block-scaled formats. The kernels
    take ragged token groups, so nothing is padded."""

    attr: str

    @dataclass(kw_only=True, slots=True)
    class Config(Configurable.Config):
        fqns: list[str] | str = field(default_factory=list)

    def __init__(self, config: Config, *, parallel_dims, model_compile_enabled: bool):
        if not has_gfx950():
            raise ValueError(f"{type(self).__name__} is only supported on gfx950 (MI355X)")
        self.fqns = _split_fqns(config.fqns)
        self.config = config

    def _matches(self, name: str) -> bool:
        return bool(name) and any(f in name for f in self.fqns)

    def convert(self, model: nn.Module) -> list[str]:
        """Switches the matching GroupedExperts; returns their names. Matching experts of other
        classes, which have no such recipe, are refused."""
        for name, mod in model.named_modules(remove_duplicate=False):
            if self._matches(name) and isinstance(mod, (GptOssGroupedExperts, *_PACKED.values(),
                                                             Int8GroupedExperts, Int8GptOssGroupedExperts)):
                raise ValueError(f"{name}: {type(mod).__name__} cannot be converted to {self.attr}")
        return _mark_experts(model, self.fqns, self.attr)

    def post_optimizer_hook(self, model) -> None:
        pass


class MXFP4Converter(_ExpertsConverter):
    """MXFP4 grouped GEMMs for the matching experts in training: every operand of the forward
    products in 4 bits, gradients straight through (ops.grouped_swiglu_mxfp4_train)."""

    attr = "mxfp4"

    @dataclass(kw_only=True, slots=True)
    class Config(_ExpertsConverter.Config):
        pass


class MXFP8ActivationCheckpointConverter(_ExpertsConverter):
    """bf16 grouped GEMMs whose x, gate and up are kept for the backward in MXFP8 instead of
    bf16 (ops.grouped_swiglu_ckpt8): (D + 2H) 33/32 bytes a routed row instead of 2D + 6H."""

    attr = "ckpt8"

    @dataclass(kw_only=True, slots=True)
    class Config(_ExpertsConverter.Config):
        pass


class MXFP4WeightConverter(_ExpertsConverter):
    """Inference on weights packed in MXFP4: replaces the matching GroupedExperts and
    GptOssGroupedExperts by MXFP4GroupedExperts / MXFP4GptOssGroupedExperts, which hold their
    packed weights in place of the parameters (17/32 of a byte per weight) and take no gradients."""

    @dataclass(kw_only=True, slots=True)
    class Config(_ExpertsConverter.Config):
        pass

    def convert(self, model: nn.Module) -> list[str]:
        """Replaces the matching experts; returns their names. Subclasses, which may compute something
        else, and modules with hooks, which would not see the calls any more, are refused."""
        matching = [(name, mod) for name, mod in model.named_modules(remove_duplicate=False)
                    if self._matches(name) and isinstance(mod, tuple(_PACKED))]
        for name, mod in matching:
            if type(mod) not in _PACKED:
                raise ValueError(f"{name}: the subclass {type(mod).__name__} has no packed form")
            if mod._forward_hooks or mod._forward_pre_hooks or mod._backward_hooks or mod._backward_pre_hooks:
                raise ValueError(f"{name} has hooks, which its packed form would not run: register them after packing")
        return _replace(model, matching, lambda mod: _PACKED[type(mod)].from_experts(mod))


def _hooked(mod: nn.Module) -> bool:
    return bool(mod._forward_hooks or mod._forward_pre_hooks or mod._backward_hooks or mod._backward_pre_hooks)


class Int8WeightConverter(_ExpertsConverter):
    """Inference on 8-bit integers: replaces the matching GroupedExperts, GptOssGroupedExperts,
    FeedForward and Linear by Int8GroupedExperts, Int8GptOssGroupedExperts, Int8FeedForward and
    Int8Linear, which hold codes and a scale per output channel in place of the parameters, quantize
    their inputs by rows and take no gradients. A FeedForward is replaced as a whole, and a router's
    gate, which decides where tokens go, is left as it is."""

    @dataclass(kw_only=True, slots=True)
    class Config(_ExpertsConverter.Config):
        pass

    def convert(self, model: nn.Module) -> list[str]:
        """Replaces the matching modules; returns their names. Refused are subclasses, which may compute
        something else, modules with hooks, which would not see the calls any more, feed-forwards
        with biases, and experts that are marked for another recipe."""
        kept = set()  # what belongs to a router
        for mod in model.modules():
            if isinstance(mod, TokenChoiceTopKRouter):
                kept.update(mod.modules())
        matching, whole = [], set()  # whole: the names replaced so far, whose parts (which may have other names too) go with them
        for name, mod in model.named_modules(remove_duplicate=False):
            if (self._matches(name) and isinstance(mod, tuple(_INT8)) and mod not in kept
                    and name.rpartition(".")[0] not in whole):
                self._check(name, mod)
                matching.append((name, mod))
                whole.add(name)
        return _replace(model, matching, lambda mod: _INT8[type(mod)](mod))

    @staticmethod
    def _check(name: str, mod: nn.Module) -> None:
        for part in (mod, *mod.children()):
            if type(part) not in _INT8:
                raise ValueError(f"{name}: the subclass {type(part).__name__} has no form on 8-bit integers")
            if _hooked(part):
                raise ValueError(f"{name} has hooks, which its form on 8-bit integers would not run: register them after "
                                 "converting")
        if isinstance(mod, FeedForward) and any(lin.bias is not None for lin in mod.children()):
            raise ValueError(f"{name}: a feed-forward with biases has no form on 8-bit integers")
        marked = [r for r in _RECIPES if getattr(mod, r, False)]
        if marked:
            raise ValueError(f"{name} is already converted to {marked[0]}")
        for part, p in mod.named_parameters():
            if "bias" in part:
                continue
            if p.dtype not in (torch.bfloat16, torch.float32):
                raise TypeError(f"{name}: 8-bit weights are made of bfloat16 and float32, {part} is {p.dtype}")
            if p.shape[-1] % ops.INT8_MULTIPLE or not ops.INT8_MULTIPLE <= p.shape[-1] <= ops.INT8_MAX_K:
                raise ValueError(f"{name}: 8-bit weights take contractions that are multiples of {ops.INT8_MULTIPLE} up to "
                                 f"{ops.INT8_MAX_K}, {part} is {list(p.shape)}")
            *experts, n, _k = _local(p).shape
            if not 1 <= n <= ops.INT8_MAX_N:
                raise ValueError(f"{name}: 8-bit weights take 1 to {ops.INT8_MAX_N} output channels, {part} is {list(p.shape)}")
            if experts and not 1 <= experts[0] <= ops.MAX_GEMM_EXPERTS:
                raise ValueError(f"{name}: 8-bit weights take 1 to {ops.MAX_GEMM_EXPERTS} experts, {part} is {list(p.shape)}")
        if isinstance(mod, FeedForward):
            w1, w2, w3 = (list(lin.weight.shape) for lin in (mod.w1, mod.w2, mod.w3))
            if w3 != w1 or w2 != w1[::-1]:
                raise ValueError(f"{name}: 8-bit weights take w1 and w3 of [H, D] and w2 of [D, H], got {w1}, {w3} and {w2}")


def find_pad_multiple(converters: list) -> int | None:
    """Token-group pad multiple needed by the configured quantized grouped GEMMs."""
    for c in converters:
        if isinstance(c, Float8GroupedMMConverter.Config):
            return PAD_MULTIPLE_MAP["float8"]
        if isinstance(c, MXFP8Converter.Config):
            return PAD_MULTIPLE_MAP["mxfp8"]
    return None
