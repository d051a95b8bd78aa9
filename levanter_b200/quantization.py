"""Low-precision training configuration (the reference's ``haliax.quantization.QuantizationConfig`` reached through
``trainer.quantization``, src/levanter/trainer.py:648, config/gpt2_small_fast_fp8.yaml:17-18).

``fp8: true`` selects fp8 GEMMs for the Linear layers named by ``targets`` (all by default): e4m3 for forward operands,
e5m2 for output gradients.  ``scaling: tensor`` (default) uses one scale per tensor taken from a rolling history of absolute
maxima (delayed scaling, as in the reference); ``scaling: block`` uses one power-of-two scale per 32 values along the
contraction dimension, applied by the tensor core (``tcgen05.mma kind::mxf8f6f4.block_scale``).  ``block_size`` is accepted
for configs that name it; the hardware's block is 32 whatever it says.
``int8: true`` selects 8-bit integer products for the forward pass (``ops/int8.py``): one scale per token and per output channel, taken from the values
themselves, gradients from bf16 products, activations and weights kept for the backward pass in 8 bits.
``quantize_linear_layers`` swaps matching ``Linear`` modules for ``Fp8Linear`` or ``Int8Linear``;
master weights, optimizer state and checkpoints are unchanged.
``quantize_for_serving`` replaces the projections of attention layers and gated MLPs by ones that hold their weights in 8 bits (``int8: true``)."""
from __future__ import annotations

import re
from dataclasses import dataclass
from typing import List, Optional, Union

import torch
import torch.nn as nn


@dataclass(frozen=True)
class QuantizationConfig:
    targets: Union[None, List[str], str] = None
    amax_history_length: int = 1024
    compute_dtype: Optional[str] = None
    fp8: bool = False
    int8: bool = False
    block_size: int = 128
    scaling: str = "tensor"  # tensor | block

    def __post_init__(self):
        if self.fp8 and self.int8:
            raise ValueError("only one of fp8 / int8 can be enabled")
        if self.scaling not in ("tensor", "block"):
            raise ValueError(f"scaling must be 'tensor' or 'block', got {self.scaling!r}")

    def matches(self, name: str) -> bool:
        if self.targets is None:
            return True
        if isinstance(self.targets, str):
            return re.search(self.targets, name) is not None
        return any(t in name.split(".") or t == name for t in self.targets)


def quantize_linear_layers(model: nn.Module, config: QuantizationConfig) -> nn.Module:
    """Replace targeted ``Linear`` modules by their fp8 or int8 counterparts (in place; returns the model)."""
    if not (config.fp8 or config.int8):
        return model
    from .nn import Linear
    from .ops.fp8 import Fp8Linear
    from .ops.int8 import Int8Linear

    for name, mod in list(model.named_modules()):
        for child_name, child in list(mod.named_children()):
            full = f"{name}.{child_name}" if name else child_name
            if type(child) is Linear and config.matches(full) and "lm_head" not in full:
                if config.int8:
                    setattr(mod, child_name, Int8Linear.from_linear(child))
                    continue
                setattr(mod, child_name, Fp8Linear.from_linear(child, block=config.block_size, amax_history_length=config.amax_history_length,
                                                                     block_scaled=config.scaling == "block"))
    return model


def quantize_for_serving(model: nn.Module, config: QuantizationConfig) -> nn.Module:
    """Hold the weights of the targeted projections of ``Attention`` layers and ``LlamaMlp`` blocks (shared experts among them) in 8 bits, one scale per output channel
    (in place; returns the model).  Other layers stay as they are: routed experts, MLPs without a gate, other mixers, embeddings and head.  The
    model serves from then on: those weights are not parameters any more, and engines made of it before (their CUDA graphs read the old weights) are done.  A model that is quantised already comes back as it is."""
    if config.fp8:
        raise ValueError("serving holds weights in 8-bit integers: use QuantizationConfig(int8=True)")
    if not config.int8:
        return model
    from .layers.attention import Attention
    from .models.llama import LlamaMlp
    from .nn import Linear
    from .ops.int8 import Int8Linear, Int8ServingLinear

    held, found = 0, []
    for name, mod in model.named_modules():
        if not isinstance(mod, (Attention, LlamaMlp)):
            continue
        if mod.tp is not None and mod.tp.size > 1:
            raise ValueError(f"{name}: int8 serving weights are not split over tensor-parallel ranks")
        for child_name, child in mod.named_children():
            held += type(child) is Int8ServingLinear
            if type(child) in (Linear, Int8Linear) and config.matches(f"{name}.{child_name}"):
                Int8ServingLinear.check_weight(child.weight)
                found.append((mod, child_name))
    if held == 0 and not found:
        raise ValueError("no projection of an attention or MLP layer matches the quantization targets")
    for mod, child_name in found:  # (nothing has been replaced where one of them is refused)
        setattr(mod, child_name, Int8ServingLinear.from_linear(getattr(mod, child_name)))
    return model


def check_not_quantized(model: nn.Module, what: str) -> None:
    """Refuses ``what`` of a model that serves: weights held in 8 bits are not parameters, so it would pass them over."""
    from .ops.int8 import Int8ServingLinear

    for name, m in model.named_modules():
        if type(m) is Int8ServingLinear:
            raise ValueError(f"{what}: the weight of {name} is held in 8 bits; use the model as it was before quantize_for_serving")
