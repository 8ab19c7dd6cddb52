"""Linear layers with 8-bit block-scaled weights, the format of FP8 checkpoints: e4m3 values [N, K] and one fp32
scale per 128 x 128 block, activations quantised per token and 128 channels in the layer
(``ops.fp8_linear``).  The attributes carry the checkpoints' names (``weight``, ``weight_scale_inv``,
``bias``), so such a state_dict loads unchanged; weight and scales keep their types when a model is moved to
another one.  Inference only.

No counterpart in the reference, which calls the model library's own FP8 layers (its patch is "FP8-safe" by
reusing them by reference, qwen_routed_attention.py:94-156).
"""
from __future__ import annotations

from typing import Optional, Sequence, Tuple

import torch
import torch.nn as nn

from . import _lib, ops


class Fp8Linear(nn.Module):
    """y = x w^T + b with an e4m3 weight and 128 x 128 block scales."""

    def __init__(self, in_features: int, out_features: int, bias: bool = False,
                 bias_dtype: torch.dtype = torch.bfloat16, device=None) -> None:
        super().__init__()
        self.in_features, self.out_features = in_features, out_features
        blk = ops.FP8_BLOCK
        self.register_buffer("weight", torch.zeros(out_features, in_features, device=device).to(torch.float8_e4m3fn))
        self.register_buffer("weight_scale_inv", torch.ones(-(-out_features // blk), -(-in_features // blk), device=device))
        self.register_buffer("bias", torch.zeros(out_features, dtype=bias_dtype, device=device) if bias else None)

    @classmethod
    def from_linear(cls, lin: nn.Linear) -> "Fp8Linear":
        """Quantise an ``nn.Linear`` (128 x 128 blocks, amax / 448)."""
        m = cls(lin.in_features, lin.out_features, lin.bias is not None, lin.weight.dtype, lin.weight.device)
        m.weight, m.weight_scale_inv = ops.fp8_quantize_weight(lin.weight.detach())
        if lin.bias is not None:
            m.bias = lin.bias.detach().clone()
        return m

    def _apply(self, fn, recurse: bool = True):
        # moves of a model reach its layers through here: devices apply to the weight and its scales, a type
        # (model.bfloat16(), .half(), .to(dtype)) to the bias alone
        held = (self.weight, self.weight_scale_inv)

        def keep(t: torch.Tensor) -> torch.Tensor:
            if any(t is h for h in held):
                probe = fn(t.new_empty(0))
                if probe.dtype != t.dtype:
                    return t.to(probe.device)
            return fn(t)

        return super()._apply(keep, recurse)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return ops.fp8_linear(x, self.weight, self.weight_scale_inv, bias=self.bias)


def fp8_weight_of(m: nn.Module) -> Optional[Tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor]]]:
    """(weight, scales, bias) of a layer that already holds an e4m3 weight with 128 x 128 fp32 block scales
    (``Fp8Linear``, the model library's block-scaled FP8 layers), else None."""
    w, s = getattr(m, "weight", None), getattr(m, "weight_scale_inv", None)
    if w is None or s is None or w.dtype != torch.float8_e4m3fn or w.dim() != 2:
        return None
    blk = ops.FP8_BLOCK
    if tuple(s.shape) != (-(-w.shape[0] // blk), -(-w.shape[1] // blk)):
        return None
    bias = getattr(m, "bias", None)
    return w.detach().contiguous(), s.detach().float().contiguous(), None if bias is None else bias.detach().contiguous()


def fp8_concat(mods: Sequence[nn.Module]) -> Optional[Tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor]]]:
    """One (weight, scales, bias) for layers that share their input, so that they run as one product: 8-bit
    layers as they are, plain ``nn.Linear`` layers quantised.  None when a layer is neither, or when a layer but
    the last ends inside a 128-feature block (its scales would not line up).  A single 8-bit layer's tensors
    come as they are, without a copy."""
    parts = []
    for i, m in enumerate(mods):
        p = fp8_weight_of(m)
        if p is None and type(m) is nn.Linear:
            p = (*ops.fp8_quantize_weight(m.weight.detach()), None if m.bias is None else m.bias.detach())
        if p is None or (i + 1 < len(mods) and p[0].shape[0] % ops.FP8_BLOCK):
            return None
        parts.append(p)
    if len({p[0].shape[1] for p in parts}) != 1:
        raise _lib.HgaError("fp8_concat: the layers differ in their input's width")
    if len(parts) == 1:
        return parts[0]
    bias = None
    if any(p[2] is not None for p in parts):
        dt = next(p[2].dtype for p in parts if p[2] is not None)
        bias = torch.cat([p[2] if p[2] is not None else torch.zeros(p[0].shape[0], device=p[0].device, dtype=dt)
                          for p in parts]).contiguous()
    w = torch.cat([p[0].view(torch.uint8) for p in parts]).view(torch.float8_e4m3fn)
    return w.contiguous(), torch.cat([p[1] for p in parts]).contiguous(), bias


__all__ = ["Fp8Linear", "fp8_concat", "fp8_weight_of"]
