"""Group norm with an activation behind it, for channels-last maps: the layers of a label head on the FPN levels, which leave the
encoder 256 channels wide.  One statistics pass and one pass that normalises, scales and activates (`lsam_group_norm_act_fwd`); the
backward recomputes the activation's argument from x instead of keeping it (`lsam_group_norm_act_bwd`)."""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn

from . import heads_autograd as HA
from . import ops
from ._C import LsamError


def group_norm_act(x: torch.Tensor, num_groups: int, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
                   eps: float = 1e-5, act: str = "none") -> torch.Tensor:
    """act(F.group_norm(x, num_groups, weight, bias, eps)) for x [N, C, *spatial] (float32 or bfloat16) laid out channels last; `act`
    is "none", "relu", "silu" or "gelu" (the erf form; bfloat16 maps: from a polynomial, off by less than 1.5e-7 |h|). Statistics,
    parameters and their gradients are fp32; the result has x's type and is channels last without gaps. x may be a channel slice of a
    wider channels-last map; any other layout (an NCHW map of the neck) is copied to channels last first. At most 8192 channels, fewer
    than 2^20 samples and 2^24 groups in all."""
    if not x.is_cuda:
        raise LsamError("group_norm_act runs on the MI355X only (no CPU or PyTorch fallback)")
    if x.dim() < 2 or x.dtype not in (torch.float32, torch.bfloat16):
        raise LsamError(f"group_norm_act: [N, C, *] in float32 or bfloat16, got {tuple(x.shape)} {x.dtype}")
    if num_groups < 1 or x.shape[1] < 1 or x.shape[1] % num_groups:
        raise LsamError(f"group_norm_act: {x.shape[1]} channels do not make {num_groups} groups")
    if act not in ops.ACTIVATIONS:
        raise LsamError(f"group_norm_act: activation {act!r}; one of {sorted(ops.ACTIVATIONS)}")
    for t, name in ((weight, "weight"), (bias, "bias")):
        if t is not None and (t.shape != x.shape[1:2] or not t.is_floating_point()):
            raise LsamError(f"group_norm_act: {name} {tuple(t.shape)} {t.dtype} does not match {x.shape[1]} channels")
    if not (x.dim() == 4 and x.is_contiguous(memory_format=torch.channels_last)) and ops.channels_last_rows(x) is None:
        x = x.movedim(1, -1).contiguous().movedim(-1, 1)
    if HA.no_derivative(x, weight, bias):
        return ops.group_norm_act_fwd(x, int(num_groups), weight, bias, float(eps), act)
    return HA.GroupNormActFn.apply(x, weight, bias, int(num_groups), float(eps), act)


class GroupNormAct(nn.GroupNorm):
    """nn.GroupNorm (same constructor, parameters and state_dict keys) with the activation fused behind it, channels last."""

    def __init__(self, num_groups: int, num_channels: int, eps: float = 1e-5, affine: bool = True, device=None, dtype=None, act: str = "none"):
        super().__init__(num_groups, num_channels, eps, affine, device, dtype)
        if act not in ops.ACTIVATIONS:
            raise LsamError(f"GroupNormAct: activation {act!r}; one of {sorted(ops.ACTIVATIONS)}")
        self.act = act

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return group_norm_act(x, self.num_groups, self.weight, self.bias, self.eps, self.act)

    def extra_repr(self) -> str:
        return f"{super().extra_repr()}, act={self.act}"
