"""Linear modules whose weights are held in 4 bits: for frozen models that only run forward (rollouts, reference and reward
models, evaluation)."""
from __future__ import annotations

from typing import Callable, Optional

import torch
import torch.nn as nn

from ..ops.w4 import w4_linear, w4_quantize


class W4Linear(nn.Module):
    """``x @ W.T + bias`` on :func:`~atorch_b200.ops.w4_linear`; codes and scales are buffers."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, in_features: int, group_size: int = 128,
                 bias: Optional[torch.Tensor] = None):
        super().__init__()
        self.in_features, self.out_features, self.group_size = in_features, codes.shape[0], group_size
        self.register_buffer("codes", codes)
        self.register_buffer("scales", scales)
        self.register_buffer("bias", bias)

    def _apply(self, fn, recurse: bool = True):
        scales = self.scales
        super()._apply(fn, recurse)
        if self.scales.dtype is not scales.dtype:      # the model is cast: scales stay what the codes were taken for
            self.scales = scales.to(self.codes.device)
        return self

    @classmethod
    def from_linear(cls, linear: nn.Linear, group_size: int = 128) -> "W4Linear":
        codes, scales = w4_quantize(linear.weight, group_size)
        return cls(codes, scales, linear.in_features, group_size, None if linear.bias is None else linear.bias.detach().clone())

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return w4_linear(x, self.codes, self.scales, self.group_size, self.bias)

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, group_size={self.group_size}"


def quantize_linears(model: nn.Module, group_size: int = 128, wanted: Optional[Callable[[str, nn.Linear], bool]] = None) -> nn.Module:
    """Replace the ``nn.Linear`` modules of ``model`` (those that ``wanted(name, module)`` picks) by :class:`W4Linear`, in place. A
    weight that is shared with another module (a tied head) is left alone."""
    seen: dict = {}
    for m in model.modules():
        for p in m._parameters.values():
            if p is not None:
                seen[p] = seen.get(p, 0) + 1
    for name, m in list(model.named_modules()):
        for child, lin in list(m.named_children()):
            full = f"{name}.{child}" if name else child
            if type(lin) is nn.Linear and seen[lin.weight] == 1 and (wanted is None or wanted(full, lin)):
                setattr(m, child, W4Linear.from_linear(lin, group_size))
    return model
