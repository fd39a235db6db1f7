"""Linear layers whose weights are held in 4 bits with a scale per group of columns (csrc/w4.cu).

``codes`` uint8 ``[N, 16 * ceil(K / 32)]``: byte ``i`` of a row holds column ``2 i`` in its low half and ``2 i + 1`` in its high one,
rows are filled up with 8s. ``scales`` bf16 ``[N, ceil(K / group)]``. A weight is ``(code - 8) * scale``: codes run from 1 to 15 as
:func:`w4_quantize` makes them, and 0 stands for -8.

For frozen weights (rollouts, reference and reward models): there is no gradient, and a tensor that asks for one is refused.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad

from .. import _lib
from .function import refuse_gradient
from .gemm import gemm

GROUPS = (32, 64, 128)
_LOW = {torch.bfloat16: 0, torch.float16: 1}
# Rows of x from which the weights are expanded to bf16 and multiplied by the GEMM, with bf16 x and K a multiple of 8. The kernel for few
# rows keeps the weights exact (up to 12 bits; bf16 has 8), so it stays until it is the slower one. Kernel, expansion and GEMM, in us:
#    outputs x inputs      33 rows      65 rows      96 rows     128 rows     256 rows
#    22016 x 4096         58,  95      89,  95      97,  95     125,  97     240, 106
#    4096 x 11008         34,  94      58,  94      71,  94      64,  95     121,  65
#    2048 x 2048          10,  18      10,  17      10,  17      10,  18      17,  17
EXPAND_ROWS = 97


def w4_quantize(weight: torch.Tensor, group_size: int = 128) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(codes, scales)`` of a ``[N, K]`` weight: the scale of a group is its largest magnitude over 7, rounded to bf16, and a code
    the nearest one of that scale."""
    _check_group(group_size)
    if weight.dim() != 2 or not weight.is_floating_point() or weight.shape[1] == 0:
        raise ValueError(f"a [N, K] weight is wanted, got {weight.dtype} {tuple(weight.shape)}")
    N, K = weight.shape
    groups, columns = -(-K // group_size), -(-K // 32) * 32
    w = torch.zeros(N, groups * group_size, dtype=torch.float32, device=weight.device)
    w[:, :K] = weight.detach()
    w = w.view(N, groups, group_size)
    scales = (w.abs().amax(-1) * (1 / 7)).to(torch.bfloat16)
    s = scales.float().unsqueeze(-1)
    code = torch.where(s > 0, torch.round(w / s).clamp(-7, 7), torch.zeros_like(w)).nan_to_num().add_(8).to(torch.uint8)
    code = torch.nn.functional.pad(code.view(N, -1), (0, max(0, columns - groups * group_size)), value=8)[:, :columns]
    return (code[:, 0::2] | (code[:, 1::2] << 4)).contiguous(), scales


def w4_dequantize(codes: torch.Tensor, scales: torch.Tensor, in_features: int, group_size: int = 128,
                  dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The ``[N, in_features]`` weight that codes and scales stand for."""
    _check(codes, scales, in_features, group_size)
    w = torch.stack([codes & 15, codes >> 4], -1).flatten(1)[:, :in_features].float() - 8
    return (w * scales.float().repeat_interleave(group_size, 1)[:, :in_features]).to(dtype)


def _check_group(group_size: int) -> None:
    if group_size not in GROUPS:
        raise ValueError(f"group_size is one of {GROUPS}, got {group_size}")


def _check(codes, scales, K, group_size) -> int:
    """Rows of a weight of K columns."""
    if group_size not in GROUPS:
        _check_group(group_size)
    shape = codes.shape
    N = shape[0] if len(shape) == 2 else -1
    if codes.dtype is not torch.uint8 or scales.dtype is not torch.bfloat16 or K < 1 or shape[1:] != ((K + 31) // 32 * 16,) \
            or scales.shape != (N, (K + group_size - 1) // group_size):
        raise ValueError(f"codes {codes.dtype} {tuple(shape)} and scales {scales.dtype} {tuple(scales.shape)} are not a "
                         f"weight of {K} columns in groups of {group_size}")
    if not (codes.is_contiguous() and scales.is_contiguous()):
        raise ValueError("codes and scales have to be contiguous")
    return N


def w4_linear_reference(x, codes, scales, group_size=128, bias=None):
    y = x.float() @ w4_dequantize(codes, scales, x.shape[-1], group_size).t()
    return (y if bias is None else y + bias.float()).to(x.dtype)


def w4_linear(x: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, group_size: int = 128,
              bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x @ W.T (+ bias)`` for ``x`` ``[..., K]`` in bf16 or fp16 and the weight that ``codes`` and ``scales`` stand for; sums in
    fp32, the result in the type of ``x``. Made for the few rows of a decode step; many bf16 rows expand the weight for the call and
    run the GEMM (the weight is rounded to bf16 there)."""
    shape, kind = x.shape, _LOW.get(x.dtype)
    K, N = shape[-1], _check(codes, scales, shape[-1], group_size)
    if kind is None:
        raise ValueError(f"x is bf16 or fp16, got {x.dtype}")
    dev = x.get_device()
    if bias is not None:
        if bias.dtype is not x.dtype or bias.shape != (N,):
            raise ValueError(f"bias is {x.dtype} [{N}], got {bias.dtype} {tuple(bias.shape)}")
        if bias.get_device() != dev:
            raise ValueError(f"bias is on {bias.device}, and x on {x.device}")
        bias = bias.contiguous()
    if x.requires_grad or (bias is not None and bias.requires_grad) or forward_ad._current_level >= 0:
        refuse_gradient("4-bit weights have no gradient: call under torch.no_grad()", x, bias)
    if codes.get_device() != dev or scales.get_device() != dev:
        raise ValueError(f"x is on {x.device}, and its weights on {codes.device} and {scales.device}")
    if dev < 0:
        return w4_linear_reference(x, codes, scales, group_size, bias)
    x2 = x if len(shape) == 2 else x.reshape(x.numel() // K, K)
    M = x2.shape[0]
    step, one = x2.stride()
    if one != 1:
        x2, step = x2.contiguous(), K
    if codes.data_ptr() % 16:          # both kernels read them in words
        codes = codes.clone()
    if M >= EXPAND_ROWS and x.dtype is torch.bfloat16 and K % 8 == 0:
        if step < K or (x2.data_ptr() | 2 * step) & 15:
            x2 = x2.clone(memory_format=torch.contiguous_format)
        wide = (N + 7) // 8 * 8            # the GEMM stores 8 columns at a time; those behind the last are cut off
        w = torch.empty(wide, K, dtype=x.dtype, device=x.device)
        rc = _lib.lib().atb_w4_expand(codes.data_ptr(), scales.data_ptr(), w.data_ptr(), N, K, group_size, kind,
                                      _lib.stream_of(dev))
        _lib.check(rc, "atb_w4_expand")
        if bias is not None and wide != N:
            bias = torch.nn.functional.pad(bias, (0, wide - N))
        y = gemm(x2, w, bias=bias)
        return (y if wide == N else y[:, :N].contiguous()).view(*shape[:-1], N)
    y = x.new_empty(M, N) if x2 is x else x.new_empty(*shape[:-1], N)
    base = x2.data_ptr()
    rc = _lib.lib().atb_w4_linear(base, codes.data_ptr(), scales.data_ptr(), _lib.addr(bias), y.data_ptr(), M, N, K, group_size, step,
                                  int((base | 2 * step) & 15 == 0), kind, _lib.stream_of(dev), _lib.status_addr(x))
    _lib.check(rc, "atb_w4_linear")
    return y
