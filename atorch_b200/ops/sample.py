"""The next token of every sequence: temperature, top-k, top-p and min-p, drawn with given random numbers (csrc/sample.cu)."""
from __future__ import annotations

import functools
import math
import struct
from typing import Tuple, Union

import torch
from torch.autograd import forward_ad

from .. import _lib
from .function import refuse_gradient

Number = Union[float, int, torch.Tensor]
# tokens of a vocabulary that the kernel takes with top-k or top-p (its counts have room for so many), and without
MOST, LARGEST = 1 << 19, 1 << 30


def sample_reference(logits, waiting, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """In 64 bits: what lies next to a border of the filters, and tokens that arrive at nearly the same time, depend on it."""
    V = logits.shape[1]
    if logits.shape[0] == 0:
        return logits.new_empty(0, dtype=torch.int64), logits.new_empty(0, dtype=torch.float32)
    T, k, p, m = (torch.as_tensor(v, dtype=torch.float64, device=logits.device).expand(logits.shape[0]).unsqueeze(1)
                  for v in (temperature, top_k, top_p, min_p))
    m = torch.where(m > 1, torch.ones_like(m), m)
    x = logits.double()
    x = torch.where(torch.isnan(x), torch.full_like(x, -math.inf), x)
    top = x.amax(-1, keepdim=True)
    best = (x == top).double().argmax(-1, keepdim=True)                    # the lowest of the largest
    below = torch.where(x == top, torch.zeros_like(x), x - top)
    w = torch.where((x > -math.inf) & (below > -math.inf), torch.exp(below / T), torch.zeros_like(x))
    at = torch.arange(V, device=x.device).expand_as(x)
    w = torch.where(T > 0, w, ((at == best) & (top > -math.inf)).double())
    if not bool(((k > 0) | (p < 1)).any()):                                # min-p alone needs no order
        w = torch.where(w < m, torch.zeros_like(w), w)
    else:
        order = x.sort(dim=-1, descending=True, stable=True).indices
        sorted_w = w.gather(1, order)
        left = ~(sorted_w < m)
        sorted_w = torch.where((k > 0) & (at >= k), torch.zeros_like(w), sorted_w)
        sums = sorted_w.cumsum(-1)
        left = left & (~(p < 1) | (sums - sorted_w < p * sums[:, -1:]) | (at == 0))
        w = torch.zeros_like(w).scatter(1, order, torch.where(left, sorted_w, torch.zeros_like(w)))
    wait = waiting.double()
    wait = torch.where(wait >= 0, wait.abs(), torch.full_like(wait, math.inf))          # (-0 is no time, as 0 is)
    score = torch.where(w > 0, w / wait, torch.full_like(w, -1.0))
    first = torch.where(score == score.amax(-1, keepdim=True), at, torch.full_like(at, V)).amin(-1)
    logprobs = torch.log(w.gather(1, first[:, None])[:, 0] / w.sum(-1))
    return first, torch.where(top[:, 0] > -math.inf, logprobs, torch.full_like(logprobs, -math.inf)).float()


def _number(name: str, v: Number, B: int, dev: int, whole: bool, low: float, high: float):
    """A parameter as the launcher takes it: the tensor whose address it gets (None: the same for all rows), and its number."""
    if isinstance(v, torch.Tensor) and v.dim() > 0:
        kinds = (torch.int32, torch.int64) if whole else (torch.float32, torch.float64)
        if v.dtype not in kinds or v.shape != (B,):
            raise ValueError(f"{name}: a number, or {'whole numbers' if whole else 'fp32'} ({B},), got {v.dtype} {tuple(v.shape)}")
        if v.get_device() != dev:
            raise ValueError(f"{name} is on {v.device}, and the logits are on {'the CPU' if dev < 0 else f'cuda:{dev}'}")
        if whole and v.dtype is torch.int64:
            v = v.clamp(-1, MOST)
        return v.to(torch.int32 if whole else torch.float32).contiguous(), 0
    v = v.item() if isinstance(v, torch.Tensor) else v
    if whole and v != int(v):
        raise ValueError(f"{name} is a whole number, got {v}")
    if not low <= v <= high:
        raise ValueError(f"{name} lies in [{low}, {high}], got {v}")
    return None, int(v) if whole else float(v)


@functools.lru_cache(maxsize=256)
def _bits(v: float) -> int:
    """A number of 64 bits as the launcher takes it."""
    return struct.unpack("q", struct.pack("d", v))[0]


def sample(logits: torch.Tensor, waiting: torch.Tensor, temperature: Number = 1.0, top_k: Number = 0, top_p: Number = 1.0,
           min_p: Number = 0.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """A token of every row of ``logits`` ``[B, V]`` (bf16, fp16 or fp32) and the logarithm of the probability that it was drawn with:
    int64 and fp32 ``[B]``. With ``top_k`` or ``top_p`` a vocabulary has 2 ** 19 tokens at most.

    A token's weight is ``exp((logit - largest logit) / temperature)`` (with a filter, below ``2 ** -1000`` it may count as none); tokens are ordered by weight, equal ones by index. ``top_k`` leaves
    that many first ones (0: all), ``top_p`` of what these weigh together the first ones whose predecessors weigh less than that
    share, ``min_p`` those of at least that weight, which the first always has. ``waiting`` (fp32 ``[B, V]``, exponentially distributed:
    ``torch.empty(...).exponential_()``) are the random numbers: the token is the first to arrive, that with the largest
    ``weight / waiting`` of those left (equal ones: the lowest index). So a token is drawn with its share of the weight that is left. A
    temperature of 0 takes the largest logit, the lowest index of equal ones, with probability 1.

    Every parameter is a number or a tensor with one for each row, fp32 (``top_k``: int32 or int64). Numbers out of range are refused; in
    a tensor, which is not looked at on the host, a temperature that is not positive counts as 0, ``top_k`` below 1 as 0, ``top_p``
    above 1 or NaN as 1 and below 0 as 0 (the first token alone),
    ``min_p`` above 1 as 1, NaN as 0.

    A NaN logit counts as ``-inf``; of logits of ``+inf`` each weighs 1 and all others nothing; where every logit is ``-inf`` the token
    is 0 and the logarithm ``-inf``. A waiting time below 0 or NaN counts as infinite."""
    if logits.dim() != 2 or logits.dtype not in _lib.DT or logits.shape[1] == 0:
        raise ValueError(f"logits are bf16, fp16 or fp32 [B, vocabulary], got {logits.dtype} {tuple(logits.shape)}")
    B, V = logits.shape
    if V > LARGEST:
        raise ValueError(f"a vocabulary of {V}: 2 ** 30 at most")
    if waiting.dtype is not torch.float32 or waiting.shape != (B, V):
        raise ValueError(f"waiting is fp32 {(B, V)}, got {waiting.dtype} {tuple(waiting.shape)}")
    dev = logits.get_device()
    if waiting.get_device() != dev:
        raise ValueError("logits and waiting are on several devices")
    t_rows, t = _number("temperature", temperature, B, dev, False, 0.0, math.inf)
    k_rows, k = _number("top_k", top_k, B, dev, True, 0, float(1 << 62))
    p_rows, p = _number("top_p", top_p, B, dev, False, 0.0, 1.0)
    m_rows, m = _number("min_p", min_p, B, dev, False, 0.0, 1.0)
    if V > MOST and (k_rows is not None or p_rows is not None or k > 0 or p < 1):
        raise ValueError(f"a vocabulary of {V}: 2 ** 19 at most with top_k or top_p")
    if logits.requires_grad or waiting.requires_grad or forward_ad._current_level >= 0:
        refuse_gradient("a draw has no gradient: call under torch.no_grad()", logits, waiting)
    if dev < 0 or not _lib.use_kernels(logits):
        return sample_reference(logits, waiting, *(v if rows is None else rows for rows, v in ((t_rows, t), (k_rows, k), (p_rows, p),
                                                                                               (m_rows, m))))
    step, one = logits.stride()
    if one != 1 and V > 1:
        logits, step = logits.contiguous(), V
    wait_step, one = waiting.stride()
    if one != 1 and V > 1:
        waiting, wait_step = waiting.contiguous(), V
    tokens = torch.empty(B, dtype=torch.int64, device=logits.device)
    logprobs = torch.empty(B, dtype=torch.float32, device=logits.device)
    rc = _lib.lib().atb_sample(logits.data_ptr(), waiting.data_ptr(), _lib.addr(t_rows), _lib.addr(k_rows), _lib.addr(p_rows),
                               _lib.addr(m_rows), tokens.data_ptr(), logprobs.data_ptr(), B, V, step, wait_step, _bits(t), _bits(p),
                               _bits(m), min(k, V),
                               _lib.DT[logits.dtype], _lib.stream_of(dev), _lib.status_addr(logits))
    _lib.check(rc, "atb_sample")
    return tokens, logprobs
