"""Paged key/value cache held in 4 bits: append with rotation, reading back, attention of the newest tokens.

A layer's cache is a pair ``(codes, scales)``: uint8 ``[pages, 2, kv_heads, page_size, head_dim / 2]`` (0: keys, 1: values; byte
``i`` holds dim ``2 i`` in its low half, ``2 i + 1`` in its high one) and bf16 ``[pages, kv_heads, page_size, 4]`` (scale and
minimum of the key, scale and minimum of the value). A value is ``code * scale + minimum``; each token has a scale and a minimum
per head, so a token and head take ``head_dim + 8`` bytes where bf16 takes ``4 * head_dim``. Row ``b`` of ``page_table`` (int32
``[sequences, pages of the longest]``) names the pages of sequence ``b``. Pages have a power of two of 16 or more tokens.

Positions, page numbers and lengths lie on the device. One that is out of range is skipped by the kernels and recorded in the
device's status word, which ``_lib.check_status`` raises; kernels of this package behind it store nothing until then.

These operators serve generation: they have no gradient, and refuse tensors that ask for one.
"""
from __future__ import annotations

import ctypes
import functools
import math
from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad

from .. import _lib
from .function import refuse_gradient

Layer = Tuple[torch.Tensor, torch.Tensor]
HEAD_DIMS = (64, 128)          # of the kernels; the CPU path takes any even one
WHOLE = 256                    # tokens up to which the kernel never cuts a sequence, and needs no workspace (csrc/kv4.cu)


class KV4Cache:
    """The 4-bit caches of ``layers`` layers over one pool of ``pages`` pages (one page table serves all layers)."""

    def __init__(self, layers: int, pages: int, page_size: int, kv_heads: int, head_dim: int, device=None):
        _check_page_size(page_size)
        self.codes = torch.zeros(layers, pages, 2, kv_heads, page_size, head_dim // 2, dtype=torch.uint8, device=device)
        self.scales = torch.zeros(layers, pages, kv_heads, page_size, 4, dtype=torch.bfloat16, device=device)
        self.page_size = page_size

    def layer(self, i: int) -> Layer:
        return self.codes[i], self.scales[i]


def _check_page_size(n: int) -> None:
    if n < 16 or n & (n - 1):
        raise ValueError(f"page_size has to be a power of two of 16 or more, got {n}")


def _cache(layer: Layer, page_table: torch.Tensor) -> Tuple[int, ...]:
    """A layer's cache and page table as the launchers take them, after the checks that all calls share: addresses of codes, scales
    and table, pages, kv_heads, page_shift, sequences, pages of a sequence, stride of the table; then head_dim and the index of the
    device (-1: the CPU)."""
    codes, scales = layer
    shape = codes.shape
    if codes.dtype is not torch.uint8 or scales.dtype is not torch.bfloat16 or len(shape) != 5 or shape[1] != 2 or 0 in shape:
        raise ValueError("a layer's cache is (uint8 [pages, 2, kv_heads, page_size, head_dim / 2], "
                         f"bf16 [pages, kv_heads, page_size, 4]), got {codes.dtype} {tuple(shape)} and {scales.dtype}")
    pages, _, kv_heads, page_size, half = shape
    if scales.shape != (pages, kv_heads, page_size, 4):
        raise ValueError(f"codes {tuple(shape)} and scales {tuple(scales.shape)} are not one cache")
    codes_at, scales_at, dev = codes.data_ptr(), scales.data_ptr(), codes.get_device()
    if not (codes.is_contiguous() and scales.is_contiguous()) or (codes_at | scales_at) & 15:
        raise ValueError("the cache has to be contiguous and begin on 16 bytes")
    if page_size < 16 or page_size & (page_size - 1):
        _check_page_size(page_size)
    steps = page_table.stride()
    if page_table.dtype is not torch.int32 or len(steps) != 2 or (steps[1] != 1 and page_table.shape[1] > 1):
        raise ValueError("page_table is int32 [sequences, pages], its rows contiguous")
    if dev >= 0 and half != 64 and half != 32:
        raise ValueError(f"head_dim {2 * half}: the kernels take {HEAD_DIMS}")
    if scales.get_device() != dev or page_table.get_device() != dev:
        _same_device(dev, scales, page_table)
    rows, width = page_table.shape
    if width * page_size > 0x7fffffff:
        raise ValueError(f"{width} pages of {page_size} tokens a sequence: positions have 31 bits")
    return (codes_at, scales_at, page_table.data_ptr(), pages, kv_heads, page_size.bit_length() - 1, rows, width, steps[0], 2 * half,
            dev)


def _same_device(dev: int, *tensors: Optional[torch.Tensor]) -> None:
    for t in tensors:
        if t is not None and t.get_device() != dev:
            raise ValueError(f"a tensor on {t.device}, and the cache on {dev if dev >= 0 else 'the CPU'}")


def _no_gradient(t: torch.Tensor) -> None:
    if t.requires_grad or forward_ad._current_level >= 0:
        refuse_gradient("the 4-bit cache has no gradient: call under torch.no_grad()", t)


def _int32(name: str, t: Optional[torch.Tensor], n: int) -> Optional[torch.Tensor]:
    if t is None or (t.dtype is torch.int32 and t.shape == (n,) and t.is_contiguous()):
        return t
    if t.dtype not in (torch.int32, torch.int64) or t.numel() != n:
        raise ValueError(f"{name}: {n} whole numbers are wanted, got {t.dtype} {tuple(t.shape)}")
    if t.dtype is torch.int64:       # what is out of range stays so
        t = t.clamp(-1 << 31, (1 << 31) - 1)
    return t.reshape(-1).to(torch.int32).contiguous()


def _aligned(t: torch.Tensor, row: int) -> bool:
    """Whether rows of ``t`` that are ``row`` elements apart can be read in 16-byte pieces."""
    return (t.data_ptr() | row * t.element_size()) & 15 == 0


# ------------------------------------------------------------------------------------------------------------------
def quantise_reference(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Codes (one a value), scale and minimum (as fp32) of the last dimension of an fp32 tensor."""
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    scale = ((high - low) * (1 / 15)).to(torch.bfloat16).float()
    low = low.to(torch.bfloat16).float()
    code = torch.where(scale > 0, torch.round((x - low) / scale).clamp(0, 15), torch.zeros_like(x))
    return torch.nan_to_num(code).to(torch.uint8), scale, low


def _places(page_table, seq, pos, page_size, T):
    b = torch.arange(T, device=pos.device) if seq is None else seq.long()
    at = pos.clamp(min=0).long()
    real = pos >= 0
    if bool(((b < 0) | (b >= page_table.shape[0]) | (at // page_size >= page_table.shape[1]))[real].any()):
        raise IndexError("a token lies outside the page table")
    page = page_table[b.clamp(0, page_table.shape[0] - 1), (at // page_size).clamp(max=page_table.shape[1] - 1)].long()
    return page, at % page_size, real


def kv4_append_reference(layer, page_table, seq, pos, qkv, n_q, cos=None, sin=None):
    codes, scales = layer
    _, _, KV, page_size, half = codes.shape
    D = 2 * half
    T = pos.numel()
    x = qkv.reshape(T, n_q + 2 * KV, D).float()
    page, slot, real = _places(page_table, seq, pos, page_size, T)
    turned = x[:, : n_q + KV]
    if cos is not None:
        at = pos.clamp(min=0).long()
        c, s = cos[at].unsqueeze(1), sin[at].unsqueeze(1)
        a, b = turned[..., :half], turned[..., half:]
        turned = torch.where(real[:, None, None], torch.cat([a * c - b * s, b * c + a * s], -1), turned)
    code, scale, low = quantise_reference(torch.stack([turned[:, n_q:], x[:, n_q + KV:]], 1))
    code = code[..., 0::2] | (code[..., 1::2] << 4)
    codes[page[real], :, :, slot[real]] = code[real]
    scales[page[real], :, slot[real]] = torch.cat([scale, low], -1).permute(0, 2, 1, 3).flatten(2)[real].to(torch.bfloat16)
    return turned[:, :n_q].to(qkv.dtype)


def kv4_append(layer: Layer, page_table: torch.Tensor, seq: Optional[torch.Tensor], pos: torch.Tensor, qkv: torch.Tensor,
               n_q: int, cos: Optional[torch.Tensor] = None, sin: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Put tokens into the cache. ``qkv`` ``[..., (n_q + 2 kv_heads) * head_dim]`` (or with heads and dims apart) is the fused
    projection of ``T`` tokens; token ``t`` goes to position ``pos[t]`` of sequence ``seq[t]`` (``seq=None``: of sequence ``t``).
    With ``cos`` / ``sin`` (fp32 ``[positions, head_dim / 2]``, see :func:`~atorch_b200.ops.rope_tables`) the query and key
    heads are turned to the position first. Returns the query heads ``[T, n_q, head_dim]`` in the type of ``qkv``. A negative
    position is padding: its token is not kept, its queries come back as they are. What two tokens at one place leave there is not defined.

    The rotation is not rounded before the codes are taken; queries are rounded once."""
    codes, scales, table, pages, KV, shift, rows, most, stride, D, dev = _cache(layer, page_table)
    shape, dtype, width = qkv.shape, _lib.DT.get(qkv.dtype), (n_q + 2 * KV) * D
    if dtype is None:
        raise ValueError(f"qkv is bf16, fp16 or fp32, got {qkv.dtype}")
    if n_q < 0 or (shape[-1:] != (width,) and shape[-2:] != (n_q + 2 * KV, D)):
        raise ValueError(f"qkv {tuple(shape)}: {n_q} + 2 x {KV} heads of {D} are wanted in a token")
    positions = 0
    if cos is not None and sin is not None:
        positions = cos.shape[0]
        if cos.dtype is not torch.float32 or sin.dtype is not torch.float32 or cos.shape != (positions, D // 2) \
                or sin.shape != (positions, D // 2):
            raise ValueError(f"cos and sin are fp32 [positions, {D // 2}]")
        if not (cos.is_contiguous() and sin.is_contiguous()) or (cos.data_ptr() | sin.data_ptr()) & 15:      # read in pieces of 16 bytes
            cos, sin = (t.clone(memory_format=torch.contiguous_format) for t in (cos, sin))
    elif cos is not sin:
        raise ValueError("cos and sin go together")
    _no_gradient(qkv)
    x = qkv if len(shape) == 2 and shape[1] == width else qkv.reshape(qkv.numel() // width, width)
    T = x.shape[0]
    seq, pos = _int32("seq", seq, T), _int32("pos", pos, T)
    _same_device(dev, qkv, pos, seq, cos, sin)
    if dev < 0:
        return kv4_append_reference(layer, page_table, seq, pos, qkv, n_q, cos, sin)
    step, one = x.stride()
    if one != 1 or not _aligned(x, step):
        x, step = x.clone(memory_format=torch.contiguous_format), width
    q = x.new_empty(T, n_q, D)
    rc = _lib.lib().atb_kv4_append(x.data_ptr(), q.data_ptr(), codes, scales, table, _lib.addr(seq), pos.data_ptr(), _lib.addr(cos),
                                   _lib.addr(sin), positions, T, n_q, KV, D, shift, pages, rows, most, stride, step, dtype,
                                   _lib.stream_of(dev), _lib.status_addr(x))
    _lib.check(rc, "atb_kv4_append")
    return q


# ------------------------------------------------------------------------------------------------------------------
def _values_reference(layer, page, slot):
    codes, scales = layer
    sc = scales[page, :, slot].float()                               # [T, KV, 4]
    b = codes[page, :, :, slot]
    b = torch.stack([b & 15, b >> 4], -1).flatten(-2).float()
    return b[:, 0] * sc[..., 0:1] + sc[..., 1:2], b[:, 1] * sc[..., 2:3] + sc[..., 3:4]


def kv4_read_reference(layer, page_table, seq, pos, dtype=torch.bfloat16):
    page, slot, real = _places(page_table, seq, pos, layer[0].shape[3], pos.numel())
    k, v = _values_reference(layer, torch.where(real, page, torch.zeros_like(page)), slot)
    return tuple(torch.where(real[:, None, None], t, torch.zeros_like(t)).to(dtype) for t in (k, v))


def kv4_read(layer: Layer, page_table: torch.Tensor, seq: Optional[torch.Tensor], pos: torch.Tensor,
             dtype: torch.dtype = torch.bfloat16) -> Tuple[torch.Tensor, torch.Tensor]:
    """Keys and values ``[T, kv_heads, head_dim]`` that the cache stands for at the positions ``pos`` of the sequences ``seq``
    (as in :func:`kv4_append`); zeros where the position is negative. A prompt's own attention runs on them, so that its tokens
    see the same keys as the tokens after it."""
    codes, scales, table, pages, KV, shift, rows, most, stride, D, dev = _cache(layer, page_table)
    kind, T = _lib.DT.get(dtype), pos.numel()
    if kind is None:
        raise ValueError(f"dtype is bf16, fp16 or fp32, got {dtype}")
    seq, pos = _int32("seq", seq, T), _int32("pos", pos, T)
    _same_device(dev, pos, seq)
    if dev < 0:
        return kv4_read_reference(layer, page_table, seq, pos, dtype)
    k = pos.new_empty((T, KV, D), dtype=dtype)
    v = torch.empty_like(k)
    rc = _lib.lib().atb_kv4_read(k.data_ptr(), v.data_ptr(), codes, scales, table, _lib.addr(seq), pos.data_ptr(), T, KV, D, shift, pages,
                                 rows, most, stride, kind, _lib.stream_of(dev), _lib.status_addr(pos))
    _lib.check(rc, "atb_kv4_read")
    return k, v


# ------------------------------------------------------------------------------------------------------------------
def kv4_attention_reference(q, layer, page_table, lengths, softmax_scale=None):
    """Returns (out, lse)."""
    codes, _ = layer
    B, S, H, D = q.shape
    KV, page_size = codes.shape[2], codes.shape[3]
    g = H // KV
    scale = softmax_scale if softmax_scale is not None else 1.0 / math.sqrt(D)
    out = torch.zeros(B, S, H, D, dtype=torch.float32, device=q.device)
    lse = torch.full((B, H, S), -math.inf, dtype=torch.float32, device=q.device)
    if lengths.numel() and int(lengths.max()) > page_table.shape[1] * page_size:
        raise IndexError("a sequence is longer than its row of the page table")
    for b, n in enumerate(lengths.tolist()):
        if n <= 0:
            continue
        t = torch.arange(n, device=q.device)
        k, v = _values_reference(layer, page_table[b, t // page_size].long(), t % page_size)
        k, v = k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)
        s = torch.einsum("ihd,thd->hit", q[b].float(), k) * scale
        for i in range(S):      # what a query does not see does not reach it, whatever stands there
            m = max(0, n - S + i + 1)
            lse[b, :, i] = torch.logsumexp(s[:, i, :m], -1)
            shift = torch.where(lse[b, :, i] == -math.inf, torch.zeros_like(lse[b, :, i]), lse[b, :, i])
            out[b, i] = torch.einsum("ht,thd->hd", torch.exp(s[:, i, :m] - shift[:, None]), v[:m])
    return out.to(q.dtype), lse


@functools.lru_cache(maxsize=256)
def _scratch(*sizes: int) -> int:
    """Floats of the attention kernels' workspace."""
    fn = _lib.lib().atb_kv4_attention_scratch
    fn.restype = ctypes.c_longlong
    return fn(*sizes)


def kv4_attention(q: torch.Tensor, layer: Layer, page_table: torch.Tensor, lengths: torch.Tensor,
                  softmax_scale: Optional[float] = None, return_lse: bool = False):
    """Attention of the newest tokens over the cache. ``q`` ``[sequences, S, n_q, head_dim]`` (bf16 or fp16) are the queries of
    the last ``S`` tokens of every sequence, ``lengths`` ``[sequences]`` its tokens in the cache, those ``S`` included: query
    ``i`` sees the keys ``j < lengths - S + i + 1``. Query heads are shared as in :func:`~atorch_b200.ops.attention` (``n_q`` a
    multiple of the cache's heads). Returns ``[sequences, S, n_q, head_dim]``, and with ``return_lse`` the logarithms of the
    denominators, fp32 ``[sequences, n_q, S]``. A query that sees nothing gives zeros (and ``-inf``)."""
    codes, scales, table, pages, KV, shift, rows, most, stride, D, dev = _cache(layer, page_table)
    if q.dim() != 4 or q.shape[3] != D or q.shape[2] % KV or q.shape[2] == 0:
        raise ValueError(f"q {tuple(q.shape)}: [sequences, S, a multiple of {KV}, {D}] is wanted")
    if q.dtype is not torch.bfloat16 and q.dtype is not torch.float16:
        raise ValueError(f"q is bf16 or fp16, got {q.dtype}")
    B, S, H, _ = q.shape
    if rows != B:
        raise ValueError(f"page_table has {rows} rows for {B} sequences")
    _no_gradient(q)
    lengths = _int32("lengths", lengths, B)
    _same_device(dev, q, lengths)
    if dev < 0:
        out, lse = kv4_attention_reference(q, layer, page_table, lengths, softmax_scale)
        return (out, lse) if return_lse else out
    q_batch, q_token, q_head, one = q.stride()
    if one != 1 or q_head != D or (q.data_ptr() | 2 * q_batch | 2 * q_token) & 15:
        q = q.clone(memory_format=torch.contiguous_format)
        q_batch, q_token = S * H * D, H * D
    out = q.new_empty(B, S, H, D)
    lse = torch.empty(B, H, S, dtype=torch.float32, device=q.device) if return_lse else None
    partial = None if most << shift <= WHOLE else torch.empty(_scratch(B, H, KV, S, D), dtype=torch.float32, device=q.device)
    rc = _lib.lib().atb_kv4_attention(
        q.data_ptr(), out.data_ptr(), _lib.addr(lse), codes, scales, table, lengths.data_ptr(), _lib.addr(partial), S, H, KV, D, shift,
        pages, B, most, stride, q_batch, q_token, D ** -0.5 if softmax_scale is None else softmax_scale, _lib.DT[q.dtype],
        _lib.stream_of(dev), _lib.status_addr(q))
    _lib.check(rc, "atb_kv4_attention")
    return (out, lse) if return_lse else out
