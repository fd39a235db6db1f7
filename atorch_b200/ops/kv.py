"""Paged key/value cache in the model's own 16 bits: append with rotation, attention of the newest tokens, and eviction of the tokens
that attention has given least weight, so that a cache keeps to a budget however long its sequence grows.

A layer's cache is one tensor ``[pages, 2, kv_heads, page_size, head_dim]`` (0: keys, 1: values), bf16 or fp16. Row ``b`` of
``page_table`` (int32 ``[sequences, pages of the longest]``) names the pages of sequence ``b``; pages have a power of two of 16 or more
tokens. A token's place in the cache is not its position in the sequence once tokens before it have been evicted: calls that write
take both.

Places, page numbers and lengths lie on the device. One that is out of range is skipped by the kernels and recorded in the device's
status word, which ``_lib.check_status`` raises; kernels of this package behind it store nothing until then.

These operators serve generation: they have no gradient, and refuse tensors that ask for one. ``ops/kv4.py`` holds the same cache in a
quarter of the memory, without eviction.
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
from .kv4 import HEAD_DIMS, _aligned, _check_page_size, _int32, _places, _same_device

DTYPES = (torch.bfloat16, torch.float16)
# Scores that attention with weights keeps at a time (256 MB). 64 prompts of 8192 tokens, 32 last tokens each, 32 heads (2 GB of scores) took
# 2947 us at once, 3117 with 1 GB, 3291 with 256 MB and 4397 with 64; 64 of 2048 with 32 heads on 8 (512 MB) 612, 649 with 256, 814 with 64.
SCORES = 1 << 26


class KVCache:
    """The caches of ``layers`` layers over one pool of ``pages`` pages (one page table serves all layers)."""

    def __init__(self, layers: int, pages: int, page_size: int, kv_heads: int, head_dim: int, dtype: torch.dtype = torch.bfloat16,
                 device=None):
        _check_page_size(page_size)
        if dtype not in DTYPES:
            raise ValueError(f"the cache is bf16 or fp16, got {dtype}")
        self.data = torch.zeros(layers, pages, 2, kv_heads, page_size, head_dim, dtype=dtype, device=device)
        self.page_size = page_size

    def layer(self, i: int) -> torch.Tensor:
        return self.data[i]


def _cache(layer: torch.Tensor, page_table: torch.Tensor) -> Tuple[int, ...]:
    """A layer's cache and page table as the launchers take them, after the checks that all calls share: addresses of cache and table,
    pages, kv_heads, page_shift, sequences, pages of a sequence, stride of the table; then head_dim and the index of the device (-1:
    the CPU)."""
    shape, at, dev = layer.shape, layer.data_ptr(), layer.get_device()
    if layer.dtype not in DTYPES or len(shape) != 5 or shape[1] != 2 or 0 in shape:
        raise ValueError(f"a layer's cache is bf16 or fp16 [pages, 2, kv_heads, page_size, head_dim], got {layer.dtype} {tuple(shape)}")
    if not layer.is_contiguous() or at & 15:
        raise ValueError("the cache has to be contiguous and begin on 16 bytes")
    pages, _, kv_heads, page_size, D = shape
    if page_size < 16 or page_size & (page_size - 1):
        _check_page_size(page_size)
    if D % 2 or (dev >= 0 and D != 128 and D != 64):
        raise ValueError(f"head_dim {D}: the kernels take {HEAD_DIMS}")
    rows, width, step = _table(page_table, page_size)
    if page_table.get_device() != dev:
        _same_device(dev, page_table)
    return at, page_table.data_ptr(), pages, kv_heads, page_size.bit_length() - 1, rows, width, step, D, dev


def _table(page_table: torch.Tensor, page_size: int) -> Tuple[int, int, int]:
    steps = page_table.stride()
    if page_table.dtype is not torch.int32 or len(steps) != 2 or (steps[1] != 1 and page_table.shape[1] > 1):
        raise ValueError("page_table is int32 [sequences, pages], its rows contiguous")
    rows, width = page_table.shape
    if width * page_size > 0x7fffffff:
        raise ValueError(f"{width} pages of {page_size} tokens a sequence: places have 31 bits")
    return rows, width, steps[0]


def _no_gradient(a: torch.Tensor, b: torch.Tensor) -> None:
    if a.requires_grad or b.requires_grad or forward_ad._current_level >= 0:
        refuse_gradient("the cache has no gradient: call under torch.no_grad()", a, b)


# ------------------------------------------------------------------------------------------------------------------
def kv_append_reference(layer, page_table, seq, pos, qkv, n_q, cos=None, sin=None, angles=None):
    """Returns (queries, keys)."""
    _, _, KV, page_size, D = layer.shape
    T = pos.numel()
    x = qkv.reshape(T, n_q + 2 * KV, D)
    page, slot, real = _places(page_table, seq, pos, page_size, T)
    turned = x[:, : n_q + KV]
    if cos is not None:
        at = pos if angles is None else angles
        if bool(((at < 0) | (at >= cos.shape[0]))[real].any()):
            raise IndexError("an angle lies outside cos and sin")
        at = at.clamp(0, cos.shape[0] - 1).long()
        c, s = cos[at].unsqueeze(1), sin[at].unsqueeze(1)
        a, b = turned[..., : D // 2].float(), turned[..., D // 2:].float()
        turned = torch.where(real[:, None, None], torch.cat([a * c - b * s, b * c + a * s], -1).to(x.dtype), turned)
    layer[page[real], :, :, slot[real]] = torch.stack([turned[:, n_q:], x[:, n_q + KV:]], 1)[real]
    return turned[:, :n_q].contiguous(), turned[:, n_q:].contiguous()


def kv_append(layer: torch.Tensor, page_table: torch.Tensor, seq: Optional[torch.Tensor], pos: torch.Tensor, qkv: torch.Tensor, n_q: int,
              cos: Optional[torch.Tensor] = None, sin: Optional[torch.Tensor] = None, angles: Optional[torch.Tensor] = None,
              return_keys: bool = False):
    """Put tokens into the cache. ``qkv`` ``[..., (n_q + 2 kv_heads) * head_dim]`` (or with heads and dims apart), in the cache's type, is
    the fused projection of ``T`` tokens; token ``t`` goes to place ``pos[t]`` of sequence ``seq[t]`` (``seq=None``: of sequence ``t``).
    With ``cos`` / ``sin`` (fp32 ``[positions, head_dim / 2]``, see :func:`~atorch_b200.ops.rope_tables`) the query and key heads are
    turned first, to position ``angles[t]`` of the sequence, which is ``pos[t]`` where it is not given. Returns the query heads
    ``[T, n_q, head_dim]``, and with ``return_keys`` the key heads ``[T, kv_heads, head_dim]`` as the cache has them (a prompt's own
    attention runs on those). A negative place is padding: its token is not kept, its queries and keys come back as they are. What two
    tokens at one place leave there is not defined.

    The rotation is evaluated in fp32, operation by operation, and rounded once; values are copied."""
    at, table, pages, KV, shift, rows, most, stride, D, dev = _cache(layer, page_table)
    shape, width = qkv.shape, (n_q + 2 * KV) * D
    if qkv.dtype is not layer.dtype:
        raise ValueError(f"qkv is in the cache's type, {layer.dtype}, got {qkv.dtype}")
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
    elif angles is not None:
        raise ValueError("angles are positions of cos and sin")
    _no_gradient(qkv, layer)
    x = qkv if len(shape) == 2 and shape[1] == width else qkv.reshape(qkv.numel() // width, width)
    T = x.shape[0]
    seq, pos, angles = _int32("seq", seq, T), _int32("pos", pos, T), _int32("angles", angles, T)
    _same_device(dev, qkv, pos, seq, angles, cos, sin)
    if dev < 0:
        q, k = kv_append_reference(layer, page_table, seq, pos, qkv, n_q, cos, sin, angles)
        return (q, k) if return_keys else q
    step, one = x.stride()
    if one != 1 or not _aligned(x, step):
        x, step = x.clone(memory_format=torch.contiguous_format), width
    q = x.new_empty(T, n_q, D)
    k = x.new_empty(T, KV, D) if return_keys else None
    rc = _lib.lib().atb_kv_append(x.data_ptr(), q.data_ptr(), _lib.addr(k), at, table, _lib.addr(seq), pos.data_ptr(), _lib.addr(angles),
                                  _lib.addr(cos), _lib.addr(sin), positions, T, n_q, KV, D, shift, pages, rows, most, stride, step,
                                  _lib.DT[x.dtype], _lib.stream_of(dev), _lib.status_addr(x))
    _lib.check(rc, "atb_kv_append")
    return (q, k) if return_keys else q


# ------------------------------------------------------------------------------------------------------------------
def kv_attention_reference(q, layer, page_table, lengths, softmax_scale=None, weights=None):
    """Returns (out, lse)."""
    B, S, H, D = q.shape
    KV, page_size = layer.shape[2], layer.shape[3]
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
        page = page_table[b, t // page_size].long()
        if bool(((page < 0) | (page >= layer.shape[0])).any()):
            raise IndexError("a page lies outside the cache")
        kv = layer[page, :, :, t % page_size].float()                   # [n, 2, KV, D]
        k, v = kv[:, 0].repeat_interleave(g, 1), kv[:, 1].repeat_interleave(g, 1)
        s = torch.einsum("ihd,thd->hit", q[b].float(), k) * scale
        for i in range(S):      # what a query does not see does not reach it, whatever stands there
            m = max(0, n - S + i + 1)
            lse[b, :, i] = torch.logsumexp(s[:, i, :m], -1)
            shift = torch.where(lse[b, :, i] == -math.inf, torch.zeros_like(lse[b, :, i]), lse[b, :, i])
            p = torch.exp(s[:, i, :m] - shift[:, None])
            out[b, i] = torch.einsum("ht,thd->hd", p, v[:m])
            if weights is not None:
                weights[b, :, :m] += p.view(KV, g, m).sum(1)
    return out.to(q.dtype), lse


@functools.lru_cache(maxsize=256)
def _scratch(*sizes: int) -> int:
    """Floats of the attention kernels' workspace."""
    fn = _lib.lib().atb_kv_attention_scratch
    fn.restype = ctypes.c_longlong
    return fn(*sizes)


def _in_pieces(q, layer, page_table, lengths, softmax_scale, return_lse, weights, each):
    """Attention with weights whose scores (`each` of a token) are too many at once: some sequences after another, or some tokens of one."""
    B, S = q.shape[:2]
    got = []
    if B > 1:
        n = max(1, SCORES // (S * each))
        for b in range(0, B, n):
            got.append(kv_attention(q[b: b + n], layer, page_table[b: b + n], lengths[b: b + n], softmax_scale, return_lse, weights[b: b + n]))
    else:
        n = max(1, SCORES // each)
        for i in range(0, S, n):
            behind = max(0, S - i - n)          # tokens that these do not see
            got.append(kv_attention(q[:, i: i + n], layer, page_table, lengths.clamp(min=0) - behind if behind else lengths, softmax_scale,
                                    return_lse, weights))
    along = 0 if B > 1 else 1
    if not return_lse:
        return torch.cat(got, along)
    return torch.cat([out for out, _ in got], along), torch.cat([lse for _, lse in got], 2 * along)


def kv_attention(q: torch.Tensor, layer: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor,
                 softmax_scale: Optional[float] = None, return_lse: bool = False, weights: Optional[torch.Tensor] = None):
    """Attention of the newest tokens over the cache. ``q`` ``[sequences, S, n_q, head_dim]``, in the cache's type, are the queries of the
    last ``S`` tokens of every sequence, ``lengths`` ``[sequences]`` its tokens in the cache, those ``S`` included: query ``i`` sees the
    places ``j < lengths - S + i + 1``. Query heads are shared as in :func:`~atorch_b200.ops.attention` (``n_q`` a multiple of the
    cache's heads). Returns ``[sequences, S, n_q, head_dim]``, and with ``return_lse`` the logarithms of the denominators, fp32
    ``[sequences, n_q, S]``. A query that sees nothing gives zeros (and ``-inf``).

    ``weights`` (fp32 ``[sequences, kv_heads, places]``, contiguous, as many places as a row of the page table has or more) takes up what
    the queries attended to, in place: the softmax weights of the ``S`` tokens and of the heads that share a key/value head are added to
    it. :func:`kv_evict` goes by them. For them the call keeps a score of 4 bytes for every sequence, query, query head and place of a row of
    the page table, 256 MB of them at a time (or those of one token of one sequence): above that it goes through sequences, then
    tokens, in pieces."""
    at, table, pages, KV, shift, rows, most, stride, D, dev = _cache(layer, page_table)
    if q.dim() != 4 or q.shape[3] != D or q.shape[2] % KV or q.shape[2] == 0:
        raise ValueError(f"q {tuple(q.shape)}: [sequences, S, a multiple of {KV}, {D}] is wanted")
    if q.dtype is not layer.dtype:
        raise ValueError(f"q is in the cache's type, {layer.dtype}, got {q.dtype}")
    B, S, H, _ = q.shape
    if rows != B:
        raise ValueError(f"page_table has {rows} rows for {B} sequences")
    _no_gradient(q, layer)
    places = 0
    if weights is not None:
        places = weights.shape[-1]
        if weights.dtype is not torch.float32 or weights.shape != (B, KV, places) or places < most << shift or not weights.is_contiguous():
            raise ValueError(f"weights are fp32 {(B, KV)} x {most << shift} places or more, contiguous, got {weights.dtype} "
                             f"{tuple(weights.shape)}")
        _no_gradient(weights, q)
    lengths = _int32("lengths", lengths, B)
    _same_device(dev, q, lengths, weights)
    if dev < 0:
        out, lse = kv_attention_reference(q, layer, page_table, lengths, softmax_scale, weights)
        return (out, lse) if return_lse else out
    if weights is not None and (S > 1 or B > 1) and B * S * H * (most << shift) > SCORES:
        return _in_pieces(q, layer, page_table, lengths, softmax_scale, return_lse, weights, H * (most << shift))
    q_batch, q_token, q_head, one = q.stride()
    if one != 1 or q_head != D or (q.data_ptr() | 2 * q_batch | 2 * q_token) & 15:
        q = q.clone(memory_format=torch.contiguous_format)
        q_batch, q_token = S * H * D, H * D
    out = q.new_empty(B, S, H, D)
    lse = torch.empty(B, H, S, dtype=torch.float32, device=q.device) if return_lse else None
    size = _scratch(B, H, KV, S, D, most << shift, int(weights is not None))
    partial = torch.empty(size, dtype=torch.float32, device=q.device) if size else None
    rc = _lib.lib().atb_kv_attention(
        q.data_ptr(), out.data_ptr(), _lib.addr(lse), at, table, lengths.data_ptr(), _lib.addr(weights), _lib.addr(partial), S, H, KV, D,
        shift, pages, B, most, stride, places, q_batch, q_token, D ** -0.5 if softmax_scale is None else softmax_scale,
        _lib.DT[q.dtype], _lib.stream_of(dev), _lib.status_addr(q))
    _lib.check(rc, "atb_kv_attention")
    return (out, lse) if return_lse else out


# ------------------------------------------------------------------------------------------------------------------
def kv_evict_reference(cache, page_table, lengths, weights, budget, recent=0):
    """``cache`` ``[layers, pages, ...]``, ``weights`` ``[layers, ...]``."""
    page_size = cache.shape[4]
    if lengths.numel() and int(lengths.max()) > page_table.shape[1] * page_size:
        raise IndexError("a sequence is longer than its row of the page table")
    for b, n in enumerate(lengths.tolist()):
        if n <= budget:
            continue
        t = torch.arange(n, device=cache.device)
        page, slot = page_table[b, t // page_size].long(), t % page_size
        if bool(((page < 0) | (page >= cache.shape[1])).any()):
            raise IndexError("a page lies outside the cache")
        w = weights[:, b, :, :n].clone()
        rank = w[..., : n - recent] + 0.0
        rank = torch.where(torch.isnan(rank), torch.full_like(rank, -math.inf), rank)
        first = rank.sort(dim=-1, descending=True, stable=True).indices[..., : budget - recent].sort(-1).values
        kept = torch.cat([first, t[n - recent:].expand(*first.shape[:-1], recent)], -1)                 # [layers, KV, budget]
        held = cache[:, page, :, :, slot]                                                               # [n, layers, 2, KV, D]
        at = kept.permute(2, 0, 1)[:, :, None, :, None].expand(budget, *held.shape[1:])
        cache[:, page[:budget], :, :, slot[:budget]] = held.gather(0, at)
        weights[:, b, :, :n] = 0
        weights[:, b, :, :budget] = w.gather(-1, kept)
    return lengths.clamp(max=budget)


def kv_evict(cache: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor, weights: torch.Tensor, budget: int,
             recent: int = 0) -> torch.Tensor:
    """Cut the sequences that have more than ``budget`` tokens in the cache down to that many, in place. Per layer and key/value head the
    ``recent`` last tokens stay, and of those before them the ``budget - recent`` with the largest ``weights`` (what
    :func:`kv_attention` added up; equal ones go to the lower place, a NaN counts as ``-inf``). They move down into the places
    ``0 ... budget - 1`` in their order, keys, values and weights; the weights of the places behind become 0, their keys and values are
    left as they are. Sequences within the budget are not touched, nor are those that are longer than their row of the page table or
    have a page that is not there, which are recorded; the others of the call are cut all the same.

    ``cache`` ``[layers, pages, 2, kv_heads, page_size, head_dim]`` (a :class:`KVCache`'s ``data``) with ``weights`` fp32
    ``[layers, sequences, kv_heads, places]``, or one layer of both; ``lengths`` ``[sequences]``. Returns the new lengths, int32. No page
    may belong to two sequences. A token's own position is needed for its rotation alone, which the kept keys have behind them."""
    if cache.dim() not in (5, 6) or weights.dim() != cache.dim() - 2:
        raise ValueError(f"cache {tuple(cache.shape)} and weights {tuple(weights.shape)}: [layers, pages, 2, kv_heads, page_size, head_dim] "
                         "and [layers, sequences, kv_heads, places] are wanted, or one layer of both")
    if cache.dim() == 5:
        cache, weights = cache.unsqueeze(0), weights.unsqueeze(0)
    layers = cache.shape[0]
    if layers == 0 or not cache.is_contiguous():
        raise ValueError("the caches of all layers have to be contiguous")
    at, table, pages, KV, shift, rows, most, stride, D, dev = _cache(cache[0], page_table)
    budget, recent = int(budget), int(recent)
    if budget < 1 or not 0 <= recent <= budget:
        raise ValueError(f"a budget of one token at least, of which {recent} last ones stay: got {budget}")
    places = weights.shape[3]
    if weights.dtype is not torch.float32 or weights.shape != (layers, rows, KV, places) or places < most << shift \
            or not weights.is_contiguous():
        raise ValueError(f"weights are fp32 {(layers, rows, KV)} x {most << shift} places or more, contiguous, got {weights.dtype} "
                         f"{tuple(weights.shape)}")
    _no_gradient(cache, weights)
    lengths = _int32("lengths", lengths, rows)
    _same_device(dev, lengths, weights)
    if dev < 0:
        return kv_evict_reference(cache, page_table, lengths, weights, budget, recent)
    out, work = torch.empty_like(lengths), None
    if budget >= most << shift:              # no row of the page table has so many places: lengths are looked at, no more
        budget, recent = most << shift, 0
    else:
        # per layer, sequence and head: the first place that changes, where the tokens come from, their weights
        work = torch.empty(layers * rows * KV * (2 * budget + 1), dtype=torch.int32, device=lengths.device)
    rc = _lib.lib().atb_kv_evict(at, table, lengths.data_ptr(), weights.data_ptr(), out.data_ptr(), _lib.addr(work), layers, KV, D, shift,
                                 pages, rows, most, stride, places, budget, recent, _lib.stream_of(dev), _lib.status_addr(weights))
    _lib.check(rc, "atb_kv_evict")
    return out
