"""One step of a beam search: the best continuations over beams and vocabulary, and the paged 4-bit cache's rows moved to their
new beams (csrc/beam.cu).

Tokens and parents of the steps are the search's result: a sequence is read back from its last step, parent by parent.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad

from .. import _lib
from .function import refuse_gradient
from .kv4 import _check_page_size

MAX_BEAMS = 32
# continuations of a sequence up to which one cluster of blocks selects among them (in one launch); above, each beam has a cluster of
# its own and a second kernel joins them: 4 beams of 32000 tokens, with the move of 8 layers, 11.0 us in one, 11.9 in two, and 4 us
# less on the host
ONE_CLUSTER = 1 << 17


def beam_select_reference(logits, scores, finished=None, eos=-1, keep=None):
    B, W, V = logits.shape
    keep = W if keep is None else keep
    x = logits.float()
    top = x.amax(-1, keepdim=True)
    lse = top + torch.log(torch.exp(x - top).sum(-1, keepdim=True))
    f = scores.unsqueeze(-1) + (x - lse)
    if finished is not None:
        done, ends = finished.unsqueeze(-1), torch.arange(V, device=x.device) == eos
        f = torch.where(done, torch.where(ends, scores.unsqueeze(-1), torch.full_like(f, -math.inf)), f)
    f = torch.where(torch.isnan(f), torch.full_like(f, -math.inf), f)
    best, at = f.view(B, W * V).sort(dim=-1, descending=True, stable=True)
    best, at = best[:, :keep], at[:, :keep]
    parents, tokens = at // V, at % V
    ended = tokens == eos
    if finished is not None:
        ended = ended | finished.gather(1, parents)
    return best, tokens, parents.to(torch.int32), ended


def beam_select(logits: torch.Tensor, scores: torch.Tensor, finished: Optional[torch.Tensor] = None, eos: int = -1,
                keep: Optional[int] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """The ``keep`` (default: as many as there are) best continuations of every sequence's beams. ``logits`` ``[B, W, V]`` (bf16,
    fp16 or fp32) of the beams' last tokens, ``scores`` fp32 ``[B, W]`` their sums of log-probabilities so far. A continuation
    scores ``scores + log_softmax(logits)``, in fp32; equal scores go to the lower beam, then the lower token, a NaN counts as
    ``-inf``. A beam with ``finished`` set goes on with ``eos`` alone, at its score.

    Returns scores fp32, tokens int64, parents int32 (the beam that a continuation goes on from) and finished bool (the parent
    was, or the token is ``eos``), each ``[B, keep]``, best first. Behind a failed kernel (see ``_lib.check_status``) nothing is
    selected: scores of ``-inf``, tokens and parents 0, all finished."""
    if logits.dim() != 3 or logits.dtype not in _lib.DT or logits.shape[2] == 0 or logits.shape[1] == 0:
        raise ValueError(f"logits are bf16, fp16 or fp32 [B, beams, vocabulary], got {logits.dtype} {tuple(logits.shape)}")
    B, W, V = logits.shape
    keep = W if keep is None else int(keep)
    if V > 1 << 27:
        raise ValueError(f"a vocabulary of {V}: 2 ** 27 at most")
    if not 1 <= keep <= W * V:
        raise ValueError(f"keep {keep} of {W} x {V} continuations")
    if scores.dtype is not torch.float32 or scores.shape != (B, W):
        raise ValueError(f"scores are fp32 {(B, W)}, got {scores.dtype} {tuple(scores.shape)}")
    if finished is not None:
        if finished.dtype is not torch.bool or finished.shape != (B, W):
            raise ValueError(f"finished is bool {(B, W)}, got {finished.dtype} {tuple(finished.shape)}")
        if not 0 <= eos < V:
            raise ValueError(f"finished beams go on with eos, and {eos} is not in the vocabulary")
    dev = logits.get_device()
    if scores.get_device() != dev or (finished is not None and finished.get_device() != dev):
        raise ValueError("logits, scores and finished are on several devices")
    if logits.requires_grad or scores.requires_grad or forward_ad._current_level >= 0:
        refuse_gradient("a selection has no gradient: call under torch.no_grad()", logits, scores)
    if dev < 0 or not _lib.use_kernels(logits):
        return beam_select_reference(logits, scores, finished, eos, keep)
    if W > MAX_BEAMS or keep > MAX_BEAMS:
        raise ValueError(f"{W} beams, {keep} kept: the kernels take {MAX_BEAMS}")
    step, row, one = logits.stride()
    if one != 1 or (B > 1 and W > 1 and step != W * row):
        logits, row, step = logits.contiguous(), V, W * V
    if W == 1:
        row = step
    base = logits.data_ptr()
    scores, finished = scores.contiguous(), None if finished is None else finished.contiguous()
    out = scores.new_empty(B, keep)
    tokens = torch.empty_like(out, dtype=torch.int64)
    parents = torch.empty_like(out, dtype=torch.int32)
    ended = torch.empty_like(out, dtype=torch.bool)
    best = None if W * V <= ONE_CLUSTER and W <= 16 else torch.empty(B * W * keep, dtype=torch.int64, device=logits.device)
    rc = _lib.lib().atb_beam_select(base, scores.data_ptr(), _lib.addr(finished), _lib.addr(best), out.data_ptr(), tokens.data_ptr(),
                                    parents.data_ptr(), ended.data_ptr(), B, W, V, row,
                                    int(base % 16 == 0 and row * logits.element_size() % 16 == 0), int(eos), keep,
                                    _lib.DT[logits.dtype], _lib.stream_of(dev), _lib.status_addr(logits))
    _lib.check(rc, "atb_beam_select")
    return out, tokens, parents, ended


def beam_reorder_reference(codes, scales, page_table, lengths, parents):
    B, W = parents.shape
    page_size = codes.shape[4]
    n = lengths.view(B, W)
    if bool((n != n[:, :1]).any()) or bool(((parents < 0) | (parents >= W)).any()):
        raise IndexError("parents out of range, or beams of different lengths")
    source = (torch.arange(B, device=parents.device).unsqueeze(1) * W + parents).flatten()
    old = page_table.clone()
    for b in range(B):
        rows = slice(b * W, (b + 1) * W)
        full, rest = divmod(int(n[b, 0]), page_size)
        if full + (rest > 0) > page_table.shape[1]:
            raise IndexError("a sequence is longer than its row of the page table")
        page_table[rows, :full] = old[source[rows], :full]
        if rest:
            to, of = old[rows, full].long(), old[source[rows], full].long()
            codes[:, to, :, :, :rest] = codes[:, of, :, :, :rest]
            scales[:, to, :, :rest] = scales[:, of, :, :rest]


def beam_reorder(codes: torch.Tensor, scales: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor,
                 parents: torch.Tensor) -> None:
    """Let the caches of all layers (``codes`` and ``scales`` of a :class:`~atorch_b200.ops.KV4Cache`) follow the beams, in place.
    Rows ``b W`` to ``b W + W - 1`` of ``page_table`` are the beams of sequence ``b``, all of ``lengths[b W]`` tokens (int32
    ``[B * W]``, equal within a sequence), ``parents`` int32 ``[B, W]``. Row ``b W + w`` takes the full pages of row
    ``b W + parents[b, w]`` by their numbers, and the tokens of its last page by copying them into its own.

    Full pages may belong to many rows: nothing is written to them any more. From the last, partly filled page on, every row
    needs pages of its own."""
    if codes.dim() != 6 or scales.dim() != 5 or codes.dtype is not torch.uint8 or scales.dtype is not torch.bfloat16 \
            or codes.shape[2] != 2 or scales.shape != (*codes.shape[:2], *codes.shape[3:5], 4) \
            or not (codes.is_contiguous() and scales.is_contiguous()):
        raise ValueError(f"codes {tuple(codes.shape)} and scales {tuple(scales.shape)} are not the caches of layers")
    if (codes.data_ptr() | scales.data_ptr()) & 15:
        raise ValueError("the cache has to begin on 16 bytes")
    layers, pages, _, KV, page_size, half = codes.shape
    _check_page_size(page_size)
    if parents.dim() != 2 or parents.dtype is not torch.int32:
        raise ValueError(f"parents are int32 [B, beams], got {parents.dtype} {tuple(parents.shape)}")
    B, W = parents.shape
    if page_table.dtype is not torch.int32 or page_table.dim() != 2 or page_table.shape[0] != B * W \
            or (page_table.stride(1) != 1 and page_table.shape[1] > 1):
        raise ValueError(f"page_table is int32 [{B * W}, pages], its rows contiguous")
    if lengths.dtype is not torch.int32 or lengths.shape != (B * W,):
        raise ValueError(f"lengths are int32 [{B * W}], got {lengths.dtype} {tuple(lengths.shape)}")
    dev = codes.get_device()
    if any(t.get_device() != dev for t in (scales, page_table, lengths, parents)):
        raise ValueError("tensors on several devices")
    if dev < 0 or not _lib.use_kernels(codes):
        return beam_reorder_reference(codes, scales, page_table, lengths, parents)
    if W > MAX_BEAMS or half % 16:
        raise ValueError(f"{W} beams, head_dim {2 * half}: the kernel takes {MAX_BEAMS} and multiples of 32")
    parents, lengths = parents.contiguous(), lengths.contiguous()
    rc = _lib.lib().atb_beam_reorder(codes.data_ptr(), scales.data_ptr(), page_table.data_ptr(), lengths.data_ptr(),
                                     parents.data_ptr(), B, W, page_table.shape[1], page_table.stride(0), layers, pages, KV,
                                     page_size.bit_length() - 1, 2 * half, _lib.stream_of(dev), _lib.status_addr(codes))
    _lib.check(rc, "atb_beam_reorder")
