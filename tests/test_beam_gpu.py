"""Beam search on the GPU: selection against 64 bits with its ties, and the cache's move to the new beams."""
import math

import pytest
import torch

from atorch_b200 import _lib, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _check(logits, scores, finished=None, eos=-1, keep=None):
    """Every kept score is that of its parent and token, the scores are the largest in 64 bits, and equal ones go by the index."""
    B, W, V = logits.shape
    got, tokens, parents, ended = ops.beam_select(logits, scores, finished, eos, keep)
    again = ops.beam_select(logits, scores, finished, eos, keep)
    assert all(torch.equal(a, b) for a, b in zip((got, tokens, parents, ended), again))
    keep = keep or W
    f = scores.double().unsqueeze(-1) + torch.log_softmax(logits.double(), -1)
    if finished is not None:
        f[finished] = -math.inf
        f[..., eos] = torch.where(finished, scores.double(), f[..., eos])
    f = torch.where(torch.isnan(f), torch.full_like(f, -math.inf), f)
    at = parents.long() * V + tokens
    want = f.flatten(1).topk(keep, -1).values
    mine = f.flatten(1).gather(1, at)
    # fp32: a sum of exponentials, its logarithm, two differences
    tol = 2.0 ** -21 * (scores.double().abs().nan_to_num(0, 0, 0).max() + logits.double().nan_to_num(0, 0, 0).abs().max() + 12)
    same = lambda a, b: ((a == b) | ((a - b).abs() <= tol)).all()  # noqa: E731
    assert same(got.double(), mine) and same(got.double(), want)
    for b in range(B):
        assert at[b].unique().numel() == keep
    later = got[:, 1:] == got[:, :-1]
    assert (got[:, 1:] <= got[:, :-1]).all() and (at[:, 1:] > at[:, :-1])[later].all()
    hit = tokens == eos
    assert torch.equal(ended, hit if finished is None else hit | finished.gather(1, parents.long()))
    _lib.check_status(got.device)
    return got, tokens, parents


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,W,V,keep", [(1, 1, 1, 1), (1, 1, 32000, 4), (2, 4, 32000, None), (3, 5, 1001, None), (1, 16, 4097, None),
                                        (2, 32, 700, None), (5, 2, 3, 6), (1, 3, 100, 32), (24, 8, 2000, 16), (1, 2, 130001, 2)])
def test_select(B, W, V, keep, dtype):
    g = _gen(B + W + V)
    logits = (torch.randn(B, W, V, generator=g, device=DEV) * 2).to(dtype)
    scores = torch.randn(B, W, generator=g, device=DEV) - 9
    if dtype == torch.float32:      # no ties, all apart: the indices are those of 64 bits
        _, tokens, parents = _check(logits, scores, keep=keep)
        f = scores.double().unsqueeze(-1) + torch.log_softmax(logits.double(), -1)
        best = f.flatten(1).topk(keep or W, -1)
        if (best.values[:, :-1] - best.values[:, 1:]).min() > 1e-4 if (keep or W) > 1 else True:
            assert torch.equal(best.indices, parents.long() * V + tokens)
    else:
        _check(logits, scores, keep=keep)
    _check(logits, scores, torch.rand(B, W, generator=g, device=DEV) < 0.4, V // 2, keep)


def test_ties_go_to_the_lower_index():
    for V in (7, 1000, 40000):
        logits = torch.zeros(2, 3, V, device=DEV).half()
        scores = torch.zeros(2, 3, device=DEV)
        keep = min(8, 3 * V)
        _, tokens, parents = _check(logits, scores, keep=keep)
        assert torch.equal(parents.long() * V + tokens, torch.arange(keep, device=DEV).expand(2, -1))
        scores[0, 1] = 1.0
        _, tokens, parents = _check(logits, scores, keep=3)
        assert (parents[0] == 1).all() and torch.equal(tokens, torch.arange(3, device=DEV).expand(2, -1))
    # logits that differ, scores so large that the sums do not
    logits = torch.randn(1, 2, 5000, generator=_gen(2), device=DEV)
    got = ops.beam_select(logits, torch.full((1, 2), -3e8, device=DEV), keep=5)
    assert torch.equal(got[1], torch.arange(5, device=DEV)[None]) and (got[2] == 0).all()


def test_what_is_impossible():
    g = _gen(3)
    logits = torch.randn(4, 3, 2000, generator=g, device=DEV)
    scores = torch.randn(4, 3, generator=g, device=DEV)
    logits[0, :, 5:] = -math.inf               # few may follow
    logits[1, 0] = -math.inf                   # none
    logits[1, 1, 9] = float("nan")             # a NaN makes the beam impossible
    logits[1, 2, 11] = math.inf
    scores[2, 1:] = -math.inf                  # the first step: one beam stands for all
    scores[3] = -math.inf
    _, tokens, parents = _check(logits, scores, keep=8)
    assert (parents[2] == 0).all()
    for b in (1, 3):                           # nothing is possible: by the index
        assert torch.equal(parents[b].long() * 2000 + tokens[b], torch.arange(8, device=DEV))
    _check(logits, scores, torch.ones(4, 3, dtype=torch.bool, device=DEV), 1)
    _check(logits.bfloat16()[:, :, :1999], scores, torch.zeros(4, 3, dtype=torch.bool, device=DEV), 0)


def test_strides_and_the_last_step_of_longer_logits():
    logits = torch.randn(6, 5, 999, generator=_gen(4), device=DEV).half()
    _check(logits[:, -1].view(2, 3, 999), torch.randn(2, 3, generator=_gen(5), device=DEV))
    _check(logits[:, 1:4], torch.randn(6, 3, generator=_gen(5), device=DEV))
    _check(logits.transpose(0, 1), torch.randn(6, 5, generator=_gen(5), device=DEV).t())
    _check(logits[:, :, 1:].transpose(1, 2)[:, 100:105].contiguous(), torch.randn(6, 5, generator=_gen(5), device=DEV))
    out = ops.beam_select(torch.zeros(0, 3, 9, device=DEV), torch.zeros(0, 3, device=DEV))
    assert [t.shape for t in out] == [(0, 3)] * 4


@pytest.mark.parametrize("B,W,length,page,KV,D,layers", [(1, 1, 5, 16, 1, 64, 1), (3, 4, 37, 16, 2, 128, 3), (2, 8, 64, 32, 3, 64, 2),
                                                         (1, 16, 15, 16, 8, 128, 2), (2, 32, 50, 64, 1, 64, 2), (4, 5, 100, 16, 2, 64, 1),
                                                         (2, 3, 0, 16, 2, 64, 1)])
def test_reorder(B, W, length, page, KV, D, layers):
    g = _gen(W + length)
    full = length // page
    pages = B * (full + W) + 2
    cache = ops.KV4Cache(layers, pages, page, KV, D, DEV)
    cache.codes.copy_(torch.randint(0, 256, cache.codes.shape, generator=g, device=DEV, dtype=torch.uint8))
    cache.scales.copy_(torch.randn(cache.scales.shape, generator=g, device=DEV))
    pool = torch.randperm(pages, generator=g, device=DEV).int()
    table = torch.full((B * W, full + 3), -5, dtype=torch.int32, device=DEV)[:, : full + 2]
    for b in range(B):
        table[b * W: (b + 1) * W, :full] = pool[torch.randint(b * full, (b + 1) * full, (W, full), generator=g, device=DEV)] if full else 0
    table[:, full] = pool[B * full: B * (full + W)]
    lengths = torch.full((B * W,), length, dtype=torch.int32, device=DEV)
    for parents in (torch.randint(0, W, (B, W), generator=g, device=DEV), torch.arange(W, device=DEV).expand(B, W),
                    torch.arange(W, device=DEV).flip(0).expand(B, W), torch.full((B, W), W - 1, device=DEV)):
        parents = parents.int()
        want = cache.codes.clone(), cache.scales.clone(), table.clone()
        ops.beam_reorder_reference(*want, lengths, parents)
        ops.beam_reorder(cache.codes, cache.scales, table, lengths, parents)
        assert torch.equal(want[0], cache.codes) and torch.equal(want[2], table)
        assert torch.equal(want[1].view(torch.int16), cache.scales.view(torch.int16))
    _lib.check_status(table.device)


def test_bad_indices_are_reported():
    cache = ops.KV4Cache(1, 6, 16, 1, 64, DEV)
    good = dict(page_table=torch.tensor([[0, 1], [0, 2]], dtype=torch.int32, device=DEV),
                lengths=torch.tensor([20, 20], dtype=torch.int32, device=DEV), parents=torch.tensor([[1, 0]], dtype=torch.int32, device=DEV))
    ops.beam_reorder(cache.codes, cache.scales, **good)
    _lib.check_status(cache.codes.device)
    for change in (dict(parents=good["parents"] + 1), dict(parents=good["parents"] - 1), dict(lengths=good["lengths"] + 20),
                   dict(lengths=good["lengths"] - 30), dict(page_table=good["page_table"] + 5), dict(page_table=good["page_table"] - 3),
                   dict(lengths=torch.tensor([20, 19], dtype=torch.int32, device=DEV))):
        ops.beam_reorder(cache.codes, cache.scales, **{**{k: v.clone() for k, v in good.items()}, **change})
        with pytest.raises(_lib.KernelError):
            _lib.check_status(cache.codes.device)


def test_refusals():
    x, s = torch.zeros(2, 3, 10, device=DEV), torch.zeros(2, 3, device=DEV)
    f = torch.zeros(2, 3, dtype=torch.bool, device=DEV)
    for bad in ((x[0], s), (x.double(), s), (x, s.half()), (x, s[:, :2]), (x, s, f.int(), 1), (x, s, f, 10), (x, s, f, -1), (x, s, None, 0, 0),
                (x, s, None, 0, 31), (x, s.cpu()), (torch.zeros(1, 33, 10, device=DEV), torch.zeros(1, 33, device=DEV)),
                (torch.zeros(1, 1, 0, device=DEV), torch.zeros(1, 1, device=DEV))):
        with pytest.raises(ValueError):
            ops.beam_select(*bad)
    with pytest.raises(RuntimeError):
        ops.beam_select(x.clone().requires_grad_(), s)
    cache = ops.KV4Cache(1, 6, 16, 1, 64, DEV)
    ok = [cache.codes, cache.scales, torch.zeros(6, 2, dtype=torch.int32, device=DEV), torch.ones(6, dtype=torch.int32, device=DEV),
          torch.zeros(2, 3, dtype=torch.int32, device=DEV)]
    for i, bad in ((0, cache.codes[0]), (1, cache.scales.float()), (2, ok[2][:5]), (2, ok[2].long()), (3, ok[3][:4]), (3, ok[3].long()),
                   (4, ok[4].long()), (4, ok[4][0]), (2, ok[2].cpu())):
        with pytest.raises(ValueError):
            ops.beam_reorder(*[bad if j == i else t for j, t in enumerate(ok)])


@pytest.mark.parametrize("B,W,V,keep", [(2, 3, 20000, None), (1, 6, 9000, None), (3, 7, 18000, 5), (1, 4, 32000, 32), (1, 11, 5000, None),
                                        (2, 16, 8192, 16), (1, 16, 8193, 16), (40, 5, 4100, None), (1, 1, 131072, 9), (1, 17, 300, None),
                                        (1, 1, 200003, 3)])
def test_select_by_one_cluster_or_by_several(B, W, V, keep):
    """Sizes on both sides of the rule that joins a sequence's beams in one cluster, and clusters of every size."""
    g = _gen(V + W)
    scores = torch.randn(B, W, generator=g, device=DEV) - 5
    for dtype in (torch.bfloat16, torch.float32):
        logits = (torch.randn(B, W, V, generator=g, device=DEV) * 3).to(dtype)
        _check(logits, scores, keep=keep)
        _check(logits, scores, torch.rand(B, W, generator=g, device=DEV) < 0.3, 0, keep)


def test_an_infinite_score():
    """A sum that is infinite whatever follows: the first tokens."""
    logits = torch.randn(1, 2, 3000, generator=_gen(9), device=DEV)
    got = ops.beam_select(logits, torch.tensor([[0.0, math.inf]], device=DEV), keep=4)
    assert (got[0] == math.inf).all() and (got[2] == 1).all() and torch.equal(got[1], torch.arange(4, device=DEV)[None])


@pytest.mark.parametrize("B,W,V,keep", [(24, 8, 20000, None), (1, 3, 100003, 7), (2, 12, 10900, None), (74, 3, 16001, 4)])
def test_select_with_a_whole_row_in_registers(B, W, V, keep):
    """Five to eight pieces of 16 bytes a thread, as clusters of a beam and of a sequence, and sizes just beyond."""
    g = _gen(V)
    scores = torch.randn(B, W, generator=g, device=DEV) - 5
    for dtype in (torch.bfloat16, torch.float16):
        logits = (torch.randn(B, W, V, generator=g, device=DEV) * 3).to(dtype)
        logits[:, 0, V // 2:] = -math.inf
        _check(logits, scores, keep=keep)
        _check(logits, scores, torch.rand(B, W, generator=g, device=DEV) < 0.3, 0, keep)


@pytest.mark.parametrize("B,W,length,page,KV,D,layers", [(24, 8, 410, 16, 8, 128, 4), (2, 3, 1000, 2048, 1, 64, 2), (70, 2, 33, 16, 1, 64, 1),
                                                         (1, 16, 1603, 16, 2, 64, 3), (1, 32, 1601, 16, 1, 64, 40), (3, 31, 63, 64, 3, 128, 5)])
def test_reorder_in_many_rounds(B, W, length, page, KV, D, layers):
    """More places, pages or layers than the warps of a sequence take at a time."""
    test_reorder(B, W, length, page, KV, D, layers)


@pytest.mark.parametrize("B,W,V,keep", [(2, 3, 40, 4), (1, 4, 32000, None), (3, 8, 4001, 5), (2, 17, 1003, 6), (1, 2, 131072, None), (24, 8, 20000, None)])
@pytest.mark.parametrize("dtype,mask", [(torch.bfloat16, torch.finfo(torch.bfloat16).min), (torch.float32, torch.finfo(torch.float32).min),
                                        (torch.bfloat16, -1e30), (torch.float32, -1e20), (torch.float32, -1e10), (torch.float16, -65504.0)])
def test_finite_masks(B, W, V, keep, dtype, mask):
    """Tokens masked by a large finite number, most of a row of them or all: the others go on as if the masked were not there."""
    g, keep = _gen(V), keep or W
    logits = (torch.randn(B, W, V, generator=g, device=DEV) * 2).to(dtype)
    scores = torch.randn(B, W, generator=g, device=DEV) - 5
    for pattern in ("few", "end", "one row", "a token each"):
        x, masked = logits.clone(), torch.zeros(B, W, V, dtype=torch.bool, device=DEV)
        if pattern == "few":
            masked |= torch.arange(V, device=DEV) % 13 != 5
        elif pattern == "end":
            masked[..., V // 3:] = True
        elif pattern == "one row":
            masked[:, W - 1] = True
        else:
            masked |= torch.arange(V, device=DEV) != V - 1
        x[masked] = mask
        got, tokens, parents, _ = ops.beam_select(x, scores, keep=keep)
        lse = torch.logsumexp(x.double(), -1)
        f = (scores.double().unsqueeze(-1) + (x.double() - lse.unsqueeze(-1))).flatten(1)
        at = parents.long() * V + tokens
        row = lambda t: t.gather(1, parents.long())  # noqa: E731
        # an fp32 sum of exponentials, its logarithm, two differences, of the numbers that enter the kept score
        tol = 2.0 ** -21 * (row(scores).double().abs() + row(lse).abs() + x.flatten(1).gather(1, at).double().abs() + 12)
        assert (torch.isfinite(got) & ((got.double() - f.gather(1, at)).abs() <= tol)).all(), pattern
        assert ((got.double() - f.topk(keep, -1).values).abs() <= tol).all(), pattern
        hit = masked.flatten(1).gather(1, at)
        if pattern == "one row":       # masked alike, none is better than another: the row is one more distribution
            hit = hit & (parents != W - 1)
        allowed = V if pattern == "one row" else int((~masked[0]).sum())
        assert (hit.sum(1) == max(0, keep - allowed)).all(), pattern
        if pattern == "a token each" and abs(mask) > 1e9:       # what is left is alike in 32 bits: by the index
            rest = max(0, keep - W)
            assert torch.equal(tokens[:, keep - rest:], torch.arange(rest, device=DEV).expand(B, -1))
            assert (parents[:, keep - rest:] == 0).all()
    _lib.check_status(got.device)


@pytest.mark.parametrize("B,W,V,keep", [(2, 3, 1000, 4), (1, 4, 32000, None), (3, 17, 500, 20), (2, 32, 8000, None), (1, 1, 200003, 3)])
def test_behind_a_failed_kernel(B, W, V, keep):
    """Nothing is selected, and what comes back are tokens and parents all the same: they go on as indices."""
    logits = torch.randn(B, W, V, generator=_gen(V), device=DEV)
    scores, n = torch.randn(B, W, generator=_gen(W), device=DEV), keep or W
    _lib.check_status(logits.device)
    used = [torch.full((B, n), 1 << 40, dtype=t, device=DEV) if t is torch.int64 else torch.full((B, n), 99, dtype=t, device=DEV)
            for t in (torch.float32, torch.int64, torch.int32, torch.uint8) for _ in range(3)]
    del used                                 # what the outputs find in their place
    _lib.status_word(logits.device).fill_(5)
    got, tokens, parents, ended = ops.beam_select(logits, scores, eos=7, keep=keep)
    assert (got == -math.inf).all() and (tokens == 0).all() and (parents == 0).all() and ended.all()
    with pytest.raises(_lib.KernelError):
        _lib.check_status(logits.device)
    _check(logits, scores, eos=7, keep=keep)
