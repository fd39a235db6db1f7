"""16-bit paged cache on the GPU against the formulas in 64 bits: append with rotation, attention with its weights, eviction."""
import math

import pytest
import torch

from atorch_b200 import _lib, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _table(rows, width, pages, seed=0):
    return torch.randperm(pages, generator=_gen(seed), device=DEV)[: rows * width].to(torch.int32).view(rows, width)


def _filled(layers, pages, page, KV, D, dtype, seed=0):
    cache = ops.KVCache(layers, pages, page, KV, D, dtype, DEV)
    cache.data.copy_(torch.randn(cache.data.shape, generator=_gen(seed), device=DEV) * 1.3)
    return cache


def _ints(*v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _poison(layer, table, lengths):
    """Places that no token fills hold anything, and entries that no token needs name no page."""
    page = layer.shape[3]
    for b, n in enumerate(lengths):
        t = torch.arange(n, -(-n // page) * page, device=DEV)
        layer[table[b, t // page].long(), :, :, t % page] = torch.tensor([float("nan"), float("inf")], device=DEV, dtype=layer.dtype)[t % 2][:, None, None, None]
        table[b, -(-n // page):] = -7


def _exact(q, layer, table, lengths, scale):
    """Output, its tolerance, logarithms of the denominators, sums of the weights and their tolerance, in 64 bits."""
    B, S, H, D = q.shape
    KV, page = layer.shape[2], layer.shape[3]
    unit = torch.finfo(q.dtype).eps / 2
    out = torch.zeros(B, S, H, D, dtype=torch.float64, device=DEV)
    tol = torch.zeros_like(out)
    lse = torch.full((B, H, S), -math.inf, dtype=torch.float64, device=DEV)
    sums = torch.zeros(B, KV, table.shape[1] * page, dtype=torch.float64, device=DEV)
    sums_tol = torch.zeros_like(sums)
    for b, n in enumerate(lengths):
        if n == 0:
            continue
        t = torch.arange(n, device=DEV)
        kv = layer[table[b, t // page].long(), :, :, t % page].double()
        k, v = kv[:, 0].repeat_interleave(H // KV, 1), kv[:, 1].repeat_interleave(H // KV, 1)
        for i in range(S):
            m = n - S + i + 1
            if m <= 0:
                continue
            s = torch.einsum("hd,thd->ht", q[b, i].double(), k[:m]) * scale
            size = torch.einsum("hd,thd->ht", q[b, i].double().abs(), k[:m].abs()) * abs(scale)
            # a score is an fp32 sum of D products; its factor and the distance to the maximum are rounded too
            off = (size * (D + 8) * 2.0 ** -24).amax(-1, keepdim=True) + 2.0 ** -20
            p = torch.softmax(s, -1)
            out[b, i] = torch.einsum("ht,thd->hd", p, v[:m])
            # weights are rounded to 16 bits for their product with the values, and the result once more
            tol[b, i] = unit * out[b, i].abs() + (2 * unit + 2 * off) * torch.einsum("ht,thd->hd", p, v[:m].abs())
            lse[b, :, i] = torch.logsumexp(s, -1)
            sums[b, :, :m] += p.view(KV, H // KV, m).sum(1)
            sums_tol[b, :, :m] += (2 * off * p).view(KV, H // KV, m).sum(1)
    return out, tol, lse, sums, sums_tol


def _check(q, layer, table, lengths, scale=None, start=None):
    n = _ints(*lengths) if lengths else _ints()
    KV, places = layer.shape[2], table.shape[1] * layer.shape[3] + 5
    before = start if start is not None else torch.rand(len(lengths), KV, places, generator=_gen(9), device=DEV) * 3
    weights = before.clone()
    out, lse = ops.kv_attention(q, layer, table, n, scale, return_lse=True)
    weighed = ops.kv_attention(q, layer, table, n.long(), scale, weights=weights)
    assert torch.equal(out, weighed)                                  # one order of sums
    again = before.clone()
    ops.kv_attention(q, layer, table, n, scale, weights=again)
    assert torch.equal(again, weights)
    want, tol, want_lse, sums, sums_tol = _exact(q, layer, table, lengths, scale if scale is not None else q.shape[3] ** -0.5)
    assert out.shape == q.shape and out.dtype == q.dtype
    off = (out.double() - want).abs() - tol
    assert (off <= 1e-30).all(), off.max()
    seen = want_lse > -math.inf
    assert torch.equal(seen, lse > -math.inf)
    assert ((lse.double() - want_lse).abs()[seen] <= (1e-5 + 2.0 ** -20 * want_lse.abs())[seen] + 1e-4).all()
    got = weights.double()[..., : sums.shape[-1]] - before.double()[..., : sums.shape[-1]]
    # added to what is there in fp32, head after head
    off = (got - sums).abs() - sums_tol - 2.0 ** -24 * (2 + q.shape[1] * q.shape[2] // KV) * (before[..., : sums.shape[-1]].double() + sums)
    assert (off <= 0).all(), off.max()
    for b, m in enumerate(lengths):
        assert torch.equal(weights[b, :, m:], before[b, :, m:])
    _lib.check_status(out.device)
    return out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,KV,S,page", [(1, 1, 1, 16), (16, 16, 1, 16), (32, 8, 1, 64), (6, 2, 3, 32), (16, 1, 1, 16), (40, 8, 9, 128),
                                         (24, 2, 2, 16), (14, 2, 31, 32)])
def test_attention(D, H, KV, S, page, dtype):
    lengths = [0, 1, 15, 16, 17, 63, 64, 65, 127, 700, 1025, 2]
    width = -(-max(lengths) // page)
    layer = _filled(2, len(lengths) * width + 3, page, KV, D, dtype, seed=D + H).layer(1)
    table = _table(len(lengths), width, len(lengths) * width + 3)
    _poison(layer, table, lengths)
    fused = (torch.randn(len(lengths), S, H + 2 * KV, D, generator=_gen(1), device=DEV) * 1.5).to(dtype)
    _check(fused[:, :, :H], layer, table, lengths)
    _check(fused[:, :, :H].contiguous(), layer, table, lengths, scale=0.3)


@pytest.mark.parametrize("lengths", [[9001], [30000, 5], [1] * 300, [64] * 37 + [4097], [0, 0], [256] * 3, [257] * 3])
def test_attention_split_over_the_gpu(lengths):
    """One sequence over many blocks, many sequences over one, both at once, none."""
    page, KV, D = 32, 2, 128
    width = max(1, -(-max(lengths) // page))
    layer = _filled(1, len(lengths) * width, page, KV, D, torch.bfloat16, seed=3).layer(0)
    q = torch.randn(len(lengths), 1, 8, D, generator=_gen(4), device=DEV).bfloat16() * 2
    _check(q, layer, _table(len(lengths), width, len(lengths) * width), lengths)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("H,S", [(4, 1), (4, 5), (16, 4)])
def test_what_a_query_does_not_see_does_not_reach_it(H, S, dtype):
    """NaN and infinities among the last tokens: queries before them are as if they were not there."""
    page, KV, D, lengths = 16, 2, 64, [3, 40, 333]
    layer = _filled(1, 64, page, KV, D, dtype, seed=8).layer(0)
    table = _table(3, 21, 64)
    q = torch.randn(3, S, H, D, generator=_gen(2), device=DEV).to(dtype)
    clean = ops.kv_attention(q, layer, table, _ints(*lengths), return_lse=True)
    weights = torch.zeros(3, KV, 21 * page, device=DEV)
    for back in range(1, S + 1):
        for which, bad in ((0, float("nan")), (1, float("nan")), (1, float("inf")), (0, float("inf"))):
            spoiled = layer.clone()
            for b, n in enumerate(lengths):
                if n - back >= 0:
                    spoiled[table[b, (n - back) // page].long(), which, 0, (n - back) % page, 3] = bad
            out, lse = ops.kv_attention(q, spoiled, table, _ints(*lengths), return_lse=True, weights=weights)
            g = H // KV
            for i in range(S):
                hit = i >= S - back                    # the query sees the place
                if not hit:
                    assert torch.equal(out[:, i], clean[0][:, i]) and torch.equal(lse[:, :, i], clean[1][:, :, i])
                else:
                    assert torch.equal(out[:, i, g:], clean[0][:, i, g:])        # the other head has nothing of it
                    for b, n in enumerate(lengths):
                        if n - back >= 0 and which == 1:
                            assert not torch.isfinite(out[b, i, :g, 3]).any() and torch.isfinite(out[b, i, :g, 4:]).all()
    _lib.check_status(q.device)


def test_scores_of_minus_infinity_and_large_ones():
    page, KV, D = 16, 1, 64
    layer = _filled(1, 40, page, KV, D, torch.bfloat16, seed=1).layer(0)
    table = _table(2, 20, 40)
    q = torch.randn(2, 1, 1, D, generator=_gen(1), device=DEV).bfloat16()
    _check(q * 200, layer, table, [300, 7])           # one weight has nearly all
    _check(q * 1e-20, layer, table, [300, 7])
    _check(q, layer, table, [300, 7], scale=0.0)
    _check(q, layer, table, [300, 7], scale=-0.2)
    # keys of -inf in a dim where the query is positive: no weight for any of them
    layer[table[1, 0].long(), 0, 0, :7, 5] = -math.inf
    q[1, 0, 0, 5] = 1.0
    weights = torch.zeros(2, 1, 320, device=DEV)
    out, lse = ops.kv_attention(q, layer, table, _ints(300, 7), return_lse=True, weights=weights)
    assert (out[1] == 0).all() and lse[1].item() == -math.inf and (weights[1] == 0).all() and torch.isfinite(out[0]).all()
    layer[table[1, 0].long(), 0, 0, 2, 5] = 0.0       # one of the places has a weight after all
    out = ops.kv_attention(q, layer, table, _ints(300, 7), weights=weights)
    assert torch.equal(out[1, 0, 0], layer[table[1, 0].long(), 1, 0, 2]) and weights[1, 0, 2] == 1 and weights[1].sum() == 1


def test_a_score_far_above_the_others_late_in_the_sequence():
    """The running maximum moves by more than a type's range; what came before has no weight left."""
    for dtype in (torch.bfloat16, torch.float16):
        layer = _filled(1, 64, 16, 1, 64, dtype, seed=2).layer(0)
        table = _table(1, 64, 64)
        flat = table[0].long()
        t = torch.arange(1024, device=DEV)
        layer[flat[t // 16], 0, 0, t % 16] = 0.01
        for late in (1, 17, 500, 1010, 1023):
            spoiled = layer.clone()
            spoiled[flat[late // 16], 0, 0, late % 16] = 60.0
            _check(torch.full((1, 1, 2, 64), 2.0, device=DEV, dtype=dtype), spoiled, table, [1024])


def test_offsets_over_32_bits():
    page, KV, D = 64, 8, 128
    pages = (1 << 31) // (2 * KV * page * D) + 300          # more than 2^31 elements, 2^32 bytes
    layer = torch.empty(pages, 2, KV, page, D, dtype=torch.bfloat16, device=DEV)
    table = torch.stack([torch.arange(pages - 20, pages, device=DEV), torch.arange(5, 25, device=DEV)]).to(torch.int32)
    layer[table.flatten().long()] = torch.randn(40, 2, KV, page, D, generator=_gen(1), device=DEV).bfloat16()
    q = torch.randn(2, 1, 16, D, generator=_gen(2), device=DEV).bfloat16()
    _check(q, layer, table, [1270, 1111])
    x = torch.randn(2, (16 + 2 * KV) * D, generator=_gen(3), device=DEV).bfloat16()
    ops.kv_append(layer, table, None, _ints(1279, 1279), x, 16)
    want = x.view(2, -1, D)[:, 16:].view(2, 2, KV, D)
    assert torch.equal(layer[table[:, 19].long(), :, :, 63], want)
    weights = torch.rand(2, KV, 1280, generator=_gen(4), device=DEV)
    keep = layer[table.flatten().long()].cpu(), weights.cpu()
    n = ops.kv_evict(layer, table, _ints(1280, 1280), weights, 700, 30)
    small = keep[0].clone()
    other = ops.kv_evict(small, torch.arange(40, dtype=torch.int32).view(2, 20), torch.tensor([1280, 1280]), keep[1], 700, 30)
    assert torch.equal(layer[table.flatten().long()].cpu(), small) and torch.equal(weights.cpu(), keep[1]) and torch.equal(n.cpu(), other)
    _lib.check_status(q.device)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,n_q,KV,page,T", [(64, 4, 2, 16, 77), (128, 32, 8, 64, 33), (128, 0, 1, 16, 5), (64, 3, 3, 32, 200),
                                             (128, 32, 32, 16, 1), (128, 32, 8, 32, 3000)])
@pytest.mark.parametrize("rope", ["none", "places", "angles"])
def test_append(D, n_q, KV, page, T, rope, dtype):
    width = -(-T // page) + 1
    cache = _filled(2, 2 * width + 2, page, KV, D, dtype, seed=5)
    table = _table(2, width, 2 * width + 2)
    pos = torch.randperm(width * page, generator=_gen(1), device=DEV)[:T]
    seq = torch.randint(0, 2, (T,), generator=_gen(2), device=DEV)
    angles = torch.randint(0, 5000, (T,), generator=_gen(3), device=DEV)
    pos[T // 2] = -1
    angles[T // 2] = -900                 # of padding: not looked at
    x = torch.randn(T, (n_q + 2 * KV) * D, generator=_gen(4), device=DEV).to(dtype)
    kw = {} if rope == "none" else dict(zip(("cos", "sin"), ops.rope_tables(5000, D, device=DEV)))
    if rope == "angles":
        kw["angles"] = angles
    before = cache.data.clone()
    q, k = ops.kv_append(cache.layer(1), table, seq, pos, x, n_q, **kw, return_keys=True)
    _lib.check_status(x.device)
    want = before[1].cpu()
    wq, wk = ops.kv_append_reference(want, table.cpu(), seq.cpu(), pos.cpu(), x.cpu(), n_q,
                                     *((kw["cos"].cpu(), kw["sin"].cpu()) if kw else ()), angles=angles.cpu() if rope == "angles" else None)
    assert torch.equal(q.cpu(), wq) and torch.equal(k.cpu(), wk)
    assert torch.equal(cache.layer(1).cpu(), want) and torch.equal(cache.layer(0), before[0])
    # against the formula in 64 bits: two roundings of fp32 products, one of their sum, one of the result
    if kw:
        at = (angles if rope == "angles" else pos).clamp(min=0)
        c, s = kw["cos"][at].double()[:, None], kw["sin"][at].double()[:, None]
        u, v = x.view(T, -1, D)[:, : n_q + KV].double().split(D // 2, -1)
        full = torch.cat([u * c - v * s, v * c + u * s], -1)
        size = torch.cat([(u * c).abs() + (v * s).abs(), (v * c).abs() + (u * s).abs()], -1)
        off = (torch.cat([q, k], 1).double() - full).abs() - torch.finfo(dtype).eps / 2 * full.abs() - 2.0 ** -22 * size
        assert (off[pos >= 0] <= 2.0 ** -25).all()           # (fp16 below its normal numbers)
    # a strided view, heads and dims apart, off its alignment
    wide = torch.zeros(T, 3 + (n_q + 2 * KV) * D, dtype=dtype, device=DEV)
    wide[:, 3:] = x
    cache.data.copy_(before)
    assert torch.equal(ops.kv_append(cache.layer(1), table, seq, pos.int(), wide[:, 3:], n_q, **kw), q)
    assert torch.equal(cache.layer(1).cpu(), want)


def _evict(layers, lengths, KV, D, page, budget, recent, weights, dtype=torch.bfloat16, seed=0):
    width = max(1, -(-max(lengths) // page))
    rows = len(lengths)
    cache = _filled(layers, rows * width + 1, page, KV, D, dtype, seed=seed)
    table = _table(rows, width, rows * width + 1, seed)
    for b, n in enumerate(lengths):
        table[b, -(-n // page):] = -3 if n > 0 else 1 << 30
    want, want_w, before = cache.data.cpu(), weights.cpu(), cache.data.clone()
    n = _ints(*lengths)
    got = ops.kv_evict(cache.data, table, n, weights, budget, recent)
    _lib.check_status(n.device)
    assert torch.equal(n, _ints(*lengths))
    new = ops.kv_evict_reference(want, table.cpu().clamp(0, rows * width), n.cpu(), want_w, budget, recent)
    assert torch.equal(got.cpu(), new) and got.dtype == torch.int32
    assert torch.equal(weights.cpu(), want_w)
    assert torch.equal(cache.data.cpu(), want)
    return before, cache.data, table


@pytest.mark.parametrize("D,page,KV", [(64, 16, 3), (128, 64, 1), (128, 16, 8)])
@pytest.mark.parametrize("budget,recent", [(1, 0), (1, 1), (17, 0), (100, 100), (100, 33), (255, 1), (256, 256), (511, 7), (700, 64)])
def test_evict(D, page, KV, budget, recent):
    lengths = [701, 0, 1, budget, budget + 1, 255, 256, 257, 512, 700]
    weights = torch.rand(2, len(lengths), KV, 704, generator=_gen(budget), device=DEV) ** 4
    _evict(2, lengths, KV, D, page, budget, recent, weights)


@pytest.mark.parametrize("kind", ["ties", "zeros", "same", "signs", "nan", "inf", "rising", "falling", "tiny"])
def test_evict_by_unusual_weights(kind):
    lengths, places = [1300, 1025, 40], 1312
    w = torch.randint(0, 4, (1, 3, 2, places), generator=_gen(1), device=DEV).float()
    if kind == "zeros":
        w.zero_()
        w[..., ::3] = -0.0
    if kind == "same":
        w.fill_(0.7)
    if kind == "signs":
        w = torch.randn(w.shape, generator=_gen(2), device=DEV)
    if kind == "nan":
        w[torch.rand(w.shape, generator=_gen(3), device=DEV) < 0.5] = float("nan")
    if kind == "inf":
        w[torch.rand(w.shape, generator=_gen(3), device=DEV) < 0.5] = float("inf")
    if kind in ("rising", "falling"):
        w = torch.arange(places, device=DEV).float().expand(w.shape) * (1 if kind == "rising" else -1)
    if kind == "tiny":
        w = torch.randint(0, 1 << 20, w.shape, generator=_gen(4), device=DEV, dtype=torch.int32).view(torch.float32)      # subnormal
    for budget, recent in ((1000, 10), (30, 30), (39, 0), (1024, 500)):
        width_w = torch.where(torch.isnan(w), torch.full_like(w, 0.0), w).clone() if kind == "nan" else w.clone()
        if kind == "nan":              # a NaN among the sums: compared as -inf
            width_w = w.clone()
            got = width_w.clone()
            cache = _filled(1, 3 * 82, 16, 2, 64, torch.float16)
            table = _table(3, 82, 3 * 82)
            want, want_w = cache.data.cpu(), width_w.cpu()
            ops.kv_evict(cache.data, table, _ints(*lengths), got, budget, recent)
            ops.kv_evict_reference(want, table.cpu(), torch.tensor(lengths), want_w, budget, recent)
            assert torch.equal(cache.data.cpu(), want) and torch.equal(torch.nan_to_num(got.cpu(), -5), torch.nan_to_num(want_w, -5))
        else:
            _evict(1, lengths, 2, 64, 16, budget, recent, width_w, torch.float16)


@pytest.mark.parametrize("layers,lengths,KV,D,page,budget,recent", [
    (1, [30011], 2, 128, 32, 15000, 100), (1, [70001, 3], 1, 64, 64, 69000, 0), (16, [300, 280] * 4, 4, 64, 16, 256, 16),
    (3, [4097] * 5, 1, 128, 16, 4096, 0), (2, [9000] * 9, 8, 128, 64, 1000, 1000)])
def test_evict_sizes(layers, lengths, KV, D, page, budget, recent):
    width = -(-max(lengths) // page)
    weights = torch.rand(layers, len(lengths), KV, width * page + 3, generator=_gen(3), device=DEV)
    _evict(layers, lengths, KV, D, page, budget, recent, weights)


def test_evict_one_layer_and_within_the_budget():
    cache = _filled(1, 8, 16, 2, 64, torch.bfloat16)
    table, n = _table(2, 4, 8), _ints(60, 20)
    weights = torch.rand(2, 2, 64, generator=_gen(1), device=DEV)
    a, b = cache.data.clone(), cache.data.clone()
    w1, w2 = weights.clone(), weights.clone()
    m1 = ops.kv_evict(a[0], table, n, w1, 31, 4)
    m2 = ops.kv_evict(b, table, n, w2[None], 31, 4)
    assert torch.equal(a, b) and torch.equal(w1, w2) and torch.equal(m1, m2) and m1.tolist() == [31, 20] and not torch.equal(a, cache.data)
    for budget in (60, 64, 1000, 1 << 31):
        m = ops.kv_evict(a, table, m1, w1[None], budget, 2)
        assert torch.equal(m, m1) and m.data_ptr() != m1.data_ptr() and torch.equal(a, b) and torch.equal(w1, w2)


def test_append_attend_and_evict_as_steps():
    """A decode loop over a budget, each step against the CPU's on the same state."""
    B, H, KV, D, page, budget, slack = 3, 8, 2, 64, 16, 40, 8
    width = -(-(budget + slack) // page)
    cache = ops.KVCache(1, B * width, page, KV, D, torch.float16, DEV)
    table = _table(B, width, B * width)
    weights = torch.zeros(1, B, KV, width * page, device=DEV)
    cos, sin = ops.rope_tables(200, D, device=DEV)
    lengths, position = _ints(0, 0, 0), 0
    for step in range(90):
        x = torch.randn(B, (H + 2 * KV) * D, generator=_gen(step), device=DEV).half()
        before = cache.data.cpu(), weights.cpu()
        q = ops.kv_append(cache.layer(0), table, None, lengths, x, H, cos, sin, angles=torch.full_like(lengths, position))
        now = lengths + 1
        out = ops.kv_attention(q.unsqueeze(1), cache.layer(0), table, now, weights=weights[0])
        cpu = before[0].clone()
        wq, _ = ops.kv_append_reference(cpu[0], table.cpu(), None, lengths.cpu(), x.cpu(), H, cos.cpu(), sin.cpu(),
                                        torch.full((B,), position))
        assert torch.equal(q.cpu(), wq) and torch.equal(cache.data.cpu(), cpu)
        w = before[1].clone()
        want, _ = ops.kv_attention_reference(wq.unsqueeze(1), cpu[0], table.cpu(), now.cpu(), weights=w[0])
        assert (out.cpu().float() - want.float()).abs().max() < 2e-2 and (weights.cpu() - w).abs().max() < 1e-3
        lengths, position = now, position + 1
        if step % slack == slack - 1:
            cpu, w = cache.data.cpu(), weights.cpu()
            lengths = ops.kv_evict(cache.data, table, lengths, weights, budget, 10)
            assert torch.equal(lengths.cpu(), ops.kv_evict_reference(cpu, table.cpu(), now.cpu(), w, budget, 10))
            assert torch.equal(cache.data.cpu(), cpu) and torch.equal(weights.cpu(), w)
    assert lengths.tolist() == [42] * 3
    _lib.check_status(x.device)


def test_captured_steps_share_nothing():
    """Two captured graphs replayed at once on two streams, and an eager call beside them, with lengths that change between replays."""
    page, KV, D, H, B = 16, 2, 128, 8, 4
    width = 100
    layer = _filled(1, B * width, page, KV, D, torch.bfloat16, seed=3).layer(0)
    table, n = _table(B, width, B * width), _ints(1590, 3, 700, 0)
    qs = [torch.randn(B, 1, H, D, generator=_gen(i), device=DEV).bfloat16() for i in range(2)]
    ws = [torch.zeros(B, KV, width * page, device=DEV) for _ in range(2)]
    for q, w in zip(qs, ws):
        ops.kv_attention(q, layer, table, n, weights=w.clone())
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for q, w in zip(qs, ws):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(ops.kv_attention(q, layer, table, n, weights=w))
        graphs.append(graph)
    for lengths in ([1590, 3, 700, 0], [5, 1600, 1, 900], [0, 0, 0, 0]):
        n.copy_(_ints(*lengths))
        want = [ops.kv_attention(q, layer, table, n) for q in qs]
        for w in ws:
            w.zero_()
        torch.cuda.synchronize()
        for _ in range(3):
            for graph, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    graph.replay()
        ops.kv_attention(qs[0], layer, table, n)
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(outs[i], want[i])
            w = torch.zeros_like(ws[i])
            for _ in range(3):
                ops.kv_attention(qs[i], layer, table, n, weights=w)
            assert torch.equal(w, ws[i])
    _lib.check_status(layer.device)


def test_a_captured_cut():
    cache = _filled(2, 30, 16, 2, 64, torch.bfloat16, seed=1)
    table, n = _table(3, 10, 30), _ints(150, 90, 33)
    weights = torch.rand(2, 3, 2, 160, generator=_gen(1), device=DEV)
    ops.kv_evict(cache.data.clone(), table, n, weights.clone(), 64, 8)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    a, w = cache.data.clone(), weights.clone()
    with torch.cuda.graph(graph):
        m = ops.kv_evict(a, table, n, w, 64, 8)
    for lengths in ([150, 90, 33], [64, 65, 160], [0, 1, 2]):
        a.copy_(cache.data), w.copy_(weights), n.copy_(_ints(*lengths))
        graph.replay()
        b, v = cache.data.clone(), weights.clone()
        assert torch.equal(m, ops.kv_evict(b, table, n, v, 64, 8)) and torch.equal(a, b) and torch.equal(w, v)


def test_indices_out_of_range_are_reported():
    D, KV = 64, 2
    cache = ops.KVCache(1, 4, 16, KV, D, device=DEV)
    layer = cache.layer(0)
    table = torch.tensor([[0, 1], [2, 9]], dtype=torch.int32, device=DEV)
    x = torch.randn(2, (2 + 2 * KV) * D, device=DEV).bfloat16()
    cos, sin = ops.rope_tables(30, D, device=DEV)
    dev = x.device
    _lib.check_status(dev)
    for seq, pos, kw in (([0, 1], [0, 20], {}), ([0, 1], [32, 0], {}), ([0, 2], [0, 0], {}), ([0, -1], [0, 0], {}), ([0, 0], [0, 31], dict(cos=cos, sin=sin)),
                         ([0, 0], [0, 1], dict(cos=cos, sin=sin, angles=_ints(0, 30))), ([0, 0], [0, 1], dict(cos=cos, sin=sin, angles=_ints(0, -1)))):
        ops.kv_append(layer, table, torch.tensor(seq, device=dev), torch.tensor(pos, device=dev), x, 2, **kw)
        with pytest.raises(_lib.KernelError):
            _lib.check_status(dev)
    q = torch.randn(2, 1, 4, D, device=dev).bfloat16()
    for lengths in ([3, 20], [33, 1]):
        ops.kv_attention(q, layer, table, _ints(*lengths))
        with pytest.raises(_lib.KernelError):
            _lib.check_status(dev)
    before = cache.data.clone()
    for lengths in ([3, 20], [1, 33]):
        weights = torch.rand(1, 2, KV, 32, device=dev)
        ops.kv_evict(cache.data, table, _ints(*lengths), weights, 10, 2)
        with pytest.raises(_lib.KernelError):
            _lib.check_status(dev)
        assert torch.equal(cache.data, before)
    # behind a failed kernel nothing is stored
    weights = torch.rand(1, 2, KV, 32, device=dev)
    kept = weights.clone()
    _lib.status_word(dev).fill_(1)
    ops.kv_append(layer, table, None, _ints(0, 0), x, 2)
    ops.kv_attention(q, layer, table, _ints(20, 3), weights=weights[0])
    ops.kv_evict(cache.data, table, _ints(20, 3), weights, 10, 2)
    with pytest.raises(_lib.KernelError):
        _lib.check_status(dev)
    assert torch.equal(cache.data, before) and torch.equal(weights, kept)
    _lib.check_status(dev)


def test_empty_calls():
    cache = ops.KVCache(1, 4, 16, 2, 64, device=DEV)
    table, none = torch.zeros(0, 2, dtype=torch.int32, device=DEV), _ints()
    assert ops.kv_append(cache.layer(0), table, None, none, torch.zeros(0, 8 * 64, device=DEV).bfloat16(), 4).shape == (0, 4, 64)
    assert ops.kv_attention(torch.zeros(0, 1, 4, 64, device=DEV).bfloat16(), cache.layer(0), table, none).shape == (0, 1, 4, 64)
    assert ops.kv_attention(torch.zeros(0, 1, 4, 64, device=DEV).bfloat16(), cache.layer(0), table, none,
                            weights=torch.zeros(0, 2, 32, device=DEV)).shape == (0, 1, 4, 64)
    assert ops.kv_evict(cache.data, table, none, torch.zeros(1, 0, 2, 32, device=DEV), 4).shape == (0,)
    # a table without columns: nothing to see
    nothing = torch.zeros(2, 0, dtype=torch.int32, device=DEV)
    q = torch.ones(2, 3, 4, 64, device=DEV).bfloat16()
    out, lse = ops.kv_attention(q, cache.layer(0), nothing, _ints(0, 0), return_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()
    assert (ops.kv_attention(q, cache.layer(0), nothing, _ints(0, 0), weights=torch.zeros(2, 2, 0, device=DEV)) == 0).all()
    assert ops.kv_evict(cache.data, nothing, _ints(0, 0), torch.zeros(1, 2, 2, 0, device=DEV), 4).tolist() == [0, 0]
    _lib.check_status(q.device)
    one = torch.zeros(1, 2, dtype=torch.int32, device=DEV)
    assert ops.kv_attention(torch.zeros(1, 0, 4, 64, device=DEV).bfloat16(), cache.layer(0), one, _ints(3)).shape == (1, 0, 4, 64)


def test_refusals():
    from test_kv_cpu import check_refusals

    check_refusals(DEV)
    odd = ops.KVCache(1, 4, 16, 2, 96, device=DEV)
    table, q = torch.zeros(1, 2, dtype=torch.int32, device=DEV), torch.zeros(1, 1, 4, 96, device=DEV).bfloat16()
    with pytest.raises(ValueError):
        ops.kv_attention(q, odd.layer(0), table, _ints(1))


@pytest.mark.parametrize("layers,KV,width,long", [(1, 2, 4, 65), (3, 40, 4, 1000), (1, 1, 300, 4801), (1, 2, 300, 1 << 30)])
@pytest.mark.parametrize("wrong", ["length", "page"])
def test_a_cut_leaves_what_is_out_of_range(layers, KV, width, long, wrong):
    """A sequence longer than its row, whose pages are all there, or with a page that is not: it stays, whole, and the others are cut."""
    D, page = 64, 16
    lengths = [width * page, long if wrong == "length" else width * page, width * page - 3, 20]
    table = _table(4, width, 4 * width)
    cache = _filled(layers, 4 * width, page, KV, D, torch.bfloat16)
    weights = torch.rand(layers, 4, KV, width * page, generator=_gen(1), device=DEV)
    if wrong == "page":
        table[1, width - 1] = 4 * width
    data, kept = cache.data.clone(), weights.clone()
    got = ops.kv_evict(cache.data, table, _ints(*lengths), weights, 30, 5)
    with pytest.raises(_lib.KernelError):
        _lib.check_status(table.device)
    rest = _ints(0, 2, 3).long()
    kept_rest = kept[:, rest].contiguous()
    want = ops.kv_evict_reference(data, table[rest], _ints(*(lengths[b] for b in (0, 2, 3))), kept_rest, 30, 5)
    assert torch.equal(got[rest], want) and (wrong == "page" or int(got[1]) == long)
    assert torch.equal(weights[:, rest], kept_rest) and torch.equal(weights[:, 1], kept[:, 1])
    assert torch.equal(cache.data, data)


def test_lengths_out_of_range_under_a_budget_that_no_sequence_is_over():
    cache = _filled(1, 4, 16, 2, 64, torch.bfloat16)
    table, weights = _table(2, 2, 4), torch.rand(1, 2, 2, 32, device=DEV)
    before = cache.data.clone(), weights.clone()
    for budget in (32, 33, 1 << 40):
        assert ops.kv_evict(cache.data, table, _ints(32, 5), weights, budget, 3).tolist() == [32, 5]
        _lib.check_status(table.device)
        ops.kv_evict(cache.data, table, _ints(5, 33), weights, budget, 3)
        with pytest.raises(_lib.KernelError):
            _lib.check_status(table.device)
    assert torch.equal(cache.data, before[0]) and torch.equal(weights, before[1])


@pytest.mark.parametrize("room", [1, 4000, 20000, 1 << 20])
def test_attention_with_weights_in_pieces(room, monkeypatch):
    """Scores that are too many at once: pieces of sequences, and of the tokens of one, down to one token."""
    monkeypatch.setattr(ops.kv, "SCORES", room)
    D, KV, page, S = 64, 2, 16, 9
    lengths = [0, 1, 5, 9, 10, 300, 77]
    layer = _filled(1, 7 * 19, page, KV, D, torch.bfloat16).layer(0)
    table = _table(7, 19, 7 * 19)
    _poison(layer, table, lengths)
    q = (torch.randn(7, S, 6, D, generator=_gen(1), device=DEV) * 1.5).bfloat16()
    before = torch.rand(7, KV, 19 * page + 3, generator=_gen(2), device=DEV)
    weights = before.clone()
    out, lse = ops.kv_attention(q, layer, table, _ints(*lengths), return_lse=True, weights=weights)
    want, tol, want_lse, sums, sums_tol = _exact(q, layer, table, lengths, D ** -0.5)
    assert out.shape == q.shape and lse.shape == (7, 6, S) and ((out.double() - want).abs() <= tol).all()
    seen = want_lse > -math.inf
    assert torch.equal(seen, lse > -math.inf) and ((lse.double() - want_lse).abs()[seen] <= 1e-4).all()
    # one rounding for every call that adds to a place
    grown = weights.double()[..., : 19 * page] - before.double()[..., : 19 * page]
    assert ((grown - sums).abs() <= sums_tol + 2.0 ** -24 * (2 + S + S * 3) * (before[..., : 19 * page].double() + sums)).all()
    for b, n in enumerate(lengths):
        assert torch.equal(weights[b, :, n:], before[b, :, n:])
    _lib.check_status(q.device)
    # a length out of range is reported from any of them
    ops.kv_attention(q, layer, table.clamp(min=0), _ints(0, 1, 5, 9, 19 * page + 1, 300, 77), weights=weights)
    with pytest.raises(_lib.KernelError):
        _lib.check_status(q.device)


def test_the_workspace_of_weights_is_bounded():
    """16 prompts of up to 32768 tokens, 32 query heads, 32 last tokens each: 2.1 GB of scores."""
    B, S, H, KV, D, page = 16, 32, 32, 8, 64, 64
    layer = _filled(1, 64, page, KV, D, torch.bfloat16).layer(0)
    table = torch.zeros(B, 512, dtype=torch.int32, device=DEV) + torch.arange(512, device=DEV, dtype=torch.int32) % 64
    lengths = _ints(32768, *range(1, 16))
    q = torch.randn(B, S, H, D, generator=_gen(1), device=DEV).bfloat16()
    weights = torch.zeros(B, KV, 32768, device=DEV)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    held = torch.cuda.memory_allocated()
    ops.kv_attention(q, layer, table, lengths, weights=weights)
    assert torch.cuda.max_memory_allocated() - held < 320 << 20
    _lib.check_status(q.device)


@pytest.mark.parametrize("KV,n,budget", [(8, 30011, 15000), (1, 50021, 49000), (18, 9000, 8990)])
def test_rounds_of_a_cluster_again_and_again(KV, n, budget):
    """Blocks of a cluster write what others have read a round before: the same tokens every time, with other work beside."""
    D, page = 128, 64
    width = -(-n // page)
    cache, table = _filled(1, width, page, KV, D, torch.bfloat16), _table(1, width, width)
    weights = torch.randn(1, 1, KV, width * page, generator=_gen(3), device=DEV).exp()
    data, sums = cache.data.clone(), weights.clone()
    ops.kv_evict_reference(data, table, _ints(n), sums, budget, 7)
    filled, kept, beside = cache.data.clone(), weights.clone(), torch.cuda.Stream()
    for _ in range(15):
        cache.data.copy_(filled)
        weights.copy_(kept)
        beside.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(beside):
            filled.clone()
        ops.kv_evict(cache.data, table, _ints(n), weights, budget, 7)
        assert torch.equal(cache.data, data) and torch.equal(weights, sums)
    torch.cuda.current_stream().wait_stream(beside)
    _lib.check_status(table.device)
