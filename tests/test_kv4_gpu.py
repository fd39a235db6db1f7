"""4-bit paged cache on the GPU against the formulas in 64 bits: append with rotation, reading back, attention."""
import math

import pytest
import torch

from atorch_b200 import _lib, ops
from atorch_b200.ops import kv4

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _table(rows, width, pages, seed=0):
    return torch.randperm(pages, generator=_gen(seed), device=DEV)[: rows * width].to(torch.int32).view(rows, width)


def _fill(codes, scales, seed, k_scale=0.4, v_scale=0.2):
    g = _gen(seed)
    codes.copy_(torch.randint(0, 256, codes.shape, generator=g, device=DEV, dtype=torch.uint8))
    s = 0.5 + torch.rand(scales.shape, generator=g, device=DEV)
    s[..., 0] *= k_scale
    s[..., 1] *= -7.5 * k_scale
    s[..., 2] *= v_scale
    s[..., 3] *= -7.5 * v_scale
    scales.copy_(s)


def _values(layer, table, b, n):
    """Keys and values [KV, n, D] of a sequence in 64 bits."""
    codes, scales = layer
    page = codes.shape[3]
    t = torch.arange(n, device=DEV)
    rows, slot = table[b, t // page].long(), t % page
    byte = codes[rows, :, :, slot].permute(1, 2, 0, 3)
    val = torch.empty(*byte.shape[:-1], 2 * byte.shape[-1], dtype=torch.float64, device=DEV)
    val[..., 0::2], val[..., 1::2] = (byte & 15).double(), (byte >> 4).double()
    sc = scales[rows, :, slot].double().transpose(0, 1)
    return val[0] * sc[..., 0:1] + sc[..., 1:2], val[1] * sc[..., 2:3] + sc[..., 3:4], sc


def _attention(q, layer, table, lengths, scale):
    B, S, H, D = q.shape
    KV = layer[0].shape[2]
    out = torch.zeros(B, S, H, D, dtype=torch.float64, device=DEV)
    lse = torch.full((B, H, S), -math.inf, dtype=torch.float64, device=DEV)
    tol = torch.zeros(B, S, H, 1, dtype=torch.float64, device=DEV)
    for b, n in enumerate(lengths):
        if n == 0:
            continue
        k, v, sc = _values(layer, table, b, n)
        k, v, vs = (t.repeat_interleave(H // KV, 0) for t in (k, v, sc[..., 2]))
        for i in range(S):
            m = n - S + i + 1
            if m <= 0:
                continue
            s = torch.einsum("hd,htd->ht", q[b, i].double(), k[:, :m]) * scale
            p = torch.softmax(s, -1)
            out[b, i] = torch.einsum("ht,htd->hd", p, v[:, :m])
            lse[b, :, i] = torch.logsumexp(s, -1)
            # p vs is rounded to 11 bits and meets codes up to 15; scores are fp32 sums of 2 D terms of up to 15 |q| ks
            size = (q[b, i].double().abs().sum(-1) * 22.5 * float(sc[..., 0].max()) * scale)[:, None]
            tol[b, i] = (2.0 ** -11) * 15 * (p * vs[:, :m]).sum(-1, keepdim=True) + size * 2.0 ** -20 * v.abs().max()
    return out, lse, tol


def _check(q, layer, table, lengths, scale=None):
    out, lse = ops.kv4_attention(q, layer, table, torch.tensor(lengths, dtype=torch.int32, device=DEV), scale, return_lse=True)
    again = ops.kv4_attention(q, layer, table, torch.tensor(lengths, device=DEV), scale)
    assert torch.equal(out, again)                  # one order of sums
    want, want_lse, tol = _attention(q, layer, table, lengths, scale if scale is not None else q.shape[3] ** -0.5)
    unit = 2.0 ** -8 if q.dtype == torch.bfloat16 else 2.0 ** -11
    assert out.shape == q.shape and out.dtype == q.dtype
    assert ((out.double() - want).abs() <= unit * want.abs() + tol + 1e-7).all(), ((out.double() - want).abs() - unit * want.abs() - tol).max()
    seen = want_lse > -math.inf
    assert torch.equal(seen, lse > -math.inf)
    assert ((lse.double() - want_lse).abs()[seen] < 1e-4).all()
    _lib.check_status(out.device)
    return out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,KV,S,page", [(1, 1, 1, 16), (16, 16, 1, 16), (32, 8, 1, 64), (6, 2, 3, 32), (16, 1, 1, 16), (40, 8, 9, 128),
                                         (24, 2, 2, 16)])
def test_attention(D, H, KV, S, page, dtype):
    lengths = [0, 1, 15, 16, 17, 63, 64, 65, 127, 700, 1025, 2]
    width = -(-max(lengths) // page)
    cache = ops.KV4Cache(2, len(lengths) * width + 3, page, KV, D, DEV)
    _fill(*cache.layer(1), seed=D + H)
    layer = cache.layer(1)
    table = _table(len(lengths), width, len(lengths) * width + 3)
    # places that no token fills hold anything, and entries that no token needs name no page
    for b, n in enumerate(lengths):
        t = torch.arange(n, -(-n // page) * page, device=DEV)
        layer[1][table[b, t // page].long(), :, t % page] = float("nan")
        table[b, -(-n // page):] = -7
    fused = torch.randn(len(lengths), S, H + 2 * KV, D, generator=_gen(1), device=DEV).to(dtype) * 1.5
    _check(fused[:, :, :H], layer, table, lengths)
    _check(fused[:, :, :H].contiguous(), layer, table, lengths, scale=0.3)


@pytest.mark.parametrize("lengths", [[9001], [30000, 5], [1] * 300, [64] * 37 + [4097], [0, 0]])
def test_attention_split_over_the_gpu(lengths):
    """One sequence over many blocks, many sequences over one, both at once, none."""
    page, KV, D = 32, 2, 128
    width = max(1, -(-max(lengths) // page))
    cache = ops.KV4Cache(1, len(lengths) * width, page, KV, D, DEV)
    _fill(*cache.layer(0), seed=3)
    q = torch.randn(len(lengths), 1, 8, D, generator=_gen(4), device=DEV).bfloat16() * 2
    _check(q, cache.layer(0), _table(len(lengths), width, len(lengths) * width), lengths)


def test_attention_scales_far_apart():
    """Value scales over 20 powers of two, the largest at tokens that get no weight; tiny and huge queries."""
    page, D, n = 16, 64, 200
    cache = ops.KV4Cache(1, 13, page, 1, D, DEV)
    codes, scales = layer = cache.layer(0)
    _fill(codes, scales, seed=5)
    table = _table(1, 13, 13)
    t = torch.arange(n, device=DEV)
    big = (t % 5 == 4)
    size = torch.where(big, torch.full_like(t, 2.0 ** 10, dtype=torch.float), torch.full_like(t, 2.0 ** -10, dtype=torch.float))
    where = table[0, t // page].long(), 0, t % page
    scales[where[0], 0, where[2], 2] = size.bfloat16()
    scales[where[0], 0, where[2], 3] = (-7 * size).bfloat16()
    # keys: all dims alike, so that the score goes by the sum of the query; large values stand at keys 40 below the others
    codes[where[0], 0, 0, where[2]] = 0
    scales[where[0], 0, where[2], 0] = 0
    scales[where[0], 0, where[2], 1] = torch.where(big, -40.0, 0.0).bfloat16()
    q = torch.ones(1, 1, 1, D, device=DEV).bfloat16()
    _check(q, layer, table, [n])
    _fill(codes, scales, seed=6)
    for f in (1e-20, 1e4):
        x = torch.randn(1, 1, 1, D, generator=_gen(7), device=DEV).bfloat16() * f
        _check(x, layer, table, [n], scale=0.1 / f)
    # constant values: no scale at all
    scales[..., 2] = 0
    out = _check(torch.randn(1, 1, 1, D, device=DEV).half(), layer, table, [n])
    assert torch.isfinite(out).all()


def test_attention_nan_goes_where_it_is_seen():
    page, D, KV = 16, 64, 2
    cache = ops.KV4Cache(1, 8, page, KV, D, DEV)
    _fill(*cache.layer(0), seed=8)
    table = _table(2, 4, 8)
    for which in (0, 1, 2, 3):
        cache.scales[0, table[0, 1].long(), 1, 3, which], keep = float("nan"), cache.scales[0, table[0, 1].long(), 1, 3, which].clone()
        q = torch.randn(2, 4, 4, D, generator=_gen(9), device=DEV).half()
        out = ops.kv4_attention(q, cache.layer(0), table, torch.tensor([23, 50], dtype=torch.int32, device=DEV))
        seen = torch.isnan(out).all(-1)        # position 19 is behind none of the four tokens; heads 2 and 3 share the one it is in
        assert torch.equal(seen[0], torch.tensor([[False, False, True, True]] * 4, device=DEV))
        out = ops.kv4_attention(q, cache.layer(0), table, torch.tensor([22, 50], dtype=torch.int32, device=DEV))
        assert torch.equal(torch.isnan(out).all(-1)[0, :, 2:].any(-1), torch.tensor([False, True, True, True], device=DEV))
        assert not torch.isnan(out[1]).any() and not torch.isnan(out[:, :, :2]).any()
        cache.scales[0, table[0, 1].long(), 1, 3, which] = keep
    _lib.check_status(out.device)


def test_offsets_over_32_bits():
    """A cache of more than 4 GB: the last pages are found."""
    page, KV, D, pages = 64, 8, 128, 66000
    cache = ops.KV4Cache(1, pages, page, KV, D, DEV)
    assert cache.codes.numel() > 1 << 32
    layer = cache.layer(0)
    at = torch.tensor([65999, 3, 65990], device=DEV)
    table = at.to(torch.int32).view(1, 3)
    codes, scales = layer[0][at], layer[1][at]
    _fill(codes, scales, seed=10)
    layer[0][at], layer[1][at] = codes, scales
    q = torch.randn(1, 1, 16, D, generator=_gen(11), device=DEV).bfloat16()
    _check(q, layer, table, [170])
    cos, sin = ops.rope_tables(200, D, device=DEV)
    qkv = torch.randn(1, 32 * D, generator=_gen(12), device=DEV).bfloat16()
    pos = torch.tensor([170], dtype=torch.int32, device=DEV)
    ops.kv4_append(layer, table, None, pos, qkv, 16, cos, sin)
    k, v = ops.kv4_read(layer, table, None, pos)
    assert (v[0].float() - qkv.view(32, D)[24:].float()).abs().max() < 0.3
    assert layer[0][65990, 1, :, 170 % 64].any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D,n_q,KV,page,rope", [(128, 32, 8, 16, True), (64, 3, 3, 32, True), (128, 1, 1, 64, False), (64, 0, 2, 16, True)])
def test_append_and_read(D, n_q, KV, page, rope, dtype):
    g = _gen(20)
    sizes, past = [1, 40, 0, 17, 129], [0, 5, 9, 47, 60]
    width = -(-200 // page)
    cache = ops.KV4Cache(1, 5 * width + 1, page, KV, D, DEV)
    layer = cache.layer(0)
    table = _table(5, width, 5 * width + 1)
    seq = torch.repeat_interleave(torch.arange(5), torch.tensor(sizes)).to(DEV)
    pos = torch.cat([torch.arange(p, p + n) for p, n in zip(past, sizes)]).to(DEV)
    pos[7] = pos[60] = -1
    order = torch.randperm(len(seq), generator=g, device=DEV)
    seq, pos = seq[order], pos[order]
    T = len(seq)
    x = (torch.randn(T, n_q + 2 * KV, D, generator=g, device=DEV) * 3).to(dtype)
    x[3, -1] = 2.5                                        # a constant head has no scale
    wide = torch.randn(T, (n_q + 2 * KV) * D + 24, device=DEV).to(dtype)
    wide[:, : (n_q + 2 * KV) * D] = x.view(T, -1)
    cos, sin = ops.rope_tables(200, D, device=DEV) if rope else (None, None)
    before = cache.codes.clone(), cache.scales.clone()
    q = ops.kv4_append(layer, table, seq, pos, wide[:, : (n_q + 2 * KV) * D], n_q, cos, sin)
    k, v = ops.kv4_read(layer, table, seq.int(), pos.int(), torch.float32)
    _lib.check_status(q.device)
    # the kernels follow the formula operation by operation: the same codes as the plain operations
    want = before[0][0], before[1][0]
    want_q = ops.kv4_append_reference(want, table, seq, pos, x, n_q, cos, sin)
    assert torch.equal(want[0], layer[0]) and torch.equal(want[1].view(torch.int16), layer[1].view(torch.int16))
    assert torch.equal(want_q, q) and q.dtype == dtype
    for a, b in zip(ops.kv4_read_reference(want, table, seq, pos, dtype), ops.kv4_read(layer, table, seq, pos, dtype)):
        assert torch.equal(a, b)
    # and stand for the rotated values: half a step, and the rounding of scale and minimum to bf16
    xd, real = x.double(), (pos >= 0)
    if rope:
        z = torch.complex(xd[:, : n_q + KV, : D // 2], xd[:, : n_q + KV, D // 2:])
        at = pos.clamp(min=0)
        z = torch.where(real[:, None, None], z * torch.complex(cos[at].double(), sin[at].double())[:, None], z)
        xd = torch.cat([torch.cat([z.real, z.imag], -1), xd[:, n_q + KV:]], 1)
    unit = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -10, torch.float32: 2.0 ** -21}[dtype]
    assert ((q.double() - xd[:, :n_q]).abs() <= unit * xd[:, :n_q].abs() + 1e-5).all()
    for got, ideal in ((k, xd[:, n_q: n_q + KV]), (v, xd[:, n_q + KV:])):
        low, high = ideal.amin(-1, keepdim=True), ideal.amax(-1, keepdim=True)
        most = (high - low) / 15 * (0.5 + 2.0 ** -8) + 2.0 ** -8 * (low.abs() + high - low) + 1e-5
        assert ((got.double() - ideal).abs() <= most)[real].all()
        assert (got[~real] == 0).all()
    # nothing else was written
    mine = torch.zeros(5 * width + 1, page, dtype=torch.bool, device=DEV)
    mine[table[seq, pos.clamp(min=0) // page].long()[real], (pos % page)[real]] = True
    assert (layer[0].permute(0, 3, 1, 2, 4)[~mine] == 0).all() and (layer[1].permute(0, 2, 1, 3)[~mine] == 0).all()


def test_append_then_attend_as_a_step():
    """The token that a step appends is seen by its own query; another stream than the default one."""
    H, KV, D, page, B = 8, 2, 128, 16, 3
    cache = ops.KV4Cache(1, B * 4, page, KV, D, DEV)
    table = _table(B, 4, B * 4)
    cos, sin = ops.rope_tables(64, D, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.no_grad():
        for t in range(20):
            qkv = torch.randn(B, (H + 2 * KV) * D, generator=_gen(t), device=DEV).bfloat16()
            q = ops.kv4_append(cache.layer(0), table, None, torch.full((B,), t, device=DEV), qkv, H, cos, sin)
            out = ops.kv4_attention(q.view(B, 1, H, D), cache.layer(0), table, torch.full((B,), t + 1, device=DEV))
    side.synchronize()
    _check(q.view(B, 1, H, D), cache.layer(0), table, [20] * B)
    assert torch.isfinite(out).all()


def test_special_values_in_a_token():
    """NaN and infinities make their head of their token NaN, and nothing else."""
    D, KV = 64, 3
    cache = ops.KV4Cache(1, 2, 16, KV, D, DEV)
    table = torch.tensor([[1]], dtype=torch.int32, device=DEV)
    x = torch.randn(4, 2 * KV, D, generator=_gen(30), device=DEV)
    x[1, 0, 5], x[2, 4, 63], x[3, 2, 0] = float("nan"), float("inf"), -float("inf")
    seq, pos = torch.zeros(4, dtype=torch.int32, device=DEV), torch.arange(4, dtype=torch.int32, device=DEV)
    ops.kv4_append(cache.layer(0), table, seq, pos, x, 0)
    k, v = ops.kv4_read(cache.layer(0), table, seq, pos, torch.float32)
    bad = torch.zeros(4, 2 * KV, dtype=torch.bool, device=DEV)
    bad[1, 0] = bad[2, 4] = bad[3, 2] = True
    assert torch.equal(torch.isnan(torch.cat([k, v], 1)).all(-1), bad) and torch.equal(torch.isnan(torch.cat([k, v], 1)).any(-1), bad)


def test_indices_out_of_range_are_reported():
    D, KV = 64, 2
    cache = ops.KV4Cache(1, 4, 16, KV, D, DEV)
    table = torch.tensor([[0, 1], [2, 9]], dtype=torch.int32, device=DEV)
    x = torch.randn(2, (2 + 2 * KV) * D, device=DEV).bfloat16()
    cos, sin = ops.rope_tables(30, D, device=DEV)
    dev = x.device
    _lib.check_status(dev)
    for seq, pos in (([0, 1], [0, 20]), ([0, 1], [32, 0]), ([0, 2], [0, 0]), ([0, -1], [0, 0]), ([0, 0], [0, 31])):
        rope = (cos, sin) if pos[1] == 31 else (None, None)
        ops.kv4_append(cache.layer(0), table, torch.tensor(seq, device=dev), torch.tensor(pos, device=dev), x, 2, *rope)
        with pytest.raises(_lib.KernelError):
            _lib.check_status(dev)
    ops.kv4_read(cache.layer(0), table, None, torch.tensor([0, 17], device=dev))
    with pytest.raises(_lib.KernelError):
        _lib.check_status(dev)
    q = torch.randn(2, 1, 4, D, device=dev).bfloat16()
    for lengths in ([3, 20], [33, 1]):
        ops.kv4_attention(q, cache.layer(0), table, torch.tensor(lengths, device=dev))
        with pytest.raises(_lib.KernelError):
            _lib.check_status(dev)
    _lib.check_status(dev)


def test_empty_calls():
    cache = ops.KV4Cache(1, 4, 16, 2, 64, DEV)
    table = torch.zeros(0, 2, dtype=torch.int32, device=DEV)
    none = torch.zeros(0, dtype=torch.int32, device=DEV)
    assert ops.kv4_append(cache.layer(0), table, None, none, torch.zeros(0, 8 * 64, device=DEV), 4).shape == (0, 4, 64)
    assert ops.kv4_read(cache.layer(0), table, None, none)[0].shape == (0, 2, 64)
    assert ops.kv4_attention(torch.zeros(0, 1, 4, 64, device=DEV).half(), cache.layer(0), table, none).shape == (0, 1, 4, 64)


def test_refusals():
    cache = ops.KV4Cache(1, 4, 16, 2, 64, DEV)
    layer, table = cache.layer(0), torch.zeros(1, 2, dtype=torch.int32, device=DEV)
    pos = torch.zeros(1, dtype=torch.int32, device=DEV)
    x, q = torch.zeros(1, 8 * 64, device=DEV), torch.zeros(1, 1, 4, 64, device=DEV).half()
    cos, sin = ops.rope_tables(4, 64, device=DEV)
    ok = dict(layer=layer, page_table=table, seq=None, pos=pos, qkv=x, n_q=4)
    for change in (dict(n_q=3), dict(qkv=x.double()), dict(pos=pos.float()), dict(pos=torch.zeros(2, device=DEV).int()), dict(cos=cos),
                   dict(cos=cos[:, :8], sin=sin[:, :8]), dict(page_table=table.long()), dict(layer=(layer[0], layer[1].float())),
                   dict(layer=(layer[0][:, :, :, :8], layer[1][:, :, :8])), dict(page_table=table.cpu()), dict(layer=(layer[0][:2], layer[1])),
                   dict(layer=(layer[0].transpose(2, 3), layer[1]))):
        with pytest.raises(ValueError):
            ops.kv4_append(**{**ok, **change})
    with pytest.raises(RuntimeError):
        ops.kv4_append(**{**ok, "qkv": x.clone().requires_grad_()})
    n = torch.ones(1, dtype=torch.int32, device=DEV)
    for bad in ((q.float(), layer, table, n), (q[..., :32], layer, table, n), (q[:, :, :3], layer, table, n), (q[0], layer, table, n),
                (q, layer, table.repeat(2, 1), n), (q, layer, table, n.float()), (q, layer, table, n.cpu())):
        with pytest.raises(ValueError):
            ops.kv4_attention(*bad)
    with pytest.raises(RuntimeError):
        ops.kv4_attention(q.clone().requires_grad_(), layer, table, n)
    odd = ops.KV4Cache(1, 4, 16, 2, 96, DEV)
    with pytest.raises(ValueError):
        ops.kv4_read(odd.layer(0), table, None, pos)
    with pytest.raises(ValueError):
        ops.KV4Cache(1, 4, 24, 2, 64, DEV)
    assert kv4.HEAD_DIMS == (64, 128)


def _check_weighted(q, layer, table, lengths, scale):
    """As :func:`_check`, with a tolerance that goes by what the weights leave of the values: a token without weight adds nothing to it,
    however large its values are."""
    out = ops.kv4_attention(q, layer, table, torch.tensor(lengths, dtype=torch.int32, device=DEV), scale)
    want, _, _ = _attention(q, layer, table, lengths, scale)
    B, S, H, D = q.shape
    unit = 2.0 ** -8 if q.dtype == torch.bfloat16 else 2.0 ** -11
    for b, n in enumerate(lengths):
        k, v, sc = (t.repeat_interleave(H // layer[0].shape[2], 0) for t in _values(layer, table, b, n))
        for i in range(S):
            m = n - S + i + 1
            p = torch.softmax(torch.einsum("hd,htd->ht", q[b, i].double(), k[:, :m]) * scale, -1)
            # p vs is rounded to 11 bits and meets codes up to 15; a score is an fp32 sum, its exponential off by 2^-22, and the weights'
            # sums with the minima are fp32
            score = (q[b, i].double().abs()[:, None] * k[:, :m].abs()).sum(-1).amax(-1) * scale
            tol = 2.0 ** -11 * 15 * (p * sc[:, :m, 2].abs()).sum(-1) + (4 * score + 64) * 2.0 ** -20 * (p * v[:, :m].abs().amax(-1)).sum(-1)
            off = (out[b, i].double() - want[b, i]).abs() - unit * want[b, i].abs() - tol[:, None]
            assert torch.isfinite(out[b, i]).all() and (off <= 0).all(), (b, i, float(off.max()))
    _lib.check_status(out.device)


@pytest.mark.parametrize("heads,S", [(1, 1), (4, 1), (4, 4)])
@pytest.mark.parametrize("apart", [12, 28, 45, 100])
def test_values_of_little_weight_do_not_blur_the_others(apart, heads, S):
    """Value scales 2^12 to 2^100 apart, the large ones at tokens whose weights make up for it, many times over or just."""
    page, D, n = 16, 64, 700
    t = torch.arange(n, device=DEV)
    for steps, large in ((1.0, t % 5 == 4), (1.0, t < 200), (1.0, t >= 640), (0.0, t % 50 == 49), (0.0, t < 3)):
        cache = ops.KV4Cache(1, 44, page, 1, D, DEV)
        codes, scales = layer = cache.layer(0)
        _fill(codes, scales, seed=21)
        table = _table(1, 44, 44)
        page_of, slot = table[0, t // page].long(), t % page
        # keys of equal dims: with a query of ones and a scale of 1 / D a score is the key's minimum. Large values stand 2^apart above the others,
        # their weights as far below them (steps 0), or twice as far and a little (steps 1)
        codes[page_of, 0, 0, slot] = 0
        scales[page_of, 0, slot, 0] = 0
        scales[page_of, 0, slot, 1] = torch.where(large, -apart * (1 + steps) * math.log(2) - 3 * steps, -0.01 * (t % 7)).bfloat16()
        size = torch.where(large, 2.0 ** (apart // 2), 2.0 ** (apart // 2 - apart)).bfloat16()
        scales[page_of, 0, slot, 2] = size
        scales[page_of, 0, slot, 3] = (-7.5 * size.float()).bfloat16()
        q = torch.ones(1, S, heads, D, device=DEV).bfloat16()
        _check_weighted(q, layer, table, [n], 1 / D)


@pytest.mark.parametrize("S,apart", [(2, 20), (3, 30), (5, 60)])
def test_values_that_a_query_does_not_see_do_not_blur_its_others(S, apart):
    """The newest token has huge values; the queries before it do not see them."""
    page, D, KV, n = 32, 128, 2, 333
    cache = ops.KV4Cache(1, 11, page, KV, D, DEV)
    codes, scales = layer = cache.layer(0)
    _fill(codes, scales, seed=22)
    table = _table(1, 11, 11)
    at = table[0, (n - 1) // page].long(), 1, (n - 1) % page
    scales[at[0], at[1], at[2], 2] = 2.0 ** apart
    scales[at[0], at[1], at[2], 3] = -7 * 2.0 ** apart
    q = torch.randn(1, S, 4, D, generator=_gen(23), device=DEV).bfloat16()
    _check_weighted(q, layer, table, [n], D ** -0.5)


def test_the_largest_values_and_queries():
    """Values up to 10^37, which bf16 holds, and queries of 10^34 against keys that are as small."""
    page, D = 16, 128
    cache = ops.KV4Cache(1, 20, page, 1, D, DEV)
    codes, scales = layer = cache.layer(0)
    table = _table(1, 20, 20)
    _fill(codes, scales, seed=24, v_scale=2.0 ** 119)
    q = torch.randn(1, 1, 8, D, generator=_gen(25), device=DEV).bfloat16()
    _check_weighted(q, layer, table, [311], D ** -0.5)
    _fill(codes, scales, seed=24, k_scale=0.4e-34)
    _check_weighted(q * 1e34, layer, table, [311], D ** -0.5)


@pytest.mark.parametrize("offset", [1, 2, 3])
def test_angles_off_their_alignment(offset):
    """Tables of angles that are contiguous and begin anywhere."""
    D, n_q, KV, T = 64, 2, 2, 9
    cos, sin = ops.rope_tables(40, D, device=DEV)
    x = torch.randn(T, (n_q + 2 * KV) * D, generator=_gen(40), device=DEV).bfloat16()
    pos = torch.arange(30, 30 + T, dtype=torch.int32, device=DEV)
    table, seq = torch.tensor([[0, 1, 2]], dtype=torch.int32, device=DEV), torch.zeros(T, dtype=torch.int32, device=DEV)
    results = []
    for off in (0, offset):
        cache = ops.KV4Cache(1, 3, 16, KV, D, DEV)
        pair = [torch.cat([torch.zeros(off, device=DEV), t.flatten()])[off:].view(t.shape) for t in (cos, sin)]
        assert all(t.is_contiguous() and t.data_ptr() % 16 == 4 * off for t in pair)
        results.append((ops.kv4_append(cache.layer(0), table, seq, pos, x, n_q, *pair), cache.codes, cache.scales.view(torch.int16)))
    assert all(torch.equal(a, b) for a, b in zip(*results))
    _lib.check_status(x.device)


@pytest.mark.parametrize("far", [1 << 32, (1 << 32) + 5, (1 << 63) - 1, -(1 << 32) + 5, -(1 << 63)])
def test_whole_numbers_of_64_bits_are_not_cut(far):
    """What is out of range in 64 bits stays out of range: skipped where it is negative, reported where it is not."""
    D, KV = 64, 2
    cache = ops.KV4Cache(1, 4, 16, KV, D, DEV)
    layer, table = cache.layer(0), torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device=DEV)
    place, one = torch.tensor([far], device=DEV), torch.zeros(1, dtype=torch.int64, device=DEV)
    x, q = torch.randn(1, (2 + 2 * KV) * D, device=DEV).bfloat16(), torch.randn(2, 1, 4, D, device=DEV).bfloat16()
    dev = x.device

    def is_reported(wanted):
        if not wanted:
            return _lib.check_status(dev)
        with pytest.raises(_lib.KernelError):
            _lib.check_status(dev)

    ops.kv4_append(layer, table, one, place, x, 2)
    is_reported(far > 0)
    k, v = ops.kv4_read(layer, table, one, place)
    is_reported(far > 0)
    assert far > 0 or ((k == 0).all() and (v == 0).all())
    out = ops.kv4_attention(q, layer, table, torch.tensor([far, 0], device=DEV))
    is_reported(far > 0)
    assert far > 0 or (out == 0).all()
    ops.kv4_append(layer, table, place, one, x, 2)
    is_reported(True)
    assert (cache.codes == 0).all() and (cache.scales == 0).all()
