"""16-bit paged cache without a GPU: the plain implementations against the formulas, and the refusals."""
import math

import pytest
import torch
from torch.autograd import forward_ad

from atorch_b200 import ops


def _filled(pages=9, page=16, KV=2, D=32, seed=0, dtype=torch.float16):
    g = torch.Generator().manual_seed(seed)
    cache = ops.KVCache(2, pages, page, KV, D, dtype)
    cache.data.copy_(torch.randn(cache.data.shape, generator=g))
    return cache, torch.randperm(pages, generator=g)[: 2 * 4].to(torch.int32).view(2, 4), g


def _rows(layer, table, b, n):
    t = torch.arange(n)
    return layer[table[b, t // layer.shape[3]].long(), :, :, t % layer.shape[3]]       # [n, 2, KV, D]


def test_rotation_is_that_of_rope_at_the_angles():
    cache, table, g = _filled(dtype=torch.bfloat16)
    cos, sin = ops.rope_tables(600, 32)
    x = torch.randn(5, 8 * 32, generator=g).bfloat16()
    pos, angles = torch.tensor([0, 3, 17, -1, 63]), torch.tensor([0, 500, 17, 9000, 599])
    before = cache.data.clone()
    q, k = ops.kv_append(cache.layer(0), table, torch.tensor([0, 1, 0, 1, 0]), pos, x, 4, cos, sin, angles, return_keys=True)
    want = ops.rope_reference(x, cos, sin, 6, 32, angles.clamp(max=599)).view(5, 8, 32)
    want[3] = x.view(5, 8, 32)[3]
    assert torch.equal(q, want[:, :4]) and torch.equal(k, want[:, 4:6])
    for t, b in ((0, 0), (1, 1), (2, 0), (4, 0)):
        assert torch.equal(cache.data[0, table[b, int(pos[t]) // 16].long(), :, :, int(pos[t]) % 16], torch.stack([want[t, 4:6], x.view(5, 8, 32)[t, 6:]]))
    assert int((cache.data != before).flatten(2).any(-1).sum()) == 4 and torch.equal(cache.data[1], before[1])


@pytest.mark.parametrize("S", [1, 3])
def test_attention_and_its_weights(S):
    cache, table, g = _filled()
    layer, n = cache.layer(1), [37, 1]
    q = torch.randn(2, S, 6, 32, generator=g).half()
    weights = torch.rand(2, 2, 70, generator=g)
    before = weights.clone()
    out, lse = ops.kv_attention(q, layer, table, torch.tensor(n), return_lse=True, weights=weights)
    for b in range(2):
        kv = _rows(layer, table, b, n[b]).double().repeat_interleave(3, 2)
        for i in range(S):
            m = n[b] - S + i + 1
            if m <= 0:
                assert (out[b, i] == 0).all() and (lse[b, :, i] == -math.inf).all()
                continue
            s = torch.einsum("hd,thd->ht", q[b, i].double(), kv[:m, 0]) / 32 ** 0.5
            p = torch.softmax(s, -1)
            assert torch.allclose(out[b, i].double(), torch.einsum("ht,thd->hd", p, kv[:m, 1]), atol=2e-3)
            assert torch.allclose(lse[b, :, i].double(), torch.logsumexp(s, -1), atol=1e-5)
            before[b, :, :m] += p.view(2, 3, m).sum(1).float()
    assert torch.allclose(weights, before, atol=1e-5)


def test_eviction_keeps_the_heaviest_and_the_last_in_order():
    cache, table, g = _filled(dtype=torch.bfloat16)
    lengths = torch.tensor([61, 20], dtype=torch.int32)
    weights = torch.randint(0, 6, (2, 2, 2, 64), generator=g).float()           # many are equal
    rows = [[_rows(cache.layer(i), table, b, 64).clone() for b in range(2)] for i in range(2)]
    old = weights.clone()
    new = ops.kv_evict(cache.data, table, lengths, weights, 24, 5)
    assert new.tolist() == [24, 20] and new.dtype == torch.int32 and lengths.tolist() == [61, 20]
    for i in range(2):
        assert torch.equal(_rows(cache.layer(i), table, 1, 64), rows[i][1]) and torch.equal(weights[i, 1], old[i, 1])
        for h in range(2):
            w = old[i, 0, h]
            kept = sorted(sorted(range(56), key=lambda j: (-w[j].item(), j))[:19]) + list(range(56, 61))
            assert torch.equal(_rows(cache.layer(i), table, 0, 24)[:, :, h], rows[i][0][kept][:, :, h])
            assert torch.equal(weights[i, 0, h, :24], w[kept]) and (weights[i, 0, h, 24:61] == 0).all()
            assert torch.equal(weights[i, 0, h, 61:], w[61:])
            assert torch.equal(_rows(cache.layer(i), table, 0, 64)[24:, :, h], rows[i][0][24:, :, h])


def check_refusals(dev):
    cache = ops.KVCache(2, 4, 16, 2, 64, device=dev)
    layer, table = cache.layer(0), torch.zeros(1, 2, dtype=torch.int32, device=dev)
    pos = torch.zeros(1, dtype=torch.int32, device=dev)
    x, q = torch.zeros(1, 8 * 64, device=dev).bfloat16(), torch.zeros(1, 1, 4, 64, device=dev).bfloat16()
    cos, sin = ops.rope_tables(4, 64, device=dev)
    off = torch.zeros(layer.numel() + 8, dtype=torch.bfloat16, device=dev)[1: layer.numel() + 1].view(layer.shape)
    layers = (dict(layer=layer.float()), dict(layer=layer[:, :, :, :8]), dict(layer=layer.transpose(2, 3)), dict(layer=off), dict(layer=cache.data),
              dict(page_table=table.long()), dict(page_table=table[0]), dict(page_table=table.repeat(1, 2)[:, ::2]))
    ok = dict(layer=layer, page_table=table, seq=None, pos=pos, qkv=x, n_q=4)
    for change in layers + (dict(n_q=3), dict(qkv=x.half()), dict(pos=pos.float()), dict(pos=torch.zeros(2, device=dev).int()), dict(cos=cos),
                            dict(cos=cos[:, :8], sin=sin[:, :8]), dict(cos=cos.double(), sin=sin.double()), dict(angles=pos), dict(seq=torch.zeros(3, device=dev).int())):
        with pytest.raises(ValueError):
            ops.kv_append(**{**ok, **change})
    n, w = torch.ones(1, dtype=torch.int32, device=dev), torch.zeros(1, 2, 32, device=dev)
    ok = dict(q=q, layer=layer, page_table=table, lengths=n, weights=w)
    for change in layers + (dict(q=q.half()), dict(q=q[..., :32]), dict(q=q[:, :, :3]), dict(q=q[0]), dict(page_table=table.repeat(2, 1)), dict(lengths=n.float()),
                            dict(weights=w.double()), dict(weights=w[..., :31]), dict(weights=w[0]), dict(weights=torch.zeros(1, 2, 64, device=dev)[..., ::2]),
                            dict(weights=torch.zeros(2, 2, 32, device=dev))):
        with pytest.raises(ValueError):
            ops.kv_attention(**{**ok, **change})
    ok = dict(cache=cache.data, page_table=table, lengths=n, weights=torch.zeros(2, 1, 2, 32, device=dev), budget=4, recent=2)
    for change in (dict(cache=cache.data.float()), dict(cache=cache.data[:, :, :, :, :8]), dict(cache=cache.data.transpose(3, 4)), dict(cache=layer),
                   dict(cache=cache.data[:, :2]), dict(weights=torch.zeros(1, 2, 32, device=dev)), dict(weights=torch.zeros(2, 1, 2, 31, device=dev)),
                   dict(weights=torch.zeros(2, 1, 2, 32, device=dev).double()), dict(weights=torch.zeros(2, 1, 2, 64, device=dev)[..., ::2]),
                   dict(budget=0), dict(budget=-3), dict(recent=5), dict(recent=-1), dict(lengths=n.float()), dict(lengths=torch.ones(2, device=dev).int()),
                   dict(page_table=table.repeat(2, 1))):
        with pytest.raises(ValueError):
            ops.kv_evict(**{**ok, **change})
    for bad in (torch.float32, torch.float64, torch.uint8):
        with pytest.raises(ValueError):
            ops.KVCache(1, 4, 16, 2, 64, bad, dev)
    with pytest.raises(ValueError):
        ops.KVCache(1, 4, 24, 2, 64, device=dev)
    if dev != "cpu":
        for call in (lambda: ops.kv_append(layer, table.cpu(), None, pos, x, 4), lambda: ops.kv_attention(q, layer, table, n.cpu()),
                     lambda: ops.kv_attention(q, layer, table, n, weights=w.cpu()), lambda: ops.kv_append(layer, table, None, pos, x.cpu(), 4),
                     lambda: ops.kv_evict(cache.data, table, n.cpu(), torch.zeros(2, 1, 2, 32, device=dev), 4),
                     lambda: ops.kv_evict(cache.data, table, n, torch.zeros(2, 1, 2, 32), 4)):
            with pytest.raises(ValueError):
                call()
    # gradients and tangents
    evict_w = torch.zeros(2, 1, 2, 32, device=dev)
    calls = {"append": ([x, layer], lambda t, c: ops.kv_append(c, table, None, pos, t, 4)),
             "attention": ([q, layer, w], lambda t, c, v: ops.kv_attention(t, c, table, n, weights=v)),
             "evict": ([cache.data, evict_w], lambda c, v: ops.kv_evict(c, table, n, v, 4))}
    for name, (tensors, call) in calls.items():
        for i in range(len(tensors)):
            asks = [t.clone().requires_grad_() if j == i else t for j, t in enumerate(tensors)]
            with pytest.raises(RuntimeError, match="gradient"):
                call(*asks)
            with torch.no_grad():
                call(*asks)
            with forward_ad.dual_level():
                dual = [forward_ad.make_dual(t, torch.ones_like(t)) if j == i else t for j, t in enumerate(tensors)]
                with torch.no_grad(), pytest.raises(RuntimeError, match="gradient"):
                    call(*dual)


def test_refusals():
    check_refusals("cpu")


def test_what_is_not_there_is_refused():
    cache, table, _ = _filled()
    layer = cache.layer(0)
    x, one = torch.zeros(1, 8 * 32).half(), torch.zeros(1, dtype=torch.int32)
    cos, sin = ops.rope_tables(8, 32)
    for seq, pos in ((2, 0), (0, 64), (-1, 0)):
        with pytest.raises(IndexError):
            ops.kv_append(layer, table, one + seq, one + pos, x, 4)
    for angle in (-1, 8):
        with pytest.raises(IndexError):
            ops.kv_append(layer, table, None, one, x, 4, cos, sin, one + angle)
    with pytest.raises(IndexError):
        ops.kv_attention(torch.zeros(2, 1, 4, 32).half(), layer, table, torch.tensor([1, 65]))
    weights = torch.zeros(2, 2, 2, 64)
    with pytest.raises(IndexError):
        ops.kv_evict(cache.data, table, torch.tensor([1, 65]), weights, 10)
    table[1, 1] = 9
    for call in (lambda n: ops.kv_attention(torch.zeros(2, 1, 4, 32).half(), layer, table, n), lambda n: ops.kv_evict(cache.data, table, n, weights, 10)):
        with pytest.raises(IndexError):
            call(torch.tensor([1, 17]))
        call(torch.tensor([1, 16]))


@pytest.mark.parametrize("far", [1 << 32, -(1 << 33) - 5, (1 << 40) + 7])
def test_whole_numbers_of_64_bits_are_not_cut(far):
    cache, table, _ = _filled()
    x = torch.zeros(1, 8 * 32).half()
    cos, sin = ops.rope_tables(8, 32)
    before = cache.data.clone()
    if far > 0:
        with pytest.raises(IndexError):
            ops.kv_append(cache.layer(0), table, None, torch.tensor([far]), x, 4)
        with pytest.raises(IndexError):
            ops.kv_attention(torch.zeros(2, 1, 4, 32).half(), cache.layer(0), table, torch.tensor([1, far]))
    else:
        ops.kv_append(cache.layer(0), table, None, torch.tensor([far]), x, 4)      # padding
        assert ops.kv_evict(cache.data, table, torch.tensor([far, 3]), torch.zeros(2, 2, 2, 64), 4)[0] < 0
    with pytest.raises(IndexError):
        ops.kv_append(cache.layer(0), table, None, torch.tensor([0]), x, 4, cos, sin, torch.tensor([far]))
    assert torch.equal(cache.data, before)
