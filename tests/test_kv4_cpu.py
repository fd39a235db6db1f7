"""4-bit paged cache without a GPU: the plain implementations and the refusals."""
import math

import pytest
import torch

from atorch_b200 import ops


def _filled(pages=9, page=16, KV=2, D=32, seed=0):
    g = torch.Generator().manual_seed(seed)
    cache = ops.KV4Cache(2, pages, page, KV, D)
    return cache, torch.randperm(pages, generator=g)[: 2 * 4].to(torch.int32).view(2, 4), g


def test_tokens_come_back_within_half_a_step():
    cache, table, g = _filled()
    x = torch.randn(30, (4 + 4) * 32, generator=g)
    seq, pos = torch.tensor([0] * 20 + [1] * 10), torch.cat([torch.arange(20), torch.arange(40, 50)])
    pos[4] = -1
    q = ops.kv4_append(cache.layer(1), table, seq, pos, x, 4)
    assert torch.equal(q, x.view(30, 8, 32)[:, :4])
    k, v = ops.kv4_read(cache.layer(1), table, seq, pos, torch.float32)
    for got, want in ((k, x.view(30, 8, 32)[:, 4:6]), (v, x.view(30, 8, 32)[:, 6:])):
        low, high = want.amin(-1, keepdim=True), want.amax(-1, keepdim=True)
        off = (got - want).abs() <= (high - low) / 30 * 1.01 + 2 ** -8 * (low.abs() + high - low)
        assert off[torch.arange(30) != 4].all() and (got[4] == 0).all()
    assert (cache.codes[0] == 0).all()


def test_rotation_is_that_of_rope():
    cache, table, g = _filled()
    cos, sin = ops.rope_tables(64, 32)
    x = torch.randn(5, 8 * 32, generator=g)
    pos = torch.tensor([0, 3, 17, 40, 63])
    q = ops.kv4_append(cache.layer(0), table, torch.tensor([0, 1, 0, 1, 0]), pos, x, 4, cos, sin)
    want = ops.rope_reference(x, cos, sin, 6, 32, pos).view(5, 8, 32)
    assert torch.equal(q, want[:, :4])


def test_attention_is_that_of_the_values():
    cache, table, g = _filled()
    layer = cache.layer(0)
    n = [37, 1]
    for b in range(2):
        ops.kv4_append(layer, table, torch.full((n[b],), b), torch.arange(n[b]), torch.randn(n[b], 4 * 32, generator=g), 0)
    q = torch.randn(2, 3, 6, 32, generator=g)
    out, lse = ops.kv4_attention(q.half(), layer, table, torch.tensor(n), return_lse=True)
    for b in range(2):
        k, v = ops.kv4_read(layer, table, torch.full((n[b],), b), torch.arange(n[b]), torch.float32)
        want = ops.attention_reference(q[b: b + 1].half().float(), k[None], v[None], causal=True)
        assert torch.allclose(out[b].float(), want[0], atol=2e-3)
    assert (out[1, :2] == 0).all() and (lse[1, :, :2] == -math.inf).all() and torch.isfinite(lse[0]).all()


def test_what_is_not_there_is_refused():
    cache, table, _ = _filled()
    x, one = torch.zeros(1, 8 * 32), torch.zeros(1, dtype=torch.int32)
    for seq, pos in ((2, 0), (0, 64), (-1, 0)):
        with pytest.raises(IndexError):
            ops.kv4_append(cache.layer(0), table, torch.tensor([seq]), torch.tensor([pos]), x, 4)
    with pytest.raises(IndexError):
        ops.kv4_attention(torch.zeros(2, 1, 4, 32).half(), cache.layer(0), table, torch.tensor([65, 1]))
    with pytest.raises(ValueError):
        ops.kv4_append(cache.layer(0), table, None, one, x, 5)
    with pytest.raises(RuntimeError):
        ops.kv4_append(cache.layer(0), table, None, one, x.clone().requires_grad_(), 4)
    with pytest.raises(ValueError):
        ops.KV4Cache(1, 4, 8, 2, 32)


@pytest.mark.parametrize("far", [1 << 32, (1 << 32) + 5, 1 << 40, (1 << 63) - 1, -(1 << 32) + 5, -(1 << 63)])
def test_whole_numbers_of_64_bits_are_not_cut(far):
    """What is out of range in 64 bits stays out of range: skipped where it is negative, refused where it is not."""
    cache, table, _ = _filled()
    layer, x = cache.layer(0), torch.randn(1, 8 * 32)
    place, one = torch.tensor([far]), torch.zeros(1, dtype=torch.int64)
    if far < 0:
        ops.kv4_append(layer, table, one, place, x, 4)
        assert all((t == 0).all() for t in ops.kv4_read(layer, table, one, place))
        out, lse = ops.kv4_attention(torch.randn(2, 1, 4, 32).half(), layer, table, torch.tensor([far, 0]), return_lse=True)
        assert (out == 0).all() and (lse == -math.inf).all()
    else:
        with pytest.raises(IndexError):
            ops.kv4_append(layer, table, one, place, x, 4)
        with pytest.raises(IndexError):
            ops.kv4_read(layer, table, one, place)
        with pytest.raises(IndexError):
            ops.kv4_attention(torch.randn(2, 1, 4, 32).half(), layer, table, torch.tensor([1, far]))
    with pytest.raises(IndexError):
        ops.kv4_append(layer, table, place, one, x, 4)
    assert (cache.codes == 0).all() and (cache.scales == 0).all()


def test_a_table_of_one_column_may_have_any_stride_there():
    cache, table, g = _filled()
    wide = table.repeat_interleave(3, 1)[:, ::3][:, :1]            # one page a sequence, the next column three places on
    assert wide.shape == (2, 1) and wide.stride(1) == 3
    x, pos = torch.randn(2, 8 * 32, generator=g), torch.tensor([3, 7])
    ops.kv4_append(cache.layer(0), wide, None, pos, x, 4)
    got = ops.kv4_read(cache.layer(0), wide, None, pos)
    want = ops.kv4_read(cache.layer(0), table, None, pos)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and got[0].any()
    ops.beam_reorder(cache.codes, cache.scales, wide, torch.full((2,), 9, dtype=torch.int32), torch.tensor([[1, 0]], dtype=torch.int32))
    after = ops.kv4_read(cache.layer(0), table, torch.tensor([1, 0]), pos)
    assert all(torch.equal(a, b) for a, b in zip(after, want))
    with pytest.raises(ValueError):
        ops.kv4_read(cache.layer(0), table.repeat_interleave(3, 1)[:, ::3], None, pos)
