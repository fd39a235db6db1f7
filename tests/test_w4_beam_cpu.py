"""4-bit weights and beam search without a GPU: the plain implementations and the refusals."""
import math

import pytest
import torch
from torch.autograd import forward_ad

from atorch_b200 import ops


@pytest.mark.parametrize("N,K,group", [(5, 64, 32), (3, 100, 64), (2, 1, 128), (7, 257, 128)])
def test_weights_come_back_and_multiply(N, K, group):
    w = torch.randn(N, K, generator=torch.Generator().manual_seed(K))
    codes, scales = ops.w4_quantize(w, group)
    assert codes.shape == (N, -(-K // 32) * 16) and scales.shape == (N, -(-K // group))
    got = ops.w4_dequantize(codes, scales, K, group)
    assert ((got - w).abs() <= scales.float().repeat_interleave(group, 1)[:, :K] * (0.5 + 7 / 256)).all()
    x, b = torch.randn(2, 3, K).half(), torch.randn(N).half()
    y = ops.w4_linear(x, codes, scales, group, b)
    assert torch.allclose(y.float(), x.float() @ got.t() + b.float(), atol=2e-2, rtol=2e-3)
    with pytest.raises(ValueError):
        ops.w4_linear(x.float(), codes, scales, group)
    with pytest.raises(RuntimeError):
        ops.w4_linear(x.clone().requires_grad_(), codes, scales, group)


def test_select_is_a_sort_of_all_continuations():
    g = torch.Generator().manual_seed(0)
    logits, scores = torch.randn(3, 4, 50, generator=g), torch.randn(3, 4, generator=g)
    finished = torch.tensor([[False, True, False, False]] * 3)
    got, tokens, parents, ended = ops.beam_select(logits, scores, finished, 7, 6)
    for b in range(3):
        every = []
        lse = torch.logsumexp(logits[b].double(), -1)
        for w in range(4):
            for v in range(50):
                f = scores[b, w].double() + (logits[b, w, v].double() - lse[w])
                if finished[b, w]:
                    f = scores[b, w].double() if v == 7 else torch.tensor(-math.inf)
                every.append((-float(f), w, v))
        every.sort()
        assert [(w, v) for _, w, v in every[:6]] == list(zip(parents[b].tolist(), tokens[b].tolist()))
        assert [v == 7 or w == 1 for _, w, v in every[:6]] == ended[b].tolist()
        assert all(abs(f + s) < 1e-5 for (f, _, _), s in zip(every, got[b].tolist()))
    with pytest.raises(ValueError):
        ops.beam_select(logits, scores, finished)


def test_reorder_moves_what_the_beams_hold():
    """Before and after: row w reads what its parent read."""
    cache = ops.KV4Cache(2, 12, 16, 1, 32)
    g = torch.Generator().manual_seed(1)
    table = torch.tensor([[0, 1, 5], [0, 2, 6], [0, 3, 7]], dtype=torch.int32)
    n = 41
    for i in range(2):
        for w in range(3):
            ops.kv4_append(cache.layer(i), table, torch.full((n,), w), torch.arange(n), torch.randn(n, 64, generator=g), 0)
    pos = torch.arange(n)
    held = [[ops.kv4_read(cache.layer(i), table, torch.full((n,), w), pos) for w in range(3)] for i in range(2)]
    parents = torch.tensor([[2, 0, 0]], dtype=torch.int32)
    ops.beam_reorder(cache.codes, cache.scales, table, torch.full((3,), n, dtype=torch.int32), parents)
    assert table[:, 2].tolist() == [5, 6, 7]
    for i in range(2):
        for w in range(3):
            k, v = ops.kv4_read(cache.layer(i), table, torch.full((n,), w), pos)
            assert torch.equal(k, held[i][parents[0, w]][0]) and torch.equal(v, held[i][parents[0, w]][1])
    with pytest.raises(IndexError):
        ops.beam_reorder(cache.codes, cache.scales, table, torch.full((3,), n, dtype=torch.int32), parents + 1)


def test_reorder_refuses_a_cache_off_its_alignment():
    """The kernel moves codes in pieces of 16 bytes and scales in pieces of 8; a layer's operators refuse the same."""
    cache = ops.KV4Cache(1, 6, 16, 1, 64)
    table, lengths = torch.zeros(2, 2, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    table[1] = 1
    parents = torch.zeros(1, 2, dtype=torch.int32)
    ops.beam_reorder(cache.codes, cache.scales, table, lengths, parents)

    def off(t, n):
        return torch.zeros(t.numel() + 16, dtype=t.dtype)[n: n + t.numel()].view(t.shape)

    for codes, scales in ((off(cache.codes, 1), cache.scales), (off(cache.codes, 8), cache.scales), (cache.codes, off(cache.scales, 1)),
                          (cache.codes, off(cache.scales, 4))):
        assert codes.is_contiguous() and scales.is_contiguous()
        with pytest.raises(ValueError):
            ops.beam_reorder(codes, scales, table, lengths, parents)
        with pytest.raises(ValueError):
            ops.kv4_read((codes[0], scales[0]), table, None, lengths)


def _calls(dev):
    """Each operator on tensors of a device, by name: the tensors that a gradient could be asked of, and the call."""
    g = torch.Generator().manual_seed(2)
    cache = ops.KV4Cache(1, 4, 16, 2, 64, dev)
    table, n = torch.tensor([[0, 1]], dtype=torch.int32, device=dev), torch.tensor([20], dtype=torch.int32, device=dev)
    qkv, q = torch.randn(1, 8 * 64, generator=g).to(dev), torch.randn(1, 1, 4, 64, generator=g).half().to(dev)
    codes, scales = (t.to(dev) for t in ops.w4_quantize(torch.randn(16, 64, generator=g), 64))
    x, bias = torch.randn(3, 64, generator=g).bfloat16().to(dev), torch.randn(16, generator=g).bfloat16().to(dev)
    logits, scores = torch.randn(1, 2, 50, generator=g).to(dev), torch.randn(1, 2, generator=g).to(dev)
    return {"append": ([qkv], lambda t: ops.kv4_append(cache.layer(0), table, None, n, t, 4)),
            "attention": ([q], lambda t: ops.kv4_attention(t, cache.layer(0), table, n)),
            "w4_linear": ([x, bias], lambda t, b: ops.w4_linear(t, codes, scales, 64, b)),
            "beam_select": ([logits, scores], lambda t, s: ops.beam_select(t, s))}


def check_gradients_are_refused(dev):
    for name, (tensors, call) in _calls(dev).items():
        with torch.no_grad():
            call(*tensors)
        for i in range(len(tensors)):
            asks = [t.clone().requires_grad_() if j == i else t for j, t in enumerate(tensors)]
            with pytest.raises(RuntimeError, match="gradient"):
                call(*asks)
            with torch.no_grad():
                call(*asks)
            with forward_ad.dual_level():
                dual = [forward_ad.make_dual(t, torch.ones_like(t)) if j == i else t for j, t in enumerate(tensors)]
                for off in (False, True):           # gradients that are switched off leave tangents as they are
                    with torch.set_grad_enabled(not off), pytest.raises(RuntimeError, match="gradient"):
                        call(*dual)
                call(*tensors)


def test_gradients_and_tangents_are_refused():
    check_gradients_are_refused("cpu")


def test_launches_are_on_the_current_device(monkeypatch):
    """The launchers launch on the current device: the stream of another one is refused."""
    from atorch_b200 import _lib

    current = [0]
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: current[0], raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda device: 1000 + device, raising=False)
    assert _lib.stream_of(0) == 1000
    with pytest.raises(ValueError, match="cuda:1"):
        _lib.stream_of(1)
    current[0] = 1
    assert _lib.stream_of(1) == 1001
