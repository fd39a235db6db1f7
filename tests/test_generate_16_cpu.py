"""Generation with the cache in 16 bits on the CPU: against the model's own forward, with a budget against lists of keys and values, and
with the filters of sampling."""
import math

import pytest
import torch

from atorch_b200 import ops
from atorch_b200.models import generate as module
from atorch_b200.models.generate import CachedSampler, Generator
from atorch_b200.models.llama import LlamaConfig, LlamaModel


def model(device="cpu", dtype=torch.bfloat16, seed=0, **kw):
    torch.manual_seed(seed)
    cfg = LlamaConfig(**{**dict(vocab_size=40, hidden_size=64, intermediate_size=96, num_hidden_layers=2, num_attention_heads=4,
                                num_key_value_heads=2, max_position_embeddings=256, initializer_range=0.1), **kw})
    return LlamaModel(cfg).to(device, dtype).eval()


def prompts(m, sizes, seed=1):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, m.config.vocab_size, (n,), generator=g).to(m.embed_tokens.weight.device) for n in sizes]


class Lists:
    """One sequence, token after token, in fp32: a list of keys, values and sums of weights for every layer and key/value head, cut when it
    is told to."""

    def __init__(self, m):
        self.m = m
        self.k = [[[] for _ in range(layer.n_kv)] for layer in m.layers]
        self.v = [[[] for _ in range(layer.n_kv)] for layer in m.layers]
        self.w = [[[] for _ in range(layer.n_kv)] for layer in m.layers]
        self.at = 0

    def token(self, t, weigh):
        m, f = self.m, lambda lin, x: x @ lin.weight.float().t()
        norm = lambda n, x: x * torch.rsqrt(x.pow(2).mean() + n.eps) * n.weight.float()
        h, d = m.embed_tokens.weight[t].float(), m.config.head_dim
        cos, sin = m.rope(self.at + 1, h.device)
        for i, layer in enumerate(m.layers):
            qkv = f(layer.qkv_proj, norm(layer.input_layernorm, h)).view(-1, d)
            n_q, n_kv = layer.n_q, layer.n_kv
            a, b = qkv[: n_q + n_kv, : d // 2], qkv[: n_q + n_kv, d // 2:]
            qk = torch.cat([a * cos[self.at] - b * sin[self.at], b * cos[self.at] + a * sin[self.at]], -1)
            out = []
            for h_kv in range(n_kv):
                k, v, w = self.k[i][h_kv], self.v[i][h_kv], self.w[i][h_kv]
                k.append(qk[n_q + h_kv]), v.append(qkv[n_q + n_kv + h_kv]), w.append(0.0)
                q = qk[h_kv * (n_q // n_kv): (h_kv + 1) * (n_q // n_kv)]
                p = torch.softmax(q @ torch.stack(k).t() / math.sqrt(d), -1)
                if weigh:
                    self.w[i][h_kv] = [x + y for x, y in zip(w, p.sum(0).tolist())]
                out.append(p @ torch.stack(v))
            h = h + f(layer.o_proj, torch.cat(out).flatten())
            gate, up = f(layer.gate_up_proj, norm(layer.post_attention_layernorm, h)).chunk(2)
            h = h + f(layer.down_proj, torch.nn.functional.silu(gate) * up)
        self.at += 1
        return f(m.lm_head, norm(m.norm, h))

    def cut(self, budget, recent, weights, off):
        """By the weights that the generation has, which are near the lists' own (those of two tokens may be nearer to each other)."""
        for i in range(len(self.k)):
            for h in range(len(self.k[i])):
                n = len(self.w[i][h])
                w, own = weights[i, h, :n].tolist(), torch.tensor(self.w[i][h])
                assert (torch.tensor(w) - own).norm() <= off * own.norm() and (weights[i, h, n:] == 0).all()
                if n <= budget:
                    continue
                kept = sorted(sorted(range(n - recent), key=lambda j: (-w[j], j))[: budget - recent]) + list(range(n - recent, n))
                for each in (self.k, self.v, self.w):
                    each[i][h] = [each[i][h][j] for j in kept]


def steps(m, ids, new, monkeypatch, **kw):
    """What a generation puts out, the logits it went by, and by which weights it cut its cache after how many of them."""
    logits, cuts, evict = [], {}, ops.kv_evict
    run = Generator._run
    monkeypatch.setattr(Generator, "_run", lambda self, *a: logits.append(run(self, *a)) or logits[-1])
    monkeypatch.setattr(module.ops, "kv_evict", lambda *a: cuts.setdefault(len(logits), a[3].clone()) is None or evict(*a))
    out = Generator(m, **kw).generate(ids, new)
    monkeypatch.undo()
    return out, logits, cuts


def check_against_lists(m, sizes, new, monkeypatch, off, **kw):
    """Logits of every step against the lists', which are cut at the same steps. In front of a cut the lists have added up the weights of the
    same queries: a prompt's last ones, then every token."""
    budget, recent = kw.get("budget"), kw.get("recent")
    ids = prompts(m, sizes)
    out, logits, cuts = steps(m, ids, new, monkeypatch, cache_bits=16, **kw)
    assert len(logits) == new
    with torch.no_grad():
        for b, (p, o) in enumerate(zip(ids, out)):
            lists = Lists(m)
            window = min(Generator.WINDOW, max(sizes))
            for n, t in enumerate(p):
                last = lists.token(t, n >= len(p) - window)
            for i in range(new):
                got = logits[i][b].float()
                assert (got - last).norm() / last.norm() < off, (b, i, float((got - last).norm() / last.norm()))
                if i + 1 in cuts:
                    lists.cut(budget, recent, cuts[i + 1][:, b].cpu(), off)
                if i + 1 < new:
                    last = lists.token(o[len(p) + i], True)
            if budget is not None:
                assert max(len(w) for layer in lists.w for w in layer) <= max(budget + kw["slack"], 1)
    return list(cuts)


def test_the_cache_alone(monkeypatch):
    assert check_against_lists(model(), (3, 37, 70), 20, monkeypatch, 0.03) == []


def test_with_a_budget(monkeypatch):
    # heads that attend to little: the sums of those that go and those that stay lie apart
    m = model(initializer_range=0.2)
    assert check_against_lists(m, (3, 37, 70), 30, monkeypatch, 0.06, budget=40, recent=8, slack=6) == [1, 7, 13, 19, 25]
    assert check_against_lists(m, (20, 20), 30, monkeypatch, 0.06, budget=16, recent=16, slack=8) == [1, 9, 17, 25]
    assert check_against_lists(m, (5,), 12, monkeypatch, 0.06, budget=64, recent=0, slack=1) == []


def test_a_budget_that_is_never_reached_changes_nothing():
    m = model()
    ids = prompts(m, (5, 40, 70))
    plain = Generator(m, cache_bits=16).generate(ids, 25)
    for a, b in zip(plain, Generator(m, cache_bits=16, budget=95).generate(ids, 25)):
        assert torch.equal(a, b)


def test_sampling_filters():
    m = model()
    ids = prompts(m, (6, 6, 6, 6))
    first = Generator(m).generate(ids, 8, temperature=1.5, top_k=1)
    for kw in (dict(top_p=1e-6), dict(top_k=7, top_p=0.0), dict(top_k=1, min_p=1.0)):       # of equal logits the lowest index
        for a, b in zip(first, Generator(m).generate(ids, 8, temperature=0.5, **kw)):
            assert torch.equal(a, b)
    torch.manual_seed(3)
    whole = Generator(m).generate(ids, 8, temperature=1.0)
    torch.manual_seed(3)
    for a, b in zip(whole, CachedSampler(m, 8, top_k=40, top_p=1.0)(None, torch.stack(ids))):
        assert torch.equal(a, b)                # the same draws: 40 tokens are all
    some = CachedSampler(m, 8, top_p=0.5, cache_bits=16, budget=8, recent=2, slack=2)(None, torch.stack(ids))
    assert some.shape == (4, 14) and (some < 40).all()


def check_refusals(m):
    ids = prompts(m, (5,))
    for kw in (dict(cache_bits=8), dict(budget=10), dict(cache_bits=16, budget=0), dict(cache_bits=16, budget=4, recent=5),
               dict(cache_bits=16, budget=4, recent=-1), dict(cache_bits=16, budget=4, slack=0)):
        with pytest.raises(ValueError):
            Generator(m, **kw)
    with pytest.raises(ValueError):
        Generator(m, cache_bits=16).generate(ids, 4, beams=2)
    for kw in (dict(top_k=3), dict(top_p=0.5), dict(min_p=0.5)):
        with pytest.raises(ValueError):
            Generator(m).generate(ids, 4, beams=2, **kw)
    for kw in (dict(top_k=-1), dict(top_p=1.5), dict(min_p=-0.5), dict(temperature=1.0, top_p=float("nan"))):
        with pytest.raises(ValueError):
            Generator(m).generate(ids, 4, **{"temperature": 1.0, **kw})


def test_refusals():
    check_refusals(model())
