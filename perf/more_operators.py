"""Generation from a key/value cache held in 16 bits that keeps to a budget, and sampling: the operators of one decode step, measured.

Four kinds of work, each over the range of sizes that rollouts and evaluation by generation meet:

``append``   tokens of a fused q|k|v projection go into a paged cache, with the rotation on the way; the angle's position is given
             apart from the place in the cache, because a cache that tokens were taken out of is shorter than its sequence
``attend``   attention of the newest tokens of every sequence over its pages; where it is weighed, the weight that every kept token
             got from them is added to a running sum per key/value head
``evict``    sequences longer than the budget keep their newest tokens and, of the others, those with the largest sums, per layer and
             key/value head; keys, values and sums move down in their order
``sample``   the next token of every sequence from its logits: temperature, top-k, top-p, min-p, with given waiting times

The cache of a layer is ``[pages, 2, kv_heads, page_size, head_dim]`` (0: keys, 1: values). The next token is the first to arrive: of the
tokens that the filters leave, that with the largest ``weight / waiting time``, where waiting times are exponentially distributed.

``listed()`` gives the fixed cases, ``draw(rng)`` another one out of the same ranges, ``exact`` the results in 64 bits.
"""
import math
import random

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
THETA = 10000.0
INF = float("inf")


def listed():
    return [
        # one token of 64 rollouts through a layer with grouped heads, from caches that have lost tokens: latency counts
        dict(name="append_step", kind="append", heads=32, kv_heads=8, dim=128, page=16, batch=64, new=1, past=2000, gone=700, lens=1,
             dtype="bf16"),
        # prompts of different lengths packed one behind another, padding among them
        dict(name="append_prompts", kind="append", heads=32, kv_heads=8, dim=128, page=64, batch=8, new=2048, past=0, gone=0, lens=2,
             dtype="bf16"),
        # one rollout of the 1.3B model: latency counts
        dict(name="attend_single", kind="attend", heads=16, kv_heads=16, dim=128, page=16, batch=1, new=1, longest=1531, weighed=False,
             lens=4, dtype="bf16"),
        # a batch of rollouts at every length up to the model's, grouped heads
        dict(name="attend_rollouts", kind="attend", heads=32, kv_heads=8, dim=128, page=16, batch=32, new=1, longest=4096, weighed=False,
             lens=5, dtype="bf16"),
        # long documents
        dict(name="attend_long", kind="attend", heads=32, kv_heads=8, dim=128, page=64, batch=2, new=1, longest=100003, weighed=False,
             lens=6, dtype="bf16"),
        # rollouts of the 7B model whose caches keep to a budget
        dict(name="attend_weighed", kind="attend", heads=32, kv_heads=32, dim=128, page=32, batch=16, new=1, longest=1152, weighed=True,
             lens=7, dtype="bf16"),
        # the last tokens of prompts say which of their tokens carry weight: 64-wide heads, prompts shorter than that among them
        dict(name="attend_window", kind="attend", heads=16, kv_heads=4, dim=64, page=32, batch=19, new=31, longest=1801, weighed=True,
             lens=8, dtype="fp16"),
        # some layers of a batch of rollouts, 128 tokens over the budget
        dict(name="evict_layers", kind="evict", layers=8, kv_heads=8, dim=128, page=16, batch=8, longest=1152, budget=1024, recent=64,
             lens=9, dtype="bf16"),
        # one layer of a long document, halved
        dict(name="evict_long", kind="evict", layers=1, kv_heads=8, dim=128, page=64, batch=1, longest=100003, budget=50001, recent=1000,
             lens=10, dtype="bf16"),
        # one sequence with both usual filters: latency counts
        dict(name="sample_single", kind="sample", batch=1, vocab=32000, temperature=0.7, top_k=50, top_p=0.95, min_p=0.0, dtype="bf16"),
        # a batch of rollouts, the nucleus alone
        dict(name="sample_nucleus", kind="sample", batch=192, vocab=32000, temperature=1.0, top_k=0, top_p=0.9, min_p=0.0, dtype="fp32"),
        # rollouts drawn from the model's own distribution, a larger vocabulary of odd size
        dict(name="sample_plain", kind="sample", batch=64, vocab=100003, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, dtype="bf16"),
    ]


def _between(rng, low, high, step=1):
    """A multiple of `step`, even over the logarithm of [low, high]."""
    v = math.exp(rng.uniform(math.log(low), math.log(high)))
    return min(high, max(low, int(round(v / step)) * step))


def draw(rng):
    kind = rng.choice(["append", "attend", "evict", "sample"])
    dtype, page, lens = rng.choice(["bf16", "bf16", "fp16"]), rng.choice([16, 32, 64]), rng.randrange(1 << 20)
    kv, dim = rng.choice([1, 2, 3, 4, 8, 16, 32]), rng.choice([64, 128])
    heads = kv * rng.choice([g for g in (1, 2, 4, 8) if kv * g <= 32])
    if kind == "append":
        batch = _between(rng, 1, 64)
        new = rng.choice([1, _between(rng, 2, max(2, 16384 * 48 // (batch * (heads + 2 * kv)) * 128 // dim))])
        past = rng.randrange(0, 2000)
        return dict(kind=kind, heads=heads, kv_heads=kv, dim=dim, page=page, batch=batch, new=min(new, 4096), past=past,
                    gone=rng.choice([0, rng.randrange(0, past + 1)]), lens=lens, dtype=dtype)
    if kind == "attend":
        batch, new = _between(rng, 1, 64), rng.choice([1, 1, 1, 2, 4, 31])
        most = min(100003, 2 * 98000 * 8 * 128 // (batch * kv * dim), 2 * 98000 * 32 * 128 // (batch * new * heads * dim))
        return dict(kind=kind, heads=heads, kv_heads=kv, dim=dim, page=page, batch=batch, new=new, longest=_between(rng, 16, max(16, most)),
                    weighed=rng.choice([True, False]), lens=lens, dtype=dtype)
    if kind == "evict":
        layers = _between(rng, 1, 32)
        batch = _between(rng, 1, max(1, min(32, 256 // layers)))
        most = max(32, min(100003, 8 * 100003 * 128 // (layers * batch * kv * dim)))
        longest = _between(rng, 32, most)
        budget = max(1, int(longest * rng.uniform(0.4, 0.97)))
        return dict(kind=kind, layers=layers, kv_heads=kv, dim=dim, page=page, batch=batch, longest=longest, budget=budget,
                    recent=rng.choice([0, rng.randrange(0, budget + 1), budget // 8]), lens=lens, dtype=dtype)
    vocab = _between(rng, 1000, 131072)
    filters = rng.choice([(0, 1.0, 0.0), (50, 1.0, 0.0), (0, 0.9, 0.0), (_between(rng, 1, 1000), 0.95, 0.0), (0, 1.0, 0.05), (20, 0.8, 0.02),
                          (0, 0.999, 0.0)])
    return dict(kind=kind, batch=_between(rng, 1, max(1, min(512, 6400000 // vocab))), vocab=vocab, temperature=rng.choice([0.3, 0.7, 1.0, 1.0, 1.5]),
                top_k=filters[0], top_p=filters[1], min_p=filters[2], dtype=rng.choice(["bf16", "fp16", "fp32"]))


def _lengths(case):
    """Tokens of each sequence, by the case alone."""
    r = random.Random(case["lens"])
    B = case["batch"]
    if case["kind"] == "append":   # (tokens in the cache before, new tokens)
        past = [r.randint(case["gone"], case["past"]) - case["gone"] for _ in range(B)]
        return past, [case["new"] if case["new"] < 2 else r.randint(case["new"] // 3, case["new"]) for _ in range(B)]
    full = case["longest"]
    if case["kind"] == "evict":    # most sequences are over the budget, as far as they may grow before they are cut
        return [full if b == 0 else r.randint(1, full) if b % 4 == 3 else r.randint(min(full, case["budget"] + 1), full) for b in range(B)]
    return [full if b == 0 else r.randint(1, full) if B > 2 else full - r.randint(0, full // 8) for b in range(B)]


def _random(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _normal(g, shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=g, device=DEV, dtype=torch.float32) * scale).to(dtype)


def _tables(length, dim):
    inv = 1.0 / (THETA ** (torch.arange(0, dim, 2, dtype=torch.float32, device=DEV) / dim))
    f = torch.outer(torch.arange(length, dtype=torch.float32, device=DEV), inv)
    return f.cos(), f.sin()


def _pages(g, lengths, page):
    """A page table whose pages lie in no order, and how many pages there are."""
    width = max(1, -(-max(lengths) // page))
    need = [-(-n // page) for n in lengths]
    pool = torch.randperm(sum(need), generator=g, device=DEV).to(torch.int32)
    table = torch.zeros(len(lengths), width, dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = pool[at: at + n]
        at += n
    return table, sum(need)


def _filled(g, shape, dtype):
    """Pages with keys and values of a sequence: some channels of the keys are larger than the others."""
    data = torch.empty(shape, dtype=dtype, device=DEV)
    kv_heads, page, dim = shape[-3:]
    channel = 1 + 3 * (torch.rand(1, kv_heads, 1, dim, generator=g, device=DEV) > 0.95).float()
    flat = data.view(-1, 2, kv_heads, page, dim)
    step = max(1, (1 << 25) // (kv_heads * page * dim))
    for a in range(0, flat.shape[0], step):
        n = min(step, flat.shape[0] - a)
        for i in range(2):
            flat[a: a + n, i] = (_normal(g, (n, kv_heads, page, dim)) * (channel if i == 0 else 0.7)).to(dtype)
    return data


def _sums(g, shape, lengths):
    """What attention has left: a few tokens have most of the weight; nothing behind a sequence."""
    w = torch.exp(_normal(g, shape, scale=2.0))
    behind = torch.arange(shape[-1], device=DEV) >= torch.tensor(lengths, device=DEV).view(-1, 1, 1)
    return torch.where(behind, torch.zeros_like(w), w)


def prepare(case, seed):
    g, c = _random(seed), case
    dtype = DTYPES[c["dtype"]]
    if c["kind"] == "append":
        past, new = _lengths(c)
        total = [a + b for a, b in zip(past, new)]
        T = sum(new)
        table, pages = _pages(g, total, c["page"])
        cache = torch.zeros(pages, 2, c["kv_heads"], c["page"], c["dim"], dtype=dtype, device=DEV)
        seq = torch.repeat_interleave(torch.arange(c["batch"], dtype=torch.int32), torch.tensor(new)).to(DEV)
        pos = torch.cat([torch.arange(a, a + b, dtype=torch.int32) for a, b in zip(past, new)])
        angles = pos + c["gone"]
        if c["new"] > 1:
            pos[torch.rand(T, generator=torch.Generator().manual_seed(c["lens"])) < 0.02] = -1      # padding
        cos, sin = _tables(max(total) + c["gone"], c["dim"])
        return dict(case=c, cache=cache, table=table, seq=seq, pos=pos.to(DEV), angles=angles.to(DEV), cos=cos, sin=sin,
                    qkv=_normal(g, (T, (c["heads"] + 2 * c["kv_heads"]) * c["dim"]), dtype))
    if c["kind"] == "attend":
        lengths = _lengths(c)
        table, pages = _pages(g, lengths, c["page"])
        return dict(case=c, cache=_filled(g, (pages, 2, c["kv_heads"], c["page"], c["dim"]), dtype), table=table,
                    lengths=torch.tensor(lengths, dtype=torch.int32, device=DEV),
                    q=_normal(g, (c["batch"], c["new"], c["heads"], c["dim"]), dtype, 1.5),
                    weights=_sums(g, (c["batch"], c["kv_heads"], table.shape[1] * c["page"]), lengths) if c["weighed"] else None)
    if c["kind"] == "evict":
        lengths = _lengths(c)
        table, pages = _pages(g, lengths, c["page"])
        shape = (c["layers"], c["batch"], c["kv_heads"], table.shape[1] * c["page"])
        learned = _sums(g, shape, lengths)
        return dict(case=c, cache=_filled(g, (c["layers"], pages, 2, c["kv_heads"], c["page"], c["dim"]), dtype), table=table,
                    lengths=torch.tensor(lengths, dtype=torch.int32, device=DEV), learned=learned, weights=torch.empty_like(learned))
    B, V = c["batch"], c["vocab"]
    logits = _normal(g, (B, V), scale=2.5)
    logits += 9.0 * (torch.rand(B, V, generator=g, device=DEV) < 8 / V)                    # likely tokens
    logits[torch.rand(B, V, generator=g, device=DEV) < 0.001] = -INF                      # tokens that may not follow
    return dict(case=c, logits=logits.to(dtype), waiting=torch.empty(B, V, device=DEV).exponential_(generator=g))


def run(state):
    return {"append": _append, "attend": _attend, "evict": _evict, "sample": _sample}[state["case"]["kind"]](state)


def _append(s):
    c = s["case"]
    if own:
        from atorch_b200 import ops

        q, k = ops.kv_append(s["cache"], s["table"], s["seq"], s["pos"], s["qkv"], c["heads"], s["cos"], s["sin"], angles=s["angles"],
                             return_keys=True)
        return q, k, s["cache"]
    H, KV, D, page = c["heads"], c["kv_heads"], c["dim"], c["page"]
    x = s["qkv"].view(-1, H + 2 * KV, D).float()
    at = s["angles"].long()
    cos, sin = s["cos"][at].unsqueeze(1), s["sin"][at].unsqueeze(1)
    a, b = x[:, : H + KV, : D // 2], x[:, : H + KV, D // 2:]
    real = s["pos"] >= 0
    turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    turned = torch.where(real[:, None, None], turned, x[:, : H + KV]).to(s["qkv"].dtype)      # padding is not turned
    place = s["pos"].clamp(min=0).long()
    to, slot = s["table"][s["seq"].long(), place // page].long()[real], (place % page)[real]
    s["cache"][to, 0, :, slot] = turned[:, H:][real]
    s["cache"][to, 1, :, slot] = s["qkv"].view(-1, H + 2 * KV, D)[:, H + KV:][real]
    return turned[:, :H].contiguous(), turned[:, H:].contiguous(), s["cache"]


def _attend(s):
    c, q = s["case"], s["q"]
    if own:
        from atorch_b200 import ops

        out = ops.kv_attention(q, s["cache"], s["table"], s["lengths"], weights=s["weights"])
        return (out, s["weights"]) if c["weighed"] else out
    B, S, H, D = q.shape
    KV = c["kv_heads"]
    held = s["cache"][s["table"].long()]                                     # [B, P, 2, KV, page, D]
    k = held[:, :, 0].transpose(1, 2).flatten(2, 3).float()                  # [B, KV, T, D]
    v = held[:, :, 1].transpose(1, 2).flatten(2, 3).float()
    T = k.shape[2]
    behind = (torch.arange(T, device=q.device) >= s["lengths"].view(B, 1)).view(B, 1, T, 1)
    k, v = k.masked_fill(behind, 0.0), v.masked_fill(behind, 0.0)
    qf = q.float().view(B, S, KV, H // KV, D).permute(0, 2, 3, 1, 4).reshape(B, KV, H // KV * S, D)
    score = torch.matmul(qf, k.transpose(-1, -2)) / math.sqrt(D)
    limit = s["lengths"].view(B, 1, 1) - S + 1 + torch.arange(S, device=q.device).view(1, S, 1)      # keys that a token sees
    seen = (torch.arange(T, device=q.device).view(1, 1, T) < limit).repeat(1, H // KV, 1).view(B, 1, H // KV * S, T)
    score = torch.where(seen, score, torch.full_like(score, -INF))
    top = score.amax(-1, keepdim=True)
    e = torch.exp(score - torch.where(top > -INF, top, torch.zeros_like(top)))
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total > 0, total, torch.ones_like(total))
    out = torch.matmul(p, v).view(B, KV, H // KV, S, D).permute(0, 3, 1, 2, 4).reshape(B, S, H, D).to(q.dtype)
    if not c["weighed"]:
        return out
    s["weights"] += p.sum(2)
    return out, s["weights"]


def _evict(s):
    c = s["case"]
    s["weights"].copy_(s["learned"])       # as the attention since the last cut has left them: every pass has the same to do
    if own:
        from atorch_b200 import ops

        lengths = ops.kv_evict(s["cache"], s["table"], s["lengths"], s["weights"], c["budget"], c["recent"])
        return s["cache"], s["weights"], lengths
    budget, page = c["budget"], c["page"]
    cut = torch.tensor([b for b, n in enumerate(_lengths(c)) if n > budget], device=DEV)      # sequences over the budget
    n, w, rows = s["lengths"][cut].view(-1, 1, 1), s["weights"][:, cut], s["table"][cut].long()
    L, B, KV, T = w.shape
    i = torch.arange(T, device=w.device)
    rank = torch.where(i < n - c["recent"], w, torch.where(i < n, torch.full_like(w, INF), torch.full_like(w, -INF)))
    kept = rank.sort(dim=-1, descending=True, stable=True).indices[..., :budget].sort(-1).values              # [L, B, KV, budget]
    held = s["cache"][:, rows].permute(0, 1, 3, 4, 2, 5, 6).flatten(4, 5)                                # [L, B, 2, KV, T, D]
    moved = held.gather(4, kept[:, :, None, :, :, None].expand(L, B, 2, KV, budget, c["dim"]))
    j = torch.arange(budget, device=w.device)
    s["cache"][:, rows[:, j // page], :, :, j % page] = moved.permute(1, 4, 0, 2, 3, 5)
    sums = torch.zeros_like(w)
    sums[..., :budget] = w.gather(3, kept)
    s["weights"][:, cut] = sums
    return s["cache"], s["weights"], s["lengths"].clamp(max=budget)


def _sample(s):
    c = s["case"]
    if own:
        from atorch_b200 import ops

        return ops.sample(s["logits"], s["waiting"], c["temperature"], c["top_k"], c["top_p"], c["min_p"])
    x = s["logits"].double()               # in 64 bits: borders of the filters, and candidates that arrive at nearly the same time
    x = torch.where(torch.isnan(x), torch.full_like(x, -INF), x)
    w = torch.exp((x - x.amax(-1, keepdim=True)) / c["temperature"])
    order = x.sort(dim=-1, descending=True, stable=True).indices
    sorted_w = w.gather(1, order)
    left = sorted_w >= c["min_p"]
    if c["top_k"] > 0:
        sorted_w = torch.where(torch.arange(c["vocab"], device=x.device) < c["top_k"], sorted_w, torch.zeros_like(sorted_w))
    if c["top_p"] < 1:
        sums = sorted_w.cumsum(-1)
        left = left & (sums - sorted_w < c["top_p"] * sums[:, -1:])
    sorted_w = torch.where(left, sorted_w, torch.zeros_like(sorted_w))
    w = torch.zeros_like(w).scatter(1, order, sorted_w)
    tokens = (w / s["waiting"].double()).argmax(-1)
    logprobs = torch.log(w.gather(1, tokens[:, None])[:, 0] / w.sum(-1))
    return tokens, logprobs.float()


def work(case):
    c, size = case, 4 if case["dtype"] == "fp32" else 2
    if c["kind"] == "append":
        past, new = _lengths(c)
        T, H, KV, D = sum(new), c["heads"], c["kv_heads"], c["dim"]
        longest = max(a + b for a, b in zip(past, new))
        return {"bytes": T * (2 * H + 5 * KV) * D * size + min(T, longest) * D * 4 + 12 * T, "flops": 3 * T * (H + KV) * D}
    if c["kind"] == "attend":
        n = sum(_lengths(c))
        io = 2 * c["batch"] * c["new"] * c["heads"] * c["dim"] * size
        return {"bytes": n * c["kv_heads"] * (2 * c["dim"] * size + (8 if c["weighed"] else 0)) + io,
                "flops": 4 * n * c["new"] * c["heads"] * c["dim"]}
    if c["kind"] == "evict":
        over = [n for n in _lengths(c) if n > c["budget"]]
        units = c["layers"] * c["kv_heads"]
        # tokens that lie before the first one that goes stay where they are: few
        return {"bytes": units * sum(8 * n + 2 * c["budget"] * 2 * c["dim"] * size for n in over), "flops": units * sum(over)}
    B, V = c["batch"], c["vocab"]
    waits = V if c["top_k"] == 0 and c["top_p"] >= 1 and c["min_p"] == 0 else min(V, c["top_k"])      # of tokens that may be drawn
    return {"bytes": B * (V * size + 4 * waits + 12), "flops": 6 * B * V}


def exact(case, seed):
    s, c = prepare(case, seed), case
    if c["kind"] == "append":
        H, KV, D = c["heads"], c["kv_heads"], c["dim"]
        x = s["qkv"].double().view(-1, H + 2 * KV, D)
        at = s["angles"].long()
        z = torch.complex(x[:, : H + KV, : D // 2], x[:, : H + KV, D // 2:])
        z = z * torch.complex(s["cos"][at].double(), s["sin"][at].double()).unsqueeze(1)
        turned = torch.cat([z.real, z.imag], -1)
        turned = torch.where((s["pos"] >= 0)[:, None, None], turned, x[:, : H + KV])
        cache = s["cache"].double()
        keep = (s["pos"] >= 0).nonzero()[:, 0]
        p = s["pos"][keep].long()
        page = s["table"][s["seq"][keep].long(), p // c["page"]].long()
        flat = cache.permute(0, 3, 1, 2, 4).reshape(-1, 2, KV, D)          # [places, 2, KV, D]
        flat[page * c["page"] + p % c["page"]] = torch.stack([turned[keep, H:], x[keep, H + KV:]], 1)
        return turned[:, :H], turned[:, H:], flat.view(-1, c["page"], 2, KV, D).permute(0, 2, 3, 1, 4)
    if c["kind"] == "attend":
        q, (B, S, H, D), KV = s["q"].double(), s["q"].shape, c["kv_heads"]
        out = torch.zeros(B, S, H, D, dtype=torch.float64, device=q.device)
        sums = s["weights"].double() if c["weighed"] else None
        for b, n in enumerate(_lengths(c)):
            rows = s["table"][b, : -(-n // c["page"])].long()
            for h in range(KV):
                kv = s["cache"][rows, :, h].transpose(0, 1).reshape(2, -1, D)[:, :n].double()
                heads = slice(h * (H // KV), (h + 1) * (H // KV))
                for i in range(S):
                    m = n - S + i + 1
                    if m > 0:
                        p = torch.softmax(q[b, i, heads] @ kv[0, :m].t() / D ** 0.5, -1)
                        out[b, i, heads] = p @ kv[1, :m]
                        if sums is not None:
                            sums[b, h, :m] += p.sum(0)
        return (out, sums) if c["weighed"] else out
    if c["kind"] == "evict":
        cache, sums = s["cache"].double(), s["learned"].double()
        lengths, page = _lengths(c), c["page"]
        for b, n in enumerate(lengths):
            if n <= c["budget"]:
                continue
            at = s["table"][b, torch.arange(n, device=DEV) // page].long()
            place = torch.arange(n, device=DEV) % page
            for layer in range(c["layers"]):
                for h in range(c["kv_heads"]):
                    w = sums[layer, b, h, :n].clone()
                    first = torch.argsort(-w[: n - c["recent"]], stable=True)[: c["budget"] - c["recent"]]
                    kept = torch.cat([first.sort().values, torch.arange(n - c["recent"], n, device=DEV)])
                    cache[layer, at[: c["budget"]], :, h, place[: c["budget"]]] = cache[layer, at[kept], :, h, place[kept]]
                    sums[layer, b, h, :n] = 0
                    sums[layer, b, h, : c["budget"]] = w[kept]
        return cache, sums, None
    logits, chosen = s["logits"].double().cpu(), []
    waiting = s["waiting"].double().cpu()
    for x, t in zip(logits, waiting):
        ids = sorted(range(c["vocab"]), key=lambda i, v=x.tolist(): -v[i])                  # (stable: the lower index first)
        if c["top_k"] > 0:
            ids = ids[: c["top_k"]]
        ids = torch.tensor(ids)
        p = torch.softmax(x[ids] / c["temperature"], 0)
        n = len(ids) if c["top_p"] >= 1 else int((p.cumsum(0) - p < c["top_p"]).sum())
        n = min(n, int((p >= c["min_p"] * p[0]).sum()))
        p = p[:n] / p[:n].sum()
        chosen.append(torch.log(p[(p / t[ids[:n]]).argmax()]))
    return None, torch.stack(chosen).to(DEV)
