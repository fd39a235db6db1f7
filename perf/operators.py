"""Generation from a key/value cache held in 4 bits: the operators of one decode step, measured.

Four kinds of work, each over the range of sizes that rollouts and evaluation by generation meet:

``append``   tokens of a fused q|k|v projection go into a paged 4-bit cache, with the rotation on the way, and are read back as
             what the cache stands for (a prompt attends to that)
``attend``   attention of the newest tokens of every sequence over its pages
``w4``       a linear layer whose weights are held in 4 bits with a scale per group
``beam``     one step of a beam search: selection over beams and vocabulary, and the cache's rows moved to their new beams

The cache of a layer is two tensors: ``codes`` uint8 ``[pages, 2, kv_heads, page_size, head_dim / 2]`` (0: keys, 1: values; byte
``i`` holds dim ``2 i`` in its low half and ``2 i + 1`` in its high one) and ``scales`` bf16 ``[pages, kv_heads, page_size, 4]``
(scale and minimum of the keys, scale and minimum of the values); a value is ``code * scale + minimum``. 4-bit weights are
``codes`` uint8 ``[rows, 16 * ceil(K / 32)]``, the same order, filled up with 8s, and ``scales`` bf16 ``[rows, ceil(K / group)]``; a
weight is ``(code - 8) * scale``.

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
        # one token of 16 rollouts through a layer of the 7B model: latency counts
        dict(name="append_step", kind="append", heads=32, kv_heads=32, dim=128, page=16, batch=16, new=1, past=2000, lens=1, dtype="bf16"),
        # prompts of different lengths packed one behind another, grouped heads
        dict(name="append_prompts", kind="append", heads=32, kv_heads=8, dim=128, page=64, batch=8, new=2048, past=0, lens=2, dtype="bf16"),
        # short pieces at odd places of their sequences, 64-wide heads, padding among them
        dict(name="append_odd", kind="append", heads=12, kv_heads=3, dim=64, page=32, batch=37, new=61, past=517, lens=3, dtype="fp16"),
        # one rollout of the 1.3B model: latency counts
        dict(name="attend_single", kind="attend", heads=16, kv_heads=16, dim=128, page=16, batch=1, new=1, longest=1531, lens=4, dtype="bf16"),
        # a batch of rollouts at every length up to the model's, grouped heads
        dict(name="attend_rollouts", kind="attend", heads=32, kv_heads=8, dim=128, page=16, batch=32, new=1, longest=4096, lens=5, dtype="bf16"),
        # long documents
        dict(name="attend_long", kind="attend", heads=32, kv_heads=8, dim=128, page=64, batch=2, new=1, longest=100003, lens=6, dtype="bf16"),
        # several new tokens per sequence, 64-wide heads, sequences shorter than that among them
        dict(name="attend_pieces", kind="attend", heads=16, kv_heads=4, dim=64, page=32, batch=19, new=5, longest=1800, lens=7, dtype="fp16"),
        # down projection of the 7B model for one sequence
        dict(name="w4_single", kind="w4", rows=1, out=4096, inner=11008, group=128, dtype="bf16"),
        # gate|up projection of the 7B model for a batch of rollouts
        dict(name="w4_batch", kind="w4", rows=16, out=22016, inner=4096, group=128, dtype="bf16"),
        # odd sizes
        dict(name="w4_odd", kind="w4", rows=5, out=5003, inner=1111, group=64, dtype="fp16"),
        # one prompt, four beams, the cache of a small model
        dict(name="beam_single", kind="beam", batch=1, beams=4, vocab=32000, layers=8, kv_heads=8, dim=128, page=16, past=203, dtype="bf16"),
        # an evaluation batch, the cache of a whole model with grouped heads
        dict(name="beam_batch", kind="beam", batch=24, beams=8, vocab=32000, layers=32, kv_heads=8, dim=128, page=16, past=410, dtype="bf16"),
    ]


def _between(rng, low, high, step=1):
    """A multiple of `step`, even over the logarithm of [low, high]."""
    v = math.exp(rng.uniform(math.log(low), math.log(high)))
    return min(high, max(low, int(round(v / step)) * step))


def draw(rng):
    kind = rng.choice(["append", "attend", "w4", "beam"])
    dtype, page, lens = rng.choice(["bf16", "bf16", "fp16"]), rng.choice([16, 32, 64]), rng.randrange(1 << 20)
    if kind == "append":
        kv = rng.choice([1, 2, 3, 4, 8, 16, 32])
        heads, dim, batch = kv * rng.choice([g for g in (1, 2, 4, 8) if kv * g <= 32]), rng.choice([64, 128]), _between(rng, 1, 64)
        new = rng.choice([1, _between(rng, 2, max(2, 16384 * 48 // (batch * (heads + 2 * kv)) * 128 // dim))])
        return dict(kind=kind, heads=heads, kv_heads=kv, dim=dim, page=page, batch=batch, new=min(new, 4096), past=rng.randrange(0, 2000), lens=lens,
                    dtype=dtype)
    if kind == "attend":
        kv = rng.choice([1, 2, 3, 4, 8, 16, 32])
        heads, dim, batch = kv * rng.choice([g for g in (1, 2, 4, 8) if kv * g <= 32]), rng.choice([64, 128]), _between(rng, 1, 64)
        most = 2 * 100003 * 8 * 128 // (batch * kv * dim)
        return dict(kind=kind, heads=heads, kv_heads=kv, dim=dim, page=page, batch=batch, new=rng.choice([1, 1, 1, 2, 4, 7]),
                    longest=_between(rng, 16, min(most, 100003)), lens=lens, dtype=dtype)
    if kind == "w4":
        out = _between(rng, 64, 32000)
        return dict(kind=kind, rows=_between(rng, 1, 32), out=out, inner=_between(rng, 64, min(16384, 22016 * 4096 // out), rng.choice([1, 32, 128])),
                    group=rng.choice([32, 64, 128]), dtype=dtype)
    beams = _between(rng, 2, 16)
    return dict(kind=kind, batch=_between(rng, 1, 192 // beams), beams=beams, vocab=_between(rng, 1000, 32000), layers=_between(rng, 1, 32),
                kv_heads=rng.choice([2, 4, 8]), dim=rng.choice([64, 128]), page=page, past=rng.randrange(1, 500), dtype=rng.choice(["bf16", "bf16", "fp32"]))


def _lengths(case):
    """Tokens of each sequence, by the case alone."""
    r = random.Random(case["lens"])
    B = case["batch"]
    if case["kind"] == "append":   # (tokens in the cache before, new tokens)
        past = [r.randint(0, case["past"]) for _ in range(B)]
        return past, [case["new"] if case["new"] < 2 else r.randint(case["new"] // 3, case["new"]) for _ in range(B)]
    full = case["longest"]
    return [full if b == 0 else r.randint(1, full) if B > 2 else full - r.randint(0, full // 8) for b in range(B)]


def _random(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _normal(g, shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=g, device=DEV, dtype=torch.float32) * scale).to(dtype)


def _tables(length, dim):
    inv = 1.0 / (THETA ** (torch.arange(0, dim, 2, dtype=torch.float32, device=DEV) / dim))
    f = torch.outer(torch.arange(length, dtype=torch.float32, device=DEV), inv)
    return f.cos(), f.sin()


def _pages(g, lengths, page, spare=0):
    """A page table whose pages lie in no order, and how many pages there are."""
    width = max(1, -(-max(lengths) // page))
    need = [-(-n // page) for n in lengths]
    pool = torch.randperm(sum(need) + spare, generator=g, device=DEV).to(torch.int32)
    table = torch.zeros(len(lengths), width, dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = pool[at: at + n]
        at += n
    return table, sum(need) + spare


def _quantise(x):
    """Codes (one a value), scale and minimum of each row of the last dimension, in 32 bits."""
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    scale = ((high - low) / 15).to(torch.bfloat16).float()
    low = low.to(torch.bfloat16).float()
    code = torch.where(scale > 0, torch.round((x - low) / scale).clamp(0, 15), torch.zeros_like(x))
    return code.to(torch.uint8), scale, low


def _pack(code):
    return code[..., 0::2] | (code[..., 1::2] << 4)


def _unpack(codes):
    return torch.stack([codes & 15, codes >> 4], -1).flatten(-2)


def _filled(g, pages, kv_heads, page, dim):
    """Pages with keys and values of a sequence: some channels of the keys are larger than the others."""
    codes = torch.empty(pages, 2, kv_heads, page, dim // 2, dtype=torch.uint8, device=DEV)
    scales = torch.empty(pages, kv_heads, page, 4, dtype=torch.bfloat16, device=DEV)
    channel = 1 + 3 * (torch.rand(1, kv_heads, 1, dim, generator=g, device=DEV) > 0.95).float()
    step = max(1, (1 << 25) // (kv_heads * page * dim))
    for a in range(0, pages, step):
        n = min(step, pages - a)
        for i in range(2):
            x = _normal(g, (n, kv_heads, page, dim)) * (channel if i == 0 else 0.7)
            code, scale, low = _quantise(x)
            codes[a: a + n, i] = _pack(code)
            scales[a: a + n, :, :, 2 * i] = scale[..., 0].to(torch.bfloat16)
            scales[a: a + n, :, :, 2 * i + 1] = low[..., 0].to(torch.bfloat16)
    return codes, scales


def prepare(case, seed):
    g, c = _random(seed), case
    dtype = DTYPES[c["dtype"]]
    if c["kind"] == "append":
        past, new = _lengths(c)
        total = [a + b for a, b in zip(past, new)]
        T = sum(new)
        table, pages = _pages(g, total, c["page"])
        codes = torch.zeros(pages, 2, c["kv_heads"], c["page"], c["dim"] // 2, dtype=torch.uint8, device=DEV)
        scales = torch.zeros(pages, c["kv_heads"], c["page"], 4, dtype=torch.bfloat16, device=DEV)
        seq = torch.repeat_interleave(torch.arange(c["batch"], dtype=torch.int32), torch.tensor(new)).to(DEV)
        pos = torch.cat([torch.arange(a, a + b, dtype=torch.int32) for a, b in zip(past, new)])
        if c["new"] > 1:
            pos[torch.rand(T, generator=torch.Generator().manual_seed(c["lens"])) < 0.02] = -1      # padding
        cos, sin = _tables(max(total), c["dim"])
        return dict(case=c, layer=(codes, scales), table=table, seq=seq, pos=pos.to(DEV), cos=cos, sin=sin,
                    qkv=_normal(g, (T, (c["heads"] + 2 * c["kv_heads"]) * c["dim"]), dtype))
    if c["kind"] == "attend":
        lengths = _lengths(c)
        table, pages = _pages(g, lengths, c["page"])
        return dict(case=c, layer=_filled(g, pages, c["kv_heads"], c["page"], c["dim"]), table=table,
                    lengths=torch.tensor(lengths, dtype=torch.int32, device=DEV),
                    q=_normal(g, (c["batch"], c["new"], c["heads"], c["dim"]), dtype, 1.5))
    if c["kind"] == "w4":
        N, K, G = c["out"], c["inner"], c["group"]
        codes = torch.randint(0, 256, (N, -(-K // 32) * 16), generator=g, device=DEV, dtype=torch.uint8)
        codes[:, (K + 1) // 2:] = 0x88
        if K % 2:
            codes[:, K // 2] = (codes[:, K // 2] & 15) | 0x80
        scales = (0.02 / 7 * (0.5 + torch.rand(N, -(-K // G), generator=g, device=DEV))).to(torch.bfloat16)
        return dict(case=c, x=_normal(g, (c["rows"], K), dtype), codes=codes, scales=scales)
    B, W, V, L = c["batch"], c["beams"], c["vocab"], c["layers"]
    logits = _normal(g, (B, W, V), torch.float32, 2.0)
    logits[torch.rand(B, W, V, generator=g, device=DEV) < 0.001] = -INF      # tokens that may not follow
    # full pages are shared by the beams of a sequence, the last one is each beam's own
    full = c["past"] // c["page"]
    table = torch.empty(B * W, full + 1, dtype=torch.int32, device=DEV)
    pool = torch.randperm(B * (full + W), generator=g, device=DEV).to(torch.int32)
    table[:, :full] = pool[: B * full].view(B, 1, full).expand(B, W, full).reshape(B * W, full)
    table[:, full] = pool[B * full:]
    one_codes, one_scales = _filled(g, B * (full + W), c["kv_heads"], c["page"], c["dim"])
    return dict(case=c, logits=logits.to(dtype), scores=-10 + _normal(g, (B, W)), finished=torch.rand(B, W, generator=g, device=DEV) < 0.1,
                codes=one_codes.expand(L, *one_codes.shape).clone(), scales=one_scales.expand(L, *one_scales.shape).clone(), table=table,
                lengths=torch.full((B * W,), c["past"], dtype=torch.int32, device=DEV))


EOS = 2


def run(state):
    return {"append": _append, "attend": _attend, "w4": _w4, "beam": _beam}[state["case"]["kind"]](state)


def _append(s):
    c = s["case"]
    if own:
        from atorch_b200 import ops

        q = ops.kv4_append(s["layer"], s["table"], s["seq"], s["pos"], s["qkv"], c["heads"], s["cos"], s["sin"])
        return q, *ops.kv4_read(s["layer"], s["table"], s["seq"], s["pos"], s["qkv"].dtype)
    codes, scales = s["layer"]
    H, KV, D, page = c["heads"], c["kv_heads"], c["dim"], c["page"]
    x = s["qkv"].view(-1, H + 2 * KV, D).float()
    at = s["pos"].clamp(min=0).long()
    cos, sin = s["cos"][at].unsqueeze(1), s["sin"][at].unsqueeze(1)
    a, b = x[:, : H + KV, : D // 2], x[:, : H + KV, D // 2:]
    turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    kv = torch.stack([turned[:, H:], x[:, H + KV:]], 1)                     # [T, 2, KV, D]
    code, scale, low = _quantise(kv)
    real = s["pos"] >= 0
    where = s["table"][s["seq"].long(), at // page].long()[real], (at % page)[real]
    codes[where[0], :, :, where[1]] = _pack(code)[real]
    scales[where[0], :, where[1]] = torch.cat([scale, low], -1).permute(0, 2, 1, 3).flatten(2)[real].to(torch.bfloat16)
    page_of, slot = s["table"][s["seq"].long(), at // page].long(), at % page
    sc = scales[page_of, :, slot].float()                                    # [T, KV, 4]
    back = _unpack(codes[page_of, :, :, slot]).float()
    k = back[:, 0] * sc[..., 0:1] + sc[..., 1:2]
    v = back[:, 1] * sc[..., 2:3] + sc[..., 3:4]
    k, v = (torch.where(real[:, None, None], t, torch.zeros_like(t)).to(s["qkv"].dtype) for t in (k, v))
    q = torch.where(real[:, None, None], turned[:, :H], x[:, :H])            # padding is not turned
    return q.to(s["qkv"].dtype), k, v


def _attend(s):
    c, q = s["case"], s["q"]
    if own:
        from atorch_b200 import ops

        return ops.kv4_attention(q, s["layer"], s["table"], s["lengths"])
    codes, scales = s["layer"]
    B, S, H, D = q.shape
    KV = c["kv_heads"]
    rows = s["table"].long()
    sc = scales[rows].transpose(2, 3).flatten(1, 2).float()                  # [B, T, KV, 4]
    held = codes[rows]                                                       # [B, P, 2, KV, page, D / 2]
    k = (_unpack(held[:, :, 0]).transpose(2, 3).flatten(1, 2).float() * sc[..., 0:1] + sc[..., 1:2]).transpose(1, 2)
    v = (_unpack(held[:, :, 1]).transpose(2, 3).flatten(1, 2).float() * sc[..., 2:3] + sc[..., 3:4]).transpose(1, 2)
    T = k.shape[2]
    qf = q.float().view(B, S, KV, H // KV, D).permute(0, 2, 3, 1, 4).reshape(B, KV, H // KV * S, D)
    score = torch.matmul(qf, k.transpose(-1, -2)) / math.sqrt(D)
    limit = s["lengths"].view(B, 1, 1) - S + 1 + torch.arange(S, device=q.device).view(1, S, 1)      # keys that a token sees
    seen = (torch.arange(T, device=q.device).view(1, 1, T) < limit).repeat(1, H // KV, 1).view(B, 1, H // KV * S, T)
    score = torch.where(seen, score, torch.full_like(score, -INF))
    top = score.amax(-1, keepdim=True)
    e = torch.exp(score - torch.where(top > -INF, top, torch.zeros_like(top)))
    total = e.sum(-1, keepdim=True)
    out = torch.matmul(e, v) / torch.where(total > 0, total, torch.ones_like(total))
    return out.view(B, KV, H // KV, S, D).permute(0, 3, 1, 2, 4).reshape(B, S, H, D).to(q.dtype)


def _w4(s):
    c, x = s["case"], s["x"]
    if own:
        from atorch_b200 import ops

        return ops.w4_linear(x, s["codes"], s["scales"], c["group"])
    K = c["inner"]
    w = (_unpack(s["codes"])[:, :K].float() - 8) * s["scales"].float().repeat_interleave(c["group"], 1)[:, :K]
    return torch.matmul(x.float(), w.t()).to(x.dtype)


def _beam(s):
    c, x = s["case"], s["logits"]
    if own:
        from atorch_b200 import ops

        scores, tokens, parents, finished = ops.beam_select(x, s["scores"], s["finished"], EOS)
        ops.beam_reorder(s["codes"], s["scales"], s["table"], s["lengths"], parents)
        return scores, tokens, parents, finished, s["table"], s["codes"], s["scales"]
    B, W, V, page = c["batch"], c["beams"], c["vocab"], c["page"]
    x = x.float()
    top = x.amax(-1, keepdim=True)
    lse = top + torch.log(torch.exp(x - top).sum(-1, keepdim=True))
    f = s["scores"].unsqueeze(-1) + (x - lse)
    f = torch.where(torch.isnan(f), torch.full_like(f, -INF), f)
    done = s["finished"].unsqueeze(-1)
    ends = torch.arange(V, device=x.device) == EOS
    f = torch.where(done, torch.where(ends, s["scores"].unsqueeze(-1), torch.full_like(f, -INF)), f)
    scores, at = torch.sort(f.view(B, W * V), dim=-1, descending=True, stable=True)
    scores, at = scores[:, :W], at[:, :W]
    parents, tokens = at // V, at % V
    finished = s["finished"].gather(1, parents) | (tokens == EOS)
    # rows of the table up to the full pages; the tokens of the last page are copied into the beam's own
    n = c["past"]
    full, rest = n // page, n % page
    source = (torch.arange(B, device=x.device).unsqueeze(1) * W + parents).flatten()
    s["table"][:, :full] = s["table"][source, :full]
    if rest:
        to, of = s["table"][:, full].long(), s["table"][source, full].long()
        s["codes"][:, to, :, :, :rest] = s["codes"][:, of, :, :, :rest]
        s["scales"][:, to, :, :rest] = s["scales"][:, of, :, :rest]
    return scores, tokens, parents.to(torch.int32), finished, s["table"], s["codes"], s["scales"]


def work(case):
    c, size = case, 4 if case["dtype"] == "fp32" else 2
    if c["kind"] == "append":
        past, new = _lengths(c)
        T, H, KV, D = sum(new), c["heads"], c["kv_heads"], c["dim"]
        longest = max(a + b for a, b in zip(past, new))
        return {"bytes": T * (2 * H + 2 * KV) * D * size + T * KV * (D + 8) + 2 * T * KV * D * size + min(T, longest) * D * 4 + 8 * T,
                "flops": 3 * T * (H + KV) * D + 8 * T * KV * D}
    if c["kind"] == "attend":
        n = sum(_lengths(c))
        io = 2 * c["batch"] * c["new"] * c["heads"] * c["dim"] * size
        return {"bytes": n * c["kv_heads"] * (c["dim"] + 8) + io, "flops": 4 * n * c["new"] * c["heads"] * c["dim"]}
    if c["kind"] == "w4":
        M, N, K = c["rows"], c["out"], c["inner"]
        return {"bytes": N * (-(-K // 2)) + 2 * N * (-(-K // c["group"])) + size * M * (N + K), "flops": 2 * M * N * K}
    rows = c["batch"] * c["beams"]
    moved = rows * (1 - 1 / c["beams"]) * c["layers"] * (c["past"] % c["page"]) * c["kv_heads"] * (c["dim"] + 8)
    return {"bytes": rows * c["vocab"] * size + 2 * moved, "flops": 4 * rows * c["vocab"]}


def exact(case, seed):
    s, c = prepare(case, seed), case
    if c["kind"] == "append":
        H, KV, D = c["heads"], c["kv_heads"], c["dim"]
        x = s["qkv"].double().view(-1, H + 2 * KV, D)
        real = (s["pos"] >= 0)[:, None, None]
        at = s["pos"].clamp(min=0).long()
        z = torch.complex(x[:, : H + KV, : D // 2], x[:, : H + KV, D // 2:])
        z = z * torch.complex(s["cos"][at].double(), s["sin"][at].double()).unsqueeze(1)
        turned = torch.cat([z.real, z.imag], -1)

        def held(t):
            low, high = t.amin(-1, keepdim=True), t.amax(-1, keepdim=True)
            step = ((high - low) / 15).to(torch.bfloat16).double()
            low = low.to(torch.bfloat16).double()
            return torch.where(real, ((t - low) / step).round().clamp(0, 15) * step + low, 0.0)

        return torch.where(real, turned[:, :H], x[:, :H]), held(turned[:, H:]), held(x[:, H + KV:])
    if c["kind"] == "attend":
        codes, scales = s["layer"]
        q, (B, S, H, D), KV = s["q"].double(), s["q"].shape, c["kv_heads"]
        out = torch.zeros(B, S, H, D, dtype=torch.float64, device=q.device)
        for b, n in enumerate(_lengths(c)):
            rows = s["table"][b, : -(-n // c["page"])].long()
            for h in range(KV):
                sc = scales[rows, h].double().reshape(-1, 4)[:n]
                byte = codes[rows, :, h].transpose(0, 1).reshape(2, -1, D // 2)[:, :n]
                val = torch.empty(2, n, D, dtype=torch.float64, device=q.device)
                val[..., 0::2], val[..., 1::2] = byte % 16, byte // 16
                val = val * sc.t()[0::2].unsqueeze(-1) + sc.t()[1::2].unsqueeze(-1)
                for i in range(S):
                    m = n - S + i + 1
                    if m > 0:
                        heads = slice(h * (H // KV), (h + 1) * (H // KV))
                        p = torch.softmax(q[b, i, heads] @ val[0, :m].t() / D ** 0.5, -1)
                        out[b, i, heads] = p @ val[1, :m]
        return out
    if c["kind"] == "w4":
        N, K, G = c["out"], c["inner"], c["group"]
        y = torch.zeros(c["rows"], N, dtype=torch.float64, device=DEV)
        for k in range(0, K, G):
            byte = s["codes"][:, k // 2: (min(K, k + G) + 1) // 2]
            w = torch.empty(N, 2 * byte.shape[1], dtype=torch.float64, device=DEV)
            w[:, 0::2], w[:, 1::2] = byte % 16, byte // 16
            n = min(K, k + G) - k
            y += s["x"][:, k: k + n].double() @ (w[:, :n] - 8).t() * s["scales"][:, k // G].double()
        return y
    x = s["logits"].double()
    f = s["scores"].double().unsqueeze(-1) + torch.log_softmax(x, -1)
    f[s["finished"]] = -INF
    f[..., EOS] = torch.where(s["finished"], s["scores"].double(), f[..., EOS])
    return torch.topk(f.flatten(1), c["beams"]).values, None, None, None, None, None, None
