"""Drawing tokens on the GPU against the definition, token after token."""
import math

import pytest
import torch

from atorch_b200 import _lib, ops
from test_sample_cpu import FILTERS, check, check_refusals, draw, special_rows, unusual_waits

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("kw", FILTERS)
@pytest.mark.parametrize("V", [1, 2, 57, 1003, 4096, 9001])
def test_sample(V, kw):
    g = torch.Generator().manual_seed(V)
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        check(special_rows(V, dtype, g), torch.empty(12, V).exponential_(generator=g), DEV, **kw)
    _lib.check_status(torch.device("cuda", 0))


@pytest.mark.parametrize("kw", [dict(), dict(top_k=50, top_p=0.95, temperature=0.7), dict(top_p=0.9), dict(top_p=0.9999, temperature=2.0), dict(top_k=20000),
                                dict(min_p=0.01), dict(top_k=1000, top_p=0.5, min_p=0.001)])
@pytest.mark.parametrize("B,V,dtype", [(1, 32000, torch.bfloat16), (3, 100003, torch.float32), (2, 131072, torch.float16), (200, 3001, torch.bfloat16),
                                       (1, 400001, torch.float32)])
def test_sizes(B, V, dtype, kw):
    g = torch.Generator().manual_seed(B + V)
    x = torch.randn(B, V, generator=g) * 2.5
    x[0, torch.randint(0, V, (5,), generator=g)] = 12.0
    wait = torch.empty(B, V).exponential_(generator=g)
    if B > 8:                       # the oracle takes its time: rows of another batch's kind, against the plain implementation in 64 bits
        x = x.to(dtype).to(DEV)
        got, want = ops.sample(x, wait.to(DEV), **kw), ops.sample_reference(x, wait.to(DEV), **kw)
        assert torch.equal(got[0], want[0]) and torch.allclose(got[1], want[1], rtol=2 ** -23, atol=2 ** -20)
    else:
        check(x.to(dtype), wait, DEV, **kw)


def test_a_border_among_many_like_values():
    """The prefix ends in the middle of thousands of equal logits: the lowest indices are left."""
    V = 20000
    x = torch.zeros(2, V)
    x[:, 777] = 3.0
    x[1, 10000:] = -4.0
    for kw in (dict(top_k=7001), dict(top_p=0.31), dict(top_k=9000, top_p=0.5)):
        order = [777] + [i for i in range(V) if i != 777]
        for b in range(2):
            # the last token that is left arrives long before the others, but for the one behind it
            n = kw.get("top_k", V)
            if "top_p" in kw:
                w = [math.exp(3.0)] + [1.0 if b == 0 or i < 10000 else math.exp(-4.0) for i in order[1:n]]
                w = [v / math.exp(3.0) for v in w]
                total, before, n = math.fsum(w), 0.0, 0
                for v in w:
                    if n and before >= kw["top_p"] * total:
                        break
                    before += v
                    n += 1
            wait = torch.ones(1, V)
            wait[0, order[n - 1]], wait[0, order[n]] = 1e-6, 1e-9
            tokens, _ = check(x[b: b + 1], wait, DEV, **kw)
            assert int(tokens[0]) == order[n - 1]


def test_tokens_that_arrive_together():
    """Arrivals closer than fp32 tells apart: 64 bits decide, then the index."""
    V = 5000
    g = torch.Generator().manual_seed(1)
    x = (torch.randn(4, V, generator=g)).float()
    w = torch.exp(x.double() - x.double().amax(-1, keepdim=True))
    wait = w.float()                                   # all scores are 1 but for the rounding of the waiting time
    check(x, wait, DEV)
    check(x, wait, DEV, top_p=0.8)
    check(torch.zeros(3, V), torch.ones(3, V), DEV)


def test_strides_offsets_and_rows_of_parameters():
    g = torch.Generator().manual_seed(5)
    x, wait = torch.randn(6, 3007, generator=g) * 2, torch.empty(6, 3007).exponential_(generator=g)
    kw = dict(temperature=torch.tensor([0.5, 0.0, -1.0, 2.0, 1.0, 1.0]), top_k=torch.tensor([3, 0, 5, -2, 400, 1 << 40]),
              top_p=torch.tensor([0.5, 0.9, 1.0, 1.5, float("nan"), -0.5]), min_p=torch.tensor([0.0, 0.5, float("nan"), 0.01, 1.5, -0.5]))
    for dtype in (torch.float32, torch.bfloat16):
        want = check(x.to(dtype), wait, DEV, **kw)
        kd = {k: v.to(DEV) for k, v in kw.items()}
        wide = torch.full((6, 3, 3019), 50.0, dtype=dtype, device=DEV)
        wide[:, 1, 5: 3012] = x.to(dtype).to(DEV)
        waits = torch.full((6, 3010), 1e-9, device=DEV)
        waits[:, 3:] = wait.to(DEV)
        for logits, w in ((wide[:, 1, 5: 3012], waits[:, 3:]), (x.to(dtype).to(DEV).t().contiguous().t(), wait.to(DEV).t().contiguous().t())):
            tokens, logprobs = ops.sample(logits, w, **kd)
            assert torch.equal(tokens, want[0]) and torch.equal(logprobs, want[1])
        assert torch.equal(ops.sample(x.to(dtype).to(DEV)[:1].expand(4, -1), wait.to(DEV)[:4])[0].cpu(),
                           torch.tensor([draw(x.to(dtype)[0].double().tolist(), w.double().tolist(), 1.0, 0, 1.0, 0.0)[0] for w in wait[:4]]))


def test_captured_and_on_two_streams():
    V, g = 32000, torch.Generator(device=DEV).manual_seed(1)
    x, wait = torch.randn(8, V, generator=g, device=DEV) * 2, torch.empty(2, 8, V, device=DEV)
    streams, graphs, outs = [torch.cuda.Stream() for _ in range(2)], [], []
    kws = (dict(top_k=40, top_p=0.9), dict(top_p=0.95))
    for i in range(2):
        ops.sample(x, wait[i].exponential_(generator=g), **kws[i])
    torch.cuda.synchronize()
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(ops.sample(x, wait[i], **kws[i]))
        graphs.append(graph)
    for _ in range(3):
        x.normal_(generator=g).mul_(3)
        wait.exponential_(generator=g)
        torch.cuda.synchronize()
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for i in range(2):
            want = ops.sample(x, wait[i], **kws[i])
            assert torch.equal(outs[i][0], want[0]) and torch.equal(outs[i][1], want[1])
            plain = ops.sample_reference(x, wait[i], **kws[i])
            assert torch.equal(want[0], plain[0]) and torch.allclose(want[1], plain[1], rtol=2 ** -23, atol=2 ** -20)


def test_behind_a_failed_kernel():
    x, wait = torch.randn(3, 40, device=DEV), torch.ones(3, 40, device=DEV)
    dev = x.device
    _lib.status_word(dev).fill_(1)
    for kw in (dict(), dict(top_k=3)):
        tokens, logprobs = ops.sample(x, wait, **kw)
        assert (tokens == 0).all() and (logprobs == -math.inf).all()
    with pytest.raises(_lib.KernelError):
        _lib.check_status(dev)
    _lib.check_status(dev)


def test_refusals():
    check_refusals(DEV)


@pytest.mark.parametrize("top_k", [9000, 20000, 30000])
@pytest.mark.parametrize("B,V", [(1, 32000), (1, 131072), (64, 32000), (64, 131072), (192, 32000)])
def test_prefixes_longer_than_the_lists(B, V, top_k):
    """Every block of a row has to take the same way through the whole shares, however far behind the others it is."""
    g = torch.Generator(device=DEV).manual_seed(V + top_k)
    x = torch.randn(B, V, generator=g, device=DEV)
    x[::2] *= 1e-3                                     # nearly flat
    x[::3] = 0.0
    for kw in (dict(top_k=top_k), dict(top_k=top_k, top_p=0.7)):
        for dtype in (torch.float32, torch.bfloat16):
            logits = x.to(dtype)
            first = None
            for repeat in range(12):
                wait = torch.empty(B, V, device=DEV).exponential_(generator=g)
                got = ops.sample(logits, wait, **kw)
                if repeat < 2:
                    want = ops.sample_reference(logits, wait, **kw)
                    assert torch.equal(got[0], want[0]) and torch.allclose(got[1], want[1], rtol=2 ** -23, atol=2 ** -20)
                else:
                    first = first or (wait, got)
                    again = ops.sample(logits, first[0], **kw)
                    assert torch.equal(again[0], first[1][0]) and torch.equal(again[1], first[1][1])
    _lib.check_status(x.device)


@pytest.mark.parametrize("kw", [dict(), dict(top_k=1), dict(top_k=5), dict(top_p=0.5), dict(top_p=0.0), dict(top_p=0.95), dict(top_k=3000), dict(top_k=5000, top_p=0.9),
                                dict(min_p=0.01), dict(temperature=0.0)])
@pytest.mark.parametrize("V", [1, 3, 200, 9001])
def test_unusual_waiting_times(V, kw):
    """Prefixes put in order, listed, and drawn from without filters."""
    g = torch.Generator().manual_seed(V)
    for dtype in (torch.float32, torch.bfloat16):
        check((torch.randn(11, V, generator=g) * 2).to(dtype), unusual_waits(V, g), DEV, **kw)
        if V == 9001:
            check((torch.randn(11, V, generator=g) * 0.01).to(dtype), unusual_waits(V, g), DEV, **kw)
    _lib.check_status(torch.device("cuda", 0))


def test_unusual_waiting_times_behind_a_prefix_too_long_to_list():
    V, g = 40000, torch.Generator().manual_seed(1)
    for b in range(11):
        check(torch.randn(1, V, generator=g) * 0.01, unusual_waits(V, g)[b: b + 1], DEV, top_k=39000)
    _lib.check_status(torch.device("cuda", 0))


@pytest.mark.parametrize("top_p", [0.3, 0.9, 0.95])
@pytest.mark.parametrize("B,V,spread,dtype", [(192, 32000, 2.5, torch.float32), (192, 32000, 2.5, torch.bfloat16), (512, 12001, 2.5, torch.float32),
                                              (40, 131072, 2.5, torch.float32), (150, 32000, 0.7, torch.float32)])
def test_the_end_of_a_nucleus(B, V, spread, dtype, top_p):
    """Thousands of unlike weights (with little spread too many to list): the end of the prefix is that of sums in 64 bits. A token next
    to it weighs 1e-5 of what is left, ten times what a logarithm may be off by; in every other batch the last token that is left arrives
    first, but for the one behind it."""
    g = torch.Generator(device=DEV).manual_seed(V)
    for batch in range(10):
        x = torch.randn(B, V, generator=g, device=DEV) * spread
        x += (9.0 if spread > 1 else 0.0) * (torch.rand(B, V, generator=g, device=DEV) < 8 / V)
        x = x.to(dtype)
        wait = torch.empty(B, V, device=DEV).exponential_(generator=g)
        if batch % 2:
            w, order = torch.softmax(x.double(), -1).sort(dim=-1, descending=True, stable=True)
            last = ((w.cumsum(-1) - w) < top_p).sum(-1, keepdim=True) - 1
            wait.scatter_(1, order.gather(1, last), 1e-12)
            wait.scatter_(1, order.gather(1, last + 1), 1e-18)
        got, want = ops.sample(x, wait, top_p=top_p), ops.sample_reference(x, wait, top_p=top_p)
        other = int((got[0] != want[0]).sum())
        far = int(((got[1] - want[1]).abs() > 2 ** -20 + 2 ** -23 * want[1].abs()).sum())
        assert other == 0 and far == 0, (batch, other, far)


@pytest.mark.parametrize("B,V,dtype", [(2, (1 << 19) + 5, torch.float32), (1, 5000011, torch.bfloat16), (40, 700001, torch.float16)])
def test_vocabularies_that_the_filters_do_not_take(B, V, dtype):
    g = torch.Generator(device=DEV).manual_seed(V)
    x, wait = (torch.randn(B, V, generator=g, device=DEV) * 2).to(dtype), torch.empty(B, V, device=DEV).exponential_(generator=g)
    for kw in (dict(), dict(temperature=0.0), dict(min_p=0.05), dict(temperature=torch.full((B,), 0.7, device=DEV))):
        got, want = ops.sample(x, wait, **kw), ops.sample_reference(x, wait, **kw)
        assert torch.equal(got[0], want[0]) and torch.allclose(got[1], want[1], rtol=2 ** -23, atol=2 ** -20)
    with pytest.raises(ValueError, match="vocabulary"):
        ops.sample(x, wait, top_p=0.5)
    _lib.check_status(x.device)
