"""Drawing tokens without a GPU: the plain implementation against the definition, token after token, and the refusals."""
import math

import pytest
import torch
from torch.autograd import forward_ad

from atorch_b200 import ops


def draw(x, wait, T, k, p, m):
    """Token and logarithm of its probability of one row, by the definition, in Python's numbers."""
    x = [-math.inf if v != v else v for v in x]
    top, m = max(x), 1.0 if m > 1 else m
    if top == -math.inf:
        return 0, -math.inf
    if not T > 0:
        return x.index(top), 0.0
    w = [1.0 if v == top else 0.0 if v == -math.inf or top == math.inf else math.exp((v - top) / T) for v in x]
    order = sorted(range(len(x)), key=lambda i: (-x[i], i))
    if k > 0:
        order = order[:k]
    total, before, left = math.fsum(w[i] for i in order), 0.0, []
    for n, i in enumerate(order):
        if n > 0 and p < 1 and before >= p * total:
            break
        before += w[i]
        if not w[i] < m:
            left.append(i)
    score = {i: math.inf if wait[i] == 0 else w[i] / wait[i] if wait[i] > 0 else 0.0 for i in left if w[i] > 0}
    token = min(score, key=lambda i: (-score[i], i))
    return token, math.log(w[token] / math.fsum(w[i] for i in left))


FILTERS = [dict(), dict(temperature=0.4), dict(temperature=3.0), dict(temperature=math.inf), dict(temperature=1e38), dict(temperature=1e38, top_k=9, top_p=0.8), dict(temperature=1e-30, top_p=0.5), dict(top_k=1), dict(top_k=7), dict(top_k=5000), dict(top_p=0.9), dict(top_p=1e-9),
           dict(top_p=0.0), dict(min_p=0.1), dict(min_p=1.0), dict(top_k=20, top_p=0.7, min_p=0.02, temperature=0.8), dict(temperature=0.0),
           dict(top_k=50, top_p=0.999, temperature=1.3)]


def check(logits, waiting, device="cpu", **kw):
    """:func:`ops.sample` against :func:`draw`. A logarithm is of a quotient of sums of fp32 or better: off by some 2^-23 of itself and 2^-20."""
    tokens, logprobs = ops.sample(logits.to(device), waiting.to(device), **{k: v.to(device) if isinstance(v, torch.Tensor) else v for k, v in kw.items()})
    assert tokens.dtype == torch.int64 and logprobs.dtype == torch.float32 and tokens.shape == logprobs.shape == (len(logits),)
    for b in range(len(logits)):
        row = [kw.get(n, d) for n, d in (("temperature", 1.0), ("top_k", 0), ("top_p", 1.0), ("min_p", 0.0))]
        row = [v[b].item() if isinstance(v, torch.Tensor) and v.dim() else v for v in row]
        token, logprob = draw(logits[b].double().tolist(), waiting[b].double().tolist(), *row)
        assert int(tokens[b]) == token, (b, int(tokens[b]), token)
        assert float(logprobs[b]) == logprob or abs(float(logprobs[b]) - logprob) <= 2 ** -20 + 2 ** -23 * abs(logprob), (b, float(logprobs[b]), logprob)
    return tokens, logprobs


def special_rows(V, dtype, g):
    """Rows at which a selection can go wrong."""
    x = torch.randn(12, V, generator=g) * 3
    x[1] = 0.0                                        # all equal
    x[2] = torch.randint(0, 3, (V,), generator=g).float()         # many equal
    x[3, torch.rand(V, generator=g) < 0.5] = -math.inf
    x[4] = -math.inf
    x[5, torch.rand(V, generator=g) < 0.3] = float("nan")
    x[6] = float("nan")
    x[7, :: 3] = math.inf
    x[8] = torch.finfo(dtype).min
    x[8, V // 2:] = 1.0
    x[9] = torch.finfo(dtype).min                     # masked by a finite number, all of it
    x[10] = -math.inf
    x[10, V - 1] = -5.0                               # one token
    x[11] = torch.where(torch.rand(V, generator=g) < 0.5, torch.tensor(0.0), torch.tensor(-0.0))
    return x.to(dtype)


@pytest.mark.parametrize("kw", FILTERS)
@pytest.mark.parametrize("V", [1, 2, 57, 1003])
def test_sample(V, kw):
    g = torch.Generator().manual_seed(V)
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        check(special_rows(V, dtype, g), torch.empty(12, V).exponential_(generator=g), **kw)


def test_waiting_times_of_zero_infinity_and_nan():
    x = torch.zeros(5, 4)
    inf, nan = math.inf, float("nan")
    wait = torch.tensor([[1, 0, 0, 2], [inf, inf, inf, inf], [nan, nan, 5, -1], [nan, nan, nan, nan], [inf, -2.0, 0.5, 0.25]])
    tokens, logprobs = check(x, wait)
    assert tokens.tolist() == [1, 0, 2, 0, 3] and torch.allclose(logprobs, torch.full((5,), -math.log(4)))


def unusual_waits(V, g):
    """Waiting times at which a draw can go wrong, a row of each kind."""
    wait = torch.empty(11, V).exponential_(generator=g)
    odd = torch.tensor([0.0, -0.0, math.inf, float("nan"), -1.0, -math.inf])
    for i in range(6):
        wait[i] = odd[i]
    wait[6] = torch.where(torch.rand(V, generator=g) < 0.5, odd[0], odd[1])
    wait[7] = odd[torch.randint(0, 6, (V,), generator=g)]
    wait[8] = odd[torch.randint(2, 6, (V,), generator=g)]
    wait[9, V // 3] = -0.0
    mixed = torch.rand(V, generator=g) < 0.5
    wait[10, mixed] = odd[torch.randint(1, 6, (int(mixed.sum()),), generator=g)]
    return wait


@pytest.mark.parametrize("kw", [dict(), dict(top_k=1), dict(top_k=5), dict(top_p=0.5), dict(top_p=0.0), dict(min_p=0.2), dict(temperature=0.0)])
@pytest.mark.parametrize("V", [1, 3, 200])
def test_unusual_waiting_times(V, kw):
    g = torch.Generator().manual_seed(V)
    check(torch.randn(11, V, generator=g) * 2, unusual_waits(V, g), **kw)


def test_a_waiting_time_of_minus_zero():
    tokens, logprobs = check(torch.tensor([[5.0, 1.0, 0.0]]), torch.tensor([[-0.0, 1.0, 1.0]]), top_k=1)
    assert tokens.tolist() == [0] and logprobs.tolist() == [0.0]


def test_parameters_of_rows():
    g = torch.Generator().manual_seed(3)
    x, wait = torch.randn(6, 300, generator=g) * 2, torch.empty(6, 300).exponential_(generator=g)
    T, k = torch.tensor([0.5, 0.0, -1.0, 2.0, 1.0, 1.0]), torch.tensor([3, 0, 5, -2, 400, 1 << 40])
    p, m = torch.tensor([0.5, 0.9, 1.0, 1.5, float("nan"), -0.5]), torch.tensor([0.0, 0.5, float("nan"), 0.01, 1.5, -0.5])
    whole = check(x, wait, temperature=T, top_k=k, top_p=p, min_p=m)
    for b in range(6):
        one = ops.sample(x[b: b + 1], wait[b: b + 1], T[b: b + 1], k[b: b + 1], p[b: b + 1], m[b: b + 1])
        assert torch.equal(one[0], whole[0][b: b + 1]) and torch.equal(one[1], whole[1][b: b + 1])
    assert torch.equal(ops.sample(x, wait, torch.tensor(0.5), torch.tensor(3))[0], ops.sample(x, wait, 0.5, 3)[0])


def test_tokens_follow_the_distribution():
    x = torch.tensor([2.0, 1.0, 0.5, -1.0, 0.0, 1.5]).expand(20000, 6)
    wait = torch.empty(20000, 6).exponential_(generator=torch.Generator().manual_seed(1))
    for kw, kept in ((dict(), [0, 1, 2, 3, 4, 5]), (dict(top_k=3), [0, 5, 1]), (dict(top_p=0.75), [0, 5, 1]), (dict(min_p=0.2), [0, 5, 1, 2])):
        want = torch.full((6,), -math.inf)
        want[kept] = x[0, kept] / 1.2
        want = torch.softmax(want, 0)
        tokens, logprobs = ops.sample(x, wait, 1.2, **kw)
        got = torch.bincount(tokens, minlength=6) / 20000
        assert ((got - want).abs() <= 5 * (want * (1 - want) / 20000).sqrt()).all()
        assert torch.allclose(logprobs, want.log()[tokens], atol=1e-6)


def check_refusals(dev):
    x, wait = torch.zeros(2, 5, device=dev), torch.ones(2, 5, device=dev)
    for bad in ((x.double(), wait), (x[0], wait[0]), (x[:, :0], wait[:, :0]), (x, wait.half()), (x, wait[:1]), (x, wait[:, :4]), (x.long(), wait)):
        with pytest.raises(ValueError):
            ops.sample(*bad)
    row, whole = torch.ones(2, device=dev), torch.ones(2, device=dev, dtype=torch.int32)
    for kw in (dict(temperature=-0.1), dict(temperature=math.nan), dict(top_k=-1), dict(top_k=1.5), dict(top_p=-0.1), dict(top_p=1.1),
               dict(top_p=math.nan), dict(min_p=-0.1), dict(min_p=1.1), dict(temperature=row[:1]), dict(temperature=whole), dict(top_k=row), dict(top_k=whole[:1]),
               dict(top_p=row.half()), dict(min_p=row[:, None])):
        with pytest.raises(ValueError):
            ops.sample(x, wait, **kw)
    if dev != "cpu":
        for call in (lambda: ops.sample(x, wait.cpu()), lambda: ops.sample(x.cpu(), wait), lambda: ops.sample(x, wait, row.cpu()), lambda: ops.sample(x, wait, 1.0, whole.cpu())):
            with pytest.raises(ValueError):
                call()
    for i in range(2):
        ts = [t.clone().requires_grad_() if j == i else t for j, t in enumerate((x, wait))]
        with pytest.raises(RuntimeError, match="gradient"):
            ops.sample(*ts)
        with torch.no_grad():
            ops.sample(*ts)
        with forward_ad.dual_level():
            dual = [forward_ad.make_dual(t, torch.ones_like(t)) if j == i else t for j, t in enumerate((x, wait))]
            with torch.no_grad(), pytest.raises(RuntimeError, match="gradient"):
                ops.sample(*dual)
    tokens, logprobs = ops.sample(x[:0], wait[:0])
    assert tokens.shape == logprobs.shape == (0,) and tokens.dtype == torch.int64 and logprobs.dtype == torch.float32


def test_refusals():
    check_refusals("cpu")


def test_vocabularies_that_the_filters_do_not_take():
    V, g = (1 << 19) + 5, torch.Generator().manual_seed(1)
    x, wait = torch.randn(2, V, generator=g), torch.empty(2, V).exponential_(generator=g)
    for kw in (dict(), dict(temperature=torch.tensor([0.5, 0.0])), dict(min_p=0.3)):
        check(x, wait, **kw)
    whole, row = torch.zeros(2, dtype=torch.int32), torch.ones(2)
    for kw in (dict(top_k=3), dict(top_p=0.5), dict(top_k=whole), dict(top_p=row)):
        with pytest.raises(ValueError, match="vocabulary"):
            ops.sample(x, wait, **kw)


def test_drawing_without_an_order_sorts_nothing(monkeypatch):
    monkeypatch.setattr(torch.Tensor, "sort", None)
    x, wait = torch.randn(3, 50), torch.empty(3, 50).exponential_()
    for kw in (dict(), dict(temperature=0.3), dict(min_p=0.1), dict(top_p=torch.ones(3), top_k=torch.zeros(3, dtype=torch.int32))):
        tokens, _ = ops.sample(x, wait, **kw)
        want = [draw(a, b, kw.get("temperature", 1.0), 0, 1.0, kw.get("min_p", 0.0))[0] for a, b in zip(x.double().tolist(), wait.double().tolist())]
        assert tokens.tolist() == want
