"""Generation with the cache in 16 bits on the GPU, as the CPU's tests have it."""
import pytest
import torch

from atorch_b200 import _lib
from atorch_b200.models.generate import CachedSampler, Generator
from test_generate_16_cpu import check_against_lists, check_refusals, model, prompts

pytestmark = pytest.mark.gpu
SHAPE = dict(vocab_size=300, hidden_size=256, intermediate_size=384, num_attention_heads=4, num_key_value_heads=2)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_the_cache_alone(dtype, monkeypatch):
    assert check_against_lists(model("cuda", dtype, **SHAPE), (3, 37, 170), 20, monkeypatch, 0.03) == []
    assert check_against_lists(model("cuda", dtype, **SHAPE), (37, 37), 5, monkeypatch, 0.03) == []
    _lib.check_status(torch.device("cuda", 0))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_with_a_budget(dtype, monkeypatch):
    m = model("cuda", dtype, **{**SHAPE, "num_attention_heads": 2, "num_key_value_heads": 1}, initializer_range=0.08)
    assert check_against_lists(m, (3, 37, 170), 30, monkeypatch, 0.06, budget=40, recent=8, slack=6) == [1, 7, 13, 19, 25]
    assert check_against_lists(m, (20, 20), 30, monkeypatch, 0.06, budget=16, recent=16, slack=8) == [1, 9, 17, 25]
    _lib.check_status(torch.device("cuda", 0))


def test_sampling_filters():
    m = model("cuda", **SHAPE)
    ids = prompts(m, (6, 6, 6, 6))
    first = Generator(m).generate(ids, 8, temperature=1.5, top_k=1)
    for kw in (dict(top_p=1e-6), dict(top_k=7, top_p=0.0), dict(top_k=1, min_p=1.0)):       # of equal logits the lowest index
        for a, b in zip(first, Generator(m).generate(ids, 8, temperature=0.5, **kw)):
            assert torch.equal(a, b)
    torch.manual_seed(3)
    whole = Generator(m).generate(ids, 8, temperature=1.0)
    torch.manual_seed(3)
    for a, b in zip(whole, CachedSampler(m, 8, top_k=300, top_p=1.0)(None, torch.stack(ids))):
        assert torch.equal(a, b)
    some = CachedSampler(m, 60, top_p=0.9, cache_bits=16, budget=24, recent=4, slack=8)(None, torch.stack(ids))
    assert some.shape == (4, 66) and (some < 300).all()
    _lib.check_status(some.device)


def test_refusals():
    check_refusals(model("cuda", **SHAPE))
