"""Generation with the 4-bit cache on the CPU: greedy, beams, sampling, 4-bit weights."""
import copy

import pytest
import torch

from atorch_b200 import ops
from atorch_b200.models.generate import CachedSampler, Generator, generate
from atorch_b200.models.llama import LlamaConfig, LlamaModel
from atorch_b200.modules.w4_linear import W4Linear, quantize_linears


def _model(seed=0, **kw):
    torch.manual_seed(seed)
    cfg = LlamaConfig(**{**dict(vocab_size=40, hidden_size=64, intermediate_size=96, num_hidden_layers=2, num_attention_heads=4,
                                num_key_value_heads=2, max_position_embeddings=128, initializer_range=0.1), **kw})
    return LlamaModel(cfg).bfloat16().eval()


def _alone(model, ids, rows=1, steps=0, seed=0):
    """A cache of its own for ``rows`` copies of a sequence, its pages in no order, after the pass over the prompt in row 0: generator,
    cache, table, angles, logits of all tokens."""
    g = Generator(model)
    S, n, dev = g.page_size, len(ids), ids.device
    width = -(-(n + steps) // S)
    table = torch.randperm(rows * width, generator=torch.Generator().manual_seed(seed)).to(torch.int32).view(rows, width).to(dev)
    cache = ops.KV4Cache(model.config.num_hidden_layers, rows * width, S, model.layers[0].n_kv, model.config.head_dim, dev)
    cos, sin = model.rope(n + steps, dev)
    seq, pos = torch.zeros(n, dtype=torch.int32, device=dev), torch.arange(n, dtype=torch.int32, device=dev)

    def attend(q, layer):
        k, v = ops.kv4_read(layer, table, seq, pos, q.dtype)
        return ops.attention(q[None], k[None], v[None], causal=True, cu_seqlens=torch.tensor([0, n], dtype=torch.int32, device=dev))

    with torch.no_grad():
        logits = g._run(ids, cache, table, seq, pos, cos, sin, attend)
    return g, cache, table, cos, sin, logits


def _step_is_the_prompt(model, ids, places):
    """A step over what the prompt left in the cache gives the prompt's logits. Only the step's own token is computed anew: some ten
    roundings of 2^-9 a layer, in another order, and its own codes."""
    g, cache, table, cos, sin, logits = _alone(model, ids)
    kept = cache.codes.clone(), cache.scales.clone()
    for t in places:
        cache.codes.copy_(kept[0]), cache.scales.copy_(kept[1])
        with torch.no_grad():
            got = g._step(ids[t: t + 1], cache, table, torch.tensor([t], dtype=torch.int32, device=ids.device), cos, sin)[0]
        off = (got.float() - logits[t].float()).norm() / logits[t].float().norm()
        assert off < 0.05, (t, off)


def _beams_with_pages_of_their_own(model, ids, beams, steps, eos=None):
    """The same search with a whole copy of the cache for every beam, moved by indexing."""
    g, cache, table, cos, sin, logits = _alone(model, ids, beams, steps, seed=1)
    n, pages = len(ids), table.long()
    cache.codes[:, pages[1:].flatten()] = cache.codes[:, pages[:1].expand(beams - 1, -1).flatten()]
    cache.scales[:, pages[1:].flatten()] = cache.scales[:, pages[:1].expand(beams - 1, -1).flatten()]
    with torch.no_grad():
        logits = g._prompts([ids], cache, table, [0], cos, sin)       # (the logits that a search begins with, in their shape)
        scores, tokens, parents, done = ops.beam_select_reference(logits.view(1, 1, -1), torch.zeros(1, 1, device=ids.device), None,
                                                                  -1 if eos is None else eos, beams)
        sequences = tokens.view(beams, 1)
        for i in range(1, steps):
            if eos is not None and bool(done.all()):
                break
            logits = g._step(tokens.view(-1), cache, table, torch.full((beams,), n + i - 1, dtype=torch.int32, device=ids.device), cos, sin)
            scores, tokens, parents, done = ops.beam_select_reference(logits.view(1, beams, -1), scores, None if eos is None else done,
                                                                      -1 if eos is None else eos)
            parent = parents[0].long()
            sequences = torch.cat([sequences[parent], tokens.view(beams, 1)], 1)
            cache.codes[:, pages.flatten()] = cache.codes[:, pages[parent].flatten()]
            cache.scales[:, pages.flatten()] = cache.scales[:, pages[parent].flatten()]
    return torch.cat([ids, sequences[0]])


def test_a_step_continues_the_prompt():
    _step_is_the_prompt(_model(), torch.randint(0, 40, (70,), generator=torch.Generator().manual_seed(1)), (1, 15, 16, 40, 69))


def test_greedy_is_one_step_after_another():
    m = _model()
    ids = torch.randint(0, 40, (21,), generator=torch.Generator().manual_seed(2))
    g, cache, table, cos, sin, logits = _alone(m, ids, 1, 15)
    with torch.no_grad():
        token, want = g._prompts([ids], cache, table, [0], cos, sin).argmax(-1), []
        for i in range(15):
            want.append(token)
            token = g._step(token, cache, table, torch.tensor([21 + i], dtype=torch.int32), cos, sin).argmax(-1) if i < 14 else token
    assert torch.equal(generate(m, [ids], 15)[0], torch.cat([ids, *want]))


@pytest.mark.parametrize("beams,n,eos", [(2, 5, None), (4, 16, None), (5, 39, 3), (3, 15, 0)])
def test_beams_share_pages_and_nothing_else(beams, n, eos):
    m = _model(vocab_size=12)
    ids = torch.randint(0, 12, (n,), generator=torch.Generator().manual_seed(n))
    want = _beams_with_pages_of_their_own(m, ids, beams, 25, eos)
    if eos is not None and (want[n:] == eos).any():
        want = want[: n + int((want[n:] == eos).nonzero()[0]) + 1]
    assert torch.equal(generate(m, [ids], 25, beams=beams, eos=eos)[0], want)


def test_end_token_and_shapes():
    m = _model(vocab_size=6)
    prompts = torch.randint(0, 6, (3, 7), generator=torch.Generator().manual_seed(3))
    for kw in (dict(), dict(beams=3), dict(temperature=1.0), dict(beams=2, length_penalty=1.0)):
        torch.manual_seed(0)
        for p, o in zip(prompts, generate(m, prompts, 12, eos=4, **kw)):
            new = o[7:]
            assert torch.equal(o[:7], p) and 1 <= len(new) <= 12
            assert (new[:-1] != 4).all() and (len(new) == 12 or new[-1] == 4)
    assert torch.equal(generate(m, prompts, 0)[1], prompts[1])
    with pytest.raises(ValueError):
        generate(m, prompts, 4, beams=2, temperature=1.0)
    with pytest.raises(ValueError):
        generate(m, [torch.tensor([], dtype=torch.long)], 4)
    with pytest.raises(ValueError):
        Generator(m.float())
    with pytest.raises(ValueError):
        CachedSampler(_model(), temperature=0.0)


def test_sampler_follows_the_distribution():
    m = _model(vocab_size=4)
    ids = torch.randint(0, 4, (5,), generator=torch.Generator().manual_seed(4))
    want = torch.softmax(_alone(m, ids)[-1][-1].float() / 0.7, -1)
    torch.manual_seed(5)
    out = CachedSampler(m, max_new_tokens=1, temperature=0.7)(None, ids.expand(4000, 5))
    assert out.shape == (4000, 6)
    got = torch.bincount(out[:, -1], minlength=4) / 4000
    # five standard deviations, and what the sums of a batch in bf16 are rounded by
    assert ((got - want).abs() < 5 * (want * (1 - want) / 4000).sqrt() + 0.01).all()


def test_quantised_linears():
    m = _model()
    before = m.layers[0].qkv_proj.weight.detach().clone()
    quantize_linears(m, 32, lambda name, lin: "lm_head" not in name)
    assert type(m.lm_head) is torch.nn.Linear
    lin = m.layers[0].qkv_proj
    assert type(lin) is W4Linear and lin.in_features == 64 and lin.out_features == before.shape[0]
    w = ops.w4_dequantize(lin.codes, lin.scales, 64, 32)
    assert (w - before.float()).abs().max() <= float(lin.scales.max()) * 0.55
    x = torch.randn(3, 64).bfloat16()
    assert torch.allclose(lin(x).float(), x.float() @ w.t(), atol=2e-2, rtol=1e-2)
    out = generate(m, [torch.tensor([1, 2, 3])], 6)[0]
    assert len(out) == 9
    tied = _model(tie_word_embeddings=True)
    quantize_linears(tied)
    assert type(tied.lm_head) is torch.nn.Linear and type(tied.layers[1].o_proj) is W4Linear


def test_sampling_is_that_of_multinomial_and_outlives_nan(monkeypatch):
    """The same tokens for a seed; logits that hold NaN (weights that have diverged) give a token of the vocabulary."""
    m = _model(vocab_size=30)
    ids = torch.randint(0, 30, (6, 5), generator=torch.Generator().manual_seed(6))
    logits = torch.randn(6, 30, generator=torch.Generator().manual_seed(7)).bfloat16()
    monkeypatch.setattr(Generator, "_run", lambda self, *a: logits)
    torch.manual_seed(8)
    want = torch.stack([torch.multinomial(torch.softmax(logits.float() / 0.8, -1), 1).squeeze(1) for _ in range(3)], 1)
    torch.manual_seed(8)
    assert torch.equal(torch.stack(generate(m, ids, 3, temperature=0.8))[:, 5:], want)
    logits[2] = float("nan")
    logits[3, 4:9] = float("nan")
    logits[4] = -float("inf")
    out = torch.stack(generate(m, ids, 3, temperature=0.8))[:, 5:]
    assert (out >= 0).all() and (out < 30).all()


def _dequantised(model):
    """The same model with the weights that the codes stand for in its ``nn.Linear`` modules."""
    for m in list(model.modules()):
        for child, lin in list(m.named_children()):
            if type(lin) is W4Linear:
                plain = torch.nn.Linear(lin.in_features, lin.out_features, bias=lin.bias is not None)
                plain.weight.data = ops.w4_dequantize(lin.codes, lin.scales, lin.in_features, lin.group_size)
                if lin.bias is not None:
                    plain.bias.data = lin.bias.float()
                setattr(m, child, plain)
    return model.float()


@pytest.mark.parametrize("tied", [False, True])
def test_a_quantised_model_runs_its_own_forward(tied):
    """As a reference or reward model does: head and all, against the weights that the codes stand for."""
    m = quantize_linears(_model(tie_word_embeddings=tied), 32)
    assert type(m.lm_head) is (torch.nn.Linear if tied else W4Linear)
    ids = torch.randint(0, 40, (3, 17), generator=torch.Generator().manual_seed(9))
    with torch.no_grad():
        loss, logits = m(ids, labels=ids)
        want_loss, want = _dequantised(copy.deepcopy(m))(ids, labels=ids)
    # some twenty roundings to bf16 in series, each of 2^-9
    assert (logits.float() - want).norm() < 20 * 2 ** -9 * want.norm() and abs(float(loss) - float(want_loss)) < 0.05 * float(want_loss)


def test_a_quantised_mixture_of_experts_runs_its_own_forward():
    from atorch_b200.models.mixtral import MixtralConfig, MixtralModel
    from atorch_b200.modules.moe.gating import TopkGate

    torch.manual_seed(3)
    m = MixtralModel(MixtralConfig.tiny_moe()).bfloat16().eval()
    quantize_linears(m, 32, lambda name, lin: "router" not in name)
    assert type(m.lm_head) is W4Linear and type(m.layers[1].qkv_proj) is W4Linear
    ids = torch.randint(0, 256, (2, 12), generator=torch.Generator().manual_seed(9))
    with torch.no_grad():
        _, logits = m(ids)
        _, want = _dequantised(copy.deepcopy(m)).bfloat16()(ids)
    assert (logits.float() - want.float()).norm() < 0.1 * want.float().norm()
    gate = quantize_linears(TopkGate(64, 4).bfloat16(), 32)
    with torch.no_grad():
        assert torch.isfinite(gate(torch.randn(10, 64).bfloat16())[0])


def test_models_that_the_generator_does_not_know_are_refused():
    from atorch_b200.models.mixtral import MixtralConfig, MixtralModel

    m = _model()
    wrapped = torch.nn.Module()
    wrapped.module = m
    other = _model()
    other.layers[1] = MixtralModel(MixtralConfig.tiny_moe()).bfloat16().layers[0]
    for bad in (MixtralModel(MixtralConfig.tiny_moe()).bfloat16(), wrapped, other):
        with pytest.raises(TypeError):
            Generator(bad)
        with pytest.raises(TypeError):
            CachedSampler(bad)


def test_layers_in_a_wrapper_that_hands_on_their_attributes():
    from atorch_b200.modules.distributed_modules.activation_checkpointing import TPCheckpointWrapper

    m, ids = _model(), torch.randint(0, 40, (2, 9), generator=torch.Generator().manual_seed(4))
    want = generate(m, ids, 5)
    m.layers[1] = TPCheckpointWrapper(m.layers[1])
    assert all(torch.equal(a, b) for a, b in zip(generate(m, ids, 5), want))


def test_scales_keep_their_type():
    """A model that is cast keeps its scales in bf16, as its codes were taken for; the bias goes with the model."""
    lin = torch.nn.Linear(64, 24)
    w4 = W4Linear.from_linear(lin.bfloat16(), 32)
    codes, scales, state = w4.codes.clone(), w4.scales.clone(), w4.state_dict().keys()
    model = torch.nn.Sequential(torch.nn.LayerNorm(64), w4)
    for cast in (lambda m: m.half(), lambda m: m.float(), lambda m: m.to(torch.float16), lambda m: m.double().bfloat16()):
        model = cast(model)
        assert w4.scales.dtype is torch.bfloat16 and torch.equal(w4.scales, scales) and torch.equal(w4.codes, codes)
        assert w4.bias.dtype is model[0].weight.dtype and w4.state_dict().keys() == state
        if w4.bias.dtype is not torch.float32:
            with torch.no_grad():
                assert w4(torch.randn(3, 64).to(w4.bias.dtype)).dtype is w4.bias.dtype
    assert copy.deepcopy(w4).to("meta").scales.is_meta
