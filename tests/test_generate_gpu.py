"""Generation on the GPU: the operators together, against one another's plain implementations and layouts."""
import pytest
import torch

from atorch_b200 import _lib, ops
from atorch_b200.models.generate import CachedSampler, Generator
from atorch_b200.models.llama import LlamaConfig, LlamaModel
from atorch_b200.modules.w4_linear import W4Linear, quantize_linears

pytestmark = pytest.mark.gpu


def _model(seed=0, **kw):
    torch.manual_seed(seed)
    cfg = LlamaConfig(**{**dict(vocab_size=1000, hidden_size=512, intermediate_size=768, num_hidden_layers=3, num_attention_heads=4,
                                num_key_value_heads=2, max_position_embeddings=512, initializer_range=0.04), **kw})
    return LlamaModel(cfg).bfloat16().cuda().eval()


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


@pytest.mark.parametrize("kw,weights", [(dict(), None), (dict(num_attention_heads=8, num_key_value_heads=8), None), (dict(), 128),
                                        (dict(num_attention_heads=8, num_key_value_heads=4), 64)])
def test_a_step_continues_the_prompt(kw, weights):
    m = _model(**kw)
    if weights:
        quantize_linears(m, weights)
    launches = _lib.launch_count
    _step_is_the_prompt(m, torch.randint(0, 1000, (300,), generator=torch.Generator().manual_seed(1)).cuda(), (1, 16, 100, 255, 299))
    assert _lib.launch_count > launches + 5 * 3 * 2


def test_prompts_of_several_lengths():
    """Every sequence begins with its prompt, and goes on with the token that its prompt alone gives, or one as likely."""
    m = _model()
    g = torch.Generator().manual_seed(2)
    prompts = [torch.randint(0, 1000, (n,), generator=g).cuda() for n in (1, 16, 45, 130)]
    for p, o in zip(prompts, Generator(m).generate(prompts, 24)):
        assert torch.equal(o[: len(p)], p) and len(o) == len(p) + 24
        logits = _alone(m, p)[-1][-1].float()
        assert logits[o[len(p)]] >= logits.max() - 0.05 * logits.norm()


@pytest.mark.parametrize("beams,n,eos", [(2, 5, None), (4, 16, None), (7, 40, 3), (16, 31, None)])
def test_beams_share_pages_and_nothing_else(beams, n, eos):
    m = _model(vocab_size=64)
    ids = torch.randint(0, 64, (n,), generator=torch.Generator().manual_seed(n)).cuda()
    want = _beams_with_pages_of_their_own(m, ids, beams, 40, eos)
    if eos is not None and (want[n:] == eos).any():
        want = want[: n + int((want[n:] == eos).nonzero()[0]) + 1]
    assert torch.equal(Generator(m).generate([ids], 40, beams=beams, eos=eos)[0], want)


def test_sampler_and_end_token():
    m = _model(vocab_size=50)
    prompt = torch.randint(0, 50, (8, 9), generator=torch.Generator().manual_seed(3)).cuda()
    torch.manual_seed(0)
    out = CachedSampler(m, max_new_tokens=12)(None, prompt)
    assert out.shape == (8, 21) and torch.equal(out[:, :9], prompt) and (out < 50).all()
    for o in Generator(m).generate(prompt, 30, eos=7, temperature=1.5):
        assert (o[9:-1] != 7).all() and (o[-1] == 7 or len(o) == 39)


@pytest.mark.parametrize("kw", [dict(), dict(beams=3), dict(temperature=1.0)])
def test_a_failed_kernel_is_reported_before_the_first_token(kw, monkeypatch):
    m = _model(vocab_size=50)
    prompt = torch.randint(0, 50, (2, 9), generator=torch.Generator().manual_seed(4)).cuda()
    run, calls = Generator._run, []
    monkeypatch.setattr(Generator, "_run", lambda self, *a: calls.append(1))
    _lib.status_word(prompt.device).fill_(1)
    with pytest.raises(_lib.KernelError):
        Generator(m).generate(prompt, 4, **kw)
    assert not calls
    monkeypatch.setattr(Generator, "_run", run)
    assert len(Generator(m).generate(prompt, 4, **kw)[1]) == 13


def test_sampling_is_that_of_multinomial_and_outlives_nan(monkeypatch):
    """The same tokens for a seed; logits that hold NaN give a token of the vocabulary, and no assertion on the device."""
    m = _model(vocab_size=300)
    ids = torch.randint(0, 300, (40, 5), generator=torch.Generator().manual_seed(6)).cuda()
    logits = torch.randn(40, 300, generator=torch.Generator().manual_seed(7)).bfloat16().cuda()
    monkeypatch.setattr(Generator, "_run", lambda self, *a: logits)
    torch.manual_seed(8)
    want = torch.stack([torch.multinomial(torch.softmax(logits.float() / 0.8, -1), 1).squeeze(1) for _ in range(4)], 1)
    torch.manual_seed(8)
    assert torch.equal(torch.stack(Generator(m).generate(ids, 4, temperature=0.8))[:, 5:], want)
    logits[2] = float("nan")
    logits[3, 4:9] = float("nan")
    logits[4] = -float("inf")
    out = torch.stack(Generator(m).generate(ids, 4, temperature=0.8))[:, 5:]
    assert (out >= 0).all() and (out < 300).all()


@pytest.mark.parametrize("shape", [(1, 5), (2, 60), (3, 100)])
def test_a_quantised_model_runs_its_own_forward(shape):
    """As a reference or reward model does, against the weights that the codes stand for, in 32 bits on the CPU."""
    m = quantize_linears(_model(), 64)
    ids = torch.randint(0, 1000, shape, generator=torch.Generator().manual_seed(9))
    plain = LlamaModel(m.config)
    plain.load_state_dict({n: t.float().cpu() for n, t in m.state_dict().items() if not n.endswith(("codes", "scales"))}, strict=False)
    for name, lin in m.named_modules():
        if type(lin) is W4Linear:
            w = ops.w4_dequantize(lin.codes, lin.scales, lin.in_features, lin.group_size).cpu()
            plain.get_submodule(name).weight.data = w
    with torch.no_grad():
        loss, logits = m(ids.cuda(), labels=ids.cuda())
        want_loss, want = plain(ids, labels=ids)
    # some thirty roundings to bf16 in series, each of 2^-9
    assert (logits.float().cpu() - want).norm() < 30 * 2 ** -9 * want.norm()
    assert abs(float(loss) - float(want_loss)) < 0.05 * float(want_loss)


@pytest.mark.parametrize("kw", [dict(), dict(num_attention_heads=8, num_key_value_heads=2)])
def test_fp16_prompts_take_no_dense_scores(kw):
    """The flash kernels take bf16 only; a prompt in fp16 attends over the cache instead of holding scores of all tokens by all tokens."""
    m = _model(max_position_embeddings=2048, **kw).half()
    g = torch.Generator().manual_seed(5)
    prompts = [torch.randint(0, 1000, (n,), generator=g).cuda() for n in (1900, 1, 700, 17, 1900)]
    Generator(m).generate(prompts[:2], 2)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    out = Generator(m).generate(prompts, 3)
    peak = torch.cuda.max_memory_allocated() - before
    # one score of a token and head in 32 bits; what is linear in the tokens takes a third of that
    assert peak < 4518 * 4518 * m.config.num_attention_heads * 4, peak
    for p, o in zip(prompts, out):
        assert torch.equal(o[: len(p)], p) and len(o) == len(p) + 3
        gen, cache, table, cos, sin, logits = _alone(m, p)                          # dense attention over the values that the cache stands for
        with torch.no_grad():
            got = gen._prompts([p], cache, table, [0], cos, sin)[0]
        # roundings in another order, and codes of the later layers that lie on the other side of a step for them
        assert (got.float() - logits[-1].float()).norm() < 0.05 * logits[-1].float().norm()
