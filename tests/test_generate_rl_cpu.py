"""Sampling with the cache where rollouts need it: in PPO, and from actors whose parameters are sharded (two ranks, gloo)."""
import copy

import pytest
import torch
import torch.nn as nn

from atorch_b200.models.generate import CachedSampler, Generator
from atorch_b200.models.llama import LlamaConfig, LlamaDecoderLayer, LlamaModel
from atorch_b200.modules.w4_linear import quantize_linears
from atorch_b200.rl import AtorchRLConfig, ModelEngine, ModelSpec, PPOConfig, PPOTrainer
from tests.dist_utils import run_distributed


def _llama(seed=0):
    torch.manual_seed(seed)
    return LlamaModel(LlamaConfig(vocab_size=24, hidden_size=64, intermediate_size=96, num_hidden_layers=2, num_attention_heads=4,
                                  num_key_value_heads=2, max_position_embeddings=64, initializer_range=0.1)).bfloat16()


class Actor(nn.Module):
    def __init__(self, model):
        super().__init__()
        self.model = model

    def forward(self, ids):
        return self.model(ids)[1]


class Critic(nn.Module):
    def __init__(self):
        super().__init__()
        self.e, self.o = nn.Embedding(24, 16), nn.Linear(16, 1)

    def forward(self, ids):
        return self.o(self.e(ids)).squeeze(-1)


class Reward(nn.Module):
    def forward(self, ids):
        return (ids == 3).float().mean(1) * 4.0


def test_ppo_with_the_cached_sampler_and_a_quantised_reference():
    model = _llama()
    ref = Actor(quantize_linears(copy.deepcopy(model), 32))
    cfg = AtorchRLConfig(actor=ModelSpec(Actor(model), optimizer_args={"lr": 1e-3}, trainable=True),
                         critic=ModelSpec(Critic(), trainable=True), ref_model=ModelSpec(ref), reward_model=ModelSpec(Reward()),
                         ppo_config=PPOConfig(num_rollouts=8, batch_size=8, ppo_epoch=1))
    prompts = [torch.randint(0, 24, (4, 5), generator=torch.Generator().manual_seed(i)) for i in range(2)]
    trainer = PPOTrainer(ModelEngine(cfg), prompts, generate_fn=CachedSampler(model, max_new_tokens=6))
    before = model.lm_head.weight.detach().clone()
    stats = trainer.train(iterations=2)
    assert len(trainer.log) == 4 and all(torch.isfinite(torch.tensor(list(s.values()))).all() for s in stats)
    assert not torch.equal(before, model.lm_head.weight)


def _sharded(rank, world, wrap):
    from atorch_b200.parallel.fsdp import FSDP

    model = _llama()
    whole = copy.deepcopy(model)
    fsdp = FSDP(Actor(model), wrap_cls=(LlamaDecoderLayer,) if wrap else None, param_dtype=torch.bfloat16)
    prompt = torch.randint(0, 24, (3, 18), generator=torch.Generator().manual_seed(1))

    def both(**kw):
        torch.manual_seed(5 + rank)                 # each rank its own rollouts
        got = Generator(model).generate(prompt, 7, **kw)
        torch.manual_seed(5 + rank)
        want = Generator(whole).generate(prompt, 7, **kw)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), kw

    sampler = CachedSampler(model, max_new_tokens=6)
    for kw in (dict(), dict(temperature=1.0), dict(beams=3)):
        both(**kw)
    with torch.no_grad():
        want = fsdp(prompt)
    assert want.shape == (3, 18, 24)
    # a step of training, and samples of the new weights
    optimizer = torch.optim.SGD(fsdp.parameters(), lr=0.5)
    fsdp(prompt).float().logsumexp(-1).mean().backward()
    fsdp.engine.finalize_grads()
    fsdp.engine.attach_shard_grads()
    optimizer.step()
    fsdp.engine.sync_working_copy()
    state = fsdp.state_dict()
    assert not torch.equal(state["model.lm_head.weight"].bfloat16(), whole.lm_head.weight)
    whole.load_state_dict({n[len("model."):]: t for n, t in state.items()})
    both()
    both(temperature=1.0)
    assert sampler(fsdp, prompt).shape == (3, 24)
    if world > 1:                                   # nothing stays gathered
        assert all(u.full.untyped_storage().size() == 0 for u in fsdp.engine.units)


@pytest.mark.parametrize("wrap", [True, False])
def test_a_sharded_actor_is_sampled_from(wrap):
    run_distributed(_sharded, 2, (wrap,))
