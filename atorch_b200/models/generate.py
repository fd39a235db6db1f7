"""Generation with a Llama-family model of this package: a paged key/value cache in 4 bits (``ops/kv4.py``), greedy decoding,
sampling or beam search (``ops/beam.py``), and, if the model's linear layers were replaced by ``modules/w4_linear.py``, 4-bit
weights. Prompts of any lengths go through the model packed one behind another; after that every step takes one token a sequence.

The prompt's own attention runs on the keys and values that the cache stands for, so that it does not depend on how a sequence
was cut into prompt and generated tokens.
"""
from __future__ import annotations

import contextlib
import math
from typing import List, Optional, Sequence, Union

import torch

from .. import _lib, ops
from .llama import LlamaDecoderLayer, LlamaModel


class Generator:
    """Holds nothing between calls but the model; every :meth:`generate` has a cache of its own."""

    def __init__(self, model: LlamaModel, page_size: int = 16):
        # (by what is used of them: a layer may be wrapped by something that hands its attributes on)
        if not all(hasattr(model, n) for n in ("embed_tokens", "layers", "norm", "lm_head", "rope", "config")) \
                or not all(hasattr(layer, n) for layer in model.layers for n in ("qkv_proj", "gate_up_proj", "down_proj", "n_kv", "_proj")):
            raise TypeError("generation runs a LlamaModel with its LlamaDecoderLayers (the model inside a wrapper, not the wrapper), and "
                            f"this is a {type(model).__name__}")
        self.model, self.page_size = model, page_size
        self.dtype = model.embed_tokens.weight.dtype
        if self.dtype not in (torch.bfloat16, torch.float16):
            raise ValueError(f"generation runs in bf16 or fp16, and the model is {self.dtype}")

    # -- one pass over tokens [T], appended to the cache -------------------------------------------------------------------
    def _layer(self, layer: LlamaDecoderLayer, h, cache, table, seq, pos, cos, sin, attend):
        n_q, d = layer.n_q, layer.config.head_dim
        qkv = layer._proj(layer.qkv_proj, layer.input_layernorm(h))
        q = ops.kv4_append(cache, table, seq, pos, qkv, n_q, cos, sin)
        h = layer._proj(layer.o_proj, attend(q, cache).reshape(h.shape[0], n_q * d), h)
        x = layer.post_attention_layernorm(h)
        if type(layer.gate_up_proj) is torch.nn.Linear and layer.gate_up_proj.bias is None:
            act = ops.linear_swiglu(x, layer.gate_up_proj.weight)
        else:
            act = ops.swiglu(layer._proj(layer.gate_up_proj, x))
        return layer._proj(layer.down_proj, act, h)

    def _run(self, tokens, cache, table, seq, pos, cos, sin, attend, last=None):
        """Logits of the tokens (or of those that ``last`` picks)."""
        m = self.model
        h = m.embed_tokens(tokens)
        for i, layer in enumerate(m.layers):
            h = self._layer(layer, h, cache.layer(i), table, seq, pos, cos, sin, attend)
        return m.layers[0]._proj(m.lm_head, m.norm(h if last is None else h[last]))

    def _prompts(self, prompts, cache, table, rows, cos, sin):
        """Logits of the prompts' last tokens; sequence ``i`` is row ``rows[i]`` of the table."""
        dev = table.device
        sizes = torch.tensor([len(p) for p in prompts])
        seq = torch.repeat_interleave(torch.tensor(rows, dtype=torch.int32), sizes).to(dev)
        pos = torch.cat([torch.arange(len(p), dtype=torch.int32) for p in prompts]).to(dev)
        cu = torch.zeros(len(prompts) + 1, dtype=torch.int32)
        cu[1:] = sizes.cumsum(0)
        last = (cu[1:] - 1).long().to(dev)
        cu = cu.to(dev)

        def attend(q, layer):
            k, v = ops.kv4_read(layer, table, seq, pos, q.dtype)
            return ops.attention(q.unsqueeze(0), k.unsqueeze(0), v.unsqueeze(0), causal=True, cu_seqlens=cu)

        def attend_over_cache(q, layer):
            # the flash kernels take bf16; dense scores of all prompts' tokens by all tokens would be 34 GB for 16 prompts of 1024 and 32 heads
            if len(set(sizes.tolist())) == 1:
                return ops.kv4_attention(q.view(len(prompts), -1, *q.shape[1:]), layer, table[rows], lengths)
            return torch.cat([ops.kv4_attention(one.unsqueeze(0), layer, table[row: row + 1], lengths[i: i + 1])[0]
                              for i, (row, one) in enumerate(zip(rows, q.split(sizes.tolist())))])

        lengths = sizes.to(torch.int32).to(dev)
        if self.dtype is not torch.bfloat16 and dev.type == "cuda":
            attend = attend_over_cache

        return self._run(torch.cat([p.to(dev) for p in prompts]), cache, table, seq, pos, cos, sin, attend, last)

    def _step(self, tokens, cache, table, lengths, cos, sin):
        """Logits of one more token of every row; ``lengths`` counts those before it."""
        now = lengths + 1
        return self._run(tokens, cache, table, None, lengths, cos, sin,
                         lambda q, layer: ops.kv4_attention(q.unsqueeze(1), layer, table, now))

    @contextlib.contextmanager
    def _whole_parameters(self):
        """All parameters in their place for the whole call: the layers' parts are called directly, past the forwards at which a
        sharded engine (``parallel/fsdp.py``) gathers them."""
        engines = {}
        for p in self.model.parameters():
            unit = getattr(p, "_atb_unit", None)
            if unit is not None:
                engines[id(unit.engine)] = unit.engine
        with contextlib.ExitStack() as stack:
            for engine in engines.values():
                stack.enter_context(engine.summon_full_params())
            for name, p in self.model.named_parameters():
                if p.numel() and p.untyped_storage().nbytes() == 0:
                    raise ValueError(f"parameter {name} is not in memory: it is sharded by something that generation does not know")
            yield

    @torch.no_grad()
    def generate(self, prompts: Union[torch.Tensor, Sequence[torch.Tensor]], max_new_tokens: int, eos: Optional[int] = None,
                 temperature: float = 0.0, beams: int = 1, length_penalty: float = 0.0) -> List[torch.Tensor]:
        """``prompts``: token ids, ``[B, T]`` or one tensor a sequence. Greedy with ``temperature`` 0, sampling above; with ``beams``
        above 1 a beam search, whose best sequence by ``score / new tokens ** length_penalty`` is returned. Sequences come back with
        their prompts, up to ``eos`` where there is one. Where the parameters are sharded (``parallel/fsdp.py``) every rank has to
        call it, each with prompts of its own; they are gathered once for the call."""
        prompts = [p.reshape(-1) for p in prompts]
        if not prompts or min(len(p) for p in prompts) == 0:
            raise ValueError("prompts have one token at least")
        if beams < 1 or (beams > 1 and temperature > 0):
            raise ValueError("a beam search does not sample")
        if max_new_tokens < 1:
            return prompts
        dev = self.model.embed_tokens.weight.device
        with torch.cuda.device(dev) if dev.type == "cuda" else contextlib.nullcontext(), self._whole_parameters():
            return self._generate(prompts, max_new_tokens, eos, temperature, beams, length_penalty)

    def _generate(self, prompts, max_new_tokens, eos, temperature, beams, length_penalty):
        m, cfg, S = self.model, self.model.config, self.page_size
        dev, B, W = m.embed_tokens.weight.device, len(prompts), beams
        if dev.type == "cuda":
            _lib.check_status(dev)           # behind a failed kernel the operators store nothing
        longest = max(len(p) for p in prompts) + max_new_tokens
        cos, sin = m.rope(longest, dev)

        # pages: a sequence's beams share those that the prompt fills, and have the others for themselves
        width, pages = -(-longest // S), 0
        table = torch.zeros(B, W, width, dtype=torch.int32)
        for b, p in enumerate(prompts):
            full, need = len(p) // S, -(-(len(p) + max_new_tokens) // S)
            table[b, :, :full] = torch.arange(pages, pages + full, dtype=torch.int32)
            pages += full
            table[b, :, full:need] = torch.arange(pages, pages + W * (need - full), dtype=torch.int32).view(W, need - full)
            pages += W * (need - full)
        table = table.view(B * W, width).to(dev)
        cache = ops.KV4Cache(cfg.num_hidden_layers, pages, S, m.layers[0].n_kv, cfg.head_dim, dev)
        lengths = torch.tensor([len(p) for p in prompts for _ in range(W)], dtype=torch.int32, device=dev)
        logits = self._prompts(prompts, cache, table, [b * W for b in range(B)], cos, sin)

        if W > 1:
            out = self._beams(logits, cache, table, lengths, cos, sin, B, W, max_new_tokens, -1 if eos is None else eos,
                              length_penalty)
        else:
            out = self._tokens(logits, cache, table, lengths, cos, sin, max_new_tokens, eos, temperature)
        if dev.type == "cuda":
            _lib.check_status(dev)
        result = []
        for p, new in zip(prompts, out):
            if eos is not None:
                at = (new == eos).nonzero()
                new = new[: int(at[0]) + 1] if len(at) else new
            result.append(torch.cat([p.to(new.device), new]))
        return result

    def _tokens(self, logits, cache, table, lengths, cos, sin, steps, eos, temperature):
        got, done = [], None
        for i in range(steps):
            if temperature > 0:
                # the first to arrive of exponential waiting times: what multinomial draws, without its assertion on the device
                weights = torch.softmax(logits.float() / temperature, -1)
                tokens = (weights / torch.empty_like(weights).exponential_()).argmax(-1)
            else:
                tokens = logits.argmax(-1)
            got.append(tokens)
            if eos is not None:
                done = tokens == eos if done is None else done | (tokens == eos)
                if bool(done.all()):
                    break
            if i + 1 < steps:
                logits = self._step(tokens, cache, table, lengths, cos, sin)
                lengths = lengths + 1
        return torch.stack(got, 1)

    def _beams(self, logits, cache, table, lengths, cos, sin, B, W, steps, eos, penalty):
        scores = torch.zeros(B, 1, dtype=torch.float32, device=table.device)
        finished, got = None, []
        for i in range(steps):
            first = i == 0
            scores, tokens, parents, finished = ops.beam_select(logits.view(B, 1 if first else W, -1), scores, finished, eos, W)
            got.append((tokens, parents))
            if eos < 0:
                finished = None
            elif bool(finished.all()):
                break
            if i + 1 < steps:
                ops.beam_reorder(cache.codes, cache.scales, table, lengths, parents)
                logits = self._step(tokens.view(-1), cache, table, lengths, cos, sin)
                lengths = lengths + 1
        # back from the last step, parent by parent
        at = torch.arange(W, device=table.device).expand(B, W)
        sequences = []
        for tokens, parents in reversed(got):
            sequences.append(tokens.gather(1, at))
            at = parents.long().gather(1, at)
        sequences = torch.stack(sequences[::-1], 2)                  # [B, W, new]
        size = torch.full((B, W), sequences.shape[2], dtype=torch.float32, device=table.device)
        if eos >= 0:
            hit = sequences == eos
            size = torch.where(hit.any(-1), hit.float().argmax(-1) + 1.0, size)
        best = (scores / size ** penalty).argmax(-1)
        return sequences[torch.arange(B, device=table.device), best]


def generate(model: LlamaModel, prompts, max_new_tokens: int, **kw) -> List[torch.Tensor]:
    """:meth:`Generator.generate` on a model."""
    return Generator(model).generate(prompts, max_new_tokens, **kw)


class CachedSampler:
    """``generate_fn`` of :class:`~atorch_b200.rl.trainer.PPOTrainer` for actors around a :class:`LlamaModel`: samples with a cache
    instead of running the whole sequence for every token. ``model`` is the model inside the actor (it is read at every call, so
    its current weights are used)."""

    def __init__(self, model: LlamaModel, max_new_tokens: int = 8, temperature: float = 1.0, page_size: int = 16):
        if not (temperature > 0 and math.isfinite(temperature)):
            raise ValueError("sampling has a positive temperature")
        self.generator, self.max_new_tokens, self.temperature = Generator(model, page_size), max_new_tokens, temperature

    def __call__(self, actor, prompt: torch.Tensor) -> torch.Tensor:
        out = self.generator.generate(prompt, self.max_new_tokens, temperature=self.temperature)
        return torch.stack(out).to(prompt.device)
