"""Generation loop of the reference (src/generation.rs) over the HIP model step.

The reference copies the logits to the host after every token, samples there with thread_rng and
uploads the token (src/generation.rs:114-124).  Here the draw happens on the device
(bdh_sample_top_k): the uniform variates come from a torch generator on the GPU, the sampled token is
fed back without leaving HBM, and the only host transfers are the ones the caller asks for (streaming
callback or the final token list).
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Callable, List, Optional, Tuple

import torch

from .model.bdh import BDH
from .model.state import ModelState
from .rules import LogitRules, apply_rules, count_tokens, token_counts
from .tokenizer import Tokenizer


@dataclass(frozen=True)
class ContextStrategy:
    """src/generation.rs:12-16: Infinite, or Sliding { window }."""

    window: Optional[int] = None  # None = Infinite

    @classmethod
    def infinite(cls) -> "ContextStrategy":
        return cls(None)

    @classmethod
    def sliding(cls, window: int) -> "ContextStrategy":
        return cls(int(window))


@dataclass
class GenerationSettings:
    """src/generation.rs:18-24."""

    max_new_tokens: Optional[int] = None
    temperature: float = 1.0
    top_k: Optional[int] = None
    strategy: ContextStrategy = ContextStrategy()


@dataclass
class GenerationConfig:
    """src/config/core.rs:20-30."""

    prompt: str = ""
    max_tokens: Optional[int] = None
    temperature: float = 1.0
    top_k: Optional[int] = None
    context_strategy: ContextStrategy = ContextStrategy()


def resolve_context_strategy(strategy: ContextStrategy, default_window: int) -> ContextStrategy:
    """src/generation.rs:243-259: a sliding window of 0 means the training block size."""
    if strategy.window is None:
        return strategy
    return ContextStrategy(max(default_window, 1) if strategy.window == 0 else strategy.window)


def normalize_max_tokens(max_tokens: Optional[int]) -> Optional[int]:
    """src/generation.rs:236-241: negative means unbounded."""
    return max_tokens if max_tokens is not None and max_tokens >= 0 else None


def sample_from_logits(model: BDH, last_logits: torch.Tensor, temperature: float, top_k: Optional[int],
                       uniforms: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """sample_from_logits_values after the temperature division (src/generation.rs:26-72,117), on the
    device.  last_logits [B,V] f32 (rows may be strided), uniforms [B] f32 in [0,1) -> tokens [B] int64."""
    assert last_logits.dim() == 2 and last_logits.stride(1) == 1 and last_logits.dtype == torch.float32
    B, V = last_logits.shape
    uniforms = uniforms.to(last_logits.device, torch.float32).contiguous()
    assert uniforms.numel() == B
    if out is None:
        out = torch.empty((B,), device=last_logits.device, dtype=torch.int64)
    ctx = model.ctx
    ctx.check(ctx.lib.bdh_sample_top_k(ctx.handle, B, V, last_logits.data_ptr(), last_logits.stride(0) if B > 1 else V,
                                       float(temperature), int(top_k) if top_k else 0, uniforms.data_ptr(),
                                       out.data_ptr()))
    return out


def prefill_state(model: BDH, prompt_tokens) -> Tuple[ModelState, torch.Tensor]:
    """src/generation.rs:74-105: runs the prompt through forward_with_state on a fresh state and
    returns the state and the logits of the last prompt token [V]."""
    prompt = torch.as_tensor(prompt_tokens, dtype=torch.int64).reshape(1, -1)
    if prompt.shape[1] == 0:
        raise ValueError("prompt must contain at least one token")
    state = model.init_state()
    logits = model.forward_with_state(prompt, state)
    if logits.shape[1] != prompt.shape[1]:
        raise RuntimeError(f"prefill produced mismatched length: expected {prompt.shape[1]}, got {logits.shape[1]}")
    return state, logits[0, -1]


def uniform_variates(n: int, device, generator: Optional[torch.Generator] = None) -> torch.Tensor:
    """n uniform variates in [0, 1) as an [n] tensor on `device`, drawn on the generator's own device (a CPU
    generator serves a GPU model)."""
    if generator is not None and generator.device.type != torch.device(device).type:
        return torch.rand((n,), device=generator.device, generator=generator).to(device)
    return torch.rand((n,), device=device, generator=generator)


class VariateStream:
    """The uniform variates of one generation run, drawn from `generator` a block at a time so that no host work
    is done per token.  Every consumer draws blocks of the same size: two runs from equal seeds see the same
    sequence whichever entry point they go through."""

    BLOCK = 256

    def __init__(self, device, generator: Optional[torch.Generator] = None):
        self.device, self.generator = device, generator
        self._buf, self._at = None, 0

    def next(self) -> torch.Tensor:
        if self._buf is None or self._at == self.BLOCK:
            self._buf, self._at = uniform_variates(self.BLOCK, self.device, self.generator), 0
        self._at += 1
        return self._buf[self._at - 1:self._at]


def sample_next_token(model: BDH, state: ModelState, last_logits: torch.Tensor, temperature: float,
                      top_k: Optional[int], generator: Optional[torch.Generator] = None,
                      variates: Optional[VariateStream] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """src/generation.rs:107-128: draws from last_logits [V], feeds the token and returns
    (token [1] int64 on the device, logits of the new token [V]).  The variate comes from `variates` when a
    run keeps a stream, else from a draw of its own."""
    u = variates.next() if variates is not None else uniform_variates(1, last_logits.device, generator)
    nxt = sample_from_logits(model, last_logits.reshape(1, -1), temperature, top_k, u)
    logits = model.forward_with_state(nxt.reshape(1, 1), state)
    return nxt, logits[0, -1]


def generate_tokens(model: BDH, prompt_tokens: List[int], settings: GenerationSettings,
                    on_token: Optional[Callable[[int], None]] = None,
                    generator: Optional[torch.Generator] = None) -> List[int]:
    """src/generation.rs:158-203.  Without a callback the tokens stay on the device until the end;
    with one, each token is copied to the host as it is produced (streaming)."""
    if settings.max_new_tokens is None and on_token is None:
        raise ValueError("an unbounded generation needs an on_token callback that eventually raises StopIteration")
    full = list(int(t) for t in prompt_tokens)
    state, last_logits = prefill_state(model, full)
    window = settings.strategy.window
    if window and state.position > window:
        state.trim(window)
    produced: List[torch.Tensor] = []
    generated = 0
    variates = VariateStream(last_logits.device, generator)
    try:
        while settings.max_new_tokens is None or generated < settings.max_new_tokens:
            nxt, last_logits = sample_next_token(model, state, last_logits, settings.temperature, settings.top_k,
                                                 generator, variates)
            generated += 1
            if on_token is not None:
                tok = int(nxt[0])
                full.append(tok)
                on_token(tok)
            else:
                produced.append(nxt)
            if window and state.position > window:
                state.trim(window)
    except StopIteration:
        pass
    if produced:
        full.extend(int(t) for t in torch.cat(produced).cpu())
    return full


def generate_samples(model: BDH, prompt_tokens: List[int], n: int, settings: GenerationSettings,
                     rules: Optional[LogitRules] = None, stop_token: Optional[int] = None, capacity: int = 64,
                     generator: Optional[torch.Generator] = None) -> List[List[int]]:
    """n continuations of one prompt, drawn together: the prompt is read once, its state is shared by all of them for the
    first `capacity` tokens of their own (BDH.share_state) and copied for each only then.  `rules` apply to the logits of
    every draw; a sequence ends with stop_token, which is part of it, where the rules allow nothing more (its logits are all
    -inf: nothing is drawn from them), or after settings.max_new_tokens, and the ended ones leave the batch every few tokens.
    Each sequence has its own variates: where others end does not change them.  Sharing is for states that are large next to
    a launch: 4 samples of 4 heads of 256 neurons take 7.0 ms for 64 tokens with capacity 1 (states of their own after 4
    tokens) and 15.2 with 64, 32 of 4 heads of 8192 138 and 58.
    Returns the new tokens of each (the reference generates one sequence at a time, src/generation.rs:158-203)."""
    if settings.max_new_tokens is None or settings.max_new_tokens < 0:
        raise ValueError("max_new_tokens says how long the samples may become")
    if n < 1:
        raise ValueError("at least one sample")
    if settings.max_new_tokens == 0:
        return [[] for _ in range(n)]
    with model.ctx.torch_stream():
        return _generate_samples(model, prompt_tokens, n, settings, rules, stop_token, capacity, generator)


def _generate_samples(model: BDH, prompt_tokens: List[int], n: int, settings: GenerationSettings, rules: Optional[LogitRules],
                      stop_token: Optional[int], capacity: int, generator: Optional[torch.Generator]) -> List[List[int]]:
    dev, V = model.device, model.vocab_size
    state, last = prefill_state(model, prompt_tokens)
    shared, own = model.share_state(state, [n], min(capacity, settings.max_new_tokens)), None
    logits = last.reshape(1, V).repeat(n, 1)
    seen = None
    if rules is not None:
        rules = rules.to(dev, n)
        if rules.penalises:
            seen = token_counts(n, V, dev)
            said = torch.as_tensor(prompt_tokens, dtype=torch.int64).reshape(1, -1).to(dev).repeat(n, 1)
            count_tokens(said, seen, prompt=True, ctx=model.ctx)
    alive = list(range(n))  # the samples that the rows of the batch are
    alive_dev = torch.arange(n, device=dev)
    produced = []  # (rows, tokens, largest logits or None) of every draw
    newest, every, largest = None, 16, None
    for step in range(settings.max_new_tokens):
        if rules is not None:
            logits = apply_rules(logits, rules, seen, newest if seen is not None else None, ctx=model.ctx)
            largest = logits.amax(1)  # looked at with the tokens: what is drawn meanwhile from a row of -inf is dropped
        if step % every == 0:
            variates = uniform_variates(every * n, dev, generator).reshape(every, n)
        newest = sample_from_logits(model, logits, settings.temperature, settings.top_k,
                                    variates[step % every].index_select(0, alive_dev))
        produced.append((alive, newest, largest))
        if step + 1 == settings.max_new_tokens:
            break
        if (stop_token is not None or rules is not None) and step % every == every - 1:
            ended = torch.zeros_like(newest, dtype=torch.bool)
            if stop_token is not None:
                ended |= (torch.stack([t for _, t, _ in produced[-every:]]) == stop_token).any(0)
            if rules is not None:
                ended |= torch.isneginf(torch.stack([m for _, _, m in produced[-every:]])).any(0)
            live = [i for i, e in enumerate(ended.tolist()) if not e]
            if not live:
                break
            if len(live) < len(alive):
                if own is None:
                    shared = model.select_shared(shared, live)
                else:
                    own = model.select_sequences(own, live)
                index = torch.tensor(live, device=dev)
                newest, alive_dev = newest.index_select(0, index), alive_dev.index_select(0, index)
                seen = None if seen is None else seen.index_select(0, index)
                rules = None if rules is None else rules.select(index)
                alive = [alive[i] for i in live]
        if own is None and shared.room == 0:
            own, shared = model.fork_shared(shared), None
        tokens = newest.reshape(-1, 1)
        logits = (model.forward_shared(tokens, shared) if own is None else model.forward_with_state(tokens, own))[:, -1]
    out: List[List[int]] = [[] for _ in range(n)]
    going = [True] * n
    for rows, tokens, most in produced:
        for i, t, empty in zip(rows, tokens.tolist(), [False] * len(rows) if most is None else torch.isneginf(most).tolist()):
            if going[i] and not empty:
                out[i].append(t)
            going[i] = going[i] and not empty and t != stop_token
    return out


def generate_text(model: BDH, tokenizer: Tokenizer, block_size: int, generation: GenerationConfig,
                  generator: Optional[torch.Generator] = None) -> str:
    """src/generation.rs:205-234."""
    strategy = resolve_context_strategy(generation.context_strategy, block_size)
    prompt_ids = tokenizer.encode(generation.prompt, False, False)
    if strategy.window is not None and len(prompt_ids) > strategy.window:
        prompt_ids = prompt_ids[len(prompt_ids) - strategy.window:]
    settings = GenerationSettings(normalize_max_tokens(generation.max_tokens), generation.temperature,
                                  generation.top_k, strategy)
    tokens = generate_tokens(model, prompt_ids, settings, None, generator)
    return tokenizer.decode([t for t in tokens if t >= 0])
