"""What a step's logits go through before a token is drawn from them (bdh_logit_rules, bdh_count_tokens): penalties for
tokens that occurred, biases, and a mask of the tokens that a grammar allows.  The reference's sampler has a temperature
and a top_k only (src/generation.rs:26-72)."""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Optional, Union

import torch

from . import ffi

Penalty = Union[None, float, torch.Tensor]


@dataclass
class LogitRules:
    """repetition, presence, frequency: a float for all sequences or an f32 tensor [B]; bias: f32 [V] or [B,V]; allowed:
    the words of pack_allowed, int32 [W] or [B,W].  None: no such rule."""

    repetition: Penalty = None
    presence: Penalty = None
    frequency: Penalty = None
    bias: Optional[torch.Tensor] = None
    allowed: Optional[torch.Tensor] = None

    def __post_init__(self):
        r, p, f = self.repetition, self.presence, self.frequency
        if r is not None and not isinstance(r, torch.Tensor) and not 2.0**-126 <= r < 2.0**128:
            raise ValueError(f"repetition divides and multiplies logits: it is positive and finite in f32, not {r}")
        if (p is not None and not isinstance(p, torch.Tensor) and not p > -math.inf) or \
                (f is not None and not isinstance(f, torch.Tensor) and not f > -math.inf):
            raise ValueError(f"a penalty is a number, or infinite where no token is said twice: presence {p}, frequency {f}")

    @property
    def penalises(self) -> bool:
        return any(p is not None for p in (self.repetition, self.presence, self.frequency))

    def to(self, device, batch: int) -> "LogitRules":
        """The rules with their penalties as tensors on `device`: a loop makes them once."""

        def row(p):
            if p is None or torch.is_tensor(p):
                return p
            return torch.full((batch,), float(p), device=device, dtype=torch.float32)

        return LogitRules(row(self.repetition), row(self.presence), row(self.frequency), self.bias, self.allowed)

    def select(self, index: torch.Tensor) -> "LogitRules":
        """The rules of the sequences `index` of the batch (rows that all share stay as they are)."""

        def pick(t, per_row):
            return t.index_select(0, index) if torch.is_tensor(t) and t.dim() == per_row else t

        return LogitRules(pick(self.repetition, 1), pick(self.presence, 1), pick(self.frequency, 1), pick(self.bias, 2),
                          pick(self.allowed, 2))


def token_counts(batch: int, vocab: int, device) -> torch.Tensor:
    """Empty counts [B,V] int32: bit 31 marks a token of the prompt, the others count how often it was produced."""
    return torch.zeros((batch, vocab), device=device, dtype=torch.int32)


def pack_allowed(allowed: torch.Tensor) -> torch.Tensor:
    """A mask [..., V] of truth values as int32 words [..., ceil(V / 32)]: token v is bit v % 32 of word v / 32."""
    V = allowed.shape[-1]
    padded = torch.zeros((*allowed.shape[:-1], (V + 31) // 32 * 32), device=allowed.device, dtype=torch.int64)
    padded[..., :V] = allowed.to(torch.int64)
    weights = torch.ones(32, dtype=torch.int64, device=allowed.device) << torch.arange(32, device=allowed.device)
    words = (padded.reshape(*allowed.shape[:-1], -1, 32) * weights).sum(-1)
    return torch.where(words >= 2**31, words - 2**32, words).to(torch.int32)


def _seen(seen: torch.Tensor, B: int, V: int, on: int) -> None:
    if seen.shape != (B, V) or seen.dtype is not torch.int32 or seen.get_device() != on or not seen.is_contiguous():
        raise ValueError(f"seen: expected a contiguous int32 tensor [{B}, {V}] on device {on}, got {seen.dtype} {tuple(seen.shape)} "
                         f"on {seen.device}")


def _row_stride(name: str, t: torch.Tensor, B: int, width: int, dtype, on: int) -> int:
    """Elements between the rows of a bias or mask: 0 for one row that all sequences share."""
    if t.dtype is not dtype or t.get_device() != on or t.dim() not in (1, 2) or t.shape[-1] != width or \
            (t.dim() == 2 and t.shape[0] != B) or (width > 1 and t.stride(-1) != 1):
        raise ValueError(f"{name}: expected {dtype} [{width}] or [{B}, {width}] on device {on}, got {t.dtype} {tuple(t.shape)} "
                         f"on {t.device}")
    return t.stride(0) if t.dim() == 2 and B > 1 else 0


def _check_row(name: str, p: Union[float, torch.Tensor], B: int, like: torch.Tensor, on: int) -> None:
    if isinstance(p, torch.Tensor) and (p.shape != (B,) or p.dtype is not torch.float32 or p.get_device() != on or not p.is_contiguous()):
        raise ValueError(f"{name}: expected f32 [{B}] on {like.device}")


def _row(p: float, B: int, like: torch.Tensor, ctx: ffi.Context) -> torch.Tensor:
    with ctx.torch_stream():
        return torch.full((B,), float(p), device=like.device, dtype=torch.float32)


def count_tokens(tokens: torch.Tensor, seen: torch.Tensor, lens: Optional[torch.Tensor] = None, prompt: bool = False,
                 ctx: Optional[ffi.Context] = None) -> None:
    """tokens [B,T] int64 (of row b the first lens[b]; lens int32 [B] on the device) into seen [B,V]: marked as tokens of
    the prompt, or counted as produced.  Ids outside the vocabulary are skipped."""
    B, T = tokens.shape
    on, V = tokens.get_device(), seen.shape[-1]
    if (B | T | V) >> 31:
        raise ValueError(f"sizes {B}, {T}, {V}: a call carries sizes below 2^31")
    _seen(seen, B, V, on)
    if tokens.dtype is not torch.int64 or (T > 1 and tokens.stride(1) != 1):
        raise ValueError("tokens: expected int64 rows")
    if lens is not None and (lens.shape != (B,) or lens.dtype is not torch.int32 or lens.get_device() != on or not lens.is_contiguous()):
        raise ValueError(f"lens: expected int32 [{B}] on {tokens.device}")
    ctx = ffi.context_on(on, ctx)
    ctx.check(ctx._lib.bdh_count_tokens(ctx.handle, B, T, V, tokens.data_ptr(), tokens.stride(0) if B > 1 else max(T, 1),
                                        None if lens is None else lens.data_ptr(), 1 if prompt else 0, seen.data_ptr()))


def apply_rules(logits: torch.Tensor, rules: LogitRules, seen: Optional[torch.Tensor] = None,
                newest: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                ctx: Optional[ffi.Context] = None) -> torch.Tensor:
    """logits [B,V] f32 (rows may be strided) under the rules -> out [B,V] (a new tensor, or `out`, which may be logits).
    seen [B,V]: the counts (token_counts) that penalties read; newest [B] int64: the tokens drawn last, counted first."""
    shape, f32 = logits.shape, torch.float32
    if len(shape) != 2 or logits.dtype is not f32:
        raise ValueError("logits: expected f32 rows [B,V]")
    B, V = shape
    if (B | V) >> 31:
        raise ValueError(f"sizes {B}, {V}: a call carries sizes below 2^31")
    on, dense = logits.get_device(), logits.is_contiguous()
    if not dense and V > 1 and logits.stride(1) != 1:
        raise ValueError("logits: expected f32 rows [B,V]")
    if seen is not None:
        _seen(seen, B, V, on)
        seen_ptr = seen.data_ptr()
    elif rules.penalises or newest is not None:
        raise ValueError("penalties need the counts of the tokens seen")
    else:
        seen_ptr = None
    if newest is not None and (newest.numel() != B or newest.dtype is not torch.int64 or newest.get_device() != on):
        raise ValueError(f"newest: expected int64 [{B}] on {logits.device}")
    repetition, presence, frequency = rules.repetition, rules.presence, rules.frequency
    if repetition is not None:
        _check_row("repetition", repetition, B, logits, on)
    if presence is not None:
        _check_row("presence", presence, B, logits, on)
    if frequency is not None:
        _check_row("frequency", frequency, B, logits, on)
    bias, allowed = rules.bias, rules.allowed
    bias_stride = 0 if bias is None else _row_stride("bias", bias, B, V, f32, on)
    allowed_stride = 0 if allowed is None else _row_stride("allowed", allowed, B, (V + 31) // 32, torch.int32, on)
    if out is None:
        out = torch.empty_like(logits) if dense else logits.new_empty(B, V)
        out_stride = V
    else:
        if out.shape != shape or out.dtype is not f32 or out.get_device() != on or (V > 1 and out.stride(1) != 1):
            raise ValueError(f"out: expected f32 rows [{B}, {V}] on {logits.device}")
        out_stride = out.stride(0) if B > 1 else V
    ctx = ffi.context_on(on, ctx)
    if newest is not None and (newest.dim() != 1 or not newest.is_contiguous()):
        with ctx.torch_stream():
            newest = newest.reshape(-1).contiguous()
    if repetition is not None and not isinstance(repetition, torch.Tensor):  # held until the call: a tensor made here has no other owner
        repetition = _row(repetition, B, logits, ctx)
    if presence is not None and not isinstance(presence, torch.Tensor):
        presence = _row(presence, B, logits, ctx)
    if frequency is not None and not isinstance(frequency, torch.Tensor):
        frequency = _row(frequency, B, logits, ctx)
    ctx.check(ctx._lib.bdh_logit_rules(
        ctx.handle, B, V, logits.data_ptr(), logits.stride(0) if B > 1 else V, seen_ptr,
        None if newest is None else newest.data_ptr(),
        None if repetition is None else repetition.data_ptr(), None if presence is None else presence.data_ptr(),
        None if frequency is None else frequency.data_ptr(), None if bias is None else bias.data_ptr(), bias_stride,
        None if allowed is None else allowed.data_ptr(), allowed_stride, out.data_ptr(), out_stride))
    return out
