"""Sequences that continue shared prompts, through the C ABI (bdh_shared_prefix_attention, bdh_shared_prefix_fork): the
state a prompt left is read once for all the sequences that continue it, and what a sequence says itself is kept beside
it as keys and values.  The sums are those of BDH::recurrent_attention (src/model/bdh.rs:288-302), cut where the prompt
ends; the reference gives every sequence a state of its own."""
from __future__ import annotations

import ctypes
from typing import Optional, Sequence

import torch

from . import ffi
from .positional import RotaryEmbedding

_DTYPES = {torch.float32: ffi.F32, torch.bfloat16: ffi.BF16}


def _check(name: str, t: torch.Tensor, shape, dtype, device: int) -> None:
    """device: the index, -1 for host memory (an int is compared in half the time of a torch.device; a call of one token
    takes the GPU as long as the host, so these checks count)"""
    if t.shape != shape or t.dtype is not dtype or t.get_device() != device or not t.is_contiguous():
        raise ValueError(f"{name}: expected a contiguous {dtype} tensor {tuple(shape)} on device {device}, got {t.dtype} "
                         f"{tuple(t.shape)} on {t.device}")


def _reshaped(t: torch.Tensor, shape, on: int, ctx: Optional[ffi.Context]) -> torch.Tensor:
    with ffi.context_on(on, ctx).torch_stream():  # it may be a copy
        return t.reshape(shape)


def _refuse_sizes(*sizes: int) -> None:
    raise ValueError(f"sizes {sizes}: a call carries sizes below 2^31")


def _prompts(counts: Optional[Sequence[int]], G: int, B: int):
    """The numbers of the prompts' sequences for the C ABI: None is all of one prompt."""
    if G == 1 and (counts is None or (len(counts) == 1 and counts[0] == B)):
        return None
    if counts is None:
        raise ValueError(f"{G} prompts need the numbers of their sequences")
    if len(counts) != G or sum(counts) != B or min(counts, default=0) < 0:
        raise ValueError(f"counts {list(counts)} do not deal {B} sequences to {G} prompts")
    return (ctypes.c_int32 * G)(*counts)


def _slopes(alibi_slopes, h: int):
    if alibi_slopes is None:
        return None
    if len(alibi_slopes) != h:
        raise ValueError(f"{len(alibi_slopes)} slopes for {h} heads")
    return (ctypes.c_float * h)(*map(float, alibi_slopes))


def shared_prefix_attention(query: torch.Tensor, value: torch.Tensor, rho: torch.Tensor, keys: torch.Tensor,
                            values: torch.Tensor, lens: torch.Tensor, freqs: Optional[torch.Tensor], position: int = 0,
                            positions: Optional[torch.Tensor] = None,
                            rotary_embedding: RotaryEmbedding = RotaryEmbedding.ROPE, alibi_slopes=None,
                            counts: Optional[Sequence[int]] = None, longest: Optional[int] = None,
                            ctx: Optional[ffi.Context] = None) -> torch.Tensor:
    """query [B,h,T,N] (un-rotated), value [B,T,d]; rho [G,h,Nq,d] (f32 or bf16, read only) the states of G prompts, of
    which prompt g is continued by counts[g] sequences in order; keys [B,h,Nq,S] and values [B,S,d] what each sequence
    has said (zeros from place lens[b] on, lens int32 [B] on the device).  Returns out [B,h,T,d] and stores the new
    tokens' keys and values at places lens[b] and on; lens itself is advanced by the caller.  position / positions: as in
    recurrent_attention, the prompt's tokens counted.  longest: an upper bound of lens (default S - T)."""
    B, h, T, N = query.shape
    on = query.get_device()
    rot = RotaryEmbedding.parse(rotary_embedding)
    Nq = 2 * N if rot == RotaryEmbedding.POPE else N
    d, S, G = value.shape[-1], keys.shape[-1], rho.shape[0]
    if (B | h | T | Nq | d | S | G) >> 31:
        _refuse_sizes(B, h, T, Nq, d, S, G)
    if rho.dtype not in _DTYPES:
        raise ValueError(f"rho is f32 or bf16, not {rho.dtype}")
    f32, int32 = torch.float32, torch.int32
    _check("query", query, (B, h, T, N), f32, on)
    if value.dim() != 3:
        value = _reshaped(value, (B, T, d), on, ctx)
    _check("value", value, (B, T, d), f32, on)
    _check("rho", rho, (G, h, Nq, d), rho.dtype, on)
    _check("keys", keys, (B, h, Nq, S), f32, on)
    _check("values", values, (B, S, d), f32, on)
    _check("lens", lens, (B,), int32, on)
    if positions is not None:
        _check("positions", positions, (B,), int32, on)
    if rot != RotaryEmbedding.ALIBI:
        if freqs is None:
            raise ValueError(f"{rot.name} needs its frequencies")
        if freqs.dim() != 1:
            freqs = _reshaped(freqs, (-1,), on, ctx)
        _check("freqs", freqs, (N,), f32, on)
    n_of = _prompts(counts, G, B)
    slopes = _slopes(alibi_slopes, h)
    ctx = ffi.context_on(on, ctx)
    out = query.new_empty(B, h, T, d)
    ctx.check(ctx._lib.bdh_shared_prefix_attention(
        ctx.handle, G, n_of, B, h, T, N, d, rot, query.data_ptr(), value.data_ptr(),
        None if rot == RotaryEmbedding.ALIBI else freqs.data_ptr(), int(position), None if positions is None else positions.data_ptr(), slopes,
        rho.data_ptr(), _DTYPES[rho.dtype], S, lens.data_ptr(), -1 if longest is None else int(longest), keys.data_ptr(),
        values.data_ptr(), out.data_ptr()))
    return out


def shared_prefix_fork(rho: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, lens: torch.Tensor,
                       rotary_embedding: RotaryEmbedding = RotaryEmbedding.ROPE, alibi_slopes=None,
                       counts: Optional[Sequence[int]] = None, longest: Optional[int] = None,
                       out: Optional[torch.Tensor] = None, ctx: Optional[ffi.Context] = None) -> torch.Tensor:
    """The states [B,h,Nq,d] (of rho's type) that the sequences of shared_prefix_attention would have had to themselves:
    the prompt's state with the sequence's own tokens added, as after the same recurrent_attention calls."""
    B, h, Nq, S = keys.shape
    on = keys.get_device()
    G, d = rho.shape[0], rho.shape[-1]
    if (B | h | Nq | S | G | d) >> 31:
        _refuse_sizes(B, h, Nq, S, G, d)
    if rho.dtype not in _DTYPES:
        raise ValueError(f"rho is f32 or bf16, not {rho.dtype}")
    _check("rho", rho, (G, h, Nq, d), rho.dtype, on)
    _check("keys", keys, (B, h, Nq, S), torch.float32, on)
    _check("values", values, (B, S, d), torch.float32, on)
    _check("lens", lens, (B,), torch.int32, on)
    if out is None:
        out = rho.new_empty(B, h, Nq, d)
    else:
        _check("out", out, (B, h, Nq, d), rho.dtype, on)
    n_of = _prompts(counts, G, B)
    slopes = _slopes(alibi_slopes, h)
    ctx = ffi.context_on(on, ctx)
    ctx.check(ctx._lib.bdh_shared_prefix_fork(
        ctx.handle, G, n_of, B, h, Nq, d, int(RotaryEmbedding.parse(rotary_embedding)), slopes,
        rho.data_ptr(), _DTYPES[rho.dtype], S, lens.data_ptr(), -1 if longest is None else int(longest), keys.data_ptr(),
        values.data_ptr(), out.data_ptr()))
    return out
