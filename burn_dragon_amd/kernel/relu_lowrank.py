"""relu_lowrank::fused_forward (reference: src/kernel/relu_lowrank.rs:7-37) on the HIP library."""
from __future__ import annotations

from typing import Optional

import torch

from .. import ffi
from ..packed import _ROWS, PackedWeights, _new, _rows_type, _workspace
from .block_sparse import BlockPattern1d


def fused_forward(input: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor], threshold: float,
                  layout: BlockPattern1d, gate: Optional[torch.Tensor] = None,
                  ctx: Optional[ffi.Context] = None) -> torch.Tensor:
    """input [B,1|h,T,d], weight [1,h,d,N] or [h,d,N], bias [h,1,N]|None -> [B,h,T,N]."""
    ctx = ctx or ffi.default_context(input.device.index or 0)
    if weight.dim() == 4:
        assert weight.shape[0] == 1
        weight = weight[0]
    B, h_in, T, d = input.shape
    h, d_w, N = weight.shape
    if d != d_w:
        raise ValueError(f"inner dimensions differ: {d} vs {d_w}")
    input, weight = input.contiguous().float(), weight.contiguous().float()
    bias_c = None if bias is None else bias.reshape(h, N).contiguous().float()
    gate_c = None if gate is None else gate.contiguous().float()
    out = torch.empty((B, h, T, N), device=input.device, dtype=torch.float32)
    blocks = layout.block_bytes(N) if layout.is_sparse() else None
    ctx.check(ctx.lib.bdh_relu_lowrank(ctx.handle, B, h_in, T, d, h, N, ffi.ptr(input), ffi.ptr(weight),
                                       ffi.ptr(bias_c), float(threshold), max(layout.block_size, 1),
                                       blocks, 0 if blocks is None else len(blocks), ffi.ptr(gate_c), ffi.ptr(out)))
    return out


def packed_forward(input: torch.Tensor, weights: PackedWeights, bias: Optional[torch.Tensor] = None, threshold: float = 0.0,
                   gate: Optional[torch.Tensor] = None, out_dtype: torch.dtype = torch.float32, out: Optional[torch.Tensor] = None,
                   ctx: Optional[ffi.Context] = None) -> torch.Tensor:
    """fused_forward through packed weights of h groups, dense layout: input [B,1|h,T,d], bias [h,1,N] or [h,N] (f32), gate
    [B,h,T,N] -> [B,h,T,N] = gate * relu(input . weight + bias - threshold), a new tensor of out_dtype or `out`.  Input, gate
    and out are f32 or bf16 each."""
    h, d, N, on = weights.groups, weights.inner, weights.outer, weights.on
    kind, given = _rows_type("input", input, on), input.shape
    if len(given) != 4 or given[3] != d or (given[1] != h and given[1] != 1) or not input.is_contiguous():
        raise ValueError(f"input: expected contiguous [B, 1 or {h}, T, {d}], got {tuple(given)} with strides {input.stride()}")
    B, h_in, T, _ = given
    if (B | T | B * T) >> 31:
        raise ValueError(f"{B} x {T} rows: a call carries numbers below 2^31")
    shape, gate_kind = (B, h, T, N), 0
    if bias is not None and (bias.dtype is not torch.float32 or bias.get_device() != on or bias.shape not in ((h, N), (h, 1, N)) or
                             not bias.is_contiguous()):
        raise ValueError(f"bias: expected contiguous f32 [{h}, {N}], got {bias.dtype} {tuple(bias.shape)} on {bias.device}")
    if gate is not None:
        gate_kind = _rows_type("gate", gate, on)
        if gate.shape != shape or not gate.is_contiguous():
            raise ValueError(f"gate: expected contiguous {shape}, got {tuple(gate.shape)}")
    ctx = ffi.context_on(on, ctx)
    if out is None:
        out = _new(input, shape, out_dtype, ctx)
    elif out.dtype not in _ROWS or out.get_device() != on or out.shape != shape or not out.is_contiguous():
        raise ValueError(f"out: expected contiguous f32 or bf16 {shape}, got {out.dtype} {tuple(out.shape)}")
    held, workspace, size = _workspace(ctx, weights, B * h_in * T, B * T, input, kind, d)
    ctx.check(ctx._lib.bdh_packed_relu_lowrank(
        ctx.handle, weights._ref, B, h_in, T, input.data_ptr(), kind, None if bias is None else bias.data_ptr(), threshold,
        None if gate is None else gate.data_ptr(), gate_kind, out.data_ptr(), _ROWS[out.dtype], workspace, size))
    return out
