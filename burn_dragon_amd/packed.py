"""Projections through weights that are packed for the matrix cores (bdh_pack_weights, bdh_packed_product,
bdh_grouped_product; the ReLU low-rank form is kernel.relu_lowrank.packed_forward): 8-bit integers with a scale for each
output channel, the rows brought to 8-bit integers with a scale each on their way, or bf16.  The reference keeps its
projections in f32 (src/model/bdh.rs:346-384, 446-449)."""
from __future__ import annotations

import ctypes
from typing import Optional, Sequence, Union

import torch

from . import ffi

_ROWS = {torch.float32: ffi.F32, torch.bfloat16: ffi.BF16}
_WEIGHTS = {torch.int8: ffi.INT8, torch.bfloat16: ffi.BF16}
MOST_INNER, MOST_OUTER, MOST_GROUPS = 131072, 1 << 24, 65535


class PackedWeights:
    """weight [K,N] or [G,K,N] (f32 or bf16, on the device) as weights of G groups for rows of K values: dtype torch.int8 or
    torch.bfloat16.  Laid out once; the tensor it was made from is not kept."""

    def __init__(self, weight: torch.Tensor, dtype: torch.dtype = torch.int8, ctx: Optional[ffi.Context] = None):
        if dtype not in _WEIGHTS:
            raise ValueError(f"packed weights are int8 or bf16, not {dtype}")
        if weight.dim() not in (2, 3) or weight.dtype not in _ROWS or not weight.is_contiguous():
            raise ValueError(f"weight: expected a contiguous f32 or bf16 tensor [K,N] or [G,K,N], got {weight.dtype} {tuple(weight.shape)}")
        self.groups, self.inner, self.outer = (1, *weight.shape) if weight.dim() == 2 else weight.shape
        if not (0 < self.inner <= MOST_INNER and 0 < self.outer <= MOST_OUTER and self.groups <= MOST_GROUPS):
            raise ValueError(f"weights [{self.groups}, {self.inner}, {self.outer}]: at most {MOST_GROUPS} groups of {MOST_INNER} x {MOST_OUTER}")
        self.dtype, self.device, self.on = dtype, weight.device, weight.get_device()
        ctx = ffi.context_on(self.on, ctx)
        lib, kind = ctx._lib, _WEIGHTS[dtype]
        with ctx.torch_stream():
            self.data = torch.empty((lib.bdh_packed_bytes(kind, self.groups, self.inner, self.outer),), device=self.device, dtype=torch.uint8)
            self.scales = torch.empty((self.groups, self.outer), device=self.device, dtype=torch.float32) if kind == ffi.INT8 else None
        ctx.check(lib.bdh_pack_weights(ctx.handle, kind, self.groups, self.inner, self.outer, weight.data_ptr(), _ROWS[weight.dtype],
                                       self.data.data_ptr(), ffi.ptr(self.scales)))
        self._c = ffi.PackedWeightsC(kind, self.groups, self.inner, self.outer, self.data.data_ptr(), ffi.ptr(self.scales))
        self._ref = ctypes.byref(self._c)
        # calls of up to this many rows a group need no workspace: asking for its size would cost a tenth of such a call
        self.few = 0
        for n in (16, 32, 64):
            if self.groups == 0 or lib.bdh_packed_workspace(ctx.handle, self._ref, n, n, None, ffi.F32, self.inner):
                break
            self.few = n

    def used_on(self, stream: torch.cuda.Stream) -> None:
        """Calls on `stream` use these weights: when they are dropped, their memory is given to others behind what is queued there
        by then (Tensor.record_stream).  For weights that are dropped while another stream than the one that made them works."""
        for t in (self.data, self.scales):
            if t is not None:
                t.record_stream(stream)

    @property
    def nbytes(self) -> int:
        return self.data.numel() + (0 if self.scales is None else 4 * self.scales.numel())


def _refuse_rows(name: str, t: torch.Tensor, on: int) -> None:
    raise ValueError(f"{name}: expected f32 or bf16 on device {on}, got {t.dtype} on {t.device}")


def _rows_type(name: str, t: torch.Tensor, on: int) -> int:
    kind = _ROWS.get(t.dtype)
    if kind is None or t.get_device() != on:
        _refuse_rows(name, t, on)
    return kind


def _workspace(ctx: ffi.Context, weights: PackedWeights, rows: int, of_group: int, x: torch.Tensor, kind: int, stride: int):
    """What the call needs beside its arguments, from torch's allocator: a captured call keeps its own."""
    if 0 <= of_group <= weights.few:
        return None, None, 0
    size = ctx._lib.bdh_packed_workspace(ctx.handle, weights._ref, rows, of_group, x.data_ptr(), kind, stride)
    if size == 0:
        return None, None, 0
    with ctx.torch_stream():
        held = torch.empty((size,), device=x.device, dtype=torch.uint8)
    return held, held.data_ptr(), size


def _new(like: torch.Tensor, shape, dtype: torch.dtype, ctx: ffi.Context) -> torch.Tensor:
    if dtype not in _ROWS:
        raise ValueError(f"out_dtype: f32 or bf16, not {dtype}")
    if ctx._follow:  # a tensor like another is a quarter faster to make than one from scratch
        return like.new_empty(shape) if dtype is like.dtype else like.new_empty(shape, dtype=dtype)
    with ctx.torch_stream():
        return like.new_empty(shape, dtype=dtype)


def _call(x: torch.Tensor, weights: PackedWeights, offsets, out_dtype, out, ctx):
    K, N, on = weights.inner, weights.outer, weights.on
    kind, shape = _rows_type("x", x, on), x.shape
    if not shape or shape[-1] != K:
        raise ValueError(f"x: expected rows of {K} values, got {tuple(shape)}")
    ctx = ffi.context_on(on, ctx)
    if len(shape) != 2 or not x.is_contiguous():
        if len(shape) != 2 or (K > 1 and x.stride(1) != 1) or (shape[0] > 1 and x.stride(0) < K):
            with ctx.torch_stream():  # it may be a copy
                x = x.reshape(-1, K).contiguous()
    M = x.shape[0]
    if out is None:
        out, out_stride = _new(x, (M, N) if len(shape) == 2 else (*shape[:-1], N), out_dtype, ctx), N
    else:
        _rows_type("out", out, on)
        dense = out.is_contiguous()
        if out.shape != (*shape[:-1], N) or not (dense or (out.dim() == 2 and out.stride(1) == 1 and out.stride(0) >= N)):
            raise ValueError(f"out: expected rows {(*shape[:-1], N)}, got {tuple(out.shape)} with strides {out.stride()}")
        out_stride = N if dense else out.stride(0)
    stride = x.stride(0) if M > 1 else K
    # (up to 32 grouped rows, on average at most 16 a group, are streamed as they are)
    of_group = M if offsets is None else 0 if M <= 32 and M <= 16 * weights.groups else -1
    held, workspace, size = _workspace(ctx, weights, M, of_group, x, kind, stride)
    if offsets is None:
        ctx.check(ctx._lib.bdh_packed_product(ctx.handle, weights._ref, M, x.data_ptr(), kind, stride, out.data_ptr(), _ROWS[out.dtype],
                                              out_stride, workspace, size))
    else:
        ctx.check(ctx._lib.bdh_grouped_product(ctx.handle, weights._ref, M, offsets.data_ptr(), x.data_ptr(), kind, stride,
                                               out.data_ptr(), _ROWS[out.dtype], out_stride, workspace, size))
    return out


def product(x: torch.Tensor, weights: PackedWeights, out_dtype: torch.dtype = torch.float32, out: Optional[torch.Tensor] = None,
            ctx: Optional[ffi.Context] = None) -> torch.Tensor:
    """x [..., K] (f32 or bf16) times weights of one group -> [..., N], a new tensor of out_dtype (f32 or bf16) or `out`."""
    if weights.groups != 1:
        raise ValueError(f"weights of {weights.groups} groups: a product takes one (grouped_product takes them all)")
    return _call(x, weights, None, out_dtype, out, ctx)


def grouped_product(x: torch.Tensor, weights: PackedWeights, offsets: Union[torch.Tensor, Sequence[int]],
                    out_dtype: torch.dtype = torch.float32, out: Optional[torch.Tensor] = None,
                    ctx: Optional[ffi.Context] = None) -> torch.Tensor:
    """x [M,K] (f32 or bf16), rows sorted by the group of weights they meet: rows offsets[g] .. offsets[g+1] - 1 meet group g
    -> [M,N], a new tensor of out_dtype or `out`, in which rows of no group are left as they are (uninitialised in a new one).
    offsets: G + 1 numbers that do not decrease; a list is checked here, an int32 tensor on the device is not (what decreases or
    leaves 0 .. M counts as the running maximum within 0 .. M)."""
    G = weights.groups
    if x.dim() != 2:
        raise ValueError(f"x: expected rows [M, {weights.inner}], got {tuple(x.shape)}")
    if not torch.is_tensor(offsets):
        offsets = [int(o) for o in offsets]
        if len(offsets) != G + 1 or offsets[0] < 0 or offsets[-1] > x.shape[0] or any(a > b for a, b in zip(offsets, offsets[1:])):
            raise ValueError(f"offsets: {len(offsets)} numbers for {G} groups of {x.shape[0]} rows that start at 0 or later and do not decrease")
        _rows_type("x", x, weights.on)
        with ffi.context_on(weights.on, ctx).torch_stream():
            offsets = torch.tensor(offsets, dtype=torch.int32, device=x.device)
    if offsets.shape != (G + 1,) or offsets.dtype is not torch.int32 or offsets.get_device() != weights.on or not offsets.is_contiguous():
        raise ValueError(f"offsets: expected int32 [{G + 1}] on {weights.device}, got {offsets.dtype} {tuple(offsets.shape)} on {offsets.device}")
    return _call(x, weights, offsets, out_dtype, out, ctx)
