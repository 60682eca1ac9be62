"""Sequences of a batch moved between the slots of the buffers that hold them (bdh_copy_slots): forked, compacted,
freed, reordered; all buffers of a batch in one launch."""
from __future__ import annotations

import math
from typing import Iterable, Optional, Sequence, Tuple, Union

import torch

from . import ffi

FREE, KEEP = -1, -2


def copy_slots(buffers: Iterable[Tuple[torch.Tensor, torch.Tensor, int]], origin: Union[torch.Tensor, Sequence[int]],
               ctx: Optional[ffi.Context] = None) -> None:
    """buffers: (destination, source, slot dimension) of each, the two alike but for the number of slots; the same tensor
    twice moves its slots in place (every slot is read as it was before the call).  origin[i], for every slot of the
    destinations: the source's slot that it takes, FREE (zeros) or KEEP (left as it is).  A list is checked here; an
    int32 tensor on the device is not, entries that name no slot leave theirs as it is."""
    buffers = list(buffers)
    if not buffers:
        return
    dst, src, dim = buffers[0]
    dev, on, n, m = dst.device, dst.get_device(), dst.shape[dim], src.shape[dim]
    if (n | m) >> 31:
        raise ValueError(f"{n} and {m} slots: a call carries numbers below 2^31")
    table = (ffi.SlotBufferC * len(buffers))()
    for k, (dst, src, dim) in enumerate(buffers):
        shape, rank = dst.shape, dst.dim()
        if not dst.is_contiguous() or dst.get_device() != on:
            raise ValueError(f"buffer {k}: every buffer is contiguous and on {dev}")
        if src is not dst and not (dst.dtype is src.dtype and rank == src.dim() and src.is_contiguous() and src.get_device() == on):
            raise ValueError(f"buffer {k}: destination and source are contiguous tensors of one type and rank on {dev}")
        if shape[dim] != n or src.shape[dim] != m:
            raise ValueError(f"buffer {k}: {shape[dim]} and {src.shape[dim]} slots, the first has {n} and {m}")
        dim %= rank
        outer, inner = shape[:dim], shape[dim + 1:]
        if src is not dst and (outer != src.shape[:dim] or inner != src.shape[dim + 1:]):
            raise ValueError(f"buffer {k}: slots of {tuple(shape)} and {tuple(src.shape)} differ")
        row = table[k]
        row.dst, row.src = dst.data_ptr(), src.data_ptr()
        before = math.prod(outer)
        if before >> 31:
            raise ValueError(f"buffer {k}: {before} rows of slots before the slot dimension: a call carries numbers below 2^31")
        row.outer, row.slot_bytes = before, math.prod(inner) * dst.element_size()
    if not torch.is_tensor(origin):
        origin = [int(o) for o in origin]
        bad = [o for o in origin if not KEEP <= o < m]
        if bad or len(origin) != n:
            raise ValueError(f"origin: {len(origin)} entries for {n} slots, naming slots {bad} of {m}")
        ctx = ffi.context_on(on, ctx)
        with ctx.torch_stream():
            origin = torch.tensor(origin, dtype=torch.int32, device=dev)
    if origin.shape != (n,) or origin.dtype != torch.int32 or origin.get_device() != on or not origin.is_contiguous():
        raise ValueError(f"origin: expected int32 [{n}] on {dev}, got {origin.dtype} {tuple(origin.shape)} on {origin.device}")
    ctx = ffi.context_on(on, ctx)
    ctx.check(ctx._lib.bdh_copy_slots(ctx.handle, table, len(buffers), n, m, origin.data_ptr()))
