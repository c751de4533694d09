"""Low-rank adapters of many requests beside a shared projection
(di_linear_lora): the projection of di_linear (reference hooks of
fused-block.js WGSL_MATMUL :54-115) with an adapter per run of rows.
"""
from __future__ import annotations

import ctypes

from .device import F16, Buffer, Device, call

ACT_NONE, ACT_GELU, ACT_GEGLU, ACT_SILU, ACT_GELU_TANH = range(5)


class _Lora(ctypes.Structure):
    """di_lora."""
    _fields_ = [(n, ctypes.c_uint64) for n in ("down", "up", "scale", "ids")] + \
               [(n, ctypes.c_uint32) for n in ("n", "rank", "rows_per_id")]


class Adapters:
    """A stack of ``n`` adapters of one rank: ``down`` [n][rank][K] and ``up``
    [n][N][rank] in the projection's dtype (smaller ranks padded with zeros),
    ``scale`` fp32 [n] or None for ones."""

    def __init__(self, down: Buffer, up: Buffer, n: int, rank: int, scale: Buffer | None = None):
        self.down, self.up, self.scale, self.n, self.rank = down, up, scale, n, rank


def linear_lora(dev: Device, x: Buffer, w: Buffer, bias: Buffer | None, adapters: Adapters,
                ids: Buffer, y: Buffer, M: int, N: int, K: int, *, residual: Buffer | None = None,
                rows_per_id: int = 1, act: int = ACT_NONE, dtype: int = F16):
    """y = act(x w^T + bias + scale[a] (x down[a]^T) up[a]^T) + residual with
    a = ids[m // rows_per_id] (int32; outside [0, n): no adapter) for row m."""
    a = _Lora(adapters.down.handle, adapters.up.handle,
              adapters.scale.handle if adapters.scale is not None else 0, ids.handle, adapters.n,
              adapters.rank, rows_per_id)
    call("di_linear_lora", dev.ctx, x.handle, w.handle, bias.handle if bias is not None else 0,
         ctypes.byref(a), residual.handle if residual is not None else 0, y.handle, M, N, K, act,
         dtype)
