"""Head norms with rotary positions, and attention to an encoder's states.

Entry points of libdrawinstant_hip beside ``di_attn_self`` / ``di_attn_cross``
(reference kernel WGSL_FUSED, fused-cross-attn.js:112-173) for denoising
transformers: ``qk_norm_rope`` (di_qk_norm_rope) and ``attn_encoder``
(di_attn_encoder).  Both take the heads of a tensor as views of a buffer
(``heads``), so the parts of a stacked projection, either attention layout and
a run of tokens in a longer sequence need no copies.
"""
from __future__ import annotations

import ctypes

from .device import BHSD, BSHD, F16, Buffer, Device, call  # noqa: F401

NORM_NONE, NORM_RMS = 0, 1
_ROPE_HALVES, _ROPE_ONE_SPECTRUM = 1, 2


class Heads(ctypes.Structure):
    """di_heads: heads [B][S][H][d] in a buffer, strides in elements."""
    _fields_ = [(n, ctypes.c_uint64) for n in ("buf", "offset", "token", "head", "batch")]


class Bias(ctypes.Structure):
    """di_attn_bias: an additive fp32 score bias [b][h][query][key], strides in
    elements, 0 to broadcast; -inf removes a key."""
    _fields_ = [(n, ctypes.c_uint64) for n in ("buf", "offset", "batch", "head", "query")]

    def __init__(self, buf: Buffer, *, offset: int = 0, batch: int = 0, head: int = 0, query: int = 0):
        super().__init__(buf.handle, offset, batch, head, query)


class Rope(ctypes.Structure):
    """di_rope: ``dims[a]`` channels of each head turn with axis ``a`` of the
    positions (all of them even); ``theta`` is one base or one per axis.

    ``halves`` pairs channel p with p + r/2 of the r rotated ones, else 2p with
    2p + 1; with ``one_spectrum`` the frequencies run on over the axes, else
    each axis starts its own.  ``pos_batch``: elements between the positions of
    two batch entries (0: one set for all)."""
    _fields_ = [("axes", ctypes.c_uint32), ("dim", ctypes.c_uint32 * 4),
                ("theta", ctypes.c_float * 4), ("flags", ctypes.c_uint32),
                ("pos_batch", ctypes.c_uint64)]

    def __init__(self, dims=(), theta=10000.0, *, halves: bool = False, one_spectrum: bool = False,
                 pos_batch: int = 0):
        dims = list(dims)
        if len(dims) > 4:
            raise ValueError(f"{len(dims)} axes (at most 4)")
        base = list(theta) if hasattr(theta, "__len__") else [theta] * len(dims)
        if len(base) != len(dims):
            raise ValueError(f"{len(base)} bases for {len(dims)} axes")
        super().__init__(len(dims), (ctypes.c_uint32 * 4)(*dims), (ctypes.c_float * 4)(*base),
                         (_ROPE_HALVES if halves else 0) | (_ROPE_ONE_SPECTRUM if one_spectrum else 0),
                         pos_batch)


def heads(buf: Buffer, S: int, H: int, d: int, layout: int = BSHD, *, offset: int = 0, start: int = 0,
          token: int | None = None, head: int | None = None, batch: int | None = None) -> Heads:
    """The view of ``H`` heads of ``d`` channels over a buffer of ``S`` tokens
    per batch entry, from token ``start`` on; any stride may be given instead
    (a stacked projection's row as ``token``, 0 as ``batch`` for one sequence
    that every entry reads)."""
    t, h, b = (H * d, d, S * H * d) if layout == BSHD else (d, S * d, H * S * d)
    t = t if token is None else token
    return Heads(buf.handle, offset + start * t, t, h if head is None else head,
                 b if batch is None else batch)


def qk_norm_rope(dev: Device, q: Heads, k: Heads | None, q_out: Heads, k_out: Heads | None,
                 pos: Buffer | None, rope: Rope, B: int, S: int, Hq: int, Hk: int, d: int, *,
                 q_gamma: Buffer | None = None, k_gamma: Buffer | None = None,
                 norm: int = NORM_RMS, eps: float = 1e-6, dtype: int = F16):
    """Norm of each head (``NORM_RMS`` with optional fp32 gammas, or
    ``NORM_NONE``) and its rotation by fp32 positions [S][axes], in one pass;
    ``q`` alone with ``k = k_out = None`` and ``Hk = 0``."""
    call("di_qk_norm_rope", dev.ctx, ctypes.byref(q), ctypes.byref(k) if k is not None else None,
         ctypes.byref(q_out), ctypes.byref(k_out) if k_out is not None else None,
         q_gamma.handle if q_gamma is not None else 0, k_gamma.handle if k_gamma is not None else 0,
         pos.handle if pos is not None else 0, ctypes.byref(rope), B, S, Hq, Hk, d, norm, eps, dtype)


def attn_encoder(dev: Device, q: Heads, k: Heads, v: Heads, o: Heads, B: int, Hq: int, Hk: int,
                 Sq: int, Skv: int, d: int, *, kv_len: Buffer | None = None,
                 bias: Bias | None = None, scale: float = 0.0, dtype: int = F16):
    """softmax(scale q k^T + bias) v over the first ``kv_len[b]`` (int32 [B])
    of ``Skv`` keys; ``scale <= 0`` selects 1/sqrt(d)."""
    call("di_attn_encoder", dev.ctx, ctypes.byref(q), ctypes.byref(k), ctypes.byref(v),
         ctypes.byref(o), kv_len.handle if kv_len is not None else 0,
         ctypes.byref(bias) if bias is not None else None, B, Hq, Hk, Sq, Skv, d, scale, dtype)
