"""Plain 64-bit forms of the attention-layer operators and the error bounds of
their kernels, element by element, from the roundings that the kernels make."""
import math

import numpy as np

U16, U32 = 2.0 ** -11, 2.0 ** -24  # half a step of fp16 / fp32, relative
TINY16 = 2.0 ** -25                # half the smallest step of fp16


def unit(dt):
    return U16 if dt == np.float16 else U32


def attention(q, k, v, lens=None, bias=None, scale=None, dt=np.float16):
    """q [B][Hq][Sq][d], k / v [B][Hk][Skv][d], bias broadcastable to
    [B][Hq][Sq][Skv] -> (o, bound).  The values of removed keys are not looked at."""
    q, k, v = (np.asarray(a, np.float64) for a in (q, k, v))
    B, Hq, Sq, d = q.shape
    Hk, Skv = k.shape[1:3]
    scale = scale or 1.0 / math.sqrt(d)
    u = unit(dt)
    o, bound = np.zeros_like(q), np.zeros_like(q)
    for b in range(B):
        n = Skv if lens is None else min(max(int(lens[b]), 0), Skv)
        for h in range(Hq):
            kk, vv = k[b, h // (Hq // Hk), :n], v[b, h // (Hq // Hk), :n]
            bb = np.zeros((Sq, n)) if bias is None else \
                np.broadcast_to(bias, (B, Hq, Sq, Skv))[b, h, :, :n].astype(np.float64)
            gone = np.isneginf(bb)
            unseen = gone.all(0)
            kk, vv = np.where(unseen[:, None], 0.0, kk), np.where(unseen[:, None], 0.0, vv)
            s = np.where(gone, -np.inf, np.where(bb <= -1e30, 0.0, scale * q[b, h] @ kk.T) + bb)
            if n == 0:
                continue
            m = s.max(1, keepdims=True)
            m = np.where(np.isneginf(m), 0.0, m)
            e = np.exp(s - m)
            z = e.sum(1, keepdims=True)
            p = e / np.where(z == 0, 1.0, z)
            o[b, h] = p @ vv
            # a score is off by the rounding of scale * q (u), of the factor
            # scale * log2(e) (2 U32) and of d + 4 fp32 sums and products, a
            # bias by its own product; a probability by twice the worst of its
            # row's scores and by u (its own rounding, fp16) and U32's of exp2
            # and of n sums; fp16 probabilities below 2^-14 by an absolute TINY16
            mag = scale * np.abs(q[b, h]) @ np.abs(kk).T
            fine = np.where(gone | (bb <= -1e30), 0.0, np.abs(bb))
            ds = ((u + (d + 6) * U32) * mag + 4 * U32 * (fine + mag)).max(1, keepdims=True)
            a = p @ np.abs(vv)
            rel = np.expm1(2 * ds) + (u if dt == np.float16 else 0) + (2 * n + 16) * U32
            flush = n * TINY16 if dt == np.float16 else 0.0
            bound[b, h] = rel * a * 1.01 + flush * np.abs(vv).max(initial=0.0) + u * np.abs(o[b, h]) + 1e-30
            if dt == np.float16:
                bound[b, h] += TINY16
    return o, bound


def qk(x, gamma, pos, dims, theta, halves, one, norm, eps, dt):
    """x [B][S][H][d], pos [B or 1][S][axes] -> (y, bound)."""
    x = np.asarray(x, np.float64)
    d = x.shape[-1]
    if norm:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
        x = x * (1.0 if gamma is None else np.asarray(gamma, np.float64))
    half = sum(dims) // 2
    freq = np.array([theta[0] ** (-p / half) for p in range(half)]) if one else \
        np.concatenate([[theta[a] ** (-2.0 * i / n) for i in range(n // 2)] for a, n in enumerate(dims)] + [[]])
    axis = np.repeat(np.arange(len(dims)), [n // 2 for n in dims])
    y, bound = x.copy(), np.abs(x)
    if half:
        ang = np.asarray(pos, np.float64)[:, :, axis] * freq
        c, s = np.cos(ang)[:, :, None], np.sin(ang)[:, :, None]
        iu, iw = (np.arange(half), np.arange(half) + half) if halves else \
            (2 * np.arange(half), 2 * np.arange(half) + 1)
        y[..., iu] = x[..., iu] * c - x[..., iw] * s
        y[..., iw] = x[..., iw] * c + x[..., iu] * s
        bound[..., iu] = bound[..., iw] = np.abs(x[..., iu]) + np.abs(x[..., iw])
    # the mean of d squares (d + 2 roundings, halved by the root), the root,
    # its reciprocal, the two products with the value and gamma; cosine and
    # sine with 5 U32 each (argument, series), the turn's products and sum
    bound = ((d + 2) / 2 + 14) * U32 * bound + unit(dt) * np.abs(y) + (TINY16 if dt == np.float16 else 1e-38)
    return y, bound


def gelu(x):
    from math import erf
    return 0.5 * x * (1.0 + np.vectorize(erf, otypes=[np.float64])(x / math.sqrt(2.0)))


def lora(x, w, b, down, up, scale, ids, run, act, res, dt):
    """-> (y, bound)."""
    x, w, down, up = (np.asarray(a, np.float64) for a in (x, w, down, up))
    M, K = x.shape
    n, R = down.shape[:2]
    u = unit(dt)
    y = x @ w.T + (0.0 if b is None else b)
    # K + R sums; fp32 products from split parts (3 U32 more each)
    err = (K + R + 8) * U32 * (np.abs(x) @ np.abs(w).T + (0.0 if b is None else np.abs(b)))
    row = np.asarray(ids)[np.arange(M) // run]
    for a in range(n):
        m = row == a
        t = (1.0 if scale is None else float(scale[a])) * (x[m] @ down[a].T)
        y[m] += t @ up[a].T
        # t: K sums and its rounding to the type
        dt_ = (K + 4) * U32 * (1.0 if scale is None else abs(float(scale[a]))) * (np.abs(x[m]) @ np.abs(down[a]).T)
        dt_ = dt_ + u * np.abs(t) + (TINY16 if dt == np.float16 else 0.0)
        err[m] += dt_ @ np.abs(up[a]).T + (K + R + 8) * U32 * (np.abs(t) @ np.abs(up[a]).T)
    # |gelu'| < 1.13; the kernel's erf is off by 1.5e-7, its exponential and
    # reciprocal by a few U32
    gerr = lambda v, e: 1.13 * e + np.abs(v) * (1.5e-7 + 8 * U32)  # noqa: E731
    if act == "gelu":
        y, err = gelu(y), gerr(y, err)
    if act == "geglu":
        y, err = y.reshape(M, -1, 2, 16), err.reshape(M, -1, 2, 16)
        h, g, eh, eg = y[:, :, 0], y[:, :, 1], err[:, :, 0], err[:, :, 1]
        y = (h * gelu(g)).reshape(M, -1)
        err = (eh * (np.abs(gelu(g)) + gerr(g, eg)) + np.abs(h) * gerr(g, eg)).reshape(M, -1)
        err = err + 2 * U32 * np.abs(y)
    if res is not None:
        y = y + np.asarray(res, np.float64)
        err = err + U32 * np.abs(y)
    return y, err + u * (np.abs(y) + err) + (TINY16 if dt == np.float16 else 0.0)


def check(got, ref, bound, what=""):
    got = np.asarray(got, np.float64)
    assert got.shape == ref.shape, (got.shape, ref.shape)
    assert np.isfinite(got).all(), f"{what}: {np.count_nonzero(~np.isfinite(got))} values are not finite"
    off = np.abs(got - ref)
    off = np.where(off == 0, 0.0, off / np.where(bound == 0, 1e-300, bound))
    at = np.unravel_index(np.argmax(off), off.shape)
    print(f"[{what}] worst error {off[at]:.3f} of its bound, rel-L2 "
          f"{np.linalg.norm(got - ref) / max(np.linalg.norm(ref), 1e-30):.2e}", flush=True)
    assert off[at] <= 1.0, f"{what}: {got[at]} for {ref[at]} at {at}, bound {bound[at]}"
