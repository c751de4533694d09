"""GPU: di_qk_norm_rope against the 64-bit form: axes, pairings, spectra, head
sizes and alignments, layouts, far positions, in place."""
import numpy as np
import pytest

from attention_layer_ref import check, qk

pytestmark = pytest.mark.gpu

F16, F32 = np.float16, np.float32


def run(dev, rng, B, S, Hq, Hk, d, dims, dt=F16, theta=10000.0, halves=False, one=False, norm=1, gammas=True,
        stacked=False, layout=0, start=0, tail=0, pos=None, per_batch=False, in_place=False, pad=0, std=1.0):
    from drawinstant import attention as at
    H = Hq + 2 * Hk if stacked else Hq + Hk
    row = H * d + pad
    x = np.full((B, S, row), 3.0, dt)
    x[:, :, :H * d] = (std * rng.standard_normal((B, S, H * d))).astype(dt)
    xq = x[:, :, :Hq * d].reshape(B, S, Hq, d)
    xk = x[:, :, Hq * d:(Hq + Hk) * d].reshape(B, S, Hk, d)
    g = [(1 + 0.3 * rng.standard_normal(d)).astype(F32) if gammas and norm else None for _ in range(2)]
    if pos is None:
        pos = rng.integers(0, 100, (B if per_batch else 1, S, max(1, len(dims)))).astype(F32)
    bx, bp = dev.storage(x), dev.storage(pos)
    bg = [dev.storage(a) if a is not None else None for a in g]
    rope = at.Rope(dims, theta, halves=halves, one_spectrum=one, pos_batch=S * len(dims) if per_batch else 0)
    q = at.heads(bx, S, Hq, d, token=row, batch=S * row)
    k = at.heads(bx, S, Hk, d, offset=Hq * d, token=row, batch=S * row) if Hk else None
    if in_place:
        qo, ko, outs = q, k, []
    else:
        total = start + S + tail
        outs = [dev.storage(np.full((B, total, h, d) if layout == 0 else (B, h, total, d), 9.0, dt))
                for h in (Hq, Hk)[:2 if Hk else 1]]
        qo = at.heads(outs[0], total, Hq, d, layout, start=start)
        ko = at.heads(outs[1], total, Hk, d, layout, start=start) if Hk else None
    at.qk_norm_rope(dev, q, k, qo, ko, bp, rope, B, S, Hq, Hk, d, q_gamma=bg[0], k_gamma=bg[1] if Hk else None,
                    norm=norm, eps=1e-6, dtype=1 if dt == F16 else 0)
    th = [theta] * len(dims) if np.isscalar(theta) else theta
    for i, (src, h) in enumerate(((xq, Hq), (xk, Hk))[:2 if Hk else 1]):
        y, bound = qk(src, g[i], pos, dims, th, halves, one, norm, 1e-6, dt)
        if in_place:
            got = dev.download(bx, dt, x.shape)
            rest = got[:, :, (Hq + Hk) * d:]
            assert np.array_equal(rest, x[:, :, (Hq + Hk) * d:])
            got = got[:, :, :Hq * d] if i == 0 else got[:, :, Hq * d:(Hq + Hk) * d]
            got = got.reshape(B, S, h, d)
        else:
            got = dev.download(outs[i], dt, (B, total, h, d) if layout == 0 else (B, h, total, d))
            got = got if layout == 0 else got.transpose(0, 2, 1, 3)
            assert (got[:, :start] == 9).all() and (got[:, start + S:] == 9).all()
            got = got[:, start:start + S]
        check(got, y, bound, f"{'qk'[i]} B={B} S={S} H={h} d={d} dims={dims}")
    for b in [bx, bp] + outs + [b for b in bg if b is not None]:
        b.destroy()


@pytest.mark.parametrize("dt", [F16, F32])
@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("one", [False, True])
@pytest.mark.parametrize("d,dims", [(64, [32, 32]), (128, [44, 42, 42]), (80, [16, 24, 24]), (40, [40]), (256, [64, 192]),
                                    (16, [2, 0, 4, 10]), (72, [24, 24, 24]), (2, [2]), (8, [6])])
def test_axes(dev, rng, dt, halves, one, d, dims):
    run(dev, rng, 2, 19, 3, 2, d, dims, dt, halves=halves, one=one)


@pytest.mark.parametrize("dt", [F16, F32])
@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("d,dims", [(18, [8, 6]), (33, [32]), (50, [50]), (254, [100, 154]), (127, [10, 20, 30, 40]), (1, [])])
def test_odd_heads(dev, rng, dt, halves, d, dims):
    """Heads that are no whole vectors."""
    run(dev, rng, 1, 33, 2, 1, d, dims, dt, halves=halves, pad=3)


@pytest.mark.parametrize("dt", [F16, F32])
@pytest.mark.parametrize("layout", [0, 1])
@pytest.mark.parametrize("stacked,start,tail", [(True, 0, 0), (True, 77, 5), (False, 3, 0)])
def test_layouts(dev, rng, dt, layout, stacked, start, tail):
    run(dev, rng, 3, 50, 8, 2, 64, [16, 24, 24], dt, stacked=stacked, layout=layout, start=start, tail=tail)


@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("d,pad", [(64, 0), (64, 5), (20, 0)])
def test_in_place(dev, rng, halves, d, pad):
    run(dev, rng, 2, 40, 4, 4, d, [d // 2, 4], F16, halves=halves, stacked=True, in_place=True, pad=pad)


@pytest.mark.parametrize("dt", [F16, F32])
@pytest.mark.parametrize("far", [0.0, 1e3, 1e6, 1.6e7, -5e5])
def test_far_positions(dev, rng, dt, far):
    """Positions past where an fp32 angle still says anything; negative and
    fractional ones."""
    pos = (far + rng.integers(0, 8, (2, 30, 2))).astype(F32)
    pos[:, 10:] += F32(0.25) if abs(far) < 1e6 else 0
    run(dev, rng, 2, 30, 3, 3, 64, [24, 40], dt, theta=[10000.0, 500.0], pos=pos, per_batch=True)


@pytest.mark.parametrize("dt", [F16, F32])
@pytest.mark.parametrize("norm,gammas", [(0, False), (1, False), (1, True)])
def test_norms(dev, rng, dt, norm, gammas):
    run(dev, rng, 2, 30, 3, 1, 96, [32, 32, 32], dt, norm=norm, gammas=gammas, std=20.0)
    run(dev, rng, 2, 30, 3, 1, 96, [], dt, norm=norm, gammas=gammas)


def test_queries_alone(dev, rng):
    run(dev, rng, 2, 64, 7, 0, 64, [32, 32])


@pytest.mark.parametrize("B,S", [(1, 1), (1, 5000), (70, 1)])
def test_lengths(dev, rng, B, S):
    run(dev, rng, B, S, 2, 1, 128, [128], F16)


def test_small_values(dev, rng):
    """Heads of zeros and of subnormals: eps keeps the norm finite."""
    from drawinstant import attention as at
    x = np.zeros((1, 4, 1, 64), F32)
    x[0, 1] = 1e-30
    x[0, 2] = 1e-3
    x[0, 3] = 1e15
    b, p, o = dev.storage(x), dev.storage(np.zeros((4, 1), F32)), dev.create_buffer(x.nbytes)
    at.qk_norm_rope(dev, at.heads(b, 4, 1, 64), None, at.heads(o, 4, 1, 64), None, p, at.Rope([64]), 1, 4, 1, 0, 64,
                    dtype=0)
    got = dev.download(o, F32, x.shape)
    y, bound = qk(x, None, np.zeros((1, 4, 1)), [64], [1e4], False, False, 1, 1e-6, F32)
    check(got, y, bound, "small")
    for t in (b, p, o):
        t.destroy()


@pytest.mark.parametrize("halves", [False, True])
def test_infinite_channels_that_do_not_turn(dev, rng, halves):
    """Without a norm the channels past the rotated ones pass whatever they hold."""
    from drawinstant import attention as at
    x = rng.standard_normal((1, 6, 2, 24)).astype(F32)
    x[0, :, 0, 20] = np.inf
    x[0, 1, 1, 17:] = np.nan
    b, p, o = dev.storage(x), dev.storage(np.arange(6, dtype=F32)), dev.create_buffer(x.nbytes)
    at.qk_norm_rope(dev, at.heads(b, 6, 2, 24), None, at.heads(o, 6, 2, 24), None, p, at.Rope([16], halves=halves),
                    1, 6, 2, 0, 24, norm=at.NORM_NONE, dtype=0)
    got = dev.download(o, F32, x.shape)
    assert np.array_equal(got[..., 16:], x[..., 16:], equal_nan=True)
    y, bound = qk(x[..., :16], None, np.arange(6).reshape(1, 6, 1), [16], [1e4], halves, False, 0, 0, F32)
    check(got[..., :16], y, bound, "rotated part")
    for t in (b, p, o):
        t.destroy()
