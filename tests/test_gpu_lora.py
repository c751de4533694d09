"""GPU: di_linear_lora against the 64-bit form: types, every path of the
projection, ranks, runs of rows, ids in any order and out of range."""
import numpy as np
import pytest

from attention_layer_ref import check, lora

pytestmark = pytest.mark.gpu

F16, F32 = np.float16, np.float32


def run(dev, rng, M, N, K, R, n, run, dt=F16, act="none", res=False, bias=True, scale=True, ids=None, x=None):
    from drawinstant import lora as lo
    x = rng.standard_normal((M, K)).astype(dt) if x is None else x
    w = (rng.standard_normal((N, K)) / np.sqrt(K)).astype(dt)
    b = rng.standard_normal(N).astype(F32) if bias else None
    down = (rng.standard_normal((n, R, K)) / np.sqrt(K)).astype(dt)
    up = (rng.standard_normal((n, N, R)) / np.sqrt(R)).astype(dt)
    sc = rng.uniform(0.5, 2.0, n).astype(F32) if scale else None
    ids = rng.integers(-1, n + 1, -(-M // run)) if ids is None else np.asarray(ids)
    nout = N // 2 if act == "geglu" else N
    r = rng.standard_normal((M, nout)).astype(dt) if res else None
    put = lambda a: dev.storage(a) if a is not None else None  # noqa: E731
    bx, bw, bb, bd, bu, bs, br = map(put, (x, w, b, down, up, sc, r))
    bi, y = dev.storage(ids.astype(np.int32)), dev.create_buffer(M * nout * x.itemsize)
    lo.linear_lora(dev, bx, bw, bb, lo.Adapters(bd, bu, n, R, bs), bi, y, M, N, K, residual=br, rows_per_id=run,
                   act={"none": 0, "gelu": 1, "geglu": 2}[act], dtype=1 if dt == F16 else 0)
    got = dev.download(y, dt, (M, nout))
    for t in (bx, bw, bb, bd, bu, bs, br, bi, y):
        if t is not None:
            t.destroy()
    live = np.where((ids >= 0) & (ids < n), ids, -1)
    check(got, *lora(x, w, b, down, up, sc, live, run, act, r, dt), f"lora {M}x{N}x{K} R={R} n={n} run={run} {act}")
    return got


@pytest.mark.parametrize("dt", [F16, F32])
@pytest.mark.parametrize("M,N,K", [(1, 64, 64), (8, 1280, 320), (200, 320, 640), (77, 96, 1024), (513, 640, 128)])
@pytest.mark.parametrize("R,n,rows", [(16, 4, 1), (8, 3, 50), (64, 2, 77), (5, 5, 7)])
def test_paths(dev, rng, dt, M, N, K, R, n, rows):
    run(dev, rng, M, N, K, R, n, rows, dt)


@pytest.mark.parametrize("dt", [F16, F32])
@pytest.mark.parametrize("M,N,K", [(30, 37, 50), (65, 33, 129), (100, 8, 24), (3, 1, 7), (129, 130, 100)])
def test_odd_sizes(dev, rng, dt, M, N, K):
    """No whole vectors, no whole stages: the bounds-checked kernels."""
    run(dev, rng, M, N, K, 6, 3, 4, dt)
    run(dev, rng, M, N, K, 32, 3, 1, dt, res=True)


@pytest.mark.parametrize("dt", [F16, F32])
@pytest.mark.parametrize("R", [1, 2, 3, 4, 7, 8, 12, 16, 17, 33, 48, 65, 100, 128, 200, 256])
def test_ranks(dev, rng, dt, R):
    run(dev, rng, 90, 128, 192, R, 3, 20, dt)


@pytest.mark.parametrize("dt", [F16, F32])
@pytest.mark.parametrize("act", ["none", "gelu", "geglu"])
@pytest.mark.parametrize("M,N,K", [(150, 320, 320), (64, 96, 1280), (40, 64, 100)])
def test_epilogues(dev, rng, dt, act, M, N, K):
    run(dev, rng, M, N, K, 16, 3, 30, dt, act=act, res=True)
    run(dev, rng, M, N, K, 16, 3, 30, dt, act=act, bias=False, scale=False)


@pytest.mark.parametrize("dt", [F16, F32])
@pytest.mark.parametrize("ids", ["none", "out", "one", "each", "shuffled"])
def test_ids(dev, rng, dt, ids):
    """No adapter at all, ids past the stack, one for all, one per row, any order."""
    M, n = 140, 140
    v = {"none": np.full(M, -1), "out": np.full(M, n), "one": np.full(M, 9), "each": np.arange(M),
         "shuffled": rng.permutation(M)}[ids]
    run(dev, rng, M, 64, 128, 8, n, 1, dt, ids=v)


@pytest.mark.parametrize("tile", range(15))
def test_every_tile(dev, rng, monkeypatch, tile):
    """Each tile shape of the projection, with and without split k."""
    monkeypatch.setenv("DI_GEMM_TILE", str(tile))
    for splits in (1, 3):
        monkeypatch.setenv("DI_GEMM_SPLITS", str(splits))
        for dt in (F16, F32):
            run(dev, rng, 150, 192, 512, 24, 4, 40, dt)


@pytest.mark.parametrize("dt", [F16, F32])
def test_no_adapter_is_the_linear(dev, rng, dt):
    """Rows without an adapter are di_linear's: both within the bound of the
    product alone (the two may sum k in another order, so not bit for bit)."""
    import drawinstant
    M, N, K = 100, 320, 320
    x = rng.standard_normal((M, K)).astype(dt)
    w = (rng.standard_normal((N, K)) / np.sqrt(K)).astype(dt)
    from drawinstant import lora as lo
    bx, bw = dev.storage(x), dev.storage(w)
    down, up = (dev.storage(rng.standard_normal(s).astype(dt)) for s in ((2, 16, K), (2, N, 16)))
    ids = dev.storage(np.array([0, -1, 1, -1], np.int32))
    y, z = (dev.create_buffer(M * N * x.itemsize) for _ in range(2))
    code = 1 if dt == F16 else 0
    lo.linear_lora(dev, bx, bw, None, lo.Adapters(down, up, 2, 16), ids, y, M, N, K, rows_per_id=25, dtype=code)
    drawinstant.call("di_linear", dev.ctx, bx.handle, bw.handle, 0, 0, z.handle, M, N, K, 0, code)
    a, b = (dev.download(t, dt, (M, N)) for t in (y, z))
    ref, bound = lora(x, w, None, np.zeros((1, 16, K)), np.zeros((1, N, 16)), None, np.full(M, -1), 1, "none", None, dt)
    for rows in (slice(25, 50), slice(75, 100)):
        check(a[rows], ref[rows], bound[rows], "without an adapter")
        check(b[rows], ref[rows], bound[rows], "di_linear")
    assert not np.array_equal(a[:25], b[:25])
    for t in (bx, bw, down, up, ids, y, z):
        t.destroy()


@pytest.mark.parametrize("dt", [F16, F32])
def test_rows_that_are_not_finite(dev, rng, dt):
    """Rows of x that are infinite or NaN stay alone with it."""
    from drawinstant import lora as lo
    M, N, K, R, n = 64, 64, 128, 8, 3
    x = rng.standard_normal((M, K)).astype(dt)
    w = (rng.standard_normal((N, K)) / np.sqrt(K)).astype(dt)
    down = (rng.standard_normal((n, R, K)) / np.sqrt(K)).astype(dt)
    up = rng.standard_normal((n, N, R)).astype(dt)
    x[5] = np.inf
    x[6, 3] = np.nan
    ids = np.array([0, 1, 2, 0] * 16, np.int32)
    bufs = [dev.storage(a) for a in (x, w, down, up, ids)] + [dev.create_buffer(M * N * x.itemsize)]
    lo.linear_lora(dev, bufs[0], bufs[1], None, lo.Adapters(bufs[2], bufs[3], n, R), bufs[4], bufs[5], M, N, K,
                   dtype=1 if dt == F16 else 0)
    got = dev.download(bufs[5], dt, (M, N))
    rows = (np.arange(M) != 5) & (np.arange(M) != 6)
    sane = np.where(np.isfinite(x), x, 0)
    ref, bound = lora(sane, w, None, down, up, None, ids, 1, "none", None, dt)
    check(got[rows], ref[rows], bound[rows], "own rows")
    assert not np.isfinite(got[~rows]).any()
    for t in bufs:
        t.destroy()
