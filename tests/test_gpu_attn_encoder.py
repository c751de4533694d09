"""GPU: di_attn_encoder against the 64-bit form: types, head sizes, shared
heads, lengths, biases, layouts and strides, few and many rows, split keys."""
import numpy as np
import pytest

from attention_layer_ref import attention, check

pytestmark = pytest.mark.gpu

F16, F32 = np.float16, np.float32


class Case:
    """Tensors of a call in chosen layouts, and the call."""

    def __init__(self, dev, rng, B, Hq, Hk, Sq, Skv, d, dt, layout=0, stacked=False, std=1.0, shared=False):
        from drawinstant import attention as at
        self.at, self.dev, self.shape, self.dt, self.layout = at, dev, (B, Hq, Hk, Sq, Skv, d), dt, layout
        self.q = (std * rng.standard_normal((B, Hq, Sq, d))).astype(dt)
        kb = 1 if shared else B
        self.k = rng.standard_normal((kb, Hk, Skv, d)).astype(dt)
        self.v = rng.standard_normal((kb, Hk, Skv, d)).astype(dt)
        self.stacked, self.shared = stacked, shared

    def put(self, x):
        return self.dev.storage(x.transpose(0, 2, 1, 3) if self.layout == 0 else x)

    def run(self, lens=None, bias=None, scale=0.0, bias_strides=None, fill=7.0):
        at, dev = self.at, self.dev
        B, Hq, Hk, Sq, Skv, d = self.shape
        bufs = [self.put(self.q)]
        q = at.heads(bufs[0], Sq, Hq, d, self.layout)
        if self.stacked:
            row = 2 * Hk * d + 24  # a row longer than its heads
            kv = np.full((self.k.shape[0], Skv, row), np.nan, self.dt)
            for i, x in enumerate((self.k, self.v)):
                kv[:, :, i * Hk * d:(i + 1) * Hk * d] = x.transpose(0, 2, 1, 3).reshape(x.shape[0], Skv, -1)
            bufs.append(dev.storage(kv))
            bs = 0 if self.shared else Skv * row
            k = at.heads(bufs[1], Skv, Hk, d, token=row, batch=bs)
            v = at.heads(bufs[1], Skv, Hk, d, offset=Hk * d, token=row, batch=bs)
        else:
            bufs += [self.put(self.k), self.put(self.v)]
            kw = {"batch": 0} if self.shared else {}
            k, v = (at.heads(b, Skv, Hk, d, self.layout, **kw) for b in bufs[1:])
        out = np.full((B, Hq, Sq, d) if self.layout else (B, Sq, Hq, d), fill, self.dt)
        bufs.append(dev.storage(out))
        o = at.heads(bufs[-1], Sq, Hq, d, self.layout)
        lb = bb = bv = None
        if lens is not None:
            lb = dev.storage(np.asarray(lens, np.int32))
            bufs.append(lb)
        if bias is not None:
            bb = dev.storage(np.ascontiguousarray(bias, np.float32))
            bufs.append(bb)
            bv = at.Bias(bb, **bias_strides)
        at.attn_encoder(dev, q, k, v, o, B, Hq, Hk, Sq, Skv, d, kv_len=lb, bias=bv, scale=scale,
                        dtype=1 if self.dt == F16 else 0)
        got = dev.download(bufs[-1] if lb is None and bb is None else bufs[-1 - (lb is not None) - (bb is not None)],
                           self.dt, out.shape)
        for b in bufs:
            b.destroy()
        return got if self.layout else got.transpose(0, 2, 1, 3)

    def kv(self):
        B = self.shape[0]
        return (np.broadcast_to(x, (B,) + x.shape[1:]) for x in (self.k, self.v))


@pytest.mark.parametrize("dt", [F16, F32])
@pytest.mark.parametrize("d", [8, 32, 40, 64, 72, 96, 128, 136, 160, 192, 200, 256])
@pytest.mark.parametrize("Sq,Skv", [(1, 5), (37, 77), (130, 200)])
def test_head_sizes(dev, rng, dt, d, Sq, Skv):
    """Every instantiation, few and many rows, ragged tiles; rows of K and V
    longer than their heads, with NaN between them."""
    c = Case(dev, rng, 2, 3, 3, Sq, Skv, d, dt, stacked=True)
    k, v = c.kv()
    check(c.run(), *attention(c.q, k, v, dt=dt), f"d={d} {Sq}x{Skv} {dt.__name__}")


@pytest.mark.parametrize("dt", [F16, F32])
@pytest.mark.parametrize("Hq,Hk,Sq", [(8, 2, 1), (16, 1, 1), (17, 1, 1), (32, 1, 3), (6, 3, 50), (7, 1, 9), (64, 1, 1)])
@pytest.mark.parametrize("layout", [0, 1])
def test_shared_heads(dev, rng, dt, Hq, Hk, Sq, layout):
    c = Case(dev, rng, 2, Hq, Hk, Sq, 150, 64, dt, layout)
    k, v = c.kv()
    check(c.run(), *attention(c.q, k, v, dt=dt), f"heads {Hq}/{Hk} Sq={Sq}")


@pytest.mark.parametrize("dt", [F16, F32])
@pytest.mark.parametrize("Sq", [1, 33, 200])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_lengths(dev, rng, dt, Sq, d):
    """None, one, a tile's end and its neighbours, all, past the end and below
    zero; what lies behind a length is NaN and infinite."""
    Skv = 197
    lens = [0, 1, 16, 63, 64, 65, 128, 196, 197, 500, -3]
    c = Case(dev, rng, len(lens), 2, 1, Sq, Skv, d, dt)
    for b, n in enumerate(lens):
        n = min(max(n, 0), Skv)
        c.k[b, :, n:] = np.nan
        c.v[b, :, n:] = np.inf
    got = c.run(lens=lens)
    ok = np.array([min(max(n, 0), Skv) for n in lens])
    k, v = np.nan_to_num(c.k, nan=0.0), np.where(np.isinf(c.v), 0, c.v)
    check(got, *attention(c.q, k, v, ok, dt=dt), f"lengths Sq={Sq} d={d}")
    assert not got[0].any() and not got[-1].any()


@pytest.mark.parametrize("dt", [F16, F32])
@pytest.mark.parametrize("Sq", [1, 40, 150])
@pytest.mark.parametrize("kind", ["key", "query", "head"])
def test_bias(dev, rng, dt, Sq, kind):
    B, Hq, Hk, Skv, d = 2, 4, 2, 131, 64  # rows of 131 floats: four-byte alignment
    c = Case(dev, rng, B, Hq, Hk, Sq, Skv, d, dt)
    shape = {"key": (B, 1, 1, Skv), "query": (B, 1, Sq, Skv), "head": (1, Hq, Sq, Skv)}[kind]
    bias = rng.standard_normal(shape).astype(np.float32) * 3
    bias[rng.random(shape) < 0.4] = -np.inf
    bias[0, 0, 0, :70] = -np.inf        # a first tile with nothing in it
    bias[-1, -1, -1, :] = -np.inf       # a row with nothing at all
    st = {"key": dict(batch=Skv), "query": dict(batch=Sq * Skv, query=Skv),
          "head": dict(head=Sq * Skv, query=Skv)}[kind]
    k, v = c.kv()
    for lens in (None, [131, 90]):
        got = c.run(lens=lens, bias=bias, bias_strides=st)
        ref, bound = attention(c.q, k, v, lens, bias, dt=dt)
        check(got, ref, bound, f"bias by {kind} Sq={Sq} lens={lens}")
        gone = np.isneginf(np.broadcast_to(bias, (B, Hq, Sq, Skv))[..., :90 if lens else None]).all(-1)
        assert not got[1][gone[1]].any()


@pytest.mark.parametrize("dt", [F16, F32])
@pytest.mark.parametrize("Sq", [1, 70])
def test_removed_keys_hold_anything(dev, rng, dt, Sq):
    """NaN and infinities in keys that a bias removes for every query."""
    c = Case(dev, rng, 2, 2, 2, Sq, 100, 80, dt)
    bias = np.zeros((2, 1, 1, 100), np.float32)
    bias[0, ..., 3:50] = bias[1, ..., 90:] = -np.inf
    bias[1, ..., :64] = -np.inf
    k, v = (x.copy() for x in c.kv())
    gone = np.isneginf(bias[:, :, 0])
    for x, bad in ((c.k, np.nan), (c.v, np.nan)):
        x[np.broadcast_to(gone[..., None], x.shape)] = bad
    c.v[1, :, 5] = np.inf
    check(c.run(bias=bias, bias_strides=dict(batch=100)), *attention(c.q, k, v, None, bias, dt=dt), "removed keys")


@pytest.mark.parametrize("dt", [F16, F32])
@pytest.mark.parametrize("low", [np.finfo(np.float32).min, -1e30, -65504.0, -1e4])
def test_lowest_values(dev, rng, dt, low):
    """Finite lowest values: they lose to any other key, and a row of nothing
    else is the mean of its values (the score is swamped) or, where the value
    is small enough to leave it, the softmax of its scores."""
    B, H, Sq, Skv, d = 1, 2, 20, 150, 64
    c = Case(dev, rng, B, H, H, Sq, Skv, d, dt)
    bias = np.zeros((B, 1, Sq, Skv), np.float32)
    bias[:, :, :, :80] = low       # whole first tiles
    bias[:, :, 3] = low            # all of a row
    bias[:, :, 4, 0] = -np.inf
    bias[:, :, 4, 1:] = low
    k, v = c.kv()
    got = c.run(bias=bias, bias_strides=dict(batch=Sq * Skv, query=Skv))
    # (the bound's own 4 U32 |bias| is the rounding that a naive sum would
    # make; here the difference of two biases is exact, so it is left out)
    ref, bound = attention(c.q, k, v, None, bias, dt=dt)
    _, plain = attention(c.q, k, v, dt=dt)
    check(got, ref, np.minimum(bound, 40 * plain) if low > -1e30 else bound, f"lowest {low}")


@pytest.mark.parametrize("dt", [F16, F32])
@pytest.mark.parametrize("growth,Sq,Skv", [(6.0, 100, 600), (12.0, 1, 900), (4.0, 16, 4000)])
def test_rising_scores(dev, rng, dt, growth, Sq, Skv):
    """Scores that rise along the keys: the running maximum is raised on the way."""
    c = Case(dev, rng, 1, 2, 2, Sq, Skv, 64, dt, std=2.0)
    ramp = 1.0 + growth * np.arange(Skv) / Skv
    c.k = (c.k * ramp[None, None, :, None]).astype(dt)
    k, v = c.kv()
    check(c.run(), *attention(c.q, k, v, dt=dt), f"rising x{growth} {Sq}x{Skv}")


@pytest.mark.parametrize("dt", [F16, F32])
@pytest.mark.parametrize("B,H,Sq,Skv,d,lens", [
    (1, 1, 1, 6000, 64, None), (1, 2, 64, 5000, 128, None), (2, 1, 16, 7001, 40, [7001, 33]),
    (3, 1, 1, 4096, 256, [0, 4096, 1]), (1, 1, 300, 3000, 160, None)])
def test_split_keys(dev, rng, dt, B, H, Sq, Skv, d, lens):
    """Few rows over many keys: key ranges on several workgroups, some empty."""
    c = Case(dev, rng, B, H, H, Sq, Skv, d, dt)
    k, v = c.kv()
    check(c.run(lens=lens), *attention(c.q, k, v, lens, dt=dt), f"split {Sq}x{Skv} d={d}")


@pytest.mark.parametrize("dt", [F16, F32])
def test_one_sequence_for_the_batch(dev, rng, dt):
    """Encoder states that every entry reads (batch stride 0), and a scale."""
    c = Case(dev, rng, 3, 4, 4, 50, 77, 64, dt, stacked=True, shared=True)
    k, v = c.kv()
    check(c.run(scale=0.3, lens=[77, 5, 40]), *attention(c.q, k, v, [77, 5, 40], scale=0.3, dt=dt), "shared")


def test_rows_outside_stay(dev, rng):
    """An output in the middle of a longer sequence; the rest is left alone."""
    from drawinstant import attention as at
    B, H, Sq, Skv, d, total = 2, 3, 21, 30, 40, 50
    c = Case(dev, rng, B, H, H, Sq, Skv, d, F16, layout=1)
    bq, bk, bv = (dev.storage(x) for x in (c.q, c.k, c.v))
    o = dev.storage(np.full((B, total, H, d), 5.0, F16))
    at.attn_encoder(dev, *(at.heads(b, s, H, d, 1) for b, s in ((bq, Sq), (bk, Skv), (bv, Skv))),
                    at.heads(o, total, H, d, start=17), B, H, H, Sq, Skv, d)
    got = dev.download(o, F16, (B, total, H, d))
    assert (got[:, :17] == 5).all() and (got[:, 17 + Sq:] == 5).all()
    check(got[:, 17:17 + Sq].transpose(0, 2, 1, 3), *attention(c.q, c.k, c.v), "middle")
    for b in (bq, bk, bv, o):
        b.destroy()


def test_same_bits_again(dev, rng):
    """No atomics: the same call gives the same bits, split keys included."""
    c = Case(dev, rng, 2, 2, 2, 5, 5000, 64, F16)
    a, b = c.run(), c.run()
    assert np.array_equal(a, b)


def test_matches_cross_attention(dev, rng):
    """Beside di_attn_cross on a call that both take."""
    import drawinstant
    c = Case(dev, rng, 2, 5, 5, 300, 77, 64, F16)
    got = c.run().transpose(0, 2, 1, 3)
    bufs = [c.put(x) for x in (c.q, c.k, c.v)] + [dev.create_buffer(c.q.nbytes)]
    drawinstant.call("di_attn_cross", dev.ctx, *(b.handle for b in bufs), 2, 5, 300, 77, 64, 0, 0.0, 1)
    ref = dev.download(bufs[3], F16, got.shape)
    _, bound = attention(c.q, c.k, c.v)
    assert (np.abs(got.astype(np.float64) - ref) <= 2 * bound.transpose(0, 2, 1, 3)).all()
    for b in bufs:
        b.destroy()


@pytest.mark.parametrize("d,Skv,kind", [(32, 45, "bias"), (40, 77, "lens"), (64, 300, "bias"), (64, 33, "none"),
                                        (72, 200, "lens"), (96, 256, "none"), (128, 300, "lens"), (128, 193, "bias")])
def test_many_rows(dev, rng, d, Skv, kind):
    """Grids that fill the chip twice over: two row groups a wavefront, the
    last one ragged, heads shared by three queries each."""
    B, Hk, G, Sq = 4, 64, 3, 67  # two blocks of 128 rows, 512 workgroups
    c = Case(dev, rng, B, Hk * G, Hk, Sq, Skv, d, F16, stacked=True)
    lens = [Skv, 1, Skv - 30, 33] if kind == "lens" else None
    bias = None
    if kind == "bias":
        bias = rng.standard_normal((B, 1, Sq, Skv)).astype(np.float32)
        bias[rng.random(bias.shape) < 0.3] = -np.inf
        bias[:, :, 5] = -np.inf
    k, v = c.kv()
    got = c.run(lens=lens, bias=bias, bias_strides=dict(batch=Sq * Skv, query=Skv))
    check(got, *attention(c.q, k, v, lens, bias), f"many rows d={d} {kind}")


@pytest.mark.parametrize("dt", [F16, F32])
@pytest.mark.parametrize("B,Hk,G,Sq,Skv,d", [(2, 3, 1, 700, 150, 40), (3, 2, 2, 333, 97, 64), (1, 5, 1, 520, 300, 128)])
def test_one_bias_for_many_heads(dev, rng, dt, B, Hk, G, Sq, Skv, d):
    """Many blocks of rows under few heads, which then go side by side."""
    c = Case(dev, rng, B, Hk * G, Hk, Sq, Skv, d, dt)
    bias = rng.standard_normal((B, 1, Sq, Skv)).astype(np.float32)
    bias[:, :, 100:110, :60] = -np.inf
    bias[:, :, 3] = -np.inf
    bias[:, :, 200, 5:9] = -2e30
    lens = [Skv - 7 * i for i in range(B)]
    k, v = c.kv()
    got = c.run(lens=lens, bias=bias, bias_strides=dict(batch=Sq * Skv, query=Skv))
    check(got, *attention(c.q, k, v, lens, bias, dt=dt), f"one bias d={d}")
    assert not got[:, :, 3].any()
