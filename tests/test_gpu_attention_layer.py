"""GPU: attention to an encoder's states as a layer runs it: projections with
an adapter per request, head norms with rotation, attention over each request's
own states, and the projection back, every step against its 64-bit form on the
values that it was given; two contexts in turn; strides past 32 bits."""
import numpy as np
import pytest

from attention_layer_ref import attention, check, lora, qk

pytestmark = pytest.mark.gpu

F16, F32 = np.float16, np.float32


class Layer:
    """Weights, adapters and inputs of one layer, and its buffers on a device."""

    def __init__(self, rng, dt, B, S, L, Hq, Hk, d, Cx, Cs, R=8, n=3):
        self.dims = B, S, L, Hq, Hk, d, Cx, Cs, R, n
        self.dt = dt
        nrm = lambda *s: rng.standard_normal(s)  # noqa: E731
        self.x, self.states = nrm(B * S, Cx).astype(dt), nrm(B * L, Cs).astype(dt)
        self.rope = [d // 4 * 2, d // 8 * 2]
        self.pos = {"x": rng.integers(0, 50, (1, S, 2)).astype(F32), "s": rng.integers(0, 50, (1, L, 2)).astype(F32)}
        self.ids = np.array([i % (n + 1) - 1 for i in range(B)], np.int32)  # the first without one
        self.lens = np.array([L, 1, 0, L - 3][:B], np.int32)
        self.bias = nrm(B, 1, 1, L).astype(F32)
        self.bias[rng.random(self.bias.shape) < 0.2] = -np.inf
        self.gam = [(1 + 0.2 * nrm(d)).astype(F32) for _ in range(2)]
        self.w = {}
        for name, N, K in (("q", Hq * d, Cx), ("kv", 2 * Hk * d, Cs), ("o", Cx, Hq * d)):
            self.w[name] = ((nrm(N, K) / np.sqrt(K)).astype(dt), nrm(N).astype(F32),
                            (nrm(n, R, K) / np.sqrt(K)).astype(dt), (nrm(n, N, R) / np.sqrt(R)).astype(dt),
                            rng.uniform(0.5, 1.5, n).astype(F32))

    def put(self, dev):
        B, S, L, Hq, Hk, d, Cx, Cs, R, n = self.dims
        es = self.x.itemsize
        b = {k: dev.storage(getattr(self, k)) for k in ("x", "states", "ids", "lens", "bias")}
        b.update(px=dev.storage(self.pos["x"]), ps=dev.storage(self.pos["s"]), gq=dev.storage(self.gam[0]),
                 gk=dev.storage(self.gam[1]), q=dev.create_buffer(B * S * Hq * d * es),
                 kv=dev.create_buffer(B * L * 2 * Hk * d * es), qr=dev.create_buffer(B * S * Hq * d * es),
                 kr=dev.create_buffer(B * L * Hk * d * es), att=dev.create_buffer(B * S * Hq * d * es),
                 y=dev.create_buffer(B * S * Cx * es))
        for name, w in self.w.items():
            b[name + "_w"] = [dev.storage(a) for a in w]
        return b

    def run(self, dev, b):
        from drawinstant import attention as at, lora as lo
        B, S, L, Hq, Hk, d, Cx, Cs, R, n = self.dims
        dtype = 1 if self.dt == F16 else 0

        def project(name, x, y, rows, res=None):
            w, bias, down, up, sc = b[name + "_w"]
            N, K = self.w[name][0].shape
            lo.linear_lora(dev, x, w, bias, lo.Adapters(down, up, n, R, sc), b["ids"], y, B * rows, N, K,
                           residual=res, rows_per_id=rows, dtype=dtype)
        project("q", b["x"], b["q"], S)
        project("kv", b["states"], b["kv"], L)
        row = 2 * Hk * d
        rope = at.Rope(self.rope)
        keys = at.heads(b["kv"], L, Hk, d, token=row, batch=L * row)
        vals = at.heads(b["kv"], L, Hk, d, offset=Hk * d, token=row, batch=L * row)
        hq, hqr = at.heads(b["q"], S, Hq, d), at.heads(b["qr"], S, Hq, d, at.BHSD)
        hkr = at.heads(b["kr"], L, Hk, d, at.BHSD)
        at.qk_norm_rope(dev, hq, None, hqr, None, b["px"], rope, B, S, Hq, 0, d, q_gamma=b["gq"], dtype=dtype)
        at.qk_norm_rope(dev, keys, None, hkr, None, b["ps"], rope, B, L, Hk, 0, d, q_gamma=b["gk"], dtype=dtype)
        at.attn_encoder(dev, hqr, hkr, vals, at.heads(b["att"], S, Hq, d), B, Hq, Hk, S, L, d, kv_len=b["lens"],
                        bias=at.Bias(b["bias"], batch=L), dtype=dtype)
        project("o", b["att"], b["y"], S, b["x"])

    def check(self, dev, b):
        B, S, L, Hq, Hk, d, Cx, Cs, R, n = self.dims
        dt = self.dt
        get = lambda k, *s: dev.download(b[k], dt, s)  # noqa: E731
        q, kv, att = get("q", B, S, Hq, d), get("kv", B, L, 2, Hk, d), get("att", B, S, Hq, d)
        qr, kr = get("qr", B, Hq, S, d), get("kr", B, Hk, L, d)
        ref = lambda name, x, rows, res=None: lora(x, *self.w[name], self.ids, rows, "none", res, dt)  # noqa: E731
        check(q.reshape(B * S, -1), *ref("q", self.x, S), "q")
        check(kv.reshape(B * L, -1), *ref("kv", self.states, L), "kv")
        for got, x, g, p in ((qr, q, 0, "x"), (kr, kv[:, :, 0], 1, "s")):
            y, bound = qk(x, self.gam[g], self.pos[p], self.rope, [1e4, 1e4], False, False, 1, 1e-6, dt)
            check(got.transpose(0, 2, 1, 3), y, bound, "norm, rotation")
        o, bound = attention(qr, kr, kv[:, :, 1].transpose(0, 2, 1, 3), self.lens, self.bias, dt=dt)
        check(att.transpose(0, 2, 1, 3), o, bound, "attention")
        assert not att[self.lens == 0].any()
        check(get("y", B * S, Cx), *ref("o", att.reshape(B * S, -1), S, self.x), "y")


def drop(b):
    for x in b.values():
        for t in x if isinstance(x, list) else [x]:
            t.destroy()


SHAPES = [(1, 1, 77, 8, 8, 64, 320, 64), (3, 1, 9, 8, 2, 40, 72, 48), (4, 50, 77, 10, 10, 64, 640, 128),
          (2, 301, 33, 6, 3, 80, 200, 104)]


@pytest.mark.parametrize("dt", [F16, F32])
@pytest.mark.parametrize("shape", SHAPES)
def test_layer(dev, rng, dt, shape):
    """Twice over on the same buffers, nothing waited for in between."""
    t = Layer(rng, dt, *shape)
    b = t.put(dev)
    t.run(dev, b)
    t.run(dev, b)
    t.check(dev, b)
    first = dev.download(b["y"], dt)
    t.run(dev, b)
    assert np.array_equal(first, dev.download(b["y"], dt))
    drop(b)


def test_two_contexts(dev, rng):
    """Two contexts' streams and workspaces side by side: each gets its own
    layer's results, the bits of a run alone."""
    import drawinstant
    other = drawinstant.Device(0)
    layers = [Layer(rng, F16, *SHAPES[2]), Layer(rng, F16, *SHAPES[3])]
    devs = [dev, other]
    bufs = [t.put(d) for t, d in zip(layers, devs)]
    alone = []
    for t, d, b in zip(layers, devs, bufs):
        t.run(d, b)
        t.check(d, b)
        alone.append(d.download(b["y"], F16))
    for _ in range(5):
        for t, d, b in zip(layers, devs, bufs):
            t.run(d, b)
    for d, b, y in zip(devs, bufs, alone):
        assert np.array_equal(d.download(b["y"], F16), y)
    for b in bufs:
        drop(b)
    other.sync()
    other.destroy()


FAR = 2 ** 31 + 64  # elements between two batch entries (heads): past 32 bits in bytes and elements


def far_put(dev, x):
    """x [2][...] in a buffer with FAR elements between its two parts."""
    b = dev.create_buffer((FAR + x[1].size) * x.itemsize)
    for i in range(2):
        dev.upload(b, np.ascontiguousarray(x[i]), offset=i * FAR * x.itemsize)
    return b


@pytest.mark.parametrize("axis", ["batch", "head"])
@pytest.mark.parametrize("Sq", [1, 100])
def test_far_views(dev, rng, axis, Sq):
    """Batch entries (heads) of a cache 4 GiB apart, read, rotated and attended to in place."""
    from drawinstant import attention as at
    Skv, d, dims = 70, 64, [32]
    B, H = (2, 1) if axis == "batch" else (1, 2)
    x = [rng.standard_normal((2, s, d)).astype(F16) for s in (Sq, Skv, Skv)]
    bufs = [far_put(dev, a) for a in x]
    bufs.append(far_put(dev, np.zeros((2, Sq, d), F16)))
    view = lambda b: at.heads(b, 0, H, d, token=d, head=FAR, batch=FAR if B == 2 else 0)  # noqa: E731
    hq, hk, hv, ho = (view(b) for b in bufs)
    pos = rng.integers(0, 50, (1, Skv, 1)).astype(F32)
    bp = dev.storage(pos)
    at.qk_norm_rope(dev, hk, None, hk, None, bp, at.Rope(dims), B, Skv, H, 0, d)
    at.attn_encoder(dev, hq, hk, hv, ho, B, H, H, Sq, Skv, d)
    got = [np.stack([dev.download(b, F16, (s, d), offset=i * FAR * 2) for i in range(2)])
           for b, s in ((bufs[1], Skv), (bufs[3], Sq))]
    y, bound = qk(x[1][:, :, None], None, np.repeat(pos, 2, 0), dims, [1e4], False, False, 1, 1e-6, F16)
    check(got[0][:, :, None], y, bound, "far keys")
    ref, bound = attention(x[0][:, None], got[0][:, None], x[2][:, None])
    check(got[1][:, None], ref, bound, "far attention")
    for b in bufs + [bp]:
        b.destroy()
