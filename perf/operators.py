"""Attention-layer operators as measurable cases: what a denoising transformer
asks of the library around its attention.

=====  =====================================================================
lora   a shared projection with the low-rank adapters of many requests beside
       it: ``act(x W^T + b + s_a (x A_a^T) B_a^T) + r``, the adapter ``a``
       taken by runs of rows (none where the id is outside the stack)
qk     RMS norm of each query and key head and the rotation of its channel
       pairs by positions of several axes, in one pass
enc    attention of image tokens to an encoder's states: lengths per image,
       additive biases, query heads that share key heads, any head size
=====  =====================================================================

``run`` computes the operators from elementary torch operations; with ``own``
set it makes the library's calls.
"""
import math
import os
import sys

import torch

own = False

INF = float("inf")


def listed():
    return [
        # one pooled token per request, each with an adapter of its own: the
        # smallest projection, where launches and latency count
        {"name": "lora_f16_tokens", "kind": "lora", "f16": True, "M": 8, "N": 1280, "K": 1280,
         "rank": 16, "n": 8, "run": 1, "act": "none", "res": False},
        # an attention's output projection at the second level, four images,
        # one of them without an adapter
        {"name": "lora_f16_out_640", "kind": "lora", "f16": True, "M": 4096, "N": 640, "K": 640,
         "rank": 32, "n": 3, "run": 1024, "act": "none", "res": True},
        # the gated feed-forward's first projection at the first level, eight
        # images with an adapter each
        {"name": "lora_f16_geglu_320", "kind": "lora", "f16": True, "M": 32768, "N": 2560, "K": 320,
         "rank": 64, "n": 8, "run": 4096, "act": "geglu", "res": False},
        # keys and values of eight prompts of 77 tokens in fp32, a rank that
        # is no multiple of a vector
        {"name": "lora_f32_prompts", "kind": "lora", "f16": False, "M": 616, "N": 1280, "K": 1024,
         "rank": 12, "n": 5, "run": 77, "act": "none", "res": False},
        # a guided pair of 16 x 16 latents, queries and keys in the stacked
        # projection: the smallest pass
        {"name": "qk_f16_16x16", "kind": "qk", "f16": True, "B": 2, "T": 1, "H": 16, "W": 16,
         "Hq": 20, "Hk": 20, "d": 64, "dims": "32,32", "halves": False, "one": False,
         "stacked": True, "bhsd": False, "start": 0, "tail": 0, "far": 0},
        # a video clip: 13 x 30 x 52 latent positions, three axes, written in
        # the head-major layout of an attention
        {"name": "qk_f16_video", "kind": "qk", "f16": True, "B": 1, "T": 13, "H": 30, "W": 52,
         "Hq": 12, "Hk": 12, "d": 128, "dims": "44,42,42", "halves": False, "one": False,
         "stacked": False, "bhsd": True, "start": 0, "tail": 0, "far": 0},
        # image tokens behind the text of a joint sequence, fp32: keys shared
        # by four query heads, halves paired, sections of one spectrum, part
        # of each head unrotated, far positions
        {"name": "qk_f32_joint", "kind": "qk", "f16": False, "B": 2, "T": 3, "H": 11, "W": 35,
         "Hq": 16, "Hk": 4, "d": 80, "dims": "16,24,24", "halves": True, "one": True,
         "stacked": True, "bhsd": False, "start": 77, "tail": 5, "far": 100000},
        # one new token per caption over an image encoder's states
        {"name": "enc_f16_token", "kind": "enc", "f16": True, "B": 16, "Sq": 1, "Skv": 1500,
         "Hq": 16, "Hk": 4, "d": 64, "lens": "ragged", "bias": "none", "bhsd": False},
        # the first level of a 512 x 512 image, a guided pair, heads of 40
        {"name": "enc_f16_4096x77", "kind": "enc", "f16": True, "B": 2, "Sq": 4096, "Skv": 77,
         "Hq": 8, "Hk": 8, "d": 40, "lens": "ragged", "bias": "none", "bhsd": False},
        # a clip of 13 x 18 x 35 positions over long prompts
        {"name": "enc_f16_8190x512", "kind": "enc", "f16": True, "B": 2, "Sq": 8190, "Skv": 512,
         "Hq": 16, "Hk": 16, "d": 128, "lens": "ragged", "bias": "none", "bhsd": True},
        # a few latent queries that sum up a long video's states
        {"name": "enc_f16_64x16384", "kind": "enc", "f16": True, "B": 1, "Sq": 64, "Skv": 16384,
         "Hq": 8, "Hk": 8, "d": 128, "lens": "full", "bias": "none", "bhsd": False},
        # prompts by image region in fp32: a bias per query and key, some
        # queries with no key at all
        {"name": "enc_f32_regions", "kind": "enc", "f16": False, "B": 2, "Sq": 1024, "Skv": 154,
         "Hq": 10, "Hk": 10, "d": 64, "lens": "full", "bias": "query", "bhsd": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_lora(rng):
    f16 = rng.random() < 0.7
    act = rng.choice(["none", "none", "none", "gelu", "geglu"])
    n = rng.choice([320, 640, 1280, 2560, 8 * rng.randint(4, 320), rng.randint(30, 1300)])
    run = rng.choice([1, 77, 256, 1024, _log(rng, 1, 4096)])
    m = min(32768, run * _log(rng, 1, 64))
    return {"kind": "lora", "f16": f16, "M": max(1, m - rng.randint(0, min(run, m) - 1)),
            "N": max(32, n // 32 * 32) if act == "geglu" else n,
            "K": rng.choice([320, 640, 1024, 1280, 8 * rng.randint(4, 320), rng.randint(30, 1300)]),
            "rank": rng.choice([4, 8, 16, 32, 64, 128, rng.randint(1, 128)]),
            "n": rng.randint(1, 16), "run": run, "act": act, "res": rng.random() < 0.4}


def _draw_qk(rng):
    d = rng.choice([64, 128, 32, 40, 72, 80, 96, 160, 256, 2 * rng.randint(8, 128)])
    axes = rng.randint(1, 3)
    rot = d // 2 if rng.random() < 0.7 else rng.randint(axes, d // 2)
    cuts = sorted(rng.sample(range(1, rot), axes - 1)) if rot > axes else list(range(1, axes))
    dims = [2 * (b - a) for a, b in zip([0] + cuts, cuts + [rot])]
    hk = rng.choice([1, 2, 4, 5, 8, 10, 12, 16, 20])
    hq = hk * rng.choice([1, 1, 1, 2, 4])
    t, h, w = rng.choice([1, 1, 5, 13]), _log(rng, 1, 64), _log(rng, 1, 64)
    return {"kind": "qk", "f16": rng.random() < 0.6, "B": rng.choice([1, 2, 3]), "T": t, "H": h, "W": w,
            "Hq": hq, "Hk": hk, "d": d, "dims": ",".join(map(str, dims)), "halves": rng.random() < 0.4,
            "one": rng.random() < 0.3, "stacked": rng.random() < 0.5, "bhsd": rng.random() < 0.5,
            "start": rng.choice([0, 0, 77, rng.randint(1, 300)]), "tail": rng.choice([0, 0, 7]),
            "far": rng.choice([0, 0, 1000, 1000000])}


def _draw_enc(rng):
    hk = rng.choice([1, 2, 4, 5, 8, 10, 16, rng.randint(1, 20)])
    return {"kind": "enc", "f16": rng.random() < 0.65, "B": rng.choice([1, 2, 2, 4, 16]),
            "Sq": rng.choice([1, _log(rng, 1, 64), _log(rng, 64, 8192), _log(rng, 64, 8192)]),
            "Skv": rng.choice([77, 154, rng.randint(1, 100), _log(rng, 64, 16384)]),
            "Hq": hk * rng.choice([1, 1, 1, 2, 4, 7]), "Hk": hk,
            "d": rng.choice([64, 64, 128, 128, 40, 80, 160, 8 * rng.randint(1, 32)]),
            "lens": rng.choice(["full", "ragged", "ragged"]),
            "bias": rng.choice(["none", "none", "key", "query"]), "bhsd": rng.random() < 0.5}


def _cost(w):
    return max(w["bytes"], w["flops"] / 50)


def draw(rng):
    kind = rng.choice(["lora", "qk", "enc"])
    top = max(_cost(work(c)) for c in listed() if c["kind"] == kind)
    while True:
        c = {"lora": _draw_lora, "qk": _draw_qk, "enc": _draw_enc}[kind](rng)
        # the plain form's scores fit the card several times over
        if _cost(work(c)) <= top and (kind != "enc" or c["B"] * c["Hq"] * c["Sq"] * c["Skv"] <= 3e8):
            return c


# ------------------------------------------------------------------ inputs --
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) & 0x7FFFFFFF)
    return g


def _inputs(c, seed):
    """The tensors of a case, on the GPU, from the seed alone."""
    g = _generator(seed)
    dt = torch.float16 if c["f16"] else torch.float32

    def normal(shape, std=1.0, mean=0.0):
        return torch.randn(shape, generator=g, device="cuda") * std + mean

    def whole(lo, hi, shape):
        return torch.randint(lo, hi, shape, generator=g, device="cuda", dtype=torch.int32)

    if c["kind"] == "lora":
        M, N, K, R, n = c["M"], c["N"], c["K"], c["rank"], c["n"]
        t = {"x": normal((M, K)).to(dt), "w": normal((N, K), K ** -0.5).to(dt),
             "b": normal((N,), 0.02),
             "down": normal((n, R, K), K ** -0.5).to(dt), "up": normal((n, N, R), 0.5 * R ** -0.5).to(dt),
             "scale": torch.rand((n,), generator=g, device="cuda") + 0.5,
             # one past the stack: a run of rows without an adapter
             "ids": whole(0, n + 1, (-(-M // c["run"]),))}
        t["ids"] = torch.where(t["ids"] == n, -1, t["ids"])
        if c["res"]:
            t["r"] = normal((M, N // 2 if c["act"] == "geglu" else N)).to(dt)
        return t
    if c["kind"] == "qk":
        B, S, d = c["B"], c["T"] * c["H"] * c["W"], c["d"]
        h = c["Hq"] + 2 * c["Hk"] if c["stacked"] else None
        t = {"qkv": normal((B, S, h, d), 2.0).to(dt)} if h else \
            {"q": normal((B, S, c["Hq"], d), 2.0).to(dt), "k": normal((B, S, c["Hk"], d), 2.0).to(dt)}
        t["gq"], t["gk"] = normal((d,), 0.1, 1.0), normal((d,), 0.1, 1.0)
        at = torch.stack(torch.meshgrid(*(torch.arange(c[a], device="cuda") for a in "THW"),
                                        indexing="ij"), -1).reshape(S, 3)
        at = at[:, 3 - len(c["dims"].split(",")):]
        far = torch.randint(0, c["far"] + 1, (at.shape[1],), generator=g, device="cuda")
        t["pos"] = (at + far).float().contiguous()
        return t
    B, Sq, Skv, Hq, Hk, d = (c[x] for x in ("B", "Sq", "Skv", "Hq", "Hk", "d"))
    t = {"q": normal((B, Hq, Sq, d) if c["bhsd"] else (B, Sq, Hq, d), 1.5).to(dt),
         "kv": normal((B, Skv, 2, Hk, d)).to(dt)}
    if c["lens"] == "ragged":
        t["len"] = whole(min(Skv, max(1, Skv // 8)), Skv + 1, (B,))
        t["len"][-1] = Skv
    if c["bias"] == "key":  # weighted prompt tokens, some taken out
        t["bias"] = torch.where(torch.rand((B, 1, Skv), generator=g, device="cuda") < 0.2, -INF,
                                normal((B, 1, Skv), 0.5))
    if c["bias"] == "query":  # each query sees the tokens of its region
        nreg = 5  # the last region has no tokens
        qr, kr = whole(0, nreg, (B, Sq, 1)), whole(0, nreg - 1, (B, 1, Skv))
        t["bias"] = torch.where(qr == kr, normal((B, 1, Skv), 0.5), -INF).contiguous()
    return t


# ------------------------------------------------------------ library side --
_kept = {}


def _library():
    """The library's modules and the one device that a program keeps."""
    if not _kept:
        at = os.path.join(os.getcwd(), "draw-instant_amd")
        if at not in sys.path:
            sys.path.insert(0, at)
        import drawinstant
        from drawinstant import attention, lora
        _kept.update(dev=drawinstant.Device(0), attention=attention, lora=lora, base=drawinstant)
    return _kept


class _Buffers:
    """Device buffers that go back to the pool with their last user."""

    def __init__(self, dev):
        self.dev, self.all = dev, []

    def put(self, t):
        self.all.append(self.dev.storage(t.cpu().numpy()))
        return self.all[-1]

    def new(self, shape, f16):
        self.all.append(self.dev.create_buffer(math.prod(shape) * (2 if f16 else 4)))
        return self.all[-1]

    def __del__(self):
        try:
            for b in self.all:
                b.destroy()
        except Exception:
            pass


class _Outputs(dict):
    """Named device buffers, read back when an entry is looked up."""

    def __init__(self, owner, f16, **specs):
        super().__init__(specs)  # name -> (buffer, shape)
        self.owner, self.f16 = owner, f16

    def __getitem__(self, name):
        import numpy as np
        buf, shape = dict.__getitem__(self, name)
        return torch.from_numpy(self.owner.dev.download(buf, np.float16 if self.f16 else np.float32, shape))


def _shapes_qk(c):
    s = c["start"] + c["T"] * c["H"] * c["W"] + c["tail"]
    return {n: (c["B"], h, s, c["d"]) if c["bhsd"] else (c["B"], s, h, c["d"])
            for n, h in (("q", c["Hq"]), ("k", c["Hk"]))}


def _own_state(c, t):
    """The case's tensors in the library's buffers, the views and outputs that
    a program keeps beside them, and the call."""
    lib = _library()
    dev, attention, lora, base = lib["dev"], lib["attention"], lib["lora"], lib["base"]
    b = _Buffers(dev)
    dt = base.F16 if c["f16"] else base.F32
    h = {n: b.put(x) for n, x in t.items()}
    if c["kind"] == "lora":
        act = {"none": lora.ACT_NONE, "gelu": lora.ACT_GELU, "geglu": lora.ACT_GEGLU}[c["act"]]
        shape = (c["M"], c["N"] // 2 if c["act"] == "geglu" else c["N"])
        y = b.new(shape, c["f16"])
        ad = lora.Adapters(h["down"], h["up"], c["n"], c["rank"], h["scale"])
        def go():
            lora.linear_lora(dev, h["x"], h["w"], h["b"], ad, h["ids"], y, c["M"], c["N"], c["K"],
                             residual=h.get("r"), rows_per_id=c["run"], act=act, dtype=dt)
        return {"go": go, "out": _Outputs(b, c["f16"], y=(y, shape))}
    if c["kind"] == "qk":
        B, S, Hq, Hk, d = c["B"], c["T"] * c["H"] * c["W"], c["Hq"], c["Hk"], c["d"]
        shapes = _shapes_qk(c)
        out = {n: b.new(s, c["f16"]) for n, s in shapes.items()}
        for n, s in shapes.items():  # rows outside the image's stay as they are
            dev.upload(out[n], torch.zeros(s, dtype=torch.float16 if c["f16"] else torch.float32).numpy())
        if c["stacked"]:
            row = (Hq + 2 * Hk) * d
            q = attention.heads(h["qkv"], S, Hq, d, token=row, batch=S * row)
            k = attention.heads(h["qkv"], S, Hk, d, offset=Hq * d, token=row, batch=S * row)
        else:
            q, k = attention.heads(h["q"], S, Hq, d), attention.heads(h["k"], S, Hk, d)
        total = c["start"] + S + c["tail"]
        lay = attention.BHSD if c["bhsd"] else attention.BSHD
        qo = attention.heads(out["q"], total, Hq, d, lay, start=c["start"])
        ko = attention.heads(out["k"], total, Hk, d, lay, start=c["start"])
        dims = [int(x) for x in c["dims"].split(",")]
        rope = attention.Rope(dims, 10000.0, halves=c["halves"], one_spectrum=c["one"])
        def go():
            attention.qk_norm_rope(dev, q, k, qo, ko, h["pos"], rope, B, S, Hq, Hk, d, q_gamma=h["gq"],
                                   k_gamma=h["gk"], eps=1e-6, dtype=dt)
        return {"go": go, "out": _Outputs(b, c["f16"], **{n: (out[n], shapes[n]) for n in out})}
    B, Sq, Skv, Hq, Hk, d = (c[x] for x in ("B", "Sq", "Skv", "Hq", "Hk", "d"))
    shape = tuple(t["q"].shape)
    y = b.new(shape, c["f16"])
    lay = attention.BHSD if c["bhsd"] else attention.BSHD
    q, o = attention.heads(h["q"], Sq, Hq, d, lay), attention.heads(y, Sq, Hq, d, lay)
    k, v = (attention.heads(h["kv"], Skv, Hk, d, offset=i * Hk * d, token=2 * Hk * d, batch=2 * Skv * Hk * d)
            for i in (0, 1))
    bias = None
    if "bias" in t:
        rows = t["bias"].shape[1]
        bias = attention.Bias(h["bias"], batch=rows * Skv, query=Skv if rows > 1 else 0)
    def go():
        attention.attn_encoder(dev, q, k, v, o, B, Hq, Hk, Sq, Skv, d, kv_len=h.get("len"), bias=bias, dtype=dt)
    return {"go": go, "out": _Outputs(b, c["f16"], y=(y, shape))}


def prepare(case, seed):
    t = _inputs(case, seed)
    if own:  # the library keeps its data in buffers of its own
        s = _own_state(case, t)
        _library()["dev"].sync()
        return s
    return dict(t, case=case)


# ------------------------------------------------------------- plain forms --
def _plain_lora(c, s):
    f = torch.Tensor.float
    M, n, R = c["M"], c["n"], c["rank"]
    y = f(s["x"]) @ f(s["w"]).t() + s["b"]
    ids = s["ids"].long().repeat_interleave(c["run"])[:M]
    # every adapter's inner products, all but the row's own at zero
    own_a = (ids[:, None] == torch.arange(n, device="cuda")) * s["scale"]
    t = (f(s["x"]) @ f(s["down"]).reshape(n * R, -1).t()).reshape(M, n, R) * own_a[:, :, None]
    y = y + t.reshape(M, n * R) @ f(s["up"]).transpose(1, 2).reshape(n * R, -1)
    gelu = lambda v: 0.5 * v * (1 + torch.erf(v * 2 ** -0.5))  # noqa: E731
    if c["act"] == "gelu":
        y = gelu(y)
    if c["act"] == "geglu":  # columns in groups of [16 hidden | 16 gate]
        y = y.reshape(M, -1, 2, 16)
        y = (y[:, :, 0] * gelu(y[:, :, 1])).reshape(M, -1)
    if "r" in s:
        y = y + f(s["r"])
    return {"y": y.to(s["x"].dtype)}


def _frequencies(c):
    """Angle per unit of position of each rotated pair, and the pair's axis."""
    dims = [int(x) for x in c["dims"].split(",")]
    axis = torch.cat([torch.full((x // 2,), i) for i, x in enumerate(dims)]).cuda()
    if c["one"]:
        e = torch.arange(sum(dims) // 2, dtype=torch.float64) * (2.0 / sum(dims))
    else:
        e = torch.cat([torch.arange(x // 2, dtype=torch.float64) * (2.0 / x) for x in dims])
    return torch.exp(-math.log(10000.0) * e.cuda()), axis


def _sources(c, s):
    if not c["stacked"]:
        return s["q"], s["k"]
    return s["qkv"][:, :, :c["Hq"]], s["qkv"][:, :, c["Hq"]:c["Hq"] + c["Hk"]]


def _plain_qk(c, s):
    freq, axis = _frequencies(c)
    angle = s["pos"].double()[:, axis] * freq
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    n = 2 * freq.numel()

    def one(x, gamma, shape):
        x = x.float()
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * gamma
        r = x[..., :n]
        a, b = (r[..., :n // 2], r[..., n // 2:]) if c["halves"] else (r[..., 0::2], r[..., 1::2])
        p, q = a * cos - b * sin, a * sin + b * cos
        r = torch.cat([p, q], -1) if c["halves"] else torch.stack([p, q], -1).flatten(-2)
        x = torch.cat([r, x[..., n:]], -1)
        y = torch.zeros(shape, device="cuda", dtype=s["pos"].dtype)
        at = slice(c["start"], c["start"] + x.shape[1])
        if c["bhsd"]:
            y[:, :, at] = x.transpose(1, 2)
        else:
            y[:, at] = x
        return y.to(torch.float16 if c["f16"] else torch.float32)

    shapes = _shapes_qk(c)
    q, k = _sources(c, s)
    return {"q": one(q, s["gq"], shapes["q"]), "k": one(k, s["gk"], shapes["k"])}


def _plain_enc(c, s):
    B, Sq, Skv, Hk, d = (c[x] for x in ("B", "Sq", "Skv", "Hk", "d"))
    q = s["q"].float()
    q = q if c["bhsd"] else q.transpose(1, 2)
    q = q.reshape(B, Hk, -1, d)  # the query heads of a key head as its rows
    k, v = s["kv"].float().permute(2, 0, 3, 1, 4)
    p = ((q * d ** -0.5) @ k.transpose(2, 3).contiguous()).reshape(B, -1, Sq, Skv)
    if "bias" in s:
        p = p + s["bias"][:, None]
    if "len" in s:
        p = torch.where(torch.arange(Skv, device="cuda") < s["len"][:, None, None, None], p, -INF)
    m = p.amax(-1, keepdim=True)
    p = torch.exp(p - torch.where(m == -INF, 0.0, m))
    z = p.sum(-1, keepdim=True)
    p = (p / torch.where(z == 0, 1.0, z)).reshape(B, Hk, -1, Skv)
    y = (p @ v.contiguous()).reshape(B, -1, Sq, d)
    y = y if c["bhsd"] else y.transpose(1, 2)
    return {"y": y.to(s["q"].dtype).contiguous()}


def run(state):
    if own:
        state["go"]()
        return state["out"]
    c = state["case"]
    return {"lora": _plain_lora, "qk": _plain_qk, "enc": _plain_enc}[c["kind"]](c, state)


# -------------------------------------------------------------------- work --
def work(case):
    c, es = case, 2 if case["f16"] else 4
    if c["kind"] == "lora":
        M, N, K, R = c["M"], c["N"], c["K"], c["rank"]
        out = M * (N // 2 if c["act"] == "geglu" else N)
        used = min(c["n"], -(-M // c["run"]))
        return {"bytes": es * (M * K + N * K + used * R * (N + K) + out * (2 if c["res"] else 1)) + 4 * N,
                "flops": 2 * M * N * K + 2 * M * R * (N + K)}
    if c["kind"] == "qk":
        n = c["B"] * c["T"] * c["H"] * c["W"] * (c["Hq"] + c["Hk"]) * c["d"]
        return {"bytes": 2 * es * n, "flops": 10 * n}
    B, Sq, Skv, Hq, Hk, d = (c[x] for x in ("B", "Sq", "Skv", "Hq", "Hk", "d"))
    # ragged lengths spread evenly from an eighth to the whole, one whole
    keys = B * Skv if c["lens"] == "full" else Skv * (1 + (B - 1) * 9 / 16)
    bias = {"none": 0, "key": B * Skv, "query": B * Sq * Skv}[c["bias"]]
    return {"bytes": es * (2 * B * Sq * Hq * d + 2 * keys * Hk * d) + 4 * bias,
            "flops": 4 * Hq * Sq * keys * d}


# ------------------------------------------------- the definition, 64 bits --
def exact(case, seed):
    c = case
    t = {n: x.double() if x.is_floating_point() else x.long() for n, x in _inputs(c, seed).items()}
    if c["kind"] == "lora":
        return {"y": _exact_lora(c, t)}
    if c["kind"] == "qk":
        q, k = _sources(c, t)
        return {"q": _exact_qk(c, t, "q", q), "k": _exact_qk(c, t, "k", k)}
    return {"y": _exact_enc(c, t)}


def _exact_lora(c, t):
    y = t["x"] @ t["w"].T.contiguous() + t["b"]
    row = torch.arange(c["M"], device="cuda") // c["run"]
    for a in range(c["n"]):  # adapter by adapter, on its own rows
        m = (t["ids"][row] == a).nonzero()[:, 0]
        y[m] += t["scale"][a] * (t["x"][m] @ t["down"][a].T.contiguous()) @ t["up"][a].T.contiguous()
    phi = lambda v: (1 + torch.special.erf(v / math.sqrt(2))) / 2  # noqa: E731
    if c["act"] == "gelu":
        y = y * phi(y)
    elif c["act"] == "geglu":
        col = torch.arange(c["N"] // 2, device="cuda")
        hid = col // 16 * 32 + col % 16
        y = y[:, hid] * y[:, hid + 16] * phi(y[:, hid + 16])
    return y + t["r"] if "r" in t else y


def _exact_qk(c, t, name, x):
    x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6) * t["g" + name]
    y = x.clone()
    dims = [int(v) for v in c["dims"].split(",")]
    half, p = sum(dims) // 2, 0
    for axis, dim in enumerate(dims):  # pair by pair
        for i in range(dim // 2):
            e = p / half if c["one"] else 2 * i / dim
            a = t["pos"][:, axis] * 10000.0 ** -e
            cs, sn = a.cos()[:, None], a.sin()[:, None]
            u, w = (p, p + half) if c["halves"] else (2 * p, 2 * p + 1)
            y[..., u] = x[..., u] * cs - x[..., w] * sn
            y[..., w] = x[..., w] * cs + x[..., u] * sn
            p += 1
    y = torch.nn.functional.pad(y, (0, 0, 0, 0, c["start"], c["tail"]))
    return y.transpose(1, 2).contiguous() if c["bhsd"] else y


def _exact_enc(c, t):
    q = t["q"] if c["bhsd"] else t["q"].transpose(1, 2)
    y = torch.zeros_like(q)
    group = c["Hq"] // c["Hk"]
    for b in range(c["B"]):  # image by image, only the keys that it has
        n = int(t["len"][b]) if "len" in t else c["Skv"]
        k = t["kv"][b, :n, 0].transpose(0, 1).repeat_interleave(group, 0)
        v = t["kv"][b, :n, 1].transpose(0, 1).repeat_interleave(group, 0)
        s = torch.bmm(q[b], k.transpose(1, 2).contiguous()) / math.sqrt(c["d"])
        if "bias" in t:
            s = s + t["bias"][b, :, :n]
        y[b] = torch.bmm(torch.softmax(s, -1).nan_to_num(0.0), v.contiguous())
    return y if c["bhsd"] else y.transpose(1, 2).contiguous()
