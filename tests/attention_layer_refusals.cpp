// Host program for tests/test_attention_layer_refusals.py: every refusal of the
// attention-layer entry points on a context without a device.  A call that
// passes its checks gets as far as the missing device (DI_EHIP), never to a launch.
#include <cmath>
#include <cstdio>
#include <cstring>

#include "di_internal.h"

static int bad = 0;
static di_ctx ctx;

static void expect(int got, int want, const char* say, const char* what) {
  const char* msg = got ? di::get_error() : "";
  if (got != want || (say && !strstr(msg, say))) {
    printf("wrong: %s: status %d (wanted %d), message '%s'\n", what, got, want, msg);
    bad = 1;
  }
}

static di_handle buffer(uint64_t bytes) {
  di::Buffer b;
  b.ptr = (void*)0x1000;  // never touched
  b.bytes = b.cap = bytes;
  ctx.bufs[ctx.next_handle] = b;
  return ctx.next_handle++;
}

static void attention() {
  const di_handle q = buffer(2 * 9 * 6 * 64 * 2), kv = buffer(2 * 7 * 2 * 3 * 64 * 2), o = buffer(2 * 9 * 6 * 64 * 2);
  const di_handle len = buffer(8), bias = buffer(2 * 9 * 7 * 4);
  struct Call {
    di_heads q, k, v, o;
    di_attn_bias bias;
    di_handle len;
    uint32_t B, Hq, Hk, Sq, Skv, d;
    float scale;
    int32_t dt;
    bool with_bias;
  };
  const Call good = {{q, 0, 6 * 64, 64, 9 * 6 * 64}, {kv, 0, 2 * 3 * 64, 64, 7 * 2 * 3 * 64},
                     {kv, 3 * 64, 2 * 3 * 64, 64, 7 * 2 * 3 * 64}, {o, 0, 6 * 64, 64, 9 * 6 * 64},
                     {bias, 0, 9 * 7, 0, 7}, len, 2, 6, 3, 9, 7, 64, 0.0f, DI_F16, true};
  auto run = [&](const Call& c) {
    return di_attn_encoder(&ctx, &c.q, &c.k, &c.v, &c.o, c.len, c.with_bias ? &c.bias : nullptr, c.B, c.Hq, c.Hk, c.Sq,
                           c.Skv, c.d, c.scale, c.dt);
  };
  expect(run(good), DI_EHIP, "hipSetDevice", "a good call");
  auto with = [&](auto f) {
    Call c = good;
    f(c);
    return run(c);
  };
#define REFUSE(code, say, ...) expect(with([&](Call& c) { __VA_ARGS__; }), code, say, #__VA_ARGS__)
  REFUSE(DI_EHIP, "", c.len = 0; c.with_bias = false);
  REFUSE(DI_EHIP, "", c.k.batch = c.v.batch = 0);
  REFUSE(DI_EHIP, "", c.bias.batch = c.bias.query = 0);
  REFUSE(DI_EINVAL, "zero dimension", c.B = 0);
  REFUSE(DI_EINVAL, "zero dimension", c.Sq = 0);
  REFUSE(DI_EINVAL, "zero dimension", c.Skv = 0);
  REFUSE(DI_EINVAL, "zero dimension", c.Hk = 0);
  REFUSE(DI_EINVAL, "zero dimension", c.d = 0);
  REFUSE(DI_EINVAL, "6 query heads over 4", c.Hk = 4);
  REFUSE(DI_EUNSUPPORTED, "head dim 60", c.d = 60);
  REFUSE(DI_EUNSUPPORTED, "head dim 264", c.d = 264);
  REFUSE(DI_EINVAL, "dtype", c.dt = 2);
  REFUSE(DI_EINVAL, "scale", c.scale = NAN);
  REFUSE(DI_EINVAL, "scale", c.scale = INFINITY);
  REFUSE(DI_EINVAL, "scale", c.scale = 3e38f);
  REFUSE(DI_EHANDLE, "handle", c.q.buf = 0);
  REFUSE(DI_EHANDLE, "handle", c.v.buf = 12345);
  REFUSE(DI_EHANDLE, "handle", c.len = 12345);
  REFUSE(DI_EHANDLE, "handle", c.bias.buf = 0);
  REFUSE(DI_EINVAL, "view q ends past", c.q.offset = 8);
  REFUSE(DI_EINVAL, "view q ends past", c.Sq = 10);
  REFUSE(DI_EINVAL, "view k ends past", c.Skv = 8);
  REFUSE(DI_EINVAL, "view v ends past", c.v.token += 8);
  REFUSE(DI_EINVAL, "view q ends past", c.dt = DI_F32);
  REFUSE(DI_EINVAL, "past 2^40", c.q.head = 1ull << 40);
  REFUSE(DI_EINVAL, "past 2^40", c.bias.query = ~0ull);
  REFUSE(DI_EINVAL, "bias ends past", c.bias.offset = 1);
  REFUSE(DI_EINVAL, "bias ends past", c.bias.head = 7);
  REFUSE(DI_EUNSUPPORTED, "multiples of 8", c.q.offset = 4; c.Sq = 8);
  REFUSE(DI_EUNSUPPORTED, "multiples of 8", c.k.head = 60);
  REFUSE(DI_EINVAL, "elements of o overlap", c.o.head = 56);
  REFUSE(DI_EINVAL, "elements of o overlap", c.o.batch = 0);
  REFUSE(DI_EINVAL, "o overlaps an input", c.o.buf = q);
  REFUSE(DI_EINVAL, "o overlaps kv_len", c.len = o);
  REFUSE(DI_EINVAL, "o overlaps bias", c.bias.buf = o; c.bias.batch = c.bias.query = 0);
  REFUSE(DI_EINVAL, "needs 8", c.len = buffer(4));
#undef REFUSE
  expect(di_attn_encoder(&ctx, nullptr, &good.k, &good.v, &good.o, 0, nullptr, 1, 1, 1, 1, 1, 64, 0, 1), DI_EINVAL,
         "null view q", "null view");
  expect(di_attn_encoder(nullptr, &good.q, &good.k, &good.v, &good.o, 0, nullptr, 1, 1, 1, 1, 1, 64, 0, 1), DI_EINVAL,
         "null context", "null context");
}

static void rope() {
  const di_handle x = buffer(2 * 5 * 9 * 16 * 4), y = buffer(2 * 5 * 9 * 16 * 4), z = buffer(2 * 5 * 3 * 16 * 4);
  const di_handle gam = buffer(64), pos = buffer(5 * 2 * 4);
  struct Call {
    di_heads q, k, qo, ko;
    di_rope r;
    di_handle gq, gk, pos;
    uint32_t B, S, Hq, Hk, d;
    int32_t norm, dt;
    float eps;
    bool key;
  };
  // queries and keys of a stacked projection: rows of 9 heads, 6 + 3
  const Call good = {{x, 0, 144, 16, 720}, {x, 96, 144, 16, 720}, {y, 0, 96, 16, 480}, {z, 0, 48, 16, 240},
                     {2, {8, 6, 0, 0}, {1e4f, 1e4f, 0, 0}, 0, 0}, gam, gam, pos, 2, 5, 6, 3, 16,
                     DI_QKN_RMS, DI_F32, 1e-6f, true};
  auto run = [&](const Call& c) {
    return di_qk_norm_rope(&ctx, &c.q, c.key ? &c.k : nullptr, &c.qo, c.key ? &c.ko : nullptr, c.gq, c.gk, c.pos, &c.r,
                           c.B, c.S, c.Hq, c.Hk, c.d, c.norm, c.eps, c.dt);
  };
  expect(run(good), DI_EHIP, "hipSetDevice", "a good call");
  auto with = [&](auto f) {
    Call c = good;
    f(c);
    return run(c);
  };
#define REFUSE(code, say, ...) expect(with([&](Call& c) { __VA_ARGS__; }), code, say, #__VA_ARGS__)
  REFUSE(DI_EHIP, "", c.qo = c.q; c.ko = c.k);              // in place
  REFUSE(DI_EHIP, "", c.key = false; c.Hk = 0);             // queries only
  REFUSE(DI_EHIP, "", c.r.axes = 0; c.pos = 0);             // the norm alone
  REFUSE(DI_EHIP, "", c.norm = DI_QKN_NONE; c.gq = c.gk = 0);
  REFUSE(DI_EHIP, "", c.qo = c.q; c.qo.buf = y; c.ko = c.k; c.ko.buf = y);  // both into one stack
  REFUSE(DI_EINVAL, "zero dimension", c.S = 0);
  REFUSE(DI_EINVAL, "come together", c.Hk = 0);
  REFUSE(DI_EINVAL, "come together", c.key = false);
  REFUSE(DI_EUNSUPPORTED, "head dim 257", c.d = 257);
  REFUSE(DI_EUNSUPPORTED, "tokens", c.S = 1u << 31);
  REFUSE(DI_EINVAL, "unknown norm", c.norm = 2);
  REFUSE(DI_EINVAL, "eps", c.eps = -1.0f);
  REFUSE(DI_EINVAL, "eps", c.eps = NAN);
  REFUSE(DI_EINVAL, "gamma without", c.norm = DI_QKN_NONE);
  REFUSE(DI_EINVAL, "5 axes", c.r.axes = 5);
  REFUSE(DI_EINVAL, "unknown flags", c.r.flags = 4);
  REFUSE(DI_EINVAL, "turns 7 channels", c.r.dim[0] = 7);
  REFUSE(DI_EINVAL, "18 rotated channels", c.r.dim[0] = 12);
  REFUSE(DI_EINVAL, "theta", c.r.theta[1] = 1.0f);
  REFUSE(DI_EINVAL, "theta", c.r.theta[0] = INFINITY);
  REFUSE(DI_EINVAL, "dtype", c.dt = 3);
  REFUSE(DI_EHANDLE, "handle", c.pos = 0);
  REFUSE(DI_EHANDLE, "handle", c.ko.buf = 999);
  REFUSE(DI_EINVAL, "needs", c.r.pos_batch = 1);
  REFUSE(DI_EINVAL, "pos_batch", c.r.pos_batch = 1ull << 40);
  REFUSE(DI_EINVAL, "needs 64", c.gk = buffer(60));
  REFUSE(DI_EINVAL, "view k ends past", c.k.offset = 112);
  REFUSE(DI_EINVAL, "view q_out ends past", c.qo.token = 1 << 20);
  REFUSE(DI_EINVAL, "elements of q_out overlap", c.qo.head = 8);
  REFUSE(DI_EINVAL, "q_out overlaps q", c.qo = c.q; c.qo.head = 32; c.Hq = 3);
  REFUSE(DI_EINVAL, "q_out overlaps", c.qo = c.q; c.qo.offset = 48);
  REFUSE(DI_EINVAL, "overlaps", c.ko = c.qo);
#undef REFUSE
  expect(di_qk_norm_rope(&ctx, &good.q, nullptr, &good.qo, nullptr, 0, 0, 0, nullptr, 1, 1, 1, 0, 16, 0, 0, 0),
         DI_EINVAL, "null rope", "null rope");
}

static void lora() {
  const di_handle x = buffer(10 * 24 * 2), w = buffer(32 * 24 * 2), y = buffer(10 * 32 * 2), b = buffer(32 * 4);
  struct Call {
    di_handle x, w, b, r, y;
    di_lora lo;
    uint32_t M, N, K;
    int32_t act, dt;
  };
  const Call good = {x, w, b, 0, y,
                     {buffer(3 * 5 * 24 * 2), buffer(3 * 5 * 32 * 2), buffer(12), buffer(16), 3, 5, 3},
                     10, 32, 24, DI_ACT_NONE, DI_F16};
  auto run = [&](const Call& c) {
    return di_linear_lora(&ctx, c.x, c.w, c.b, &c.lo, c.r, c.y, c.M, c.N, c.K, c.act, c.dt);
  };
  expect(run(good), DI_EHIP, "hipSetDevice", "a good call");
  auto with = [&](auto f) {
    Call c = good;
    f(c);
    return run(c);
  };
#define REFUSE(code, say, ...) expect(with([&](Call& c) { __VA_ARGS__; }), code, say, #__VA_ARGS__)
  REFUSE(DI_EHIP, "", c.b = c.lo.scale = 0);
  REFUSE(DI_EHIP, "", c.r = c.y);
  REFUSE(DI_EINVAL, "zero dimension", c.M = 0);
  REFUSE(DI_EINVAL, "zero dimension", c.lo.n = 0);
  REFUSE(DI_EINVAL, "zero dimension", c.lo.rank = 0);
  REFUSE(DI_EINVAL, "zero dimension", c.lo.rows_per_id = 0);
  REFUSE(DI_EUNSUPPORTED, "rank 257", c.lo.rank = 257);
  REFUSE(DI_EINVAL, "adapters", c.lo.n = 1u << 31);
  REFUSE(DI_EINVAL, "unknown act", c.act = 5);
  REFUSE(DI_EINVAL, "GEGLU", c.act = DI_ACT_GEGLU; c.N = 24);
  REFUSE(DI_EINVAL, "dtype", c.dt = DI_F32W16);
  REFUSE(DI_EINVAL, "needs", c.dt = DI_F32);
  REFUSE(DI_EINVAL, "needs", c.lo.n = 4);
  REFUSE(DI_EINVAL, "needs", c.lo.rank = 6);
  REFUSE(DI_EINVAL, "needs 20", c.lo.rows_per_id = 2);
  REFUSE(DI_EHANDLE, "handle", c.lo.down = 0);
  REFUSE(DI_EHANDLE, "handle", c.lo.ids = 0);
  REFUSE(DI_EHANDLE, "handle", c.lo.up = 4321);
  REFUSE(DI_EHANDLE, "handle", c.lo.scale = 4321);
  REFUSE(DI_EINVAL, "Y is an operand", c.N = 24; c.y = c.x);
  REFUSE(DI_EINVAL, "Y is an operand", c.y = c.w);
  REFUSE(DI_EINVAL, "Y is an operand", c.M = 1; c.lo.rows_per_id = 1; c.y = c.b);
  REFUSE(DI_EINVAL, "Y is an operand", c.y = c.lo.up; c.M = 1; c.lo.rows_per_id = 1);
#undef REFUSE
  expect(di_linear_lora(&ctx, x, w, b, nullptr, 0, y, 10, 32, 24, 0, 1), DI_EINVAL, "null adapters", "null adapters");
}

int main() {
  ctx.device = 0;
  ctx.num_cus = 256;
  attention();
  rope();
  lora();
  ctx.bufs.clear();
  puts(bad ? "FAILED" : "OK");
  return bad;
}
