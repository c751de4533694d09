// Attention to an encoder's states: the fp16 instantiations of k_attn_enc.h,
// the choice of form and key split, and the C ABI (di_attn_encoder).
#include <algorithm>
#include <cmath>

#include "di_views.h"
#include "k_attn_enc.h"

namespace di {

void launch_attn_enc_f16(const AttnEncArgs& a, uint32_t B, int form, hipStream_t s) {
  launch_enc<f16>(a, B, form, s);
}

AttnEncForm attn_enc_form_f16(uint32_t d, int form) { return enc_form<f16>(d, form); }

}  // namespace di

using namespace di;

extern "C" int32_t di_attn_encoder(di_ctx* ctx, const di_heads* q, const di_heads* k, const di_heads* v,
                                   const di_heads* o, di_handle kv_len, const di_attn_bias* bias,
                                   uint32_t B, uint32_t Hq, uint32_t Hk, uint32_t Sq, uint32_t Skv,
                                   uint32_t d, float scale, int32_t dt) {
  const char* fn = "di_attn_encoder";
  DI_REQUIRE(ctx != nullptr, DI_EINVAL, "null context");
  DI_DTYPE(dt);
  DI_REQUIRE(B && Hq && Hk && Sq && Skv && d, DI_EINVAL, "%s: zero dimension (B=%u Hq=%u Hk=%u Sq=%u Skv=%u d=%u)",
             fn, B, Hq, Hk, Sq, Skv, d);
  DI_REQUIRE(Hq % Hk == 0, DI_EINVAL, "%s: %u query heads over %u key heads", fn, Hq, Hk);
  DI_REQUIRE(d % 8 == 0 && d <= 256, DI_EUNSUPPORTED, "%s: head dim %u (a multiple of 8 up to 256)", fn, d);
  DI_REQUIRE(std::isfinite(scale * kLog2E), DI_EINVAL, "%s: scale %g", fn, (double)scale);
  DI_REQUIRE(Skv < 1u << 31, DI_EUNSUPPORTED, "%s: %u keys", fn, Skv);
  HeadsPtr pq, pk, pv, po;
  int rc = check_heads(ctx, q, fn, "q", B, Sq, Hq, d, dt, &pq);
  if (!rc) rc = check_heads(ctx, k, fn, "k", B, Skv, Hk, d, dt, &pk);
  if (!rc) rc = check_heads(ctx, v, fn, "v", B, Skv, Hk, d, dt, &pv);
  if (!rc) rc = check_heads(ctx, o, fn, "o", B, Sq, Hq, d, dt, &po);
  if (rc) return rc;
  DI_REQUIRE(heads_aligned(pq, 8) && heads_aligned(pk, 8) && heads_aligned(pv, 8) && heads_aligned(po, 8),
             DI_EUNSUPPORTED, "%s: offsets and strides must be multiples of 8 elements", fn);
  DI_REQUIRE(heads_distinct(po, B, Sq, Hq, d), DI_EINVAL, "%s: elements of o overlap", fn);
  DI_REQUIRE(heads_apart(po, pq) && heads_apart(po, pk) && heads_apart(po, pv), DI_EINVAL, "%s: o overlaps an input",
             fn);
  // a tile's rows are addressed with 31-bit byte offsets from its first key
  DI_REQUIRE(pk.token < 1ull << 22 && pv.token < 1ull << 22, DI_EUNSUPPORTED,
             "%s: keys more than 2^22 elements apart", fn);
  AttnEncArgs a = {};
  a.q = pq.p, a.k = pk.p, a.v = pv.p, a.o = po.p;
  a.ldq = pq.token, a.hq = pq.head, a.bq = pq.batch;
  a.ldk = pk.token, a.hk = pk.head, a.bk = pk.batch;
  a.ldv = pv.token, a.hv = pv.head, a.bv = pv.batch;
  a.ldo = po.token, a.ho = po.head, a.bo = po.batch;
  if (kv_len) {
    DI_BUF(ctx, kv_len, lb, (uint64_t)B * 4);
    DI_REQUIRE(kv_len != o->buf, DI_EINVAL, "%s: o overlaps kv_len", fn);
    a.len = (const int32_t*)lb->ptr;
  }
  if (bias) {
    DI_REQUIRE(bias->offset < kMaxStride && bias->batch < kMaxStride && bias->head < kMaxStride &&
                   bias->query < kMaxStride,
               DI_EINVAL, "%s: offset or stride of bias past 2^40 elements", fn);
    Buffer* bb = nullptr;
    rc = lookup(ctx, bias->buf, &bb);
    if (rc) return rc;
    const unsigned __int128 end = (unsigned __int128)bias->offset + (unsigned __int128)(B - 1) * bias->batch +
                                  (unsigned __int128)(Hq - 1) * bias->head +
                                  (unsigned __int128)(Sq - 1) * bias->query + Skv;
    DI_REQUIRE(end * 4 <= bb->bytes, DI_EINVAL, "%s: bias ends past its buffer of %llu bytes", fn,
               (unsigned long long)bb->bytes);
    DI_REQUIRE(bias->buf != o->buf, DI_EINVAL, "%s: o overlaps bias", fn);
    a.bias = (const float*)bb->ptr + bias->offset;
    a.bias_b = bias->batch, a.bias_h = bias->head, a.bias_q = bias->query;
  }
  a.Hk = Hk, a.G = Hq / Hk, a.Sq = Sq, a.Skv = Skv, a.d = d;
  a.scale_log2 = (scale > 0.0f ? scale : 1.0f / sqrtf((float)d)) * kLog2E;
  const uint64_t rows = (uint64_t)Sq * a.G;
  a.prows = rows * B * Hk;
  const bool f32 = dt == DI_F32;
  // Two row groups a wavefront where that still leaves two workgroups a CU and,
  // with over 64 channels, keys enough to pay for the longer start: 2 x 16 heads
  // of 8192 x 512 keys of 128 80 us and with one group 87, 256 keys 48.8 and
  // 49.7, 154 keys 41.2 and 38.1; 8 heads of 4096 x 77 keys of 40 6.8 and 7.6; 24
  // heads of 1000 x 512 keys of 128, 192 workgroups, 15.9 and 13.9.  Not with a
  // bias, whose values take the registers of a workgroup per CU: 2 x 10 heads of
  // 4096 x 2048 keys of 64 168 us and with one group 156, x 77 keys 15.8 and 12.2
  // (past 64 channels it would spill).
  int kind = rows <= 16 ? ENC_FEW : ENC_MID;
  if (!f32 && rows > 64 && (d <= 64 || (d <= 128 && Skv > 192)) && !bias &&
      (rows + 127) / 128 * B * Hk >= 2ull * ctx->num_cus)
    kind = ENC_MANY;
  const AttnEncForm form = f32 ? attn_enc_form_f32(d, kind) : attn_enc_form_f16(d, kind);
  const uint32_t R = form.rows, KT = form.tile, WK = form.groups;
  const uint64_t blocks = (rows + R - 1) / R, groups = blocks * B * Hk;
  DI_REQUIRE(rows < 1ull << 31 && groups < 1ull << 24, DI_EUNSUPPORTED, "%s: %llu rows per key head, %llu workgroups",
             fn, (unsigned long long)rows, (unsigned long long)groups);
  a.rows = (uint32_t)rows;
  a.blocks = (uint32_t)blocks;
  // Key ranges, at most a workgroup per CU and two to four tiles each, by what
  // they save (a tile takes a wavefront 0.5 us on a CU of its own) less what the
  // merge costs (3 us and the parts' bytes at 4 TB/s).  16 heads' single tokens over
  // 8000 keys of 64 18.0 us in one piece, 8.4 in 16 ranges; 8 heads of 64 queries
  // over 16384 keys of 128 281, 20.7 in 32 ranges, 23.5 in 64; 64 heads' tokens
  // over 1500 keys, six tiles a wavefront, 7.0 and in four ranges 8.2.
  const uint64_t n_tiles = (Skv + KT - 1) / KT;
  uint64_t most = n_tiles / (kind == ENC_FEW ? 2 * WK : 4);
  most = std::min<uint64_t>({most, ctx->num_cus / groups, 64});
  a.splits = 1;
  double best = 0.0;
  for (uint32_t sp = 2; sp <= most; sp++) {
    const double gain = (double)n_tiles / WK * (1.0 - 1.0 / sp) * 0.5 - 3.0 - (double)sp * a.prows * d * 8 / 4e6;
    if (gain > best) best = gain, a.splits = sp;
  }
  if (bias && bias->head == 0) {
    // One bias for all heads: they go side by side where the workgroups that an
    // XCD holds then touch fewer bytes of keys, values and bias in its L2.  2 x 10
    // heads of 4096 x 2048 keys of 64 140 us and head by head 156, 2 x 5 of 9216 x
    // 9216 755 and 886; 24 of 1000 x 512 of 128, whose keys pass the L2 so, 22.8 and
    // 20.1.
    const uint64_t run = std::min<uint64_t>((groups * a.splits + 7) / 8, ctx->num_cus / 4);
    const uint64_t kv = (uint64_t)Skv * d * 2 * dtype_size(dt);
    const uint64_t bi = (bias->query ? std::max<uint64_t>(R / a.G, 1) : 1) * Skv * 4;
    const uint64_t by_head = (run + blocks - 1) / blocks * kv + std::min(run, blocks * a.splits) * bi;
    const uint64_t by_block = std::min<uint64_t>(run, Hk) * kv + (run + Hk - 1) / Hk * bi;
    a.heads_first = by_block < by_head;
  }
  DI_HIP(hipSetDevice(ctx->device));
  void* ws = nullptr;
  uint64_t cap = 0;
  if (a.splits > 1) {
    const uint64_t ob = a.splits * a.prows * d * 4;
    rc = pool_alloc(ctx, ob + a.splits * a.prows * 8, &ws, &cap);
    if (rc) return rc;
    a.part_o = (float*)ws;
    a.part_ml = (float*)((char*)ws + ob);
  }
  if (f32) launch_attn_enc_f32(a, B, kind, ctx->stream);
  else launch_attn_enc_f16(a, B, kind, ctx->stream);
  if (ws) pool_release(ctx, ws, cap);
  DI_LAUNCH_CHECK();
  return DI_OK;
}
