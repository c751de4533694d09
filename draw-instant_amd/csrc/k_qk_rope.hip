// Norm of each query and key head and the rotation of its channel pairs by
// positions of several axes, in one pass over the heads (di_qk_norm_rope).
//
//   u = x * rsqrt(mean(x^2) + eps) * gamma            (over the d channels)
//   (u_a, u_b) -> (u_a cos - u_b sin, u_b cos + u_a sin)   for each pair
//
// One row is the d channels of one head of one token.  LPR lanes (a power of
// two) hold a row, 16 bytes each, so a wavefront moves 64 / LPR rows at a
// time; the sum of squares is reduced by lane shuffles.  A wavefront takes one
// token at a time and walks its query, then its key heads: the cosines and
// sines of the lane's own pairs are formed once per token and serve every
// head.  Pairs (2p, 2p+1) lie in one lane; pairs (p, p + r/2) are exchanged
// through the wavefront's own strip of LDS.
//
// An angle is position * frequency: far positions (10^6) times a frequency
// rounded to fp32 would be off by whole hundredths of a turn, so the product
// is taken in 64 bits, in turns, and reduced to an eighth of a turn either
// side of a multiple of a quarter; what is left goes to fp32 and there to the
// Taylor series of sine and cosine (to x^9 and x^10 on [-pi/4, pi/4]: the next
// terms are below 2e-9 and 2e-10).  A frequency theta^(-2i/n) is the i-th power of the
// axis' ratio theta^(-2/n), raised by squaring in 64 bits at the kernel's start.
//
// The bound is HBM: every value is read and written once.
#include <cmath>

#include "di_device.h"
#include "di_views.h"

namespace di {

namespace {

struct RopeRow {  // one of the two tensors
  const void* x;
  void* y;
  const float* gamma;
  uint64_t xt, xh, xb, yt, yh, yb;  // strides in elements
  uint32_t H;
};

struct RopeArgs {
  RopeRow t[2];
  const float* pos;
  uint64_t pos_batch;
  double ratio[4];        // of each axis' neighbouring frequencies
  uint32_t pair_end[4];   // first pair past the axis
  uint32_t axes, pairs;   // pairs in all: r / 2
  uint32_t one_spectrum;
  uint32_t B, S, d, norm;
  float eps;
};

// sin and cos of 2 pi turns
__device__ __forceinline__ void sincos_turns(double turns, float& sn, float& cs) {
  const double q = __builtin_rint(turns * 4.0);
  const float x = (float)(turns * 4.0 - q) * 1.57079632679489662f;  // [-pi/4, pi/4]
  const int n = (int)(q - 4.0 * __builtin_floor(q * 0.25));  // 0 to 3
  const float z = x * x;
  const float s = x + x * z * (-1.0f / 6 + z * (1.0f / 120 + z * (-1.0f / 5040 + z * (1.0f / 362880))));
  const float c = 1.0f + z * (-0.5f + z * (1.0f / 24 + z * (-1.0f / 720 + z * (1.0f / 40320 + z * (-1.0f / 3628800)))));
  const float a = n & 1 ? c : s, b = n & 1 ? s : c;
  sn = n & 2 ? -a : a;
  cs = (n == 1 || n == 2) ? -b : b;
}

// Orders LDS accesses of one wavefront's lanes, which the hardware keeps in
// order by itself, for the compiler.
__device__ __forceinline__ void wave_lds_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

template <typename T>
struct Vec;
template <>
struct Vec<f16> {
  typedef f16x8 type;
};
template <>
struct Vec<float> {
  typedef f32x4 type;
};

// LPR lanes per row; HALVES: pairs (p, p + pairs); VEC: rows are whole 16-byte
// vectors at aligned places (else element by element)
template <typename T, int LPR, bool HALVES, bool VEC>
__global__ __launch_bounds__(256) void k_qk_rope(RopeArgs a) {
  constexpr int V = 16 / sizeof(T), RPW = 64 / LPR;
  typedef typename Vec<T>::type vec;
  constexpr int NP = HALVES ? V : V / 2;  // pairs that a lane turns
  __shared__ float strip[HALVES ? 4 * 64 * V : 1];
  kernarg_warm(a);

  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t sub = lane % LPR, row = lane / LPR, c0 = sub * V;  // first channel of this lane
  const bool in = c0 < a.d;

  // this lane's pairs: axis and turns per unit of position
  double freq[NP];
  uint32_t axis[NP];
#pragma unroll
  for (int i = 0; i < NP; i++) {
    const uint32_t c = c0 + (HALVES ? i : 2 * i);
    const uint32_t p = HALVES ? (c < a.pairs ? c : c - a.pairs) : c / 2;
    uint32_t ax = 0, first = 0;
#pragma unroll
    for (uint32_t k = 1; k < 4; k++)
      if (k < a.axes && p >= a.pair_end[k - 1]) {
        ax = k;
        first = a.pair_end[k - 1];
      }
    uint32_t e = a.one_spectrum ? p : p - first;
    double b = a.one_spectrum ? a.ratio[0] : ax == 0 ? a.ratio[0] : ax == 1 ? a.ratio[1] : ax == 2 ? a.ratio[2] : a.ratio[3];
    double f = 0.15915494309189533577;  // 1 / (2 pi)
#pragma unroll
    for (int k = 0; k < 7; k++) {  // e < 128
      if (e & 1) f *= b;
      b *= b;
      e >>= 1;
    }
    axis[i] = ax;
    freq[i] = f;
  }
  float gam[2][V];
#pragma unroll
  for (int t = 0; t < 2; t++)
#pragma unroll
    for (int j = 0; j < V; j++) gam[t][j] = a.t[t].gamma && c0 + j < a.d ? a.t[t].gamma[c0 + j] : 1.0f;

  const uint32_t tokens = a.B * a.S, step = gridDim.x * 4;
  const float inv_d = 1.0f / (float)a.d;
  for (uint32_t tok = blockIdx.x * 4 + wave; tok < tokens; tok += step) {
    const uint32_t b = tok / a.S, s = tok - b * a.S;
    float cs[NP], sn[NP];
    const float* pos = a.pos + b * a.pos_batch + (uint64_t)s * a.axes;
#pragma unroll
    for (int i = 0; i < NP; i++) {
      cs[i] = 1.0f;
      sn[i] = 0.0f;
      if (c0 + (HALVES ? i : 2 * i) < 2 * a.pairs) sincos_turns((double)pos[axis[i]] * freq[i], sn[i], cs[i]);
    }
#pragma unroll
    for (int t = 0; t < 2; t++) {
      const RopeRow& R = a.t[t];
      for (uint32_t h = row; h < (R.H + RPW - 1) / RPW * RPW; h += RPW) {
        const bool ok = in && h < R.H;
        const T* x = (const T*)R.x + b * R.xb + (uint64_t)s * R.xt + (uint64_t)h * R.xh + c0;
        float u[V];
        vec xv = {};
        if (ok) {
          if constexpr (VEC) {
            xv = *(const vec*)x;
          } else {
#pragma unroll
            for (int j = 0; j < V; j++)
              if (c0 + j < a.d) xv[j] = x[j];
          }
        }
        float q = 0.0f;
#pragma unroll
        for (int j = 0; j < V; j++) {
          u[j] = (float)xv[j];
          q = fmaf(u[j], u[j], q);
        }
        if (a.norm) {
#pragma unroll
          for (int o = LPR / 2; o > 0; o >>= 1) q += __shfl_xor(q, o);
          const float r = 1.0f / sqrtf(q * inv_d + a.eps);
#pragma unroll
          for (int j = 0; j < V; j++) u[j] *= r * gam[t][j];
        }
        if constexpr (!HALVES) {
#pragma unroll
          for (int i = 0; i < NP; i++) {
            const float p = u[2 * i], w = u[2 * i + 1];
            u[2 * i] = p * cs[i] - w * sn[i];
            u[2 * i + 1] = w * cs[i] + p * sn[i];
          }
        } else {
          // the wavefront's own strip: written and read by the same 64 lanes
          float* st = strip + wave * 64 * V + row * LPR * V;
#pragma unroll
          for (int j = 0; j < V; j++) st[c0 + j] = u[j];
          wave_lds_fence();
#pragma unroll
          for (int j = 0; j < V; j++) {
            const uint32_t c = c0 + j;
            if (c < a.pairs) u[j] = u[j] * cs[j] - st[c + a.pairs] * sn[j];
            else if (c < 2 * a.pairs) u[j] = u[j] * cs[j] + st[c - a.pairs] * sn[j];
          }
          wave_lds_fence();
        }
        if (ok) {
          T* y = (T*)R.y + b * R.yb + (uint64_t)s * R.yt + (uint64_t)h * R.yh + c0;
          if constexpr (VEC) {
            vec o;
#pragma unroll
            for (int j = 0; j < V; j++) o[j] = (T)u[j];
            *(vec*)y = o;
          } else {
#pragma unroll
            for (int j = 0; j < V; j++)
              if (c0 + j < a.d) y[j] = (T)u[j];
          }
        }
      }
    }
  }
}

template <typename T, int LPR>
void launch_lpr(const RopeArgs& a, bool halves, bool vec, uint32_t blocks, hipStream_t s) {
  if (halves && vec) k_qk_rope<T, LPR, true, true><<<blocks, 256, 0, s>>>(a);
  else if (halves) k_qk_rope<T, LPR, true, false><<<blocks, 256, 0, s>>>(a);
  else if (vec) k_qk_rope<T, LPR, false, true><<<blocks, 256, 0, s>>>(a);
  else k_qk_rope<T, LPR, false, false><<<blocks, 256, 0, s>>>(a);
}

template <typename T>
void launch_rope(const RopeArgs& a, bool halves, bool vec, int num_cus, hipStream_t s) {
  constexpr uint32_t V = 16 / sizeof(T);
  const uint32_t need = (a.d + V - 1) / V;
  const uint64_t tokens = (uint64_t)a.B * a.S, cap = (uint64_t)num_cus * 8;
  const uint32_t blocks = (uint32_t)((tokens + 3) / 4 < cap ? (tokens + 3) / 4 : cap);
  if (need <= 2) launch_lpr<T, 2>(a, halves, vec, blocks, s);
  else if (need <= 4) launch_lpr<T, 4>(a, halves, vec, blocks, s);
  else if (need <= 8) launch_lpr<T, 8>(a, halves, vec, blocks, s);
  else if (need <= 16) launch_lpr<T, 16>(a, halves, vec, blocks, s);
  else if (need <= 32) launch_lpr<T, 32>(a, halves, vec, blocks, s);
  else launch_lpr<T, 64>(a, halves, vec, blocks, s);
}

}  // namespace

}  // namespace di

using namespace di;

extern "C" int32_t di_qk_norm_rope(di_ctx* ctx, const di_heads* q, const di_heads* k, const di_heads* q_out,
                                   const di_heads* k_out, di_handle q_gamma, di_handle k_gamma,
                                   di_handle pos, const di_rope* rope, uint32_t B, uint32_t S, uint32_t Hq,
                                   uint32_t Hk, uint32_t d, int32_t norm, float eps, int32_t dt) {
  const char* fn = "di_qk_norm_rope";
  DI_REQUIRE(ctx != nullptr, DI_EINVAL, "null context");
  DI_DTYPE(dt);
  DI_REQUIRE(B && S && Hq && d, DI_EINVAL, "%s: zero dimension (B=%u S=%u Hq=%u d=%u)", fn, B, S, Hq, d);
  DI_REQUIRE(!k == !k_out && !k == !Hk, DI_EINVAL, "%s: k, k_out and Hk come together", fn);
  DI_REQUIRE(d <= 256, DI_EUNSUPPORTED, "%s: head dim %u above 256", fn, d);
  DI_REQUIRE((uint64_t)B * S < 1ull << 31, DI_EUNSUPPORTED, "%s: %llu tokens", fn, (unsigned long long)B * S);
  DI_REQUIRE(norm == DI_QKN_NONE || norm == DI_QKN_RMS, DI_EINVAL, "%s: unknown norm %d", fn, norm);
  DI_REQUIRE(norm == DI_QKN_NONE || (eps >= 0.0f && std::isfinite(eps)), DI_EINVAL, "%s: eps %g", fn, (double)eps);
  DI_REQUIRE(norm == DI_QKN_RMS || (!q_gamma && !k_gamma), DI_EINVAL, "%s: gamma without a norm", fn);
  DI_REQUIRE(rope != nullptr, DI_EINVAL, "%s: null rope", fn);
  DI_REQUIRE(rope->axes <= 4, DI_EINVAL, "%s: %u axes (at most 4)", fn, rope->axes);
  DI_REQUIRE((rope->flags & ~(uint32_t)(DI_ROPE_HALVES | DI_ROPE_ONE_SPECTRUM)) == 0, DI_EINVAL,
             "%s: unknown flags 0x%x", fn, rope->flags);
  RopeArgs a = {};
  uint64_t r = 0;
  for (uint32_t i = 0; i < rope->axes; i++) {
    DI_REQUIRE(rope->dim[i] % 2 == 0 && rope->dim[i] <= d, DI_EINVAL, "%s: axis %u turns %u channels of %u",
               fn, i, rope->dim[i], d);
    const float theta = rope->theta[rope->flags & DI_ROPE_ONE_SPECTRUM ? 0 : i];
    DI_REQUIRE(theta > 1.0f && std::isfinite(theta), DI_EINVAL, "%s: theta %g of axis %u", fn, (double)theta, i);
    r += rope->dim[i];
    a.pair_end[i] = (uint32_t)(r / 2);
  }
  DI_REQUIRE(r <= d, DI_EINVAL, "%s: %llu rotated channels of %u", fn, (unsigned long long)r, d);
  a.axes = rope->axes;
  a.pairs = (uint32_t)(r / 2);
  a.one_spectrum = rope->flags & DI_ROPE_ONE_SPECTRUM ? 1 : 0;
  for (uint32_t i = 0; i < rope->axes; i++) {
    const double n = a.one_spectrum ? (double)r : (double)rope->dim[i];
    a.ratio[i] = n > 0 ? std::pow((double)rope->theta[a.one_spectrum ? 0 : i], -2.0 / n) : 1.0;
  }
  HeadsPtr v[2], w[2];
  const di_heads* in[2] = {q, k};
  const di_heads* out[2] = {q_out, k_out};
  const uint32_t H[2] = {Hq, Hk};
  const di_handle gm[2] = {q_gamma, k_gamma};
  const char* names[4] = {"q", "k", "q_out", "k_out"};
  const int nt = k ? 2 : 1;
  const uint64_t va = dt == DI_F32 ? 4 : 8;
  bool vec = d % va == 0;
  for (int t = 0; t < nt; t++) {
    int rc = check_heads(ctx, in[t], fn, names[t], B, S, H[t], d, dt, &v[t]);
    if (rc) return rc;
    rc = check_heads(ctx, out[t], fn, names[2 + t], B, S, H[t], d, dt, &w[t]);
    if (rc) return rc;
    DI_REQUIRE(heads_distinct(w[t], B, S, H[t], d), DI_EINVAL, "%s: elements of %s overlap", fn, names[2 + t]);
    vec = vec && heads_aligned(v[t], va) && heads_aligned(w[t], va);
    if (gm[t]) {
      DI_BUF(ctx, gm[t], g, (uint64_t)d * 4);
      a.t[t].gamma = (const float*)g->ptr;
    }
    a.t[t].x = v[t].p;
    a.t[t].y = w[t].p;
    a.t[t].xt = v[t].token, a.t[t].xh = v[t].head, a.t[t].xb = v[t].batch;
    a.t[t].yt = w[t].token, a.t[t].yh = w[t].head, a.t[t].yb = w[t].batch;
    a.t[t].H = H[t];
  }
  for (int t = 0; t < nt; t++)
    for (int u = 0; u < nt; u++) {
      DI_REQUIRE((t == u && heads_same(w[t], v[u])) || heads_apart(w[t], v[u]), DI_EINVAL, "%s: %s overlaps %s", fn,
                 names[2 + t], names[u]);
      DI_REQUIRE(t == u || heads_apart(w[t], w[u]), DI_EINVAL, "%s: q_out overlaps k_out", fn);
    }
  if (a.pairs) {
    DI_REQUIRE(rope->pos_batch < kMaxStride, DI_EINVAL, "%s: pos_batch past 2^40 elements", fn);
    DI_BUF(ctx, pos, pb, ((uint64_t)(B - 1) * rope->pos_batch + (uint64_t)S * rope->axes) * 4);
    a.pos = (const float*)pb->ptr;
    a.pos_batch = rope->pos_batch;
  }
  a.B = B, a.S = S, a.d = d, a.eps = eps;
  a.norm = norm == DI_QKN_RMS;
  const bool halves = (rope->flags & DI_ROPE_HALVES) && a.pairs;
  DI_HIP(hipSetDevice(ctx->device));
  if (dt == DI_F16) launch_rope<f16>(a, halves, vec, ctx->num_cus, ctx->stream);
  else launch_rope<float>(a, halves, vec, ctx->num_cus, ctx->stream);
  DI_LAUNCH_CHECK();
  return DI_OK;
}
