// Norm of each query and key head and the rotation of its channel pairs by
// positions of several axes, in one pass over the heads (di_qk_norm_rope).
//
//   u = x * rsqrt(mean(x^2) + eps) * gamma            (over the d channels)
//   (u_a, u_b) -> (u_a cos - u_b sin, u_b cos + u_a sin)   for each pair
//
// One row is the d channels of one head of one token.  LPR lanes (a power of
// two) hold a row, 16 bytes each, so a wavefront moves 64 / LPR rows at a
// time; the sum of squares is reduced by lane moves.  A wavefront takes up
// to U such steps of one token's query and key heads: all their loads first, then
// the cosines and sines of the lane's own pairs, which serve every head, while
// the loads are on their way.  Pairs (2p, 2p+1) lie in one lane; pairs (p, p +
// r/2) are exchanged through the wavefront's own strip of LDS.
//
// An angle is position * frequency: far positions (10^6) times a frequency
// rounded to fp32 would be off by whole hundredths of a turn, so the product
// is taken in 64 bits, in turns, and reduced to an eighth of a turn either
// side of a multiple of a quarter; what is left goes to fp32 and there to the
// Taylor series of sine and cosine (to x^9 and x^10 on [-pi/4, pi/4]: the next
// terms are below 2e-9 and 2e-10).  A frequency theta^(-2i/n) is the i-th power of
// the axis' ratio theta^(-2/n), raised by squaring in 64 bits, one pair a thread,
// at the kernel's start.
//
// The bound is HBM: every value is read and written once.  20280 tokens of 12
// query and 12 key heads of 128 fp16 channels: 52 us, 4.8 TB/s (60 and 4.1 with
// inputs that no cache holds; a large copy reaches 5.2); 512 tokens of 40 heads
// of 64 take 5.7 us, of which 5.0 pass before a launch of anything returns.
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
  uint32_t steps_q, steps, segs, run;  // steps over the query and all heads of a token, in segs runs
  float eps;
};

// sin and cos of t quarter turns
__device__ __forceinline__ void sincos_quarters(double t, float& sn, float& cs) {
  const double q = __builtin_rint(t);
  const float x = (float)(t - q) * 1.57079632679489662f;  // [-pi/4, pi/4]
  const int n = (int)(__builtin_amdgcn_fract(q * 0.25) * 4.0);  // 0 to 3
  const float z = x * x;
  const float s = x + x * z * (-1.0f / 6 + z * (1.0f / 120 + z * (-1.0f / 5040 + z * (1.0f / 362880))));
  const float c = 1.0f + z * (-0.5f + z * (1.0f / 24 + z * (-1.0f / 720 + z * (1.0f / 40320 + z * (-1.0f / 3628800)))));
  const float a = n & 1 ? c : s, b = n & 1 ? s : c;
  sn = n & 2 ? -a : a;
  cs = (n == 1 || n == 2) ? -b : b;
}

// 1 / sqrt(v): the hardware's (1 ulp) is for normal numbers
__device__ __forceinline__ float rsqrt_f(float v) {
  const bool low = v < 0x1p-100f;
  return __builtin_amdgcn_rsqf(low ? v * 0x1p64f : v) * (low ? 0x1p32f : 1.0f);
}

// Sum over the LPR lanes of a row, in every one of them: neighbours within four
// lanes, then the mirrored half of eight and of sixteen (whose lanes all hold
// the same by then), in the adds' own lane moves; then across the rows of
// sixteen.
template <int CTRL>
__device__ __forceinline__ float add_dpp(float x) {
  return x + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, true));
}
template <int LPR>
__device__ __forceinline__ float row_sum(float x) {
  x = add_dpp<0xB1>(x);                   // quad_perm 1 0 3 2
  if (LPR >= 4) x = add_dpp<0x4E>(x);     // quad_perm 2 3 0 1
  if (LPR >= 8) x = add_dpp<0x141>(x);    // row_half_mirror
  if (LPR >= 16) x = add_dpp<0x140>(x);   // row_mirror
  if (LPR >= 32) {
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  }
  if (LPR >= 64) {
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  }
  return x;
}

// A barrier that waits for the wavefront's LDS operations only: loads stay in flight.
__device__ __forceinline__ void lds_barrier() {
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
  __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0); vmcnt, expcnt not waited on
  __builtin_amdgcn_s_barrier();
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
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

// LPR lanes per row; up to U steps per wavefront; HALVES: pairs (p, p + pairs); VEC:
// rows are whole 16-byte vectors at aligned places (else element by element)
template <typename T, int LPR, int U, bool HALVES, bool VEC>
__global__ __launch_bounds__(256) void k_qk_rope(RopeArgs a) {
  constexpr int V = 16 / sizeof(T), RPW = 64 / LPR;
  typedef typename Vec<T>::type vec;
  constexpr int NP = HALVES ? V : V / 2;  // pairs that a lane turns
  __shared__ __attribute__((aligned(16))) float strip[HALVES ? 4 * 64 * V : 4];
  __shared__ double sfreq[128];
  __shared__ uint32_t saxis[128];
  kernarg_warm(a);

  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t sub = lane % LPR, row = lane / LPR, c0 = sub * V;  // first channel of this lane
  const bool in = c0 < a.d;
  const RopeRow &Q = a.t[0], &K = a.t[1];

  // this lane's place in a step's rows
  const uint64_t lxq = row * Q.xh + c0, lxk = row * K.xh + c0, lyq = row * Q.yh + c0, lyk = row * K.yh + c0;
  // A unit is a run of steps of one token: query heads, then key heads.  The
  // run's rows start at a scalar address that moves on from step to step.
  struct Unit {
    uint32_t b, s, j0, n;
  };
  auto unit_of = [&](uint32_t unit) {
    const uint32_t tok = unit / a.segs, j0 = (unit - tok * a.segs) * a.run, b = tok / a.S;
    const uint32_t left = a.steps - j0;
    return Unit{b, tok - b * a.S, j0, a.run < left ? a.run : left};
  };
  auto walk = [&](const Unit& n, const char* q0, const char* k0, uint64_t dq, uint64_t dk, auto f) {
    const char* p = n.j0 >= a.steps_q ? k0 + (n.j0 - a.steps_q) * dk : q0 + n.j0 * dq;
#pragma unroll
    for (int u = 0; u < U; u++) {
      const uint32_t j = n.j0 + u;
      if (u > 0) p = j == a.steps_q ? k0 : p + (j > a.steps_q ? dk : dq);
      if ((uint32_t)u >= n.n) break;
      const bool key = j >= a.steps_q;
      f(u, key, p, in && (key ? j - a.steps_q : j) * RPW + row < (key ? K.H : Q.H));
    }
  };
  vec xv[U];
  auto load = [&](const Unit& n) {
    const T* q0 = (const T*)Q.x + (n.b * Q.xb + n.s * Q.xt);
    const T* k0 = (const T*)K.x + (n.b * K.xb + n.s * K.xt);
    walk(n, (const char*)q0, (const char*)k0, Q.xh * (RPW * sizeof(T)), K.xh * (RPW * sizeof(T)),
         [&](int u, bool key, const char* p, bool ok) {
           const T* x = (const T*)p + (key ? lxk : lxq);
           xv[u] = vec{};
           if (!ok) return;
           if constexpr (VEC) {
             xv[u] = *(const vec*)x;
           } else {
#pragma unroll
             for (int j = 0; j < V; j++)
               if (c0 + j < a.d) xv[u][j] = x[j];
           }
         });
  };
  const uint32_t units = a.B * a.S * a.segs, step = gridDim.x * 4;
  uint32_t unit = blockIdx.x * 4 + wave;
  Unit n = unit_of(unit < units ? unit : 0);
  if (unit < units) load(n);

  float gam[2][V];
#pragma unroll
  for (int t = 0; t < 2; t++)
#pragma unroll
    for (int j = 0; j < V; j++) gam[t][j] = a.t[t].gamma && c0 + j < a.d ? a.t[t].gamma[c0 + j] : 1.0f;
  // quarter turns per unit of position and axis of each pair
  if (threadIdx.x < a.pairs) {
    const uint32_t p = threadIdx.x;
    uint32_t ax = 0, first = 0;
    double b = a.ratio[0];
#pragma unroll
    for (uint32_t k = 1; k < 4; k++)
      if (k < a.axes && p >= a.pair_end[k - 1]) {
        ax = k;
        first = a.pair_end[k - 1];
        if (!a.one_spectrum) b = a.ratio[k];
      }
    uint32_t e = a.one_spectrum ? p : p - first;
    double f = 0.63661977236758134308;  // 2 / pi
#pragma unroll
    for (int k = 0; k < 7; k++) {  // e < 128
      if (e & 1) f *= b;
      b *= b;
      e >>= 1;
    }
    sfreq[p] = f;
    saxis[p] = ax;
  }
  lds_barrier();  // (leaves the loads in flight)

  const float inv_d = 1.0f / (float)a.d;
  while (unit < units) {
    float cs[NP], sn[NP];
    const float* pos = a.pos + n.b * a.pos_batch + (uint64_t)n.s * a.axes;
#pragma unroll
    for (int i = 0; i < NP; i++) {
      const uint32_t c = c0 + (HALVES ? i : 2 * i);
      cs[i] = 1.0f;
      sn[i] = 0.0f;
      if (c < 2 * a.pairs) {
        const uint32_t p = HALVES ? (c < a.pairs ? c : c - a.pairs) : c / 2;
        sincos_quarters((double)pos[saxis[p]] * sfreq[p], sn[i], cs[i]);
        if (HALVES && c < a.pairs) sn[i] = -sn[i];  // the sign of the partner's part
      }
    }
    T* q0 = (T*)Q.y + (n.b * Q.yb + n.s * Q.yt);
    T* k0 = (T*)K.y + (n.b * K.yb + n.s * K.yt);
    walk(n, (const char*)q0, (const char*)k0, Q.yh * (RPW * sizeof(T)), K.yh * (RPW * sizeof(T)),
         [&](int u, bool key, const char* p, bool ok) {
      float w[V];
      float q = 0.0f;
#pragma unroll
      for (int j = 0; j < V; j++) {
        w[j] = (float)xv[u][j];
        q = fmaf(w[j], w[j], q);
      }
      if (a.norm) {
        q = row_sum<LPR>(q);
        const float r = rsqrt_f(fmaf(q, inv_d, a.eps));
#pragma unroll
        for (int j = 0; j < V; j++) w[j] *= r * (key ? gam[1][j] : gam[0][j]);
      }
      if constexpr (!HALVES) {
#pragma unroll
        for (int i = 0; i < NP; i++) {
          const float x = w[2 * i], z = w[2 * i + 1];
          const bool turn = c0 + 2 * i < 2 * a.pairs;  // (an infinite neighbour stays out of the others)
          w[2 * i] = turn ? x * cs[i] - z * sn[i] : x;
          w[2 * i + 1] = turn ? z * cs[i] + x * sn[i] : z;
        }
      } else {
        // the wavefront's own strip: written and read by the same 64 lanes
        float* st = strip + wave * 64 * V + row * LPR * V;
#pragma unroll
        for (int j = 0; j < V; j += 4) *(f32x4*)(st + c0 + j) = f32x4{w[j], w[j + 1], w[j + 2], w[j + 3]};
        wave_lds_fence();
        float z[V];
        if (a.pairs % V == 0) {  // the partners of a lane's channels lie in one other lane
          const uint32_t pc = c0 < a.pairs ? c0 + a.pairs : c0 < 2 * a.pairs ? c0 - a.pairs : c0;
#pragma unroll
          for (int j = 0; j < V; j += 4) {
            const f32x4 t = *(const f32x4*)(st + pc + j);
#pragma unroll
            for (int k = 0; k < 4; k++) z[j + k] = t[k];
          }
        } else {
#pragma unroll
          for (int j = 0; j < V; j++) {
            const uint32_t c = c0 + j;
            z[j] = st[c < a.pairs ? c + a.pairs : c < 2 * a.pairs ? c - a.pairs : c];
          }
        }
        wave_lds_fence();
#pragma unroll
        for (int j = 0; j < V; j++) w[j] = c0 + j < 2 * a.pairs ? w[j] * cs[j] + z[j] * sn[j] : w[j];
      }
      if (!ok) return;
      T* y = (T*)p + (key ? lyk : lyq);
      if constexpr (VEC) {
        vec o;
#pragma unroll
        for (int j = 0; j < V; j++) o[j] = (T)w[j];
        *(vec*)y = o;
      } else {
#pragma unroll
        for (int j = 0; j < V; j++)
          if (c0 + j < a.d) y[j] = (T)w[j];
      }
    });
    unit += step;
    if (unit >= units) break;
    n = unit_of(unit);
    load(n);
  }
}

template <typename T, int LPR, int U>
void launch_u(const RopeArgs& a, bool halves, bool vec, uint32_t blocks, hipStream_t s) {
  if (halves && vec) k_qk_rope<T, LPR, U, true, true><<<blocks, 256, 0, s>>>(a);
  else if (halves) k_qk_rope<T, LPR, U, true, false><<<blocks, 256, 0, s>>>(a);
  else if (vec) k_qk_rope<T, LPR, U, false, true><<<blocks, 256, 0, s>>>(a);
  else k_qk_rope<T, LPR, U, false, false><<<blocks, 256, 0, s>>>(a);
}

template <typename T, int LPR>
void launch_lpr(RopeArgs a, bool halves, bool vec, int num_cus, hipStream_t s) {
  constexpr uint32_t RPW = 64 / LPR;
  const uint32_t sq = (a.t[0].H + RPW - 1) / RPW, steps = sq + (a.t[1].H + RPW - 1) / RPW;
  const uint64_t tokens = (uint64_t)a.B * a.S;
  // Steps per wavefront: long runs share one token's sines and keep more loads
  // in flight, as long as they leave every CU eight wavefronts.  2, 4 and 8
  // steps: 20280 tokens of 24 heads of 128 fp16 channels 60.7, 53.0 and 50.8 us,
  // 2048 tokens of 40 of 64 11.4, 9.5 and 8.3; 512 tokens (8 leave half the CUs
  // without work) 5.9, 5.7 and 6.1, 8 tokens 5.6, 5.7 and 6.2.
  auto units = [&](uint32_t u) { return tokens * ((steps + u - 1) / u); };
  const uint64_t enough = 8ull * num_cus;
  const uint32_t u = units(8) >= enough ? 8 : units(4) >= enough ? 4 : 2;
  a.steps_q = sq;
  a.steps = steps;
  a.segs = (steps + u - 1) / u;
  a.run = (steps + a.segs - 1) / a.segs;
  a.segs = (steps + a.run - 1) / a.run;
  const uint64_t n = (tokens * a.segs + 3) / 4, cap = (uint64_t)num_cus * 8;
  const uint32_t blocks = (uint32_t)(n < cap ? n : cap);
  if (u == 8) launch_u<T, LPR, 8>(a, halves, vec, blocks, s);
  else if (u == 4) launch_u<T, LPR, 4>(a, halves, vec, blocks, s);
  else launch_u<T, LPR, 2>(a, halves, vec, blocks, s);
}

template <typename T>
void launch_rope(const RopeArgs& a, bool halves, bool vec, int num_cus, hipStream_t s) {
  constexpr uint32_t V = 16 / sizeof(T);
  const uint32_t need = (a.d + V - 1) / V;
  if (need <= 2) launch_lpr<T, 2>(a, halves, vec, num_cus, s);
  else if (need <= 4) launch_lpr<T, 4>(a, halves, vec, num_cus, s);
  else if (need <= 8) launch_lpr<T, 8>(a, halves, vec, num_cus, s);
  else if (need <= 16) launch_lpr<T, 16>(a, halves, vec, num_cus, s);
  else if (need <= 32) launch_lpr<T, 32>(a, halves, vec, num_cus, s);
  else launch_lpr<T, 64>(a, halves, vec, num_cus, s);
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
  // (wavefront units, at most one per head, are counted in 32 bits)
  DI_REQUIRE((unsigned __int128)B * S * ((uint64_t)Hq + Hk) < 1ull << 31, DI_EUNSUPPORTED,
             "%s: %u x %u tokens of %llu heads", fn, B, S, (unsigned long long)Hq + Hk);
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
