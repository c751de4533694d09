// The first product of low-rank adapters beside a projection: the scaled inner
// products t[m][r] = scale[a] sum_k x[m][k] down[a][r][k] of each row with its
// own adapter's first factor (the second product runs as further k stages of
// the projection itself, k_gemm_kernel.h).
//
// D = down x^T on the 16x16 MFMAs: a wavefront holds 16 rows of x (columns of
// D) and RT tiles of 16 ranks, operands straight from memory as 16-byte
// vectors along k (fp32: v_mfma_f32_16x16x4 on four registers, whose k index
// runs over k = 4g + j); lane l then holds row l%16 and four consecutive ranks,
// one store.  Rows of one block may name several adapters: each distinct one
// is a slot, computed by a workgroup of its own (grid z) for all 16 rows and
// stored for the rows that name it, so a batch of single tokens with an adapter
// each runs them side by side.  KW wavefronts share a block's k (summed through
// LDS in order) where the blocks alone leave the chip idle.
#include "di_device.h"
#include "di_gemm.h"
#include "di_internal.h"

namespace di {

namespace {

struct LoraDownArgs {
  const void *x, *down;
  const float* scale;
  const int32_t* ids;
  void* t;
  uint32_t M, K, n, rank, ld, run;
};

template <typename T>
struct LoraMma;
template <>
struct LoraMma<f16> {
  typedef f16x8 frag;
  static constexpr int V = 8, KM = 32;  // values per lane and k per step
  __device__ static f32x4 mma(frag a, frag b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};
template <>
struct LoraMma<float> {
  typedef f32x4 frag;
  static constexpr int V = 4, KM = 16;
  __device__ static f32x4 mma(frag a, frag b, f32x4 c) {
#pragma unroll
    for (int j = 0; j < 4; j++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
    return c;
  }
};

// VEC: rows of x and down are whole 16-byte vectors
template <typename T, int RT, int KW, bool VEC>
__global__ __launch_bounds__(256) void k_lora_down(LoraDownArgs a) {
  typedef LoraMma<T> MM;
  typedef typename MM::frag frag;
  constexpr int V = MM::V, KM = MM::KM;
  __shared__ float red[KW > 1 ? (KW - 1) * RT * 256 : 1];
  kernarg_warm(a);
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
  const uint32_t kw = KW > 1 ? wave : 0, mb = KW > 1 ? blockIdx.x : blockIdx.x * 4 + wave;
  const uint32_t m = mb * 16 + r, rk0 = blockIdx.y * RT * 16;
  // the slot's adapter: the z-th distinct one of the block's rows
  int32_t id = -1;
  if (m < a.M) {
    id = a.ids[m / a.run];
    if ((uint32_t)id >= a.n) id = -1;
  }
  int32_t rest = id, ad = -1;
  for (uint32_t z = 0;; z++) {
    const uint64_t todo = __builtin_amdgcn_ballot_w64(rest >= 0);
    if (todo == 0) return;  // (all KW wavefronts of a block alike)
    ad = __builtin_amdgcn_readlane(rest, __builtin_ctzll(todo));
    if (z == blockIdx.z) break;
    if (rest == ad) rest = -1;
  }
  const T* X = (const T*)a.x + (uint64_t)(m < a.M ? m : 0) * a.K;
  const T* D = (const T*)a.down + (uint64_t)ad * a.rank * a.K;
  auto load = [&](const T* p, bool ok, uint32_t k) {
    frag v = {};
    if constexpr (VEC) {
      if (ok && k < a.K) v = *(const frag*)(p + k);
    } else if (ok) {
#pragma unroll
      for (int j = 0; j < V; j++)
        if (k + j < a.K) v[j] = p[k + j];
    }
    return v;
  };
  f32x4 acc[RT];
#pragma unroll
  for (int t = 0; t < RT; t++) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  // U steps' loads are issued together; steps past the last k load zeros
  constexpr int U = RT == 4 ? 2 : 4;
  for (uint32_t k0 = kw * KM; k0 < a.K; k0 += U * KW * KM) {
    frag xv[U], dv[U][RT];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const uint32_t k = k0 + u * KW * KM + g * V;
      xv[u] = load(X, true, k);
#pragma unroll
      for (int t = 0; t < RT; t++) {
        const uint32_t rk = rk0 + t * 16 + r;
        dv[u][t] = load(D + (uint64_t)(rk < a.rank ? rk : 0) * a.K, rk < a.rank, k);
      }
    }
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int t = 0; t < RT; t++) acc[t] = MM::mma(dv[u][t], xv[u], acc[t]);
  }
  if constexpr (KW > 1) {
    if (kw > 0)
#pragma unroll
      for (int t = 0; t < RT; t++)
#pragma unroll
        for (int j = 0; j < 4; j++) red[(((kw - 1) * RT + t) * 4 + j) * 64 + lane] = acc[t][j];
    __syncthreads();
    if (kw > 0) return;
#pragma unroll
    for (int w = 0; w < KW - 1; w++)
#pragma unroll
      for (int t = 0; t < RT; t++)
#pragma unroll
        for (int j = 0; j < 4; j++) acc[t][j] += red[((w * RT + t) * 4 + j) * 64 + lane];
  }
  if (id != ad) return;
  const float sc = a.scale ? a.scale[ad] : 1.0f;
#pragma unroll
  for (int t = 0; t < RT; t++) {
    const uint32_t rk = rk0 + t * 16 + g * 4;
    if (rk >= a.ld) continue;
    // (ld is a multiple of four; ranks past the last are zeros of zero rows)
    T* o = (T*)a.t + (uint64_t)m * a.ld + rk;
#pragma unroll
    for (int j = 0; j < 4; j++) o[j] = (T)(rk + j < a.rank ? acc[t][j] * sc : 0.0f);
  }
}

template <typename T, int RT, int KW>
void launch_down_vec(const LoraDownArgs& a, dim3 grid, hipStream_t s) {
  if (a.K % LoraMma<T>::V == 0) k_lora_down<T, RT, KW, true><<<grid, 256, 0, s>>>(a);
  else k_lora_down<T, RT, KW, false><<<grid, 256, 0, s>>>(a);
}

template <typename T>
void launch_down(const LoraDownArgs& a, int num_cus, hipStream_t s) {
  const uint32_t blocks = (a.M + 15) / 16, tiles = (a.rank + 15) / 16;
  // distinct adapters of 16 rows: no more than runs they can touch
  const uint32_t runs = a.run >= 16 ? 2 : a.run == 1 ? 16 : 15 / a.run + 2;
  const uint32_t slots = runs < a.n ? runs : a.n;
  const uint32_t rt = tiles >= 3 ? 4 : tiles;
  const bool split = blocks <= (uint32_t)num_cus * 4;
  const dim3 grid(split ? blocks : (blocks + 3) / 4, (tiles + rt - 1) / rt, slots < 16 ? slots : 16);
  if (split) {
    if (rt == 1) launch_down_vec<T, 1, 4>(a, grid, s);
    else if (rt == 2) launch_down_vec<T, 2, 4>(a, grid, s);
    else launch_down_vec<T, 4, 4>(a, grid, s);
  } else {
    if (rt == 1) launch_down_vec<T, 1, 1>(a, grid, s);
    else if (rt == 2) launch_down_vec<T, 2, 1>(a, grid, s);
    else launch_down_vec<T, 4, 1>(a, grid, s);
  }
}

}  // namespace

void launch_lora_down(const void* x, const void* down, const float* scale, const int32_t* ids, void* t,
                      uint32_t M, uint32_t K, uint32_t n, uint32_t rank, uint32_t ld, uint32_t run,
                      int elem, int num_cus, hipStream_t s) {
  const LoraDownArgs a{x, down, scale, ids, t, M, K, n, rank, ld, run};
  if (elem == DI_F32) launch_down<float>(a, num_cus, s);
  else launch_down<f16>(a, num_cus, s);
}

}  // namespace di
