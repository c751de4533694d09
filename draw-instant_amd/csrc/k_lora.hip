// The first product of low-rank adapters beside a projection: the scaled inner
// products t[m][r] = scale[a] sum_k x[m][k] down[a][r][k] of each row with its
// own adapter's first factor (the second product runs as further k stages of
// the projection itself, k_gemm_kernel.h).
//
// D = down x^T on the 16x16 MFMAs: a wavefront holds RF x 16 rows of x (columns
// of D) and RT x 16 ranks, operands straight from memory as 16-byte vectors along
// k (fp32: v_mfma_f32_16x16x4 on four registers, whose k index runs over k = 4g +
// j); lane l then holds row l%16 and four consecutive ranks, one store.  The
// four wavefronts of a workgroup take a quarter of k each, so that no operand
// passes the CU's load path twice, and are summed through LDS in order.  Rows
// of one block may name several adapters: each distinct one is a slot, computed
// by a workgroup of its own (grid z) for all its rows and stored for the rows that
// name it, so a batch of single tokens with an adapter each runs them side by
// side.  The first steps' rows of x are fetched before the ids are known.
// The work is little: a workgroup's few rounds of loads, one after the other, bound it
// (8192 rows of 1280 with rank 32, 21 MB, take 11.3 us, 1.9 TB/s), not HBM.
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
template <typename T, int RF, int RT, bool VEC>
__global__ __launch_bounds__(256) void k_lora_down(LoraDownArgs a) {
  typedef LoraMma<T> MM;
  typedef typename MM::frag frag;
  constexpr int V = MM::V, KM = MM::KM, KW = 4, NF = RF * RT, U = NF >= 16 ? 1 : NF >= 4 ? 2 : 4;
  __shared__ float red[(KW - 1) * NF * 256];
  kernarg_warm(a);
  const uint32_t lane = threadIdx.x & 63, kw = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t r = lane & 15, g = lane >> 4;
  const uint32_t m0 = blockIdx.x * RF * 16 + r, rk0 = blockIdx.y * RT * 16;
  // 16 bytes at element k of a row.  VEC: buffer loads, which read zeros where the
  // row or k is past the last without a branch around them; else element by element.
  constexpr uint32_t kOut = 0x80000000u;
  auto rsrc = [](const T* p, uint64_t n) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(p), (short)0, (int)(uint32_t)(n * sizeof(T)), 0x00020000);
  };
  // a row's place: its byte offset, without VEC its number
  auto row_at = [&](uint32_t row, bool ok) {
    return !ok ? kOut : VEC ? row * a.K * (uint32_t)sizeof(T) : row;
  };
  auto load = [&](__amdgpu_buffer_rsrc_t rs, const T* base, uint32_t at, uint32_t k) {
    if constexpr (VEC) {
      const uint32_t off = k < a.K ? at + k * (uint32_t)sizeof(T) : kOut;
      return __builtin_bit_cast(frag, __builtin_amdgcn_raw_buffer_load_b128(rs, off, 0, 0));
    } else {
      frag v = {};
      if (at != kOut) {
        const T* p = base + (uint64_t)at * a.K + k;
#pragma unroll
        for (int j = 0; j < V; j++)
          if (k + j < a.K) v[j] = p[j];
      }
      return v;
    }
  };
  // Adapters of the rows: two scalar loads where a run is as long as the block
  int32_t id[RF], rest[RF], a0 = -1, a1 = -1;
  const uint32_t first = blockIdx.x * RF * 16, q0 = __builtin_amdgcn_readfirstlane(first / a.run);
  const uint32_t cross = a.run - (first - q0 * a.run);  // first row of the next run
  const bool two = a.run >= RF * 16;
  if (two) {
    a0 = a.ids[q0];
    a1 = cross < min((uint32_t)(RF * 16), a.M - first) ? a.ids[q0 + 1] : a0;
    a0 = (uint32_t)a0 < a.n ? a0 : -1;
    a1 = (uint32_t)a1 < a.n ? a1 : -1;
  }
#pragma unroll
  for (int f = 0; f < RF; f++) {
    const uint32_t m = m0 + f * 16;
    id[f] = -1;
    if (m < a.M) {
      id[f] = two ? (f * 16 + r < cross ? a0 : a1) : a.ids[m / a.run];
      if ((uint32_t)id[f] >= a.n) id[f] = -1;
    }
    rest[f] = id[f];
  }
  // U steps' operands, loaded together; steps past the last k load zeros.  Two
  // sets, so that one is on its way while the other is multiplied (moved from one to
  // the other they would be waited for).
  struct Set {
    frag x[U][RF], d[U][RT];
  } s0, s1;
  const T* X = (const T*)a.x + (uint64_t)first * a.K;
  const __amdgpu_buffer_rsrc_t rX = rsrc(X, (uint64_t)min(a.M - first, (uint32_t)(RF * 16)) * a.K);
  uint32_t xat[RF];
#pragma unroll
  for (int f = 0; f < RF; f++) xat[f] = row_at(f * 16 + r, m0 + f * 16 < a.M);
  auto load_x = [&](Set& t, uint32_t k0) {
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int f = 0; f < RF; f++) t.x[u][f] = load(rX, X, xat[f], k0 + u * KW * KM + g * V);
  };
  load_x(s0, kw * KM);
  // the slot's adapter: the z-th distinct one of the block's rows
  int32_t ad = -1;
  if (two) {
    ad = blockIdx.z == 0 ? (a0 >= 0 ? a0 : a1) : a0 >= 0 && a1 != a0 ? a1 : -1;
    if (ad < 0) return;
  } else {
    for (uint32_t z = 0;; z++) {
      ad = -1;
#pragma unroll
      for (int f = 0; f < RF; f++) {
        const uint64_t todo = __builtin_amdgcn_ballot_w64(rest[f] >= 0);
        if (ad < 0 && todo != 0) ad = __builtin_amdgcn_readlane(rest[f], __builtin_ctzll(todo));
      }
      if (ad < 0) return;  // (all wavefronts of a workgroup alike)
      if (z == blockIdx.z) break;
#pragma unroll
      for (int f = 0; f < RF; f++)
        if (rest[f] == ad) rest[f] = -1;
    }
  }
  const T* D = (const T*)a.down + (uint64_t)ad * a.rank * a.K;
  const __amdgpu_buffer_rsrc_t rD = rsrc(D, (uint64_t)a.rank * a.K);
  uint32_t dat[RT];
#pragma unroll
  for (int t = 0; t < RT; t++) dat[t] = row_at(rk0 + t * 16 + r, rk0 + t * 16 + r < a.rank);
  auto load_d = [&](Set& s, uint32_t k0) {
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int t = 0; t < RT; t++) s.d[u][t] = load(rD, D, dat[t], k0 + u * KW * KM + g * V);
  };
  load_d(s0, kw * KM);
  f32x4 acc[RF][RT];
#pragma unroll
  for (int f = 0; f < RF; f++)
#pragma unroll
    for (int t = 0; t < RT; t++) acc[f][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto multiply = [&](const Set& s) {
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int f = 0; f < RF; f++)
#pragma unroll
        for (int t = 0; t < RT; t++) acc[f][t] = MM::mma(s.d[u][t], s.x[u][f], acc[f][t]);
  };
  constexpr uint32_t STEP = U * KW * KM;
  for (uint32_t k0 = kw * KM; k0 < a.K; k0 += 2 * STEP) {
    load_x(s1, k0 + STEP);
    load_d(s1, k0 + STEP);
    __builtin_amdgcn_sched_barrier(0);
    multiply(s0);
    load_x(s0, k0 + 2 * STEP);
    load_d(s0, k0 + 2 * STEP);
    __builtin_amdgcn_sched_barrier(0);
    multiply(s1);
  }
  if (kw > 0) {
#pragma unroll
    for (int f = 0; f < RF; f++)
#pragma unroll
      for (int t = 0; t < RT; t++)
#pragma unroll
        for (int j = 0; j < 4; j++) red[(((kw - 1) * NF + f * RT + t) * 4 + j) * 64 + lane] = acc[f][t][j];
  }
  __syncthreads();
  if (kw > 0) return;
  const float sc = a.scale ? a.scale[ad] : 1.0f;
  typedef T out4 __attribute__((ext_vector_type(4)));
#pragma unroll
  for (int f = 0; f < RF; f++)
#pragma unroll
    for (int t = 0; t < RT; t++) {
      f32x4 v = acc[f][t];
#pragma unroll
      for (int w = 0; w < KW - 1; w++)
#pragma unroll
        for (int j = 0; j < 4; j++) v[j] += red[((w * NF + f * RT + t) * 4 + j) * 64 + lane];
      const uint32_t rs = rk0 + t * 16 + g * 4;  // first of this lane's ranks
      if (id[f] != ad || rs >= a.ld) continue;
      // (ld is a multiple of four; ranks past the last are zeros of zero rows)
      out4 o;
#pragma unroll
      for (int j = 0; j < 4; j++) o[j] = (T)(rs + j < a.rank ? v[j] * sc : 0.0f);
      *(out4*)((T*)a.t + (uint64_t)(m0 + f * 16) * a.ld + rs) = o;
    }
}

template <typename T, int RF, int RT>
void launch_down_rt(const LoraDownArgs& a, hipStream_t s) {
  const uint32_t rows = RF * 16, tiles = (a.rank + 15) / 16;
  // distinct adapters of a block's rows: no more than the runs they can touch
  const uint32_t runs = a.run >= rows ? 2 : a.run == 1 ? rows : (rows - 1) / a.run + 2;
  const uint32_t slots = runs < a.n ? runs : a.n;
  const dim3 grid((a.M + rows - 1) / rows, (tiles + RT - 1) / RT, slots < rows ? slots : rows);
  // (a block's rows and an adapter's ranks are addressed with 31-bit offsets)
  const bool vec = a.K % LoraMma<T>::V == 0 && (uint64_t)a.K * (a.rank > rows ? a.rank : rows) * sizeof(T) < 0x7fff0000ull;
  if (vec) k_lora_down<T, RF, RT, true><<<grid, 256, 0, s>>>(a);
  else k_lora_down<T, RF, RT, false><<<grid, 256, 0, s>>>(a);
}

template <typename T>
void launch_down(const LoraDownArgs& a, uint32_t num_cus, hipStream_t s) {
  const uint32_t tiles = (a.rank + 15) / 16;
  // 64 rows a workgroup, an adapter's factor then read once for 64 rows and not
  // for 16, where those workgroups are half the CUs or more: 8192 rows of 1280 with
  // rank 32 11.3 us and by 16 rows 12.4, 16384 of 320 with rank 16 6.4 and 8.5,
  // 32768 of 320 with rank 64 13.5 and 22.9; 4096 of 640 with rank 32 8.3 and 5.5.
  const bool tall = a.M / 64 >= num_cus / 2u && a.run >= 64;
  if (tall) {
    if (tiles == 1) launch_down_rt<T, 4, 1>(a, s);
    else if (tiles == 2) launch_down_rt<T, 4, 2>(a, s);
    else launch_down_rt<T, 4, 4>(a, s);
  } else {
    if (tiles == 1) launch_down_rt<T, 1, 1>(a, s);
    else if (tiles == 2) launch_down_rt<T, 1, 2>(a, s);
    else launch_down_rt<T, 1, 4>(a, s);
  }
}

// Few rows: a workgroup takes one row and 256 columns, first the row's inner
// products (a rank per wavefront at a time, lanes along k), then its columns,
// one per thread.  Every workgroup of a row forms the products again: they are
// small, and the adapters' share of the projection is one launch.
__global__ __launch_bounds__(256) void k_lora_rows(LoraDownArgs a, const f16* up, float* d, uint32_t N) {
  __shared__ float st[256];
  kernarg_warm(a);
  const uint32_t m = blockIdx.y, n = blockIdx.x * 256 + threadIdx.x;
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int32_t id = a.ids[m / a.run];
  if ((uint32_t)id >= a.n) {
    if (n < N) d[(uint64_t)m * N + n] = 0.0f;
    return;
  }
  const f16* x = (const f16*)a.x + (uint64_t)m * a.K;
  const f16* D = (const f16*)a.down + (uint64_t)id * a.rank * a.K;
  const float sc = a.scale ? a.scale[id] : 1.0f;
  const bool vec = a.K % 8 == 0;
  constexpr int U = 4;  // ranks of a wavefront whose loads are issued together
  for (uint32_t r0 = wave * U; r0 < a.rank; r0 += 4 * U) {
    float s[U] = {};
    if (vec) {
      for (uint32_t k = lane * 8; k < a.K; k += 512) {
        const f16x8 xv = *(const f16x8*)(x + k);
        f16x8 dv[U];
#pragma unroll
        for (int u = 0; u < U; u++) dv[u] = *(const f16x8*)(D + (uint64_t)min(r0 + u, a.rank - 1) * a.K + k);
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
          for (int j = 0; j < 8; j++) s[u] = fmaf((float)xv[j], (float)dv[u][j], s[u]);
      }
    } else {
      for (uint32_t k = lane; k < a.K; k += 64)
#pragma unroll
        for (int u = 0; u < U; u++)
          s[u] = fmaf((float)x[k], (float)D[(uint64_t)min(r0 + u, a.rank - 1) * a.K + k], s[u]);
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      const float t = wave_sum(s[u]);
      if (lane == 0 && r0 + u < a.rank) st[r0 + u] = (float)(f16)(t * sc);
    }
  }
  __syncthreads();
  if (n >= N) return;
  const f16* p = up + ((uint64_t)id * N + n) * a.rank;
  float y = 0.0f;
  if (a.rank % 8 == 0) {
    for (uint32_t r = 0; r < a.rank; r += 8) {
      const f16x8 v = *(const f16x8*)(p + r);
#pragma unroll
      for (int j = 0; j < 8; j++) y = fmaf(st[r + j], (float)v[j], y);
    }
  } else {
    for (uint32_t r = 0; r < a.rank; r++) y = fmaf(st[r], (float)p[r], y);
  }
  d[(uint64_t)m * N + n] = y;
}

}  // namespace

void launch_lora_rows(const void* x, const void* down, const void* up, const float* scale, const int32_t* ids,
                      float* d, uint32_t M, uint32_t N, uint32_t K, uint32_t n, uint32_t rank, uint32_t run,
                      hipStream_t s) {
  const LoraDownArgs a{x, down, scale, ids, nullptr, M, K, n, rank, 0, run};
  k_lora_rows<<<dim3((N + 255) / 256, M), 256, 0, s>>>(a, (const f16*)up, d, N);
}

void launch_lora_down(const void* x, const void* down, const float* scale, const int32_t* ids, void* t,
                      uint32_t M, uint32_t K, uint32_t n, uint32_t rank, uint32_t ld, uint32_t run,
                      int elem, int num_cus, hipStream_t s) {
  const LoraDownArgs a{x, down, scale, ids, t, M, K, n, rank, ld, run};
  if (elem == DI_F32) launch_down<float>(a, (uint32_t)num_cus, s);
  else launch_down<f16>(a, (uint32_t)num_cus, s);
}

}  // namespace di
