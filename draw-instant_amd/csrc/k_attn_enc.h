// Flash attention to an encoder's states: any head size up to 256, lengths per
// batch entry, additive biases, query heads that share key heads; fp16 on the
// fp16 MFMA, fp32 on the fp32 MFMA.
//
//   o = softmax(scale q k^T + bias) v
//
// Rows.  The G query heads that share a key head are rows beside its queries:
// row = query * G + head, so that one read of a key serves all of them, and a
// single token's heads fill a 16-row MFMA tile together.
//
// MFMA mapping, as in k_attn.hip: S^T = K Q^T, the C layout leaving lane l row
// l%16 and keys 4g..4g+3 (g = l/16) of each 16-key tile; scale * log2(e) comes
// in with the maximum, one fma before the exp2 (folded into Q it would cost no
// instruction less here and round fp16 queries a second time: 4.3e-4 instead of
// 3.0e-4 off 64 bits at 512 keys);
// O^T += V^T P^T takes those probabilities as its B operand without moving
// them.  fp16: v_mfma_f32_16x16x32_f16, the V^T operand by transposed LDS
// reads.  fp32: v_mfma_f32_16x16x4_f32 on four registers of a 16-byte read,
// whose k index runs over channels (keys) 4g + j for j = 0..3.
//
// Softmax in one pass: a running maximum m per row, taken from the first keys
// that a row has and raised only when a lane's probabilities of a tile pass
// 2^15 (fp16-safe), then the tile is redone; row sums once, at the end.  m stays
// at kNone until a row has seen a key, so rows that a mask leaves empty end
// with a zero sum and store zeros.
//
// Keys come in tiles of KT through LDS (loads go straight to LDS; 16-byte
// chunks XOR-swizzled by row so that fragment reads meet no bank twice).  Rows
// are padded to DK channels in registers and to a power of two of chunks in LDS;
// chunks past d and keys past the length are never read from memory and land
// as zeros.  The loop is pipelined over tiles: the scores of tile t + 1 are
// multiplied before the exponentials of tile t, which do not wait for them, then
// tile t's probabilities meet its values; of two wavefronts on a SIMD one then
// has matrix work while the other has vector work.  (Matrix and exponential
// instructions of one wavefront in alternation were slower: 2 x 16 x 8190 rows of
// 128 over 512 keys 88.8 -> 93.2 us, 8 heads of 2048 x 1024 of 256 27.9 -> 34.3.)
// K is therefore fetched two tiles ahead and V one, each into two buffers.
//
// Biases.  A wavefront's tile without a value at or below kSwamped only has its
// products with log2(e) taken; else scores and values are looked at one by one,
// and the keys that no row sees are found by an or over the rows' bit masks: only
// a tile with such a key has its values masked (2 x 10 heads of 2048 x 1024 keys of
// 64, a third of the keys removed at random: 53 -> 46 us, fp32 140 -> 127; none
// removed 43 -> 40).
//
// WM wavefronts share a tile, each with QG groups of 16 rows; WK such groups
// of wavefronts walk different tiles of the same rows and are merged through
// LDS.  Forms: many rows, WM = 4 and QG = 2 (two groups share every fragment
// read); up to 64 rows, WM = 4 and QG = 1; few rows (a token, a handful of
// latents), WM = 1 and WK = 2 to 8, so that every wavefront streams keys of its own.
// Where the rows still leave CUs idle the keys are split over workgroups as
// well and k_attn_enc_merge joins the parts.
#pragma once

#include <type_traits>

#include "di_attn_enc.h"
#include "di_device.h"

namespace di {

namespace {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef __attribute__((address_space(3))) void* lds_ptr;
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

constexpr float kNone = -3.402823466e38f;  // maximum of a row without a key so far
constexpr float kSwamped = -1e30f;         // a bias that replaces its score
constexpr float kLowest = -3.0e38f;        // the lowest one in log2 units: above kNone
// a lane's probabilities of one tile sum to at most this without a rescale,
// so none exceeds it either (fp16 max is 65504)
constexpr uint32_t kLaneSumMaxBits = 0x47000000u;  // 32768.0f
constexpr float kLog2E = 1.4426950408889634f;
// s_waitcnt: all but the last n vector memory operations; the same and all LDS
// operations
constexpr int wait_vm(int n) { return (n & 15) | (n >> 4) << 14 | 7 << 4 | 15 << 8; }
constexpr int wait_vm_lds(int n) { return (n & 15) | (n >> 4) << 14 | 7 << 4; }

template <int N>
using Int = std::integral_constant<int, N>;

__device__ __forceinline__ __amdgpu_buffer_rsrc_t enc_rsrc(const void* p, uint32_t bytes) {
  // raw buffer, stride 0; dword3 0x00020000 is the gfx9-family data format
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), (short)0, (int)bytes, 0x00020000);
}

// 16 bytes per lane at off of r straight to LDS, lane l's at p + 16 l
__device__ __forceinline__ void load_lds16(__amdgpu_buffer_rsrc_t r, unsigned char* p, uint32_t off) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_ptr)p, 16, off, 0, 0, 0);
}

// Orders LDS accesses of one wavefront's lanes, which the hardware keeps in
// order by itself, for the compiler.
__device__ __forceinline__ void enc_lds_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// lanes l, l^16, l^32, l^48 hold the same row
__device__ __forceinline__ float enc_max4(float x) {
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float enc_sum4(float x) {
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// or of the 16 lanes that hold one group's rows
template <int CTRL>
__device__ __forceinline__ uint32_t enc_or_dpp(uint32_t x) {
  return x | (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xf, 0xf, true);
}
__device__ __forceinline__ uint32_t enc_or16(uint32_t x) {
  x = enc_or_dpp<0xB1>(x);    // quad_perm 1 0 3 2
  x = enc_or_dpp<0x4E>(x);    // quad_perm 2 3 0 1
  x = enc_or_dpp<0x141>(x);   // row_half_mirror
  return enc_or_dpp<0x140>(x);  // row_mirror
}

// Shapes of one instantiation.
template <typename T, int DK, int FORM>
struct EncShape {
  static constexpr bool F32 = sizeof(T) == 4;
  static constexpr bool FEW = FORM == ENC_FEW;
  static constexpr int EPC = 16 / sizeof(T);  // elements per 16-byte chunk
  // chunks of an LDS row: a power of two
  static constexpr int C0 = DK / EPC;
  static constexpr int CPR = C0 <= 4 ? 4 : C0 <= 8 ? 8 : C0 <= 16 ? 16 : C0 <= 32 ? 32 : 64;
  // Keys per tile: 32 where the wavefronts share out whole loads, 16 where an
  // fp32 tile would pass 16 KiB.  (64 at up to 128 channels: 2 x 16 x 8192 rows
  // over 512 keys 81.3 us at 128 channels and 49.8 at 64, 80.3 and 45.8 so, with
  // room for more workgroups on a CU.)
  static constexpr int KT = CPR == 4 && !FEW ? 64 : F32 && CPR >= (FEW ? 32 : 64) ? 16 : 32;
  static constexpr int TILE = KT * CPR * 16;  // bytes of a K (V) tile
  static constexpr int WM = FEW ? 1 : 4;
  // as many wavefronts' buffers as fit the 160 KiB of LDS
  static constexpr int WK = !FEW ? 1 : TILE * 4 * 8 <= 128 * 1024 ? 8 : TILE * 4 * 4 <= 128 * 1024 ? 4 : 2;
  // two row groups where their accumulators leave room for two wavefronts a SIMD
  static constexpr int QG = FORM == ENC_MANY && !F32 && DK <= 128 ? 2 : 1;
  static constexpr int ROWS = WM * QG * 16;
  static constexpr int NT = WM * WK * 64;
  static constexpr int LDS = WK * 4 * TILE;  // [key group][K | V][buffer]
  // wavefronts per SIMD that registers are kept for: what the LDS lets reside
  // (fp32 at 256 channels takes more than half of a SIMD's registers)
  static constexpr int WAVES = LDS * 2 <= 160 * 1024 && !(F32 && DK > 192) ? 2 : 1;
};

template <typename T, int DK, int FORM, bool BIAS>
__global__ __launch_bounds__((EncShape<T, DK, FORM>::NT), (EncShape<T, DK, FORM>::WAVES))
void k_attn_enc(AttnEncArgs a) {
  typedef EncShape<T, DK, FORM> Sh;
  constexpr bool F32 = Sh::F32;
  constexpr int EPC = Sh::EPC, CPR = Sh::CPR, KT = Sh::KT, TILE = Sh::TILE, WM = Sh::WM, WK = Sh::WK;
  constexpr int QG = Sh::QG, NKT = KT / 16, NDT = DK / 16;
  constexpr int RB = CPR * 16;                // bytes of an LDS row
  constexpr int QC = F32 ? DK / 16 : DK / 32; // K fragment reads per 16-key tile
  __shared__ __attribute__((aligned(16))) unsigned char smem[Sh::LDS];
  kernarg_warm(a);

  const uint32_t tid = threadIdx.x, lane = tid & 63;
  const uint32_t wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t wm = wv % WM, kg = wv / WM;
  const uint32_t r = lane & 15, g = lane >> 4;

  // XCD-aware numbering: block i runs on XCD i % 8; XCD x takes the x-th
  // contiguous run of the work list, so a head's keys stay in one L2
  const uint32_t T_ = gridDim.x, bid = blockIdx.x, xcd = bid & 7u, idx = bid >> 3;
  const uint32_t per = T_ >> 3, extra = T_ & 7u;
  const uint32_t w = xcd < extra ? xcd * (per + 1) + idx : extra * (per + 1) + (xcd - extra) * per + idx;
  // (heads_first: the heads of a block of rows side by side instead, as they
  // read one bias)
  const bool hf = BIAS && a.heads_first;
  const uint32_t n0 = hf ? a.Hk : a.blocks, r0 = w / n0, i0 = w - r0 * n0;
  const uint32_t n1 = hf ? a.blocks : a.splits, r1 = r0 / n1, i1 = r0 - r1 * n1;
  const uint32_t n2 = hf ? a.splits : a.Hk, b = r1 / n2, i2 = r1 - b * n2;
  const uint32_t mb = hf ? i1 : i0, split = hf ? i2 : i1, h = hf ? i0 : i2, hb = b * a.Hk + h;

  // this entry's keys; its tiles [t0, t1) of this workgroup's range and key group
  uint32_t nk = a.Skv;
  if (a.len) {
    const int n = a.len[b];
    nk = n <= 0 ? 0u : min((uint32_t)n, a.Skv);
  }
  nk = __builtin_amdgcn_readfirstlane(nk);
  const int n_tiles = (int)((nk + KT - 1) / KT);
  const int tps = (n_tiles + (int)a.splits - 1) / (int)a.splits;
  const int w0 = min((int)split * tps, n_tiles), w1 = min(w0 + tps, n_tiles);
  const int tpg = (w1 - w0 + WK - 1) / WK;
  const int t0 = min(w0 + (int)kg * tpg, w1), t1 = min(t0 + tpg, w1);

  const T* K = (const T*)a.k + b * a.bk + h * a.hk;
  const T* V = (const T*)a.v + b * a.bv + h * a.hv;

  // rows of this lane
  uint32_t row[QG], qh[QG], qi_[QG];
  bool live[QG];
#pragma unroll
  for (int i = 0; i < QG; i++) {
    row[i] = mb * Sh::ROWS + (wm * QG + i) * 16 + r;
    live[i] = row[i] < a.rows;
    const uint32_t rr = live[i] ? row[i] : 0;
    qi_[i] = a.G == 1 ? rr : rr / a.G;
    qh[i] = h * a.G + (rr - qi_[i] * a.G);
  }

  // Q' fragments: fp16 lane (r, g) channels 32 c + 8 g .. + 7, fp32 16 c + 4 g .. + 3
  typedef typename std::conditional<F32, f32x4, f16x8>::type frag;
  frag qf[QG][QC];
#pragma unroll
  for (int i = 0; i < QG; i++) {
    const T* p = (const T*)a.q + b * a.bq + qh[i] * a.hq + (uint64_t)qi_[i] * a.ldq;
#pragma unroll
    for (int c = 0; c < QC; c++) {
      const uint32_t e = (c * 4 + g) * EPC;
      qf[i][c] = frag{};
      if (live[i] && e < a.d) qf[i][c] = *(const frag*)(p + e);
    }
  }
  const float* bp[QG];
  if constexpr (BIAS) {
#pragma unroll
    for (int i = 0; i < QG; i++)
      bp[i] = a.bias + b * a.bias_b + qh[i] * a.bias_h + qi_[i] * a.bias_q;
  }

  // LDS swizzles, on 16-byte chunks.  K: the 16 rows that one pass of a
  // fragment read takes at one chunk land on all 64 banks.  V, fp16: a
  // 32-lane pass of a transposed read covers 8 rows x 2 chunks; fp32: the four
  // rows 4g + j of a read cover 64 bytes each.
  auto kswz = [](uint32_t row) -> uint32_t {
    if constexpr (CPR == 4) return (row >> 2) & 3u;
    else if constexpr (CPR == 8) return (row >> 1) & 7u;
    else return row & 15u;
  };
  auto vswz = [](uint32_t row) -> uint32_t {
    if constexpr (F32) return (((row >> 2) & 3u) << 2) & (CPR - 1);
    else if constexpr (CPR == 4) return ((row >> 2) & 1u) << 1;
    else if constexpr (CPR == 8) return row & 7u;
    else return (row & 7u) << 1;
  };

  // loads of a tile: 64 chunks (1 KiB of LDS) per instruction, lane l's chunk
  // at base + 16 l; a chunk past d gets an offset out of range
  constexpr int NI = TILE / (1024 * WM);
  static_assert(NI >= 1 && NI * 1024 * WM == TILE, "whole instructions per wavefront");
  uint32_t dk[NI], dv[NI];
#pragma unroll
  for (int i = 0; i < NI; i++) {
    const uint32_t f = (wm * NI + i) * 64 + lane, kr = f / CPR, sl = f % CPR;
    const uint32_t ck = sl ^ kswz(kr), cv = sl ^ vswz(kr);
    dk[i] = ck * EPC < a.d ? kr * (uint32_t)(a.ldk * sizeof(T)) + ck * 16u : 0x80000000u;
    dv[i] = cv * EPC < a.d ? kr * (uint32_t)(a.ldv * sizeof(T)) + cv * 16u : 0x80000000u;
  }
  unsigned char* const lds = smem + kg * 4 * TILE;
  auto fetch_k = [&](int t, auto buf_c) {
    const uint32_t key0 = (uint32_t)t * KT, left = min(nk - key0, (uint32_t)KT);
    const __amdgpu_buffer_rsrc_t rs = enc_rsrc(K + (uint64_t)key0 * a.ldk,
                                               (uint32_t)(((left - 1) * a.ldk + a.d) * sizeof(T)));
    unsigned char* base = lds + decltype(buf_c)::value * TILE + wm * NI * 1024;
#pragma unroll
    for (int i = 0; i < NI; i++) load_lds16(rs, base + i * 1024, dk[i]);
  };
  auto fetch_v = [&](int t, auto buf_c) {
    const uint32_t key0 = (uint32_t)t * KT, left = min(nk - key0, (uint32_t)KT);
    const __amdgpu_buffer_rsrc_t rs = enc_rsrc(V + (uint64_t)key0 * a.ldv,
                                               (uint32_t)(((left - 1) * a.ldv + a.d) * sizeof(T)));
    unsigned char* base = lds + (2 + decltype(buf_c)::value) * TILE + wm * NI * 1024;
#pragma unroll
    for (int i = 0; i < NI; i++) load_lds16(rs, base + i * 1024, dv[i]);
  };

  // K fragment c of 16-key tile kt: row kt * 16 + r, chunk 4 c + g
  uint32_t k_rd[QC];
#pragma unroll
  for (int c = 0; c < QC; c++) k_rd[c] = r * RB + (((4 * c + g) ^ kswz(r)) << 4);
  // V^T fragments.  fp16, 16 channels dt: lane r of group g reads 4 channels
  // of row 4g + r/4 at 16 dt + 4 (r%4).  fp32: channel 16 dt + r of row 4g + j.
  uint32_t v_rd[NDT];
#pragma unroll
  for (int dt = 0; dt < NDT; dt++) {
    if constexpr (F32)
      v_rd[dt] = 2 * TILE + 4 * g * RB + (((4 * dt + (r >> 2)) ^ vswz(4 * g)) << 4) + (r & 3) * 4;
    else
      v_rd[dt] = 2 * TILE + (4 * g + (r >> 2)) * RB +
                 (((2 * dt + ((r & 3) >> 1)) ^ vswz(4 * g + (r >> 2))) << 4) + (r & 1) * 8;
  }

  float m[QG], l[QG];
  f32x4 o[QG][NDT];
#pragma unroll
  for (int i = 0; i < QG; i++) {
    m[i] = kNone;
    l[i] = 0.0f;
#pragma unroll
    for (int dt = 0; dt < NDT; dt++) o[i][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  // q k^T of tile t, in K buffer `buf`; keys past the last are -inf
  auto scores = [&](int t, auto buf_c, f32x4 (&s)[QG][NKT]) {
    const unsigned char* sb = lds + decltype(buf_c)::value * TILE;
#pragma unroll
    for (int kt = 0; kt < NKT; kt++) {
#pragma unroll
      for (int i = 0; i < QG; i++) s[i][kt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < QC; c++) {
        const frag kf = *(const frag*)(sb + k_rd[c] + kt * 16 * RB);
#pragma unroll
        for (int i = 0; i < QG; i++) {
          if constexpr (F32) {
#pragma unroll
            for (int j = 0; j < 4; j++)
              s[i][kt] = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[j], qf[i][c][j], s[i][kt], 0, 0, 0);
          } else {
            s[i][kt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[i][c], s[i][kt], 0, 0, 0);
          }
        }
      }
    }
  };
  auto cut = [&](int t, f32x4 (&s)[QG][NKT]) {
    const uint32_t key0 = (uint32_t)t * KT;
    if (key0 + KT <= nk) return;
#pragma unroll
    for (int kt = 0; kt < NKT; kt++)
#pragma unroll
      for (int j = 0; j < 4; j++)
        if (key0 + kt * 16 + 4 * g + j >= nk) {
#pragma unroll
          for (int i = 0; i < QG; i++) s[i][kt][j] = -INFINITY;
        }
  };
  // the bias of tile t on its way (past the last key: unread), and the current one
  f32x4 bb[BIAS ? QG : 1][BIAS ? NKT : 1], bn[BIAS ? QG : 1][BIAS ? NKT : 1];
  auto load_bias = [&](int t) {
    if constexpr (BIAS) {
      const uint32_t key0 = (uint32_t)t * KT;
#pragma unroll
      for (int i = 0; i < QG; i++)
#pragma unroll
        for (int kt = 0; kt < NKT; kt++) {
          const uint32_t key = key0 + kt * 16 + 4 * g;
          if (key0 + KT <= nk) {
            bn[i][kt] = *(const f32x4u*)(bp[i] + key);
          } else {
#pragma unroll
            for (int j = 0; j < 4; j++) bn[i][kt][j] = key + j < nk ? bp[i][key + j] : -INFINITY;
          }
        }
    }
  };
  // The loaded bias becomes the current one; whether a value of the wavefront
  // needs more than its product with log2(e).
  auto take_bias = [&]() -> bool {
    float low = 0.0f;
    if constexpr (BIAS) {
#pragma unroll
      for (int i = 0; i < QG; i++)
#pragma unroll
        for (int kt = 0; kt < NKT; kt++) {
          bb[i][kt] = bn[i][kt];
#pragma unroll
          for (int j = 0; j < 4; j++) low = fminf(low, bb[i][kt][j]);
        }
    }
    return BIAS && __builtin_amdgcn_ballot_w64(low <= kSwamped) != 0;
  };
  // The current bias in log2 units and its effect on scores that do not count;
  // the keys that some row of this wavefront sees: bit 4 kt + j for key kt * 16 + 4g
  // + j.
  constexpr uint32_t ALL = (1u << (4 * NKT)) - 1;
  auto apply_bias = [&](f32x4 (&s)[QG][NKT], bool low) -> uint32_t {
    uint32_t seen = ALL;
    if constexpr (BIAS) {
      if (low) {
        seen = 0;
#pragma unroll
        for (int i = 0; i < QG; i++) {
          uint32_t own = 0;
#pragma unroll
          for (int kt = 0; kt < NKT; kt++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
              const float x = bb[i][kt][j];
              const bool gone = x == -INFINITY;
              own |= gone ? 0u : 1u << (4 * kt + j);
              if (x <= kSwamped) s[i][kt][j] = 0.0f;  // whatever the score: it may be NaN
              // (the product of a finite bias stays finite)
              bb[i][kt][j] = gone ? x : fmaxf(x * kLog2E, kLowest);
            }
          seen |= live[i] ? own : 0u;
        }
        seen = enc_or16(seen);
      } else {
#pragma unroll
        for (int i = 0; i < QG; i++)
#pragma unroll
          for (int kt = 0; kt < NKT; kt++) bb[i][kt] *= kLog2E;
      }
    }
    return seen;
  };
  // raise the running maximum to this tile's where that is larger
  auto raise = [&](int i, f32x4 (&s)[QG][NKT]) {
    float mx = -INFINITY;
#pragma unroll
    for (int kt = 0; kt < NKT; kt++)
#pragma unroll
      for (int j = 0; j < 4; j++)
        mx = fmaxf(mx, BIAS ? fmaf(s[i][kt][j], a.scale_log2, bb[i][kt][j]) : s[i][kt][j]);
    mx = fmaxf(BIAS ? enc_max4(mx) : enc_max4(mx) * a.scale_log2, m[i]);
    const float al = m[i] == kNone ? 0.0f : __builtin_amdgcn_exp2f(m[i] - mx);
    m[i] = mx;
    l[i] *= al;
#pragma unroll
    for (int dt = 0; dt < NDT; dt++) o[i][dt] *= al;
  };
  // probabilities, and their sum over this lane's keys.  A row without a key
  // so far has m = kNone: its first ones come out infinite.
  float pr[QG][NKT][4], ts[QG];
  auto probs = [&](int i, f32x4 (&s)[QG][NKT]) {
    ts[i] = 0.0f;
#pragma unroll
    for (int kt = 0; kt < NKT; kt++)
#pragma unroll
      for (int j = 0; j < 4; j++) {
        // with a bias, (bias - m) first: it is exact where they are close
        pr[i][kt][j] = __builtin_amdgcn_exp2f(fmaf(s[i][kt][j], a.scale_log2, BIAS ? bb[i][kt][j] - m[i] : -m[i]));
        ts[i] += pr[i][kt][j];
      }
  };
  // O^T += V^T P^T with tile t's values, in V buffer `buf`.  MASKED: the values
  // of keys that none of this wavefront's rows sees (not in `seen`) become zeros, as
  // 0 * NaN would not vanish.
  auto values = [&](auto buf_c, auto masked_c, uint32_t seen) {
    constexpr bool MASKED = decltype(masked_c)::value != 0;
    const unsigned char* sb = lds + decltype(buf_c)::value * TILE;
    if constexpr (F32) {
#pragma unroll
      for (int kt = 0; kt < NKT; kt++)
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
          for (int dt = 0; dt < NDT; dt++) {
            float vf = *(const float*)(sb + v_rd[dt] + (kt * 16 + j) * RB);
            if constexpr (MASKED) vf = (seen >> (4 * kt + j)) & 1u ? vf : 0.0f;
#pragma unroll
            for (int i = 0; i < QG; i++)
              o[i][dt] = __builtin_amdgcn_mfma_f32_16x16x4f32(vf, pr[i][kt][j], o[i][dt], 0, 0, 0);
          }
    } else {
#pragma unroll
      for (int c = 0; c < NKT / 2; c++) {
        f16x8 pf[QG];
#pragma unroll
        for (int i = 0; i < QG; i++)
#pragma unroll
          for (int j = 0; j < 8; j++) pf[i][j] = (f16)pr[i][2 * c + j / 4][j % 4];
        u32x4 keep = {~0u, ~0u, ~0u, ~0u};
        if constexpr (MASKED) {
#pragma unroll
          for (int j = 0; j < 4; j++)
            keep[j] = ((seen >> (8 * c + 2 * j)) & 1u ? 0xffffu : 0u) |
                      ((seen >> (8 * c + 2 * j + 1)) & 1u ? 0xffff0000u : 0u);
        }
#pragma unroll
        for (int dt = 0; dt < NDT; dt++) {
          const unsigned char* vp = sb + v_rd[dt] + c * 32 * RB;
          const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)vp);
          const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(vp + 16 * RB));
          f16x8 vf = __builtin_bit_cast(f16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
          if constexpr (MASKED) vf = __builtin_bit_cast(f16x8, __builtin_bit_cast(u32x4, vf) & keep);
#pragma unroll
          for (int i = 0; i < QG; i++)
            o[i][dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pf[i], o[i][dt], 0, 0, 0);
        }
      }
    }
  };
  // Every load but the last n of this wavefront's has landed, and its LDS reads
  // are done; wavefronts that share tiles meet.
  auto meet = [&](auto n_c) {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_waitcnt(wait_vm_lds(decltype(n_c)::value));
    if constexpr (WM > 1) __builtin_amdgcn_s_barrier();
    else __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
  };

  // Tile t with its scores in `s`; those of t + 1 go to `sn`.
  auto step = [&](auto cur_c, int t, f32x4 (&s)[QG][NKT], f32x4 (&sn)[QG][NKT]) {
    constexpr int cur = decltype(cur_c)::value;
    if (t + 2 < t1) fetch_k(t + 2, Int<cur>{});
    if (t + 1 < t1) fetch_v(t + 1, Int<cur ^ 1>{});
    const bool low = take_bias();
    if (t + 1 < t1) {
      load_bias(t + 1);
      scores(t + 1, Int<cur ^ 1>{}, sn);
    }
    const uint32_t seen = apply_bias(s, low);
#pragma unroll
    for (int i = 0; i < QG; i++) probs(i, s);
#pragma unroll
    for (int i = 0; i < QG; i++) {
      // a probability above 2^15 (or inf / NaN) shows in its lane's sum; the
      // bits' order puts finite < inf < NaN
      if (__builtin_amdgcn_ballot_w64((__float_as_uint(ts[i]) & 0x7fffffffu) > kLaneSumMaxBits) != 0) {
        raise(i, s);
        probs(i, s);
      }
      l[i] += ts[i];
    }
    if (BIAS && __builtin_amdgcn_ballot_w64(seen != ALL) != 0) {
      values(cur_c, Int<1>{}, seen);
    } else {
      values(cur_c, Int<0>{}, 0u);
    }
    if (t + 1 < t1) {
      cut(t + 1, sn);
      meet(Int<0>{});
    }
  };

  if (t0 < t1) {
    fetch_k(t0, Int<0>{});
    fetch_v(t0, Int<0>{});
    if (t0 + 1 < t1) {
      fetch_k(t0 + 1, Int<1>{});
      meet(Int<2 * NI>{});
    } else {
      meet(Int<NI>{});
    }
    f32x4 s0[QG][NKT], s1[QG][NKT];
    load_bias(t0);
    scores(t0, Int<0>{}, s0);
    cut(t0, s0);
    meet(Int<0>{});
    bool first = true;
    // two tiles per iteration so that each LDS buffer has fixed offsets
    for (int t = t0; t < t1; t += 2) {
      if (!BIAS && first) {
#pragma unroll
        for (int i = 0; i < QG; i++) raise(i, s0);
        first = false;
      }
      step(Int<0>{}, t, s0, s1);
      if (t + 1 < t1) step(Int<1>{}, t + 1, s1, s0);
    }
  }
#pragma unroll
  for (int i = 0; i < QG; i++) l[i] = enc_sum4(l[i]);

  if constexpr (WK > 1) {
    // merge the key groups: groups 1.. leave (o, m, l) in LDS, float f of lane
    // l at [f][l]; group 0 rescales every part to the largest maximum
    static_assert(WK == 1 || QG == 1, "key groups with one row group");
    constexpr int NF = NDT * 4 + 2;
    static_assert((WK - 1) * WM * NF * 64 * 4 <= Sh::LDS, "the parts fit the buffers");
    float* xs = reinterpret_cast<float*>(smem);
    __syncthreads();  // the buffers are free
    if (kg > 0) {
      float* dst = xs + ((kg - 1) * WM + wm) * NF * 64 + lane;
#pragma unroll
      for (int dt = 0; dt < NDT; dt++)
#pragma unroll
        for (int j = 0; j < 4; j++) dst[(dt * 4 + j) * 64] = o[0][dt][j];
      dst[NDT * 4 * 64] = m[0];
      dst[(NDT * 4 + 1) * 64] = l[0];
    }
    __syncthreads();
    if (kg > 0) return;
    float mx = m[0];
#pragma unroll
    for (int k = 1; k < WK; k++) mx = fmaxf(mx, xs[((k - 1) * WM + wm) * NF * 64 + NDT * 4 * 64 + lane]);
    float wk = __builtin_amdgcn_exp2f(m[0] - mx);
    l[0] *= wk;
#pragma unroll
    for (int dt = 0; dt < NDT; dt++) o[0][dt] *= wk;
#pragma unroll
    for (int k = 1; k < WK; k++) {
      const float* src = xs + ((k - 1) * WM + wm) * NF * 64 + lane;
      wk = __builtin_amdgcn_exp2f(src[NDT * 4 * 64] - mx);
      l[0] += src[(NDT * 4 + 1) * 64] * wk;
#pragma unroll
      for (int dt = 0; dt < NDT; dt++)
#pragma unroll
        for (int j = 0; j < 4; j++) o[0][dt][j] += src[(dt * 4 + j) * 64] * wk;
    }
    m[0] = mx;
  }

  // lane (r, g) holds channels 16 dt + 4 g .. + 3 of its rows.  fp16 outputs
  // of several wavefronts go through a strip of LDS each (the tiles' memory is
  // free by then), so that a wavefront writes rows of whole 16-byte vectors and
  // not 32 bytes of sixteen rows at a time (2 x 16 x 8192 rows of 128 over 64
  // keys: 40.5 -> 33.9 us).
  constexpr bool SWAP = !F32 && WM > 1;
  constexpr int SP = DK * 2 + 16;  // bytes between a strip's rows
  static_assert(!SWAP || 4 * 16 * SP <= Sh::LDS, "the strips fit the buffers");
  unsigned char* const strip = smem + wm * 16 * SP;
  if constexpr (SWAP) __syncthreads();
#pragma unroll
  for (int i = 0; i < QG; i++) {
    if (a.splits > 1) {
      if (!live[i]) continue;
      const uint64_t prow = (uint64_t)split * a.prows + (uint64_t)hb * a.rows + row[i];
      float* dst = a.part_o + prow * a.d;
#pragma unroll
      for (int dt = 0; dt < NDT; dt++)
        if (dt * 16 + g * 4 < a.d) *(f32x4*)(dst + dt * 16 + g * 4) = o[i][dt];
      if (g == 0) *(float2*)(a.part_ml + prow * 2) = float2{m[i], l[i]};
      continue;
    }
    const float inv = l[i] == 0.0f ? 0.0f : 1.0f / l[i];
    if constexpr (SWAP) {
#pragma unroll
      for (int dt = 0; dt < NDT; dt++) {
        const f32x4 v = o[i][dt] * inv;
        *(f16x4*)(strip + r * SP + dt * 32 + g * 8) = f16x4{(f16)v[0], (f16)v[1], (f16)v[2], (f16)v[3]};
      }
      enc_lds_fence();
      constexpr int CH = DK / 8;  // 16-byte chunks of a row
      const uint32_t row0 = mb * Sh::ROWS + (wm * QG + i) * 16;
#pragma unroll
      for (int it = 0; it < 16 * CH / 64; it++) {
        const uint32_t x = it * 64 + lane, rr = x / CH, c = x % CH, row = row0 + rr;
        const f16x8 v = *(const f16x8*)(strip + rr * SP + c * 16);
        if (row >= a.rows || c * 8 >= a.d) continue;
        const uint32_t qi = a.G == 1 ? row : row / a.G, qh = h * a.G + (row - qi * a.G);
        *(f16x8*)((f16*)a.o + b * a.bo + qh * a.ho + (uint64_t)qi * a.ldo + c * 8) = v;
      }
      enc_lds_fence();
    } else {
      if (!live[i]) continue;
      T* dst = (T*)a.o + b * a.bo + qh[i] * a.ho + (uint64_t)qi_[i] * a.ldo;
#pragma unroll
      for (int dt = 0; dt < NDT; dt++) {
        if (dt * 16 + g * 4 >= a.d) continue;
        const f32x4 v = o[i][dt] * inv;
        if constexpr (F32) *(f32x4*)(dst + dt * 16 + g * 4) = v;
        else *(f16x4*)(dst + dt * 16 + g * 4) = f16x4{(f16)v[0], (f16)v[1], (f16)v[2], (f16)v[3]};
      }
    }
  }
}

// Joins the key ranges.  A workgroup of 256 threads takes rows of d / 4 vectors:
// SG threads per vector, thread g of them the ranges g, g + SG, .. in order,
// then their partial sums through LDS in order of g.
template <typename T>
__global__ __launch_bounds__(256) void k_attn_enc_merge(AttnEncArgs a, uint32_t SG) {
  __shared__ float sm[256 * 6];
  kernarg_warm(a);
  const uint32_t vpr = a.d / 4, per = 256 / SG;  // vectors per workgroup
  const uint32_t sg = threadIdx.x / per, vi = threadIdx.x % per;
  const uint64_t i = (uint64_t)blockIdx.x * per + vi, total = a.prows * vpr;
  const bool ok = i < total && sg < SG;
  const uint64_t row = ok ? i / vpr : 0;
  const uint32_t c = ok ? (uint32_t)(i - row * vpr) * 4 : 0;
  float mx = kNone, l = 0.0f;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (uint32_t s0 = sg; ok && s0 < a.splits; s0 += SG * 4) {
    float2 ml[4];
    f32x4 v[4];
#pragma unroll
    for (uint32_t u = 0; u < 4; u++) {
      const uint64_t p = (uint64_t)min(s0 + u * SG, a.splits - 1) * a.prows + row;
      ml[u] = *(const float2*)(a.part_ml + p * 2);
      v[u] = *(const f32x4*)(a.part_o + p * a.d + c);
    }
    float m2 = mx;
#pragma unroll
    for (uint32_t u = 0; u < 4; u++) m2 = fmaxf(m2, ml[u].x);
    const float al = __builtin_amdgcn_exp2f(mx - m2);
    l *= al;
    acc *= al;
    mx = m2;
#pragma unroll
    for (uint32_t u = 0; u < 4; u++) {
      if (s0 + u * SG >= a.splits || ml[u].y == 0.0f) continue;  // (an empty range adds nothing)
      const float wt = __builtin_amdgcn_exp2f(ml[u].x - mx);
      l += wt * ml[u].y;
      acc += wt * v[u];
    }
  }
  float* own = sm + threadIdx.x * 6;
  own[0] = mx;
  own[1] = l;
#pragma unroll
  for (int j = 0; j < 4; j++) own[2 + j] = acc[j];
  __syncthreads();
  if (!ok || sg > 0) return;
  float m2 = mx;
  for (uint32_t k = 1; k < SG; k++) m2 = fmaxf(m2, sm[(k * per + vi) * 6]);
  float wt = __builtin_amdgcn_exp2f(mx - m2);
  l *= wt;
  acc *= wt;
  for (uint32_t k = 1; k < SG; k++) {
    const float* o = sm + (k * per + vi) * 6;
    if (o[1] == 0.0f) continue;
    wt = __builtin_amdgcn_exp2f(o[0] - m2);
    l += wt * o[1];
#pragma unroll
    for (int j = 0; j < 4; j++) acc[j] += wt * o[2 + j];
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  const uint32_t rr = (uint32_t)(row % a.rows), q = rr / a.G;
  const uint64_t hb = row / a.rows;
  const uint64_t h = (hb % a.Hk) * a.G + (rr - q * a.G), b = hb / a.Hk;
  T* dst = (T*)a.o + b * a.bo + h * a.ho + (uint64_t)q * a.ldo + c;
  const f32x4 v = acc * inv;
  if constexpr (sizeof(T) == 4) *(f32x4*)dst = v;
  else *(f16x4*)dst = f16x4{(f16)v[0], (f16)v[1], (f16)v[2], (f16)v[3]};
}

template <typename T, int DK, int FORM>
void launch_enc_form(const AttnEncArgs& a, uint32_t B, hipStream_t s) {
  typedef EncShape<T, DK, FORM> Sh;
  const dim3 grid(a.blocks * a.splits * a.Hk * B);
  if constexpr (FORM != ENC_MANY)
    if (a.bias) {
      k_attn_enc<T, DK, FORM, true><<<grid, Sh::NT, 0, s>>>(a);
      return;
    }
  k_attn_enc<T, DK, FORM, false><<<grid, Sh::NT, 0, s>>>(a);
}

template <typename T, int DK>
void launch_enc_dk(const AttnEncArgs& a, uint32_t B, int form, hipStream_t s) {
  if (form == ENC_FEW) {
    launch_enc_form<T, DK, ENC_FEW>(a, B, s);
    return;
  }
  // (one row group a wavefront in either form: one kernel)
  if constexpr (EncShape<T, DK, ENC_MANY>::QG > 1) {
    if (form == ENC_MANY) {
      launch_enc_form<T, DK, ENC_MANY>(a, B, s);
      return;
    }
  }
  launch_enc_form<T, DK, ENC_MID>(a, B, s);
}

// d padded to the channels of an instantiation
inline uint32_t enc_channels(uint32_t d) { return d <= 192 ? (d + 31) / 32 * 32 : 256; }

template <typename T, int DK>
AttnEncForm enc_form_dk(int form) {
  auto of = [](auto s) {
    typedef decltype(s) S;
    return AttnEncForm{S::ROWS, S::KT, S::WK};
  };
  return form == ENC_FEW ? of(EncShape<T, DK, ENC_FEW>{})
                         : form == ENC_MID ? of(EncShape<T, DK, ENC_MID>{}) : of(EncShape<T, DK, ENC_MANY>{});
}

template <typename T>
AttnEncForm enc_form(uint32_t d, int form) {
  switch (enc_channels(d)) {
    case 32: return enc_form_dk<T, 32>(form);
    case 64: return enc_form_dk<T, 64>(form);
    case 96: return enc_form_dk<T, 96>(form);
    case 128: return enc_form_dk<T, 128>(form);
    case 160: return enc_form_dk<T, 160>(form);
    case 192: return enc_form_dk<T, 192>(form);
    default: return enc_form_dk<T, 256>(form);
  }
}

template <typename T>
void launch_enc(const AttnEncArgs& a, uint32_t B, int form, hipStream_t s) {
  switch (enc_channels(a.d)) {
    case 32: launch_enc_dk<T, 32>(a, B, form, s); break;
    case 64: launch_enc_dk<T, 64>(a, B, form, s); break;
    case 96: launch_enc_dk<T, 96>(a, B, form, s); break;
    case 128: launch_enc_dk<T, 128>(a, B, form, s); break;
    case 160: launch_enc_dk<T, 160>(a, B, form, s); break;
    case 192: launch_enc_dk<T, 192>(a, B, form, s); break;
    default: launch_enc_dk<T, 256>(a, B, form, s); break;
  }
  if (a.splits > 1) {
    // threads per vector: four ranges each
    const uint32_t sg = a.splits <= 4 ? 1 : a.splits <= 8 ? 2 : a.splits <= 16 ? 4 : 8, per = 256 / sg;
    k_attn_enc_merge<T><<<(uint32_t)((a.prows * (a.d / 4) + per - 1) / per), 256, 0, s>>>(a, sg);
  }
}

}  // namespace

}  // namespace di
