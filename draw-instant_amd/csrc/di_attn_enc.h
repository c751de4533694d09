// Argument block and launch API of the encoder attention kernels
// (k_attn_enc.h).  Raw device pointers; callers validate shapes.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace di {

struct AttnEncArgs {
  const void *q, *k, *v;
  void* o;
  // strides in elements: token (ld), head, batch
  uint64_t ldq, hq, bq, ldk, hk, bk, ldv, hv, bv, ldo, ho, bo;
  const int32_t* len;  // keys per batch entry, null: Skv
  const float* bias;   // null: none
  uint64_t bias_b, bias_h, bias_q;
  uint32_t Hk, G;  // key heads, query heads per key head
  uint32_t Sq, Skv, d;
  uint32_t rows;    // Sq * G: query rows of one key head
  uint32_t blocks;  // row blocks per key head
  uint32_t splits;  // key ranges
  uint32_t heads_first;  // order of the workgroups, with a bias
  uint64_t prows;   // rows of the whole call: B * Hk * rows
  float scale_log2;
  float* part_o;   // [splits][prows][d], splits > 1
  float* part_ml;  // [splits][prows][2]
};

// The three forms (see k_attn_enc.h): rows per workgroup, keys per tile and key
// groups inside a workgroup.
enum { ENC_FEW = 0, ENC_MID = 1, ENC_MANY = 2 };
struct AttnEncForm {
  int rows, tile, groups;
};
AttnEncForm attn_enc_form_f16(uint32_t d, int form);
AttnEncForm attn_enc_form_f32(uint32_t d, int form);
// fp32 tensors and matrix products (k_attn_enc_f32.hip), or fp16.
void launch_attn_enc_f16(const AttnEncArgs& a, uint32_t B, int form, hipStream_t s);
void launch_attn_enc_f32(const AttnEncArgs& a, uint32_t B, int form, hipStream_t s);

}  // namespace di
