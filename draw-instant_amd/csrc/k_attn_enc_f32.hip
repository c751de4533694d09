// k_attn_enc instantiations: fp32 tensors on the fp32 MFMA.
#include "k_attn_enc.h"

namespace di {

void launch_attn_enc_f32(const AttnEncArgs& a, uint32_t B, int form, hipStream_t s) {
  launch_enc<float>(a, B, form, s);
}

AttnEncForm attn_enc_form_f32(uint32_t d, int form) { return enc_form<float>(d, form); }

}  // namespace di
