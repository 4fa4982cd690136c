// Attention over the paged 8-bit cache: which kernel a call takes (layout: mmnb_kv8.h).
#include "mmnb_kv8_attn.h"

namespace xrgpu {

uint64_t kv8_attention_workspace(const Kv8& p) { return kv8_attn_mma_workspace(p); }

cudaError_t launch_kv8_attention(const Kv8& p, void* ws, cudaStream_t s) {
  return p.e4m3 ? launch_kv8_attn_mma_e4m3(p, ws, s) : launch_kv8_attn_mma_int8(p, ws, s);
}

}  // namespace xrgpu
