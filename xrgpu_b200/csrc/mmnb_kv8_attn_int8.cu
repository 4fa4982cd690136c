// The mma.sync attention over caches of int8 codes.
#include "mmnb_kv8_attn_mma.cuh"

namespace xrgpu {

uint64_t kv8_attn_mma_workspace(const Kv8& p) {
  if (cluster_split(p)) return 0;
  return static_cast<uint64_t>(starts_bytes(p.seqs) + 4ll * device_sm_count() * part_floats(8 * row_tiles(p), p.D) * 4);
}

cudaError_t launch_kv8_attn_mma_int8(const Kv8& p, void* ws, cudaStream_t s) { return launch_code<false>(p, ws, s); }

}  // namespace xrgpu
