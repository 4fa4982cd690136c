// The mma.sync attention over caches of e4m3 codes.
#include "mmnb_kv8_attn_mma.cuh"

namespace xrgpu {

cudaError_t launch_kv8_attn_mma_e4m3(const Kv8& p, void* ws, cudaStream_t s) { return launch_code<true>(p, ws, s); }

}  // namespace xrgpu
