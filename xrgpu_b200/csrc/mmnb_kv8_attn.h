// Launchers behind xrgpu_kv8_attention (mmnb_kv8_attn.cu chooses).
#pragma once

#include "mmnb_kv8.h"

namespace xrgpu {

// mma.sync form (mmnb_kv8_attn_mma.cuh): any rows; bytes of its workspace, its launch.
uint64_t kv8_attn_mma_workspace(const Kv8& p);
cudaError_t launch_kv8_attn_mma_int8(const Kv8& p, void* ws, cudaStream_t s);
cudaError_t launch_kv8_attn_mma_e4m3(const Kv8& p, void* ws, cudaStream_t s);

// tcgen05 form (mmnb_kv8_attn_sm100.cu): float16 rows of the sequences with more than p.few_rows rows.
cudaError_t launch_kv8_attn_prompt(const Kv8& p, cudaStream_t s);

}  // namespace xrgpu
