// Attention over the paged 8-bit cache (layout: mmnb_kv8.h):
//   o[row, h] = sum_j p_j v_j, p = softmax_j(scale * q . k_j) over the tokens j that the row sees:
//   j <= pos (causal) or j < kv_len, and j > pos - window when a window is given; a row that sees
//   nothing gives zeros.
// First form: a warp a (row, query head), one pass with the running maximum and sum.
#include <cstdint>

#include "mmnb_kv8.cuh"

namespace xrgpu {
namespace {

template <bool E4M3, int PER>
__global__ void __launch_bounds__(256) attn_kernel(const Kv8 p) {
  const int lane = threadIdx.x & 31;
  const int64_t warp = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
  const int row = static_cast<int>(warp / p.hq), h = static_cast<int>(warp % p.hq);
  if (row >= p.tokens) return;
  int b = -1;
  if (p.uniform) {
    b = row / (p.tokens / p.seqs);
    if (b >= p.seqs) return;
  } else {
    for (int b0 = 0; b0 < p.seqs && b < 0; b0 += 32) {
      const bool here = b0 + lane < p.seqs && p.cu[b0 + lane] <= row && row < p.cu[b0 + lane + 1];
      const unsigned m = __ballot_sync(~0u, here);
      if (m) b = b0 + __ffs(m) - 1;
    }
    if (b < 0) return;
  }
  const SeqRows r = seq_rows(p, b, true);
  if (r.n == 0) return;
  const int pos = r.len - r.n + (row - r.row0), D = p.D, kvh = h / (p.hq / p.hkv);
  const int hi = p.causal ? min(pos + 1, r.len) : r.len, lo = p.window > 0 ? max(0, pos - p.window + 1) : 0;
  float q[PER], acc[PER], m = -INFINITY, l = 0.0f;
  const int64_t qat = static_cast<int64_t>(row) * p.qs + h * D, oat = static_cast<int64_t>(row) * p.os + h * D;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    q[i] = load_f(p.q, p.f16, qat + lane * PER + i) * p.scale;
    acc[i] = 0.0f;
  }
  int id = -1;
  float ks = 0.0f, vs = 0.0f;
  for (int j = lo; j < hi; ++j) {
    if (j == lo || (j & (p.page - 1)) == 0) {
      id = page_id(p, b, j >> p.page_log2);
      if (id >= 0) {
        ks = p.k_scale[static_cast<int64_t>(id) * p.hkv + kvh];
        vs = p.v_scale[static_cast<int64_t>(id) * p.hkv + kvh];
      }
    }
    if (id < 0) continue;
    const int64_t at = (((static_cast<int64_t>(id) * p.hkv + kvh) << p.page_log2) + (j & (p.page - 1))) * D + lane * PER;
    float x = 0.0f;
#pragma unroll
    for (int i = 0; i < PER; ++i) x = fmaf(q[i], code_value<E4M3>(p.k_cache[at + i]), x);
#pragma unroll
    for (int d = 16; d; d >>= 1) x += __shfl_xor_sync(~0u, x, d);
    x *= ks;
    const float mn = fmaxf(m, x), up = __expf(m - mn), w = __expf(x - mn);
    l = l * up + w;
    m = mn;
#pragma unroll
    for (int i = 0; i < PER; ++i) acc[i] = acc[i] * up + w * vs * code_value<E4M3>(p.v_cache[at + i]);
  }
  const float inv = l > 0.0f ? 1.0f / l : (l == l ? 0.0f : l);
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const float o = acc[i] * inv;
    if (p.f16) static_cast<__half*>(p.o)[oat + lane * PER + i] = __float2half_rn(o);
    else static_cast<float*>(p.o)[oat + lane * PER + i] = o;
  }
}

}  // namespace

uint64_t kv8_attention_workspace(const Kv8&) { return 0; }

cudaError_t launch_kv8_attention(const Kv8& p, void*, cudaStream_t s) {
  if (p.tokens == 0 || p.seqs == 0) return cudaSuccess;
  const unsigned grid = static_cast<unsigned>((static_cast<int64_t>(p.tokens) * p.hq + 7) / 8);
  if (p.D == 128) {
    if (p.e4m3) attn_kernel<true, 4><<<grid, 256, 0, s>>>(p);
    else attn_kernel<false, 4><<<grid, 256, 0, s>>>(p);
  } else {
    if (p.e4m3) attn_kernel<true, 2><<<grid, 256, 0, s>>>(p);
    else attn_kernel<false, 2><<<grid, 256, 0, s>>>(p);
  }
  return cudaGetLastError();
}

}  // namespace xrgpu
