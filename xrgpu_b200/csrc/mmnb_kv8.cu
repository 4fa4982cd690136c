// Append to and read back from the paged 8-bit key/value cache (layout: mmnb_kv8.h).
//
// Append. A block is one page of one head. With a = max |x| over the block's new values, L = 127
// (int8) or 448 (e4m3), s_old the stored scale if the page holds older tokens of the sequence, else 0:
//   s = max(s_old, a / L);  new codes = round(x / s);  older codes c -> round(c * s_old / s) if s > s_old,
// rounding to nearest, ties to even. So a block's scale always covers what it holds, and appending a
// prompt at once or token by token differs only by what re-rounding older codes costs. A NaN or an
// infinity in the new values makes the block's scale NaN (so that what reads it is NaN); s = 0 gives codes 0.
// The quotients are rounded as the real numbers they are: x / s in float32 can land on a border that
// x / s lies next to, so the remainder x - q s (exact in one fma) decides.
#include <cstdint>

#include "mmnb_kv8.cuh"

namespace xrgpu {
namespace {

constexpr int kThreads = 128;

// round(x / s) as a code byte, s > 0 and finite, |x| <= L s up to rounding.
template <bool E4M3>
__device__ __forceinline__ uint32_t quotient_code(float x, float s) {
  float q = x / s;
  if (E4M3) {
    const float r = fmaf(-q, s, x);
    const uint32_t u = __float_as_uint(q);
    // move q off a border, to the side where x / s is (an odd last bit is never a border)
    if (r != 0.0f && q != 0.0f && !(u & 1u)) q = __uint_as_float(((r > 0.0f) == (q > 0.0f)) ? u + 1u : u - 1u);
    return __nv_cvt_float_to_fp8(q, __NV_SATFINITE, __NV_E4M3);
  }
  q = rintf(q);
  const float r = fmaf(-q, s, x), h = 0.5f * s;
  const bool odd = static_cast<int>(q) & 1;
  if (r > h || (r == h && odd)) q += 1.0f;
  else if (r < -h || (r == -h && odd)) q -= 1.0f;
  q = fminf(fmaxf(q, -127.0f), 127.0f);
  return static_cast<uint32_t>(static_cast<int>(q)) & 255u;
}

// An older code under a larger scale: round(c * s_old / s), in float64 (rare: only when a block's scale grows).
template <bool E4M3>
__device__ __forceinline__ uint32_t rescaled_code(uint32_t byte, double s_old, double s) {
  const double d = static_cast<double>(code_value<E4M3>(byte)) * s_old / s;
  if (E4M3) {
    float f = __double2float_rz(d);
    if (static_cast<double>(f) != d) f = __uint_as_float(__float_as_uint(f) | 1u);  // sticky bit: rounds once
    return __nv_cvt_float_to_fp8(f, __NV_SATFINITE, __NV_E4M3);
  }
  return static_cast<uint32_t>(__double2int_rn(d)) & 255u;
}

template <bool F16, bool VEC>
__device__ __forceinline__ void load8(const void* src, int64_t at, float (&v)[8]) {
  if (VEC && F16) {
    const uint4 w = *reinterpret_cast<const uint4*>(static_cast<const __half*>(src) + at);
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  } else if (VEC) {
    const float4* s = reinterpret_cast<const float4*>(static_cast<const float*>(src) + at);
    const float4 a = s[0], b = s[1];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = load_f(src, F16, at + i);
  }
}

// Touched pages of sequence b.
__device__ __forceinline__ int touched_pages(const Kv8& p, int b) {
  const SeqRows r = seq_rows(p, b, false);
  return r.n == 0 ? 0 : ((r.len - 1) >> p.page_log2) - ((r.len - r.n) >> p.page_log2) + 1;
}

// CTA (slot, head, side): slot counts the touched pages of all sequences in order.
template <bool E4M3, bool F16, bool VEC>
__global__ void __launch_bounds__(kThreads) append_kernel(const Kv8 p) {
  __shared__ int found_b, found_j, warp_sum[kThreads / 32];
  __shared__ uint32_t warp_max[kThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, slot = blockIdx.x;
  if (tid == 0) found_b = -1;
  __syncthreads();
  int before = 0;
  for (int b0 = 0; b0 < p.seqs; b0 += kThreads) {
    const int b = b0 + tid, t = b < p.seqs ? touched_pages(p, b) : 0;
    int sum = t;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(~0u, sum, d);
      if (lane >= d) sum += o;
    }
    if (lane == 31) warp_sum[warp] = sum;
    __syncthreads();
    int total = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w < warp) sum += warp_sum[w];
      total += warp_sum[w];
    }
    const int at = slot - before - (sum - t);
    if (at >= 0 && at < t) {
      found_b = b;
      found_j = at;
    }
    before += total;
    __syncthreads();
    if (before > slot) break;
  }
  const int b = found_b;
  if (b < 0) return;
  const SeqRows r = seq_rows(p, b, false);
  const int start = r.len - r.n, j = (start >> p.page_log2) + found_j;
  const int lo = max(start, j << p.page_log2), hi = min(r.len, (j + 1) << p.page_log2);
  const int id = page_id(p, b, j);
  if (id < 0) return;
  const int head = blockIdx.y, D = p.D, held = lo - (j << p.page_log2), rows = hi - lo;
  const bool side_v = blockIdx.z != 0;
  const void* src = side_v ? p.v : p.k;
  const int64_t stride = side_v ? p.vs : p.ks;
  const int64_t block = static_cast<int64_t>(id) * p.hkv + head;
  uint8_t* codes = (side_v ? p.v_cache : p.k_cache) + ((block << p.page_log2) * D);
  float* scale_at = (side_v ? p.v_scale : p.k_scale) + block;
  const int64_t row0 = r.row0 + (lo - start);
  const int per_row = D >> 3, items = rows * per_row;

  uint32_t amax = 0;
  for (int i = tid; i < items; i += kThreads) {
    float v[8];
    load8<F16, VEC>(src, (row0 + i / per_row) * stride + head * D + (i % per_row) * 8, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) amax = max(amax, __float_as_uint(v[e]) & 0x7fffffffu);
  }
  amax = __reduce_max_sync(~0u, amax);
  if (lane == 0) warp_max[warp] = amax;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) amax = max(amax, warp_max[w]);
  const float s_old = held ? *scale_at : 0.0f;
  const bool bad = amax >= 0x7f800000u || !(fabsf(s_old) <= 3.4028234e38f);
  const float s = bad ? __uint_as_float(0x7fc00000u) : fmaxf(s_old, __uint_as_float(amax) / (E4M3 ? 448.0f : 127.0f));
  __syncthreads();  // everyone has read the stored scale
  if (tid == 0) *scale_at = s;

  if (!bad && held && s > s_old) {
    const double ds = s, dold = s_old;
    uint32_t* c = reinterpret_cast<uint32_t*>(codes);
    for (int i = tid; i < held * (D >> 2); i += kThreads) {
      const uint32_t w = c[i];
      uint32_t o = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) o |= rescaled_code<E4M3>((w >> (8 * e)) & 255u, dold, ds) << (8 * e);
      c[i] = o;
    }
  }
  const bool zero = bad || s == 0.0f;
  for (int i = tid; i < items; i += kThreads) {
    const int t = i / per_row, d = (i % per_row) * 8;
    uint32_t w[2] = {0, 0};
    if (!zero) {
      float v[8];
      load8<F16, VEC>(src, (row0 + t) * stride + head * D + d, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e >> 2] |= quotient_code<E4M3>(v[e], s) << (8 * (e & 3));
    }
    *reinterpret_cast<uint2*>(codes + (held + t) * D + d) = make_uint2(w[0], w[1]);
  }
}

// The sequence of a row (found by a warp), -1 if it belongs to none.
__device__ __forceinline__ int sequence_of(const Kv8& p, int row, int lane) {
  if (p.uniform) return row / (p.tokens / p.seqs);
  for (int b0 = 0; b0 < p.seqs; b0 += 32) {
    const bool here = b0 + lane < p.seqs && p.cu[b0 + lane] <= row && row < p.cu[b0 + lane + 1];
    const unsigned m = __ballot_sync(~0u, here);
    if (m) return b0 + __ffs(m) - 1;
  }
  return -1;
}

// One warp a (row, side), all heads: PER codes a lane.
template <bool E4M3, bool F16, int PER>
__global__ void __launch_bounds__(256) read_kernel(const Kv8 p) {
  constexpr int D = 32 * PER;
  const int lane = threadIdx.x & 31, row = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (row >= p.tokens) return;
  const bool side_v = blockIdx.y != 0;
  const int b = sequence_of(p, row, lane);
  const SeqRows r = b < 0 ? SeqRows{0, 0, 0} : seq_rows(p, b, false);
  const int pos = r.len - r.n + (row - r.row0), id = r.n ? page_id(p, b, pos >> p.page_log2) : -1;
  if (id < 0 && !p.zero_rest) return;
  const int64_t block = static_cast<int64_t>(id) * p.hkv;
  const float* scales = (side_v ? p.v_scale : p.k_scale) + block;
  const uint8_t* codes = (side_v ? p.v_cache : p.k_cache) + ((block << p.page_log2) + (pos & (p.page - 1))) * D + lane * PER;
  void* dst = side_v ? p.v : p.k;
  int64_t at = static_cast<int64_t>(row) * (side_v ? p.vs : p.ks) + lane * PER;
#pragma unroll 4
  for (int h = 0; h < p.hkv; ++h, at += D) {
    uint32_t w = 0;
    float s = 0.0f;
    if (id >= 0) {
      const uint8_t* src = codes + (static_cast<int64_t>(h) << p.page_log2) * D;
      w = PER == 4 ? *reinterpret_cast<const uint32_t*>(src) : *reinterpret_cast<const uint16_t*>(src);
      s = scales[h];
    }
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      const float v = id < 0 ? 0.0f : code_value<E4M3>((w >> (8 * e)) & 255u) * s;
      if (F16) static_cast<__half*>(dst)[at + e] = __float2half_rn(v);
      else static_cast<float*>(dst)[at + e] = v;
    }
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace

cudaError_t launch_kv8_append(const Kv8& p, cudaStream_t s) {
  if (p.tokens == 0 || p.seqs == 0) return cudaSuccess;
  // A touched page takes at least one row, and a sequence's n rows touch at most n / page + 2 pages.
  const int64_t most = p.tokens / p.page + 2 * static_cast<int64_t>(p.seqs);
  const dim3 grid(static_cast<unsigned>(most < p.tokens ? most : p.tokens), static_cast<unsigned>(p.hkv), 2);
  const int64_t es = p.f16 ? 2 : 4;
  const bool vec = aligned16(p.k) && aligned16(p.v) && (p.ks * es) % 16 == 0 && (p.vs * es) % 16 == 0;
  const int form = (p.e4m3 ? 4 : 0) | (p.f16 ? 2 : 0) | (vec ? 1 : 0);
  switch (form) {
    case 0: append_kernel<false, false, false><<<grid, kThreads, 0, s>>>(p); break;
    case 1: append_kernel<false, false, true><<<grid, kThreads, 0, s>>>(p); break;
    case 2: append_kernel<false, true, false><<<grid, kThreads, 0, s>>>(p); break;
    case 3: append_kernel<false, true, true><<<grid, kThreads, 0, s>>>(p); break;
    case 4: append_kernel<true, false, false><<<grid, kThreads, 0, s>>>(p); break;
    case 5: append_kernel<true, false, true><<<grid, kThreads, 0, s>>>(p); break;
    case 6: append_kernel<true, true, false><<<grid, kThreads, 0, s>>>(p); break;
    default: append_kernel<true, true, true><<<grid, kThreads, 0, s>>>(p); break;
  }
  return cudaGetLastError();
}

cudaError_t launch_kv8_read(const Kv8& p, cudaStream_t s) {
  if (p.tokens == 0 || p.seqs == 0) return cudaSuccess;
  const dim3 grid(static_cast<unsigned>((static_cast<int64_t>(p.tokens) + 7) / 8), 2);
  switch ((p.D == 128 ? 4 : 0) | (p.e4m3 ? 2 : 0) | (p.f16 ? 1 : 0)) {
    case 0: read_kernel<false, false, 2><<<grid, 256, 0, s>>>(p); break;
    case 1: read_kernel<false, true, 2><<<grid, 256, 0, s>>>(p); break;
    case 2: read_kernel<true, false, 2><<<grid, 256, 0, s>>>(p); break;
    case 3: read_kernel<true, true, 2><<<grid, 256, 0, s>>>(p); break;
    case 4: read_kernel<false, false, 4><<<grid, 256, 0, s>>>(p); break;
    case 5: read_kernel<false, true, 4><<<grid, 256, 0, s>>>(p); break;
    case 6: read_kernel<true, false, 4><<<grid, 256, 0, s>>>(p); break;
    default: read_kernel<true, true, 4><<<grid, 256, 0, s>>>(p); break;
  }
  return cudaGetLastError();
}

}  // namespace xrgpu
