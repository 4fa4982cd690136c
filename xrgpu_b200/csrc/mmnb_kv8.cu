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

// Codes round(x / s) of 8 values, s > 0 and finite, |x| <= L s up to s's rounding. A product with 1 / s lies within 2 ulp of
// x / s (inv = 0, where that would leave the normal range: a division). Only where a border between two codes is nearer
// than that is the remainder looked at; the inputs being short numbers, a third of the warps have such a value. (A
// division a value costs 40 instructions and bounded the kernel: 20 us for 11 M values.)
template <bool E4M3>
__device__ __forceinline__ uint2 codes8(float (&v)[8], float s, float inv) {
  uint32_t w[2] = {0, 0};
  float q[8];
  if (inv != 0.0f) {
#pragma unroll
    for (int e = 0; e < 8; ++e) q[e] = v[e] * inv;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (!E4M3) v[e] = fminf(fmaxf(v[e], -127.0f * s), 127.0f * s);  // a subnormal s may be far below |x| / 127
      q[e] = v[e] / s;
    }
  }
  if (E4M3) {
    uint32_t least = ~0u;
#pragma unroll
    for (int e = 0; e < 8; ++e) least = min(least, (__float_as_uint(q[e]) + 4u) & 0x7ffffu);  // borders have at most 4 significant bits
    if (least <= 8u) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        q[e] = fmaf(fmaf(-q[e], s, v[e]), inv, q[e]);  // no number lies between this and x / s
        const float r = fmaf(-q[e], s, v[e]);
        const uint32_t u = __float_as_uint(q[e]);
        // off a border, to the side where x / s is (an odd last bit is never a border)
        if (r != 0.0f && q[e] != 0.0f && !(u & 1u)) q[e] = __uint_as_float(((r > 0.0f) == (q[e] > 0.0f)) ? u + 1u : u - 1u);
      }
    }
#pragma unroll
    for (int e = 0; e < 8; e += 2)
      w[e >> 2] |= static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(make_float2(q[e], q[e + 1]), __NV_SATFINITE, __NV_E4M3)) << (8 * (e & 2));
  } else {
    constexpr float kMagic = 12582912.0f;  // 1.5 * 2^23: the sum's low bits are the rounded integer
    float most = 0.0f;
    uint32_t t[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float m = q[e] + kMagic;
      t[e] = __float_as_uint(m);
      q[e] = fmaf(kMagic - m, s, v[e]);  // the remainder, exactly
      most = fmaxf(most, fabsf(q[e]));
    }
    if (!(most + most < s)) {  // twice the remainder: half of a subnormal s would be rounded
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const bool odd = t[e] & 1u;
        const float r = q[e] + q[e];
        if (r > s || (r == s && odd)) ++t[e];
        else if (r < -s || (r == -s && odd)) --t[e];
      }
    }
#pragma unroll
    for (int e = 0; e < 8; e += 4) w[e >> 2] = __byte_perm(__byte_perm(t[e], t[e + 1], 0x40), __byte_perm(t[e + 2], t[e + 3], 0x40), 0x5410);
  }
  return make_uint2(w[0], w[1]);
}

// An older code under a larger scale: round(c * s_old / s) in float64.
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

// Four of them: float32 products with s_old / s (`ratio`), float64 where a border is nearer than their error.
template <bool E4M3>
__device__ __forceinline__ uint32_t rescaled_word(uint32_t w, float ratio, float s_old, float s) {
  uint32_t o = 0, t[4];
  float q[4];
  bool near = false;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    q[e] = code_value<E4M3>((w >> (8 * e)) & 255u) * ratio;
    const float m = q[e] + 12582912.0f;
    t[e] = __float_as_uint(m);
    near = near || (E4M3 ? q[e] != 0.0f && ((__float_as_uint(q[e]) + 4u) & 0x7ffffu) <= 8u : fabsf(q[e] - (m - 12582912.0f)) > 0.4999f);
  }
  if (near) {
#pragma unroll 1
    for (int e = 0; e < 4; ++e) o |= rescaled_code<E4M3>((w >> (8 * e)) & 255u, s_old, s) << (8 * e);
    return o;
  }
  if (E4M3) {
    o = static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(make_float2(q[0], q[1]), __NV_SATFINITE, __NV_E4M3)) |
        static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(make_float2(q[2], q[3]), __NV_SATFINITE, __NV_E4M3)) << 16;
  } else {
    o = __byte_perm(__byte_perm(t[0], t[1], 0x40), __byte_perm(t[2], t[3], 0x40), 0x5410);
  }
  return o;
}

// 8 values as they lie in memory.
template <bool F16>
struct Raw8 {
  uint32_t u[F16 ? 4 : 8];
};
template <bool F16, bool VEC>
__device__ __forceinline__ Raw8<F16> load8(const void* src, int64_t at) {
  Raw8<F16> r;
  if (VEC) {
    const uint4* p = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(src) + at * (F16 ? 2 : 4));
#pragma unroll
    for (int i = 0; i < (F16 ? 1 : 2); ++i) {
      const uint4 w = p[i];
      r.u[4 * i] = w.x;
      r.u[4 * i + 1] = w.y;
      r.u[4 * i + 2] = w.z;
      r.u[4 * i + 3] = w.w;
    }
  } else if (F16) {
    const uint16_t* p = static_cast<const uint16_t*>(src) + at;
#pragma unroll
    for (int i = 0; i < 4; ++i) r.u[i] = p[2 * i] | (static_cast<uint32_t>(p[2 * i + 1]) << 16);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) r.u[i] = static_cast<const uint32_t*>(src)[at + i];
  }
  return r;
}
template <bool F16>
__device__ __forceinline__ void values8(const Raw8<F16>& r, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < (F16 ? 4 : 8); ++i) {
    if (F16) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&r.u[i]));
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    } else {
      v[i] = __uint_as_float(r.u[i]);
    }
  }
}
// The larger of `most` and the magnitudes of 8 values, as the bits of a float32 (of two halves for F16); NaN stays.
template <bool F16>
__device__ __forceinline__ uint32_t max8(uint32_t most, const Raw8<F16>& r) {
#pragma unroll
  for (int i = 0; i < (F16 ? 4 : 8); ++i) {
    if (F16) {
      const __half2 m = __hmax2_nan(*reinterpret_cast<const __half2*>(&most), __habs2(*reinterpret_cast<const __half2*>(&r.u[i])));
      most = *reinterpret_cast<const uint32_t*>(&m);
    } else {
      most = max(most, r.u[i] & 0x7fffffffu);
    }
  }
  return most;
}

// Touched pages of sequence b.
__device__ __forceinline__ int touched_pages(const Kv8& p, int b) {
  const SeqRows r = seq_rows(p, b, false);
  return r.n == 0 ? 0 : ((r.len - 1) >> p.page_log2) - ((r.len - r.n) >> p.page_log2) + 1;
}

// CTA (slot, two blocks): slot counts the touched pages of all sequences in order; two warps each take a block (a head's K
// or V), so that two share the search for the sequence. 5400 tokens of five sequences, 8 heads of 128 halves, pages of 32, e4m3
// (33 MB): 12.8 us, 2.6 TB/s (a warp a block 13.9, four 14.5); 64 single tokens into pages of 64: 3.5 us (3.9, 4.2), a chain
// of dependent loads. Bound by latency and instructions (half of the issue slots). Held in registers between the passes,
// the values cost more occupancy than reading them again from the L1 cache does (15.6 us).
template <bool E4M3, bool F16, bool VEC, int D>
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
  const int part = blockIdx.y * 2 + (warp >> 1);
  const int head = part >> 1, held = lo - (j << p.page_log2), rows = hi - lo;
  const bool side_v = part & 1;
  const void* src = side_v ? p.v : p.k;
  const int64_t stride = side_v ? p.vs : p.ks;
  const int64_t block = static_cast<int64_t>(id) * p.hkv + head;
  uint8_t* codes = (side_v ? p.v_cache : p.k_cache) + ((block << p.page_log2) * D);
  float* scale_at = (side_v ? p.v_scale : p.k_scale) + block;
  // a thread takes the same 8 columns of every kStep-th row
  constexpr int kSize = 64, kStep = kSize / (D / 8);
  const int gid = tid & (kSize - 1);
  const int t0 = gid / (D / 8), d0 = (gid % (D / 8)) * 8;
  auto sync = [&] {  // constant barriers: with one by a register the kernel counts as using all 16, and 4 CTAs fit an SM
    if (warp < 2) asm volatile("bar.sync 1, 64;" ::: "memory");
    else asm volatile("bar.sync 2, 64;" ::: "memory");
  };
  const int64_t at0 = (r.row0 + (lo - start) + t0) * stride + head * D + d0;

  uint32_t amax = 0;
#pragma unroll 4
  for (int t = t0; t < rows; t += kStep) amax = max8(amax, load8<F16, VEC>(src, at0 + (t - t0) * stride));
  if (F16) {
    const uint32_t m = max(amax & 0xffffu, amax >> 16);
    amax = __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(m))));
  }
  amax = __reduce_max_sync(~0u, amax);
  if (lane == 0) warp_max[warp] = amax;
  sync();
  amax = max(amax, warp_max[warp ^ 1]);
  const float s_old = held ? *scale_at : 0.0f;
  const bool bad = amax >= 0x7f800000u || !(fabsf(s_old) <= 3.4028234e38f);
  const float s = bad ? __uint_as_float(0x7fc00000u) : fmaxf(s_old, __uint_as_float(amax) / (E4M3 ? 448.0f : 127.0f));
  sync();  // everyone has read the stored scale
  if (gid == 0) *scale_at = s;

  if (!bad && held && s > s_old) {
    const float ratio = s_old / s;
    uint32_t* c = reinterpret_cast<uint32_t*>(codes);
#pragma unroll 2
    for (int i = gid; i < held * (D >> 2); i += kSize) c[i] = rescaled_word<E4M3>(c[i], ratio, s_old, s);
  }
  const bool zero = bad || s == 0.0f;
  const float inv = s > 0x1p-60f && s < 0x1p60f ? 1.0f / s : 0.0f;
  uint8_t* dst = codes + (held + t0) * D + d0;
#pragma unroll 2
  for (int t = 0; t < rows - t0; t += kStep) {  // the values come from the L1 cache
    uint2 w = make_uint2(0, 0);
    const Raw8<F16> raw = load8<F16, VEC>(src, at0 + t * stride);
    if (!zero) {
      float v[8];
      values8(raw, v);
      w = codes8<E4M3>(v, s, inv);
    }
    *reinterpret_cast<uint2*>(dst + t * D) = w;
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

// One warp a (row, side), all heads: PER codes a lane. 5500 rows of 8 heads of 128 halves (34 MB): 8.7 us, 3.9 TB/s (13.2 with
// halves stored one by one).
template <bool E4M3, bool F16, int PER, bool VEC>
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
    float v[PER];
#pragma unroll
    for (int e = 0; e < PER; ++e) v[e] = id < 0 ? 0.0f : code_value<E4M3>((w >> (8 * e)) & 255u) * s;
    if (VEC && F16) {
      uint32_t u[PER / 2];
#pragma unroll
      for (int e = 0; e < PER; e += 2) {
        const __half2 x = __floats2half2_rn(v[e], v[e + 1]);
        u[e / 2] = *reinterpret_cast<const uint32_t*>(&x);
      }
      if (PER == 4) *reinterpret_cast<uint2*>(static_cast<__half*>(dst) + at) = make_uint2(u[0], u[PER / 2 - 1]);
      else *reinterpret_cast<uint32_t*>(static_cast<__half*>(dst) + at) = u[0];
    } else if (VEC) {
      if (PER == 4) *reinterpret_cast<float4*>(static_cast<float*>(dst) + at) = make_float4(v[0], v[1], v[PER - 2], v[PER - 1]);
      else *reinterpret_cast<float2*>(static_cast<float*>(dst) + at) = make_float2(v[0], v[1]);
    } else {
#pragma unroll
      for (int e = 0; e < PER; ++e) {
        if (F16) static_cast<__half*>(dst)[at + e] = __float2half_rn(v[e]);
        else static_cast<float*>(dst)[at + e] = v[e];
      }
    }
  }
}

template <bool E4M3, bool F16, int PER>
void launch_read(const Kv8& p, dim3 grid, bool vec, cudaStream_t s) {
  if (vec) read_kernel<E4M3, F16, PER, true><<<grid, 256, 0, s>>>(p);
  else read_kernel<E4M3, F16, PER, false><<<grid, 256, 0, s>>>(p);
}

template <bool E4M3, bool F16, bool VEC>
void launch_append(const Kv8& p, dim3 grid, cudaStream_t s) {
  if (p.D == 128) append_kernel<E4M3, F16, VEC, 128><<<grid, kThreads, 0, s>>>(p);
  else append_kernel<E4M3, F16, VEC, 64><<<grid, kThreads, 0, s>>>(p);
}

// Rows of k and v start on 16 bytes.
bool rows_aligned16(const Kv8& p) {
  const int64_t es = p.f16 ? 2 : 4;
  return ((reinterpret_cast<uintptr_t>(p.k) | reinterpret_cast<uintptr_t>(p.v)) & 15u) == 0 && (p.ks * es) % 16 == 0 && (p.vs * es) % 16 == 0;
}

}  // namespace

cudaError_t launch_kv8_append(const Kv8& p, cudaStream_t s) {
  if (p.tokens == 0 || p.seqs == 0) return cudaSuccess;
  // A touched page takes at least one row, and a sequence's n rows touch at most n / page + 2 pages.
  const int64_t most = p.tokens / p.page + 2 * static_cast<int64_t>(p.seqs);
  const dim3 grid(static_cast<unsigned>(most < p.tokens ? most : p.tokens), static_cast<unsigned>(p.hkv));
  const bool vec = rows_aligned16(p);
  const int form = (p.e4m3 ? 4 : 0) | (p.f16 ? 2 : 0) | (vec ? 1 : 0);
  switch (form) {
    case 0: launch_append<false, false, false>(p, grid, s); break;
    case 1: launch_append<false, false, true>(p, grid, s); break;
    case 2: launch_append<false, true, false>(p, grid, s); break;
    case 3: launch_append<false, true, true>(p, grid, s); break;
    case 4: launch_append<true, false, false>(p, grid, s); break;
    case 5: launch_append<true, false, true>(p, grid, s); break;
    case 6: launch_append<true, true, false>(p, grid, s); break;
    default: launch_append<true, true, true>(p, grid, s); break;
  }
  return cudaGetLastError();
}

cudaError_t launch_kv8_read(const Kv8& p, cudaStream_t s) {
  if (p.tokens == 0 || p.seqs == 0) return cudaSuccess;
  const dim3 grid(static_cast<unsigned>((static_cast<int64_t>(p.tokens) + 7) / 8), 2);
  const bool vec = rows_aligned16(p);
  switch ((p.D == 128 ? 4 : 0) | (p.e4m3 ? 2 : 0) | (p.f16 ? 1 : 0)) {
    case 0: launch_read<false, false, 2>(p, grid, vec, s); break;
    case 1: launch_read<false, true, 2>(p, grid, vec, s); break;
    case 2: launch_read<true, false, 2>(p, grid, vec, s); break;
    case 3: launch_read<true, true, 2>(p, grid, vec, s); break;
    case 4: launch_read<false, false, 4>(p, grid, vec, s); break;
    case 5: launch_read<false, true, 4>(p, grid, vec, s); break;
    case 6: launch_read<true, false, 4>(p, grid, vec, s); break;
    default: launch_read<true, true, 4>(p, grid, vec, s); break;
  }
  return cudaGetLastError();
}

}  // namespace xrgpu
