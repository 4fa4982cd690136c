// Rows as 8-bit codes with one scale, and sums of rows by weights (format: mmnb_int8.h).
//
// Quantisation of a row: s = max|x| / 127 in float32, code = x / s rounded to nearest, ties to even. The quotient is
// not computed: t = x * (1 / s) is off by less than 3e-5 (|t| <= 127, one rounding each of 1 / s and the product), so
// round(t) is the code unless t lies that near to a border; there the border itself is compared, 2 |x| with (2 m + 1) s, exactly
// in 64 bits (24 + 8 bits). A row with a NaN or an infinity has scale NaN and codes 0.
#include <cuda_fp16.h>

#include "mmnb_common.cuh"
#include "mmnb_int8.h"

namespace xrgpu {
namespace {

constexpr int kUnit = 16;                    // values of a thread at a time: 16 bytes of codes
constexpr int kRowThreads = 512;             // of a row at the most
constexpr unsigned kErrOrder = 0x702;
constexpr float kMagic = 12582912.0f;        // 1.5 * 2^23: t + kMagic rounds t to a whole number
constexpr float kNearBorder = 0.49996f;
constexpr float kSmallScale = 7.9e-31f;      // about 2^-100: below, 1 / s is not used

// code of x for scale s, from the exact quotient.
__device__ __forceinline__ int exact_code(float x, float s) {
  const double a = 2.0 * fabs(static_cast<double>(x)), d = static_cast<double>(s);
  double m = floor(a / (2.0 * d));
  m = m > 127.0 ? 127.0 : m;
  const double border = (2.0 * m + 1.0) * d;  // of m and m + 1
  int c = static_cast<int>(m);
  if (a > border || (a == border && (c & 1))) ++c;
  c = min(c, 127);
  return x < 0.0f ? -c : c;
}

__device__ __forceinline__ uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return prmt(prmt(a, b, 0x0040), prmt(c, d, 0x0040), 0x5410);
}

// The 16 codes of a thread.
__device__ __forceinline__ uint4 codes16(const float (&v)[kUnit], float s, float inv) {
  uint32_t b[kUnit];
  float worst = 0.0f;
#pragma unroll
  for (int i = 0; i < kUnit; ++i) {
    const float t = v[i] * inv, r = t + kMagic;
    b[i] = __float_as_uint(r);
    worst = fmaxf(worst, fabsf(t - (r - kMagic)));
  }
  if (worst > kNearBorder) {
#pragma unroll
    for (int i = 0; i < kUnit; ++i) {
      const float t = v[i] * inv, r = t + kMagic;
      if (fabsf(t - (r - kMagic)) > kNearBorder) b[i] = static_cast<uint32_t>(exact_code(v[i], s));
    }
  }
  return make_uint4(pack4(b[0], b[1], b[2], b[3]), pack4(b[4], b[5], b[6], b[7]), pack4(b[8], b[9], b[10], b[11]),
                    pack4(b[12], b[13], b[14], b[15]));
}

// 16 values from k0 on of a row, zeros behind K, as they are held (raw) and as floats.
template <bool F16, bool VEC>
struct Unit {
  uint4 raw[F16 ? 2 : 4];
  __device__ __forceinline__ void load(const void* x, int64_t row_at, int64_t k0, int64_t K) {
    constexpr int es = F16 ? 2 : 4;
    if (k0 >= K) {
#pragma unroll
      for (int i = 0; i < (F16 ? 2 : 4); ++i) raw[i] = make_uint4(0, 0, 0, 0);
    } else if (VEC && k0 + kUnit <= K) {
      const uint4* src = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(x) + (row_at + k0) * es);
#pragma unroll
      for (int i = 0; i < (F16 ? 2 : 4); ++i) raw[i] = src[i];
    } else {
      uint32_t u[F16 ? 8 : 16];
#pragma unroll
      for (int i = 0; i < (F16 ? 8 : 16); ++i) {
        if (F16) {
          const uint16_t* h = static_cast<const uint16_t*>(x) + row_at + k0;
          const uint32_t lo = k0 + 2 * i < K ? h[2 * i] : 0, hi = k0 + 2 * i + 1 < K ? h[2 * i + 1] : 0;
          u[i] = lo | hi << 16;
        } else {
          u[i] = k0 + i < K ? static_cast<const uint32_t*>(x)[row_at + k0 + i] : 0;
        }
      }
#pragma unroll
      for (int i = 0; i < (F16 ? 2 : 4); ++i) raw[i] = make_uint4(u[4 * i], u[4 * i + 1], u[4 * i + 2], u[4 * i + 3]);
    }
  }
  // the bits of the largest magnitude as float32 (NaN > infinity > numbers)
  __device__ __forceinline__ uint32_t amax() const {
    const uint32_t* u = reinterpret_cast<const uint32_t*>(raw);
    if (F16) {
      __half2 m = __float2half2_rn(0.0f);
#pragma unroll
      for (int i = 0; i < 8; ++i) m = __hmax2_nan(m, __habs2(*reinterpret_cast<const __half2*>(&u[i])));
      return __float_as_uint(__half2float(__hmax_nan(__low2half(m), __high2half(m)))) & 0x7fffffffu;
    }
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < (F16 ? 8 : 16); ++i) m = max(m, u[i] & 0x7fffffffu);
    return m;
  }
  __device__ __forceinline__ void floats(float (&v)[kUnit]) const {
    const uint32_t* u = reinterpret_cast<const uint32_t*>(raw);
#pragma unroll
    for (int i = 0; i < kUnit; ++i) {
      if (F16) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i >> 1]));
        v[i] = (i & 1) ? f.y : f.x;
      } else {
        v[i] = __uint_as_float(u[F16 ? 0 : i]);
      }
    }
  }
};

// The row that row r stands for, -1 where it fits none (recorded).
__device__ __forceinline__ int64_t source_row(const RowOrder& f, int64_t r) {
  if (!f.order) return r;
  const int o = f.order[r], t = o / f.top_k;
  if (o >= 0 && t < f.rows) return t;
  record_device_error(f.err, kErrOrder);
  return -1;
}

// blockDim.x threads (whole warps) a row, blockDim.y rows a CTA. HELD: a row is at most UNITS units a thread, kept in
// registers between the two passes; else it is read twice.
template <bool F16, bool VEC, int UNITS, bool HELD>
__global__ void __launch_bounds__(kRowThreads) quantize_kernel(const Int8Rows p) {
  __shared__ uint32_t part[32];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // a product's weights may start to load
  const int64_t row = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y;
  const bool real = row < p.rows;
  const int64_t from = real ? source_row(p.from, row) : 0, row_at = max(from, static_cast<int64_t>(0)) * p.ldx, units = real ? (p.K + kUnit - 1) / kUnit : 0;
  const int64_t read = real && from >= 0 ? p.K : 0;  // values of x that count
  Unit<F16, VEC> u[UNITS];
  uint32_t amax = 0;
  if (HELD) {
#pragma unroll
    for (int i = 0; i < UNITS; ++i) u[i].load(p.x, row_at, (threadIdx.x + static_cast<int64_t>(i) * blockDim.x) * kUnit, read);
#pragma unroll
    for (int i = 0; i < UNITS; ++i) amax = max(amax, u[i].amax());
  } else {
    for (int64_t at = threadIdx.x; at < units; at += blockDim.x) {
      u[0].load(p.x, row_at, at * kUnit, read);
      amax = max(amax, u[0].amax());
    }
  }
  amax = __reduce_max_sync(~0u, amax);
  const int warps = blockDim.x >> 5;
  if (warps > 1) {
    const int w = threadIdx.x >> 5;
    if ((threadIdx.x & 31) == 0) part[threadIdx.y * warps + w] = amax;
    __syncthreads();
    const int lane = threadIdx.x & 31;
    amax = __reduce_max_sync(~0u, lane < warps ? part[threadIdx.y * warps + lane] : 0u);
  }
  if (!real) return;
  const bool bad = amax >= 0x7f800000u;
  const float s = bad ? __uint_as_float(0x7fc00000u) : __fdiv_rn(__uint_as_float(amax), 127.0f);
  if (threadIdx.x == 0) p.scales[row] = s;
  const bool none = bad || s == 0.0f;
  const float inv = none ? 0.0f : __fdiv_rn(1.0f, s);
  uint4* dst = reinterpret_cast<uint4*>(p.codes + row * p.ldc);
  auto store = [&](const Unit<F16, VEC>& x, int64_t at) {
    float v[kUnit];
    x.floats(v);
    if (none) {
      dst[at] = make_uint4(0, 0, 0, 0);
    } else if (!F16 && s < kSmallScale) {
      uint32_t b[kUnit];
#pragma unroll
      for (int i = 0; i < kUnit; ++i) b[i] = static_cast<uint32_t>(exact_code(v[i], s));
      dst[at] = make_uint4(pack4(b[0], b[1], b[2], b[3]), pack4(b[4], b[5], b[6], b[7]), pack4(b[8], b[9], b[10], b[11]),
                           pack4(b[12], b[13], b[14], b[15]));
    } else {
      dst[at] = codes16(v, s, inv);
    }
  };
  if (HELD) {
#pragma unroll
    for (int i = 0; i < UNITS; ++i)
      if (threadIdx.x + static_cast<int64_t>(i) * blockDim.x < units) store(u[i], threadIdx.x + static_cast<int64_t>(i) * blockDim.x);
  } else {
    for (int64_t at = threadIdx.x; at < units; at += blockDim.x) {
      u[0].load(p.x, row_at, at * kUnit, read);
      store(u[0], at);
    }
  }
}

__global__ void __launch_bounds__(256) gather_kernel(const Int8Gather p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int64_t row = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y;
  if (row >= p.rows) return;
  const int64_t from = source_row(p.from, row);
  if (threadIdx.x == 0) p.scales[row] = from >= 0 ? p.a_scales[from] : 0.0f;
  const uint4* src = reinterpret_cast<const uint4*>(p.a + max(from, static_cast<int64_t>(0)) * p.lds);
  uint4* dst = reinterpret_cast<uint4*>(p.codes + row * p.ldc);
  const int64_t whole = p.K / kUnit;
#pragma unroll 4
  for (int64_t at = threadIdx.x; at < whole; at += blockDim.x) dst[at] = src[at];
  for (int64_t k = whole * kUnit + threadIdx.x; k < p.K; k += blockDim.x) p.codes[row * p.ldc + k] = reinterpret_cast<const int8_t*>(src)[k];
}

template <bool F16, bool VEC>
__global__ void __launch_bounds__(256) dequantize_kernel(const Int8Rows p) {
  const int64_t row = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y;
  if (row >= p.rows) return;
  const float s = p.scales[row];
  const int8_t* src = p.codes + row * p.ldc;
  if (VEC) {  // K a multiple of 16
    for (int64_t at = threadIdx.x; at < p.K / kUnit; at += blockDim.x) {
      const uint4 c = reinterpret_cast<const uint4*>(src)[at];
      const uint32_t w[4] = {c.x, c.y, c.z, c.w};
      float v[kUnit];
#pragma unroll
      for (int i = 0; i < kUnit; ++i) v[i] = static_cast<float>(static_cast<int8_t>(w[i >> 2] >> (8 * (i & 3)))) * s;
      if (F16) {
        uint32_t h[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const __half2 x = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
          h[i] = *reinterpret_cast<const uint32_t*>(&x);
        }
        uint4* d = reinterpret_cast<uint4*>(static_cast<__half*>(p.out) + row * p.K + at * kUnit);
        d[0] = make_uint4(h[0], h[1], h[2], h[3]);
        d[1] = make_uint4(h[4], h[5], h[6], h[7]);
      } else {
        float4* d = reinterpret_cast<float4*>(static_cast<float*>(p.out) + row * p.K + at * kUnit);
#pragma unroll
        for (int i = 0; i < 4; ++i) d[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
      }
    }
  } else {
    for (int64_t k = threadIdx.x; k < p.K; k += blockDim.x) {
      const float v = static_cast<float>(src[k]) * s;
      if (F16) static_cast<__half*>(p.out)[row * p.K + k] = __float2half_rn(v);
      else static_cast<float*>(p.out)[row * p.K + k] = v;
    }
  }
}

// One thread 4 columns of a token.
constexpr int kSumThreads = 256;
template <bool F16>
__global__ void __launch_bounds__(kSumThreads) weighted_rows_kernel(const WeightedRows p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int64_t t = blockIdx.x, n = 4 * (static_cast<int64_t>(blockIdx.y) * kSumThreads + threadIdx.x);
  if (n >= p.N) return;
  float r[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 8
  for (int j = 0; j < p.top_k; ++j) {
    const int32_t slot = p.slots[t * p.top_k + j];
    const float w = p.weights[t * p.top_k + j];
    if (slot < 0 || slot >= p.rows) continue;
    const float4 v = *reinterpret_cast<const float4*>(p.y + slot * p.ldy + n);
    r[0] = fmaf(w, v.x, r[0]);
    r[1] = fmaf(w, v.y, r[1]);
    r[2] = fmaf(w, v.z, r[2]);
    r[3] = fmaf(w, v.w, r[3]);
  }
  const int64_t at = t * p.ldo + n;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (n + i >= p.N) break;
    if (F16) static_cast<__half*>(p.out)[at + i] = __float2half_rn(r[i]);
    else static_cast<float*>(p.out)[at + i] = r[i];
  }
}

template <bool F16, bool VEC>
cudaError_t quantize(const Int8Rows& p, cudaStream_t s) {
  // Units a thread: a row has about 256 threads, and it stays in registers (8 or 16 of them a unit).
  const int64_t units = ceil_div(p.K, kUnit);
  const int64_t per = units <= 256 ? 1 : units <= 512 ? 2 : 4;
  const int64_t threads = align_up(ceil_div(units, per), 32);
  const bool held = threads <= kRowThreads;
  const unsigned tx = static_cast<unsigned>(held ? threads : kRowThreads), ty = tx < 256 ? 256 / tx : 1;
  const int64_t blocks = ceil_div(p.rows, ty);
  if (blocks > 0x7fffffff) return cudaErrorInvalidValue;
  const dim3 grid(static_cast<unsigned>(blocks)), block(tx, ty);
  if (!held) quantize_kernel<F16, VEC, 1, false><<<grid, block, 0, s>>>(p);
  else if (per == 1) quantize_kernel<F16, VEC, 1, true><<<grid, block, 0, s>>>(p);
  else if (per == 2) quantize_kernel<F16, VEC, 2, true><<<grid, block, 0, s>>>(p);
  else quantize_kernel<F16, VEC, 4, true><<<grid, block, 0, s>>>(p);
  return cudaGetLastError();
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace

cudaError_t launch_int8_quantize(const Int8Rows& p, cudaStream_t s) {
  const bool vec = aligned16(p.x) && (p.ldx * (p.f16 ? 2 : 4)) % 16 == 0;
  if (p.f16) return vec ? quantize<true, true>(p, s) : quantize<true, false>(p, s);
  return vec ? quantize<false, true>(p, s) : quantize<false, false>(p, s);
}

cudaError_t launch_int8_dequantize(const Int8Rows& p, cudaStream_t s) {
  const bool vec = p.K % kUnit == 0 && aligned16(p.out);
  const int64_t items = vec ? p.K / kUnit : p.K;
  const unsigned tx = items >= 256 ? 256 : static_cast<unsigned>(align_up(items, 32)), ty = 256 / tx;
  const int64_t blocks = ceil_div(p.rows, ty);
  if (blocks > 0x7fffffff) return cudaErrorInvalidValue;
  const dim3 grid(static_cast<unsigned>(blocks)), block(tx, ty);
  if (p.f16) vec ? dequantize_kernel<true, true><<<grid, block, 0, s>>>(p) : dequantize_kernel<true, false><<<grid, block, 0, s>>>(p);
  else vec ? dequantize_kernel<false, true><<<grid, block, 0, s>>>(p) : dequantize_kernel<false, false><<<grid, block, 0, s>>>(p);
  return cudaGetLastError();
}

cudaError_t launch_int8_gather(const Int8Gather& p, cudaStream_t s) {
  const int64_t units = ceil_div(p.K, kUnit);
  const unsigned tx = units >= 256 ? 256 : static_cast<unsigned>(align_up(units, 32)), ty = 256 / tx;
  const int64_t blocks = ceil_div(p.rows, ty);
  if (blocks > 0x7fffffff) return cudaErrorInvalidValue;
  gather_kernel<<<static_cast<unsigned>(blocks), dim3(tx, ty), 0, s>>>(p);
  return cudaGetLastError();
}

cudaError_t launch_weighted_rows(const WeightedRows& p, cudaStream_t s) {
  const int64_t parts = ceil_div(p.N, 4 * kSumThreads);
  if (p.tokens > 0x7fffffff || parts > 65535) return cudaErrorInvalidValue;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(p.tokens), static_cast<unsigned>(parts));
  cfg.blockDim = dim3(kSumThreads);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return p.f16 ? cudaLaunchKernelEx(&cfg, weighted_rows_kernel<true>, p) : cudaLaunchKernelEx(&cfg, weighted_rows_kernel<false>, p);
}

}  // namespace xrgpu
