// Rows as 8-bit codes with one scale, and sums of rows by weights (format: mmnb_int8.h).
#include <cuda_fp16.h>

#include "mmnb_int8.cuh"
#include "mmnb_int8.h"

namespace xrgpu {
namespace {

constexpr int kUnit = 16;                    // codes of 16 bytes
constexpr int kRowThreads = 1024;            // of a row at the most
constexpr unsigned kErrOrder = 0x702;

// The row that row r stands for, -1 where it fits none (recorded).
__device__ __forceinline__ int64_t source_row(const RowOrder& f, int64_t r) {
  if (!f.order) return r;
  const int o = f.order[r], t = o / f.by_top_k;
  if (o >= 0 && t < f.rows) return t;
  record_device_error(f.err, kErrOrder);
  return -1;
}

// blockDim.x threads (whole warps) a row, blockDim.y rows a CTA. HELD: a row is at most UNITS units a thread, kept in
// registers between the two passes; else it is read twice. What bounds it is the stream, then instructions (12 a value before pairs of
// float32 numbers were one: 2048 x 14336 halves 19.3 us, now 17.2, 88 MB, 5.1 TB/s; 16384 x 4096 floats 54 us, 6.2 TB/s).
template <bool F16, bool VEC, int UNITS, bool HELD>
__global__ void __launch_bounds__(kRowThreads) quantize_kernel(const Int8Rows p) {
  using U = Unit<F16, VEC>;
  __shared__ uint32_t part[32];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // a product's weights may start to load
  const int64_t row = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y;
  const bool real = row < p.rows;
  const int64_t from = real ? source_row(p.from, row) : -1;
  const uint8_t* x = static_cast<const uint8_t*>(p.x) + max(from, static_cast<int64_t>(0)) * p.ldx * (F16 ? 2 : 4);
  const int read = from >= 0 ? static_cast<int>(p.K) : 0;  // values of x that count
  const int units = real ? static_cast<int>((p.K + U::kValues - 1) / U::kValues) : 0;
  U u[UNITS];
  Largest<F16> largest;
  if (HELD) {
#pragma unroll
    for (int i = 0; i < UNITS; ++i) u[i].load(x, (threadIdx.x + i * blockDim.x) * U::kValues, read);
#pragma unroll
    for (int i = 0; i < UNITS; ++i) u[i].largest(largest);
  } else {
    for (int at = threadIdx.x; at < units; at += blockDim.x) {
      u[0].load(x, at * U::kValues, read);
      u[0].largest(largest);
    }
  }
  uint32_t amax = __reduce_max_sync(~0u, largest.bits());
  const int warps = blockDim.x >> 5;
  if (warps > 1) {
    const int lane = threadIdx.x & 31;
    if (lane == 0) part[threadIdx.y * warps + (threadIdx.x >> 5)] = amax;
    __syncthreads();
    amax = __reduce_max_sync(~0u, lane < warps ? part[threadIdx.y * warps + lane] : 0u);
  }
  if (!real) return;
  Scale c;
  bool none;
  const float s = row_scale_of<F16>(amax, &c, &none);
  if (threadIdx.x == 0) p.scales[row] = s;
  int8_t* codes = p.codes + row * p.ldc;
  auto store = [&](const U& x, int at) {
    uint32_t w[2];
    x.codes(c, w);
    if (F16) reinterpret_cast<uint2*>(codes)[at] = none ? make_uint2(0, 0) : make_uint2(w[0], w[1]);
    else reinterpret_cast<uint32_t*>(codes)[at] = none ? 0 : w[0];
  };
  if (HELD) {
#pragma unroll
    for (int i = 0; i < UNITS; ++i) {
      const int at = threadIdx.x + i * blockDim.x;
      if (at < units) store(u[i], at);
    }
  } else {
    for (int at = threadIdx.x; at < units; at += blockDim.x) {
      u[0].load(x, at * U::kValues, read);
      store(u[0], at);
    }
  }
}

// blockDim.x threads take kGatherRows rows at a time, blockDim.y such sets a CTA: their entries of the order, then their codes, are
// loaded side by side (one row at a time: 45 us for 16384 rows of 4096 codes).
constexpr int kGatherRows = 4;
__global__ void __launch_bounds__(256) gather_kernel(const Int8Gather p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int64_t row = (static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y) * kGatherRows;
  const int rows = static_cast<int>(min(p.rows - row, static_cast<int64_t>(kGatherRows)));
  int64_t from[kGatherRows];
#pragma unroll
  for (int i = 0; i < kGatherRows; ++i) from[i] = i < rows ? source_row(p.from, row + i) : -1;
  if (static_cast<int>(threadIdx.x) < rows) {
    int64_t f = from[0];
#pragma unroll
    for (int i = 1; i < kGatherRows; ++i) f = threadIdx.x == i ? from[i] : f;
    p.scales[row + threadIdx.x] = f >= 0 ? p.a_scales[f] : 0.0f;
  }
  const int whole = static_cast<int>(p.K / kUnit);
  for (int at = threadIdx.x; at < whole; at += blockDim.x) {
    uint4 v[kGatherRows];
#pragma unroll
    for (int i = 0; i < kGatherRows; ++i)  // a row that fits none: any codes, its scale is 0
      if (i < rows) v[i] = reinterpret_cast<const uint4*>(p.a + max(from[i], static_cast<int64_t>(0)) * p.lds)[at];
#pragma unroll
    for (int i = 0; i < kGatherRows; ++i)
      if (i < rows) reinterpret_cast<uint4*>(p.codes + (row + i) * p.ldc)[at] = v[i];
  }
  for (int64_t k = static_cast<int64_t>(whole) * kUnit + threadIdx.x; k < p.K; k += blockDim.x) {  // the last row may end with its codes
#pragma unroll
    for (int i = 0; i < kGatherRows; ++i)
      if (i < rows) p.codes[(row + i) * p.ldc + k] = p.a[max(from[i], static_cast<int64_t>(0)) * p.lds + k];
  }
}

// VEC: 16 bytes of values a thread at a time (K a multiple of 16). 2048 x 14336 halves 13.9 us, 6.3 TB/s.
template <bool F16, bool VEC>
__global__ void __launch_bounds__(256) dequantize_kernel(const Int8Rows p) {
  const int64_t row = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y;
  if (row >= p.rows) return;
  const float s = p.scales[row];
  const int8_t* src = p.codes + row * p.ldc;
  if (VEC) {
    const int items = static_cast<int>(p.K / (F16 ? 8 : 4));
#pragma unroll 4
    for (int at = threadIdx.x; at < items; at += blockDim.x) {
      uint32_t w[2];
      if (F16) {
        const uint2 c = reinterpret_cast<const uint2*>(src)[at];
        w[0] = c.x;
        w[1] = c.y;
      } else {
        w[0] = reinterpret_cast<const uint32_t*>(src)[at];
      }
      uint32_t o[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (F16) {
          const uint32_t pair = w[i >> 1] >> (16 * (i & 1));
          const __half2 h = __floats2half2_rn(static_cast<float>(static_cast<int8_t>(pair)) * s, static_cast<float>(static_cast<int8_t>(pair >> 8)) * s);
          o[i] = *reinterpret_cast<const uint32_t*>(&h);
        } else {
          o[i] = __float_as_uint(static_cast<float>(static_cast<int8_t>(w[0] >> (8 * i))) * s);
        }
      }
      reinterpret_cast<uint4*>(static_cast<uint8_t*>(p.out) + row * p.K * (F16 ? 2 : 4))[at] = make_uint4(o[0], o[1], o[2], o[3]);
    }
  } else {
    for (int64_t k = threadIdx.x; k < p.K; k += blockDim.x) {
      const float v = static_cast<float>(src[k]) * s;
      if (F16) static_cast<__half*>(p.out)[row * p.K + k] = __float2half_rn(v);
      else static_cast<float*>(p.out)[row * p.K + k] = v;
    }
  }
}

// One thread 4 columns of a token. Bound by the stream, and by what the product before it still writes back (4096 tokens by 4 rows of
// 4096: 301 MB, 71 us).
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
  // Units a thread, in registers while a row has no more than 1024 threads of 8. Many rows: four, so that a thread has some loads under
  // way and few threads meet for a row (16384 x 2048 halves 27.3 -> 19.6 us, 32768 x 1024 27.3 -> 17.9); few rows: as many
  // threads as a row feeds.
  const int64_t units = ceil_div(p.K, Unit<F16, VEC>::kValues);
  const int64_t per = p.rows >= 8 * device_sm_count() ? (units <= 32 ? 1 : units <= 64 ? 2 : units <= 1024 ? 4 : 8)
                                                      : (units <= 256 ? 1 : units <= 512 ? 2 : units <= 1024 ? 4 : 8);
  const int64_t threads = align_up(ceil_div(units, per), 32);
  const bool held = threads <= kRowThreads;
  const unsigned tx = static_cast<unsigned>(held ? threads : kRowThreads), ty = tx < 256 ? 256 / tx : 1;
  const int64_t blocks = ceil_div(p.rows, ty);
  if (blocks > 0x7fffffff) return cudaErrorInvalidValue;
  const dim3 grid(static_cast<unsigned>(blocks)), block(tx, ty);
  if (!held) quantize_kernel<F16, VEC, 1, false><<<grid, block, 0, s>>>(p);
  else if (per == 1) quantize_kernel<F16, VEC, 1, true><<<grid, block, 0, s>>>(p);
  else if (per == 2) quantize_kernel<F16, VEC, 2, true><<<grid, block, 0, s>>>(p);
  else if (per == 4) quantize_kernel<F16, VEC, 4, true><<<grid, block, 0, s>>>(p);
  else quantize_kernel<F16, VEC, 8, true><<<grid, block, 0, s>>>(p);
  return cudaGetLastError();
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace

cudaError_t launch_int8_quantize(const Int8Rows& p, cudaStream_t s) {
  const bool vec = aligned16(p.x) && (p.ldx * (p.f16 ? 2 : 4)) % 16 == 0 && p.K % (p.f16 ? 8 : 4) == 0;
  if (p.f16) return vec ? quantize<true, true>(p, s) : quantize<true, false>(p, s);
  return vec ? quantize<false, true>(p, s) : quantize<false, false>(p, s);
}

cudaError_t launch_int8_dequantize(const Int8Rows& p, cudaStream_t s) {
  const bool vec = p.K % kUnit == 0 && aligned16(p.out);
  const int64_t items = vec ? p.K / (p.f16 ? 8 : 4) : p.K;
  const unsigned tx = items >= 256 ? 256 : static_cast<unsigned>(align_up(items, 32)), ty = 256 / tx;
  const int64_t blocks = ceil_div(p.rows, ty);
  if (blocks > 0x7fffffff) return cudaErrorInvalidValue;
  const dim3 grid(static_cast<unsigned>(blocks)), block(tx, ty);
  if (p.f16) vec ? dequantize_kernel<true, true><<<grid, block, 0, s>>>(p) : dequantize_kernel<true, false><<<grid, block, 0, s>>>(p);
  else vec ? dequantize_kernel<false, true><<<grid, block, 0, s>>>(p) : dequantize_kernel<false, false><<<grid, block, 0, s>>>(p);
  return cudaGetLastError();
}

cudaError_t launch_int8_gather(const Int8Gather& p, bool early, cudaStream_t s) {
  const int64_t units = ceil_div(p.K, kUnit);
  const unsigned tx = units >= 256 ? 256 : static_cast<unsigned>(align_up(units, 32)), ty = 256 / tx;
  const int64_t blocks = ceil_div(p.rows, ty * kGatherRows);
  if (blocks > 0x7fffffff) return cudaErrorInvalidValue;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
  cfg.blockDim = dim3(tx, ty);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = early ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, gather_kernel, p);
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
