// Microscaled 4-bit floating point: quantisation, dequantisation, scale layout (format: mmnb_mxfp4.h).
//
// Quantisation of a block: a = max |x|, E = max(floor(log2 a) - 2, -127) (2 is the exponent of the
// largest code, 6 = 1.5 * 2^2), code = x * 2^-E rounded to nearest, ties to the even code, saturating
// at 6, the sign of x kept. floor(log2 a) is a's exponent field, so nothing is approximated: x * 2^-E is
// exact and the conversion rounds once. A block that holds a NaN or an infinity has scale byte 255
// and codes 0.
#include <cuda_fp16.h>

#include "mmnb_common.cuh"
#include "mmnb_mxfp4.h"

namespace xrgpu {
namespace {

__device__ __forceinline__ int64_t scale_offset(int64_t row, int64_t blk, int64_t kb) {
  return ((row >> 7) * ((kb + 3) >> 2) + (blk >> 2)) * 512 + (row & 31) * 16 + ((row >> 5) & 3) * 4 + (blk & 3);
}

// Two codes in a byte: lo in the low nibble.
__device__ __forceinline__ uint32_t to_e2m1x2(float lo, float hi) {
  uint32_t r;
  asm("{\n\t.reg .b8 t;\n\tcvt.rn.satfinite.e2m1x2.f32 t, %2, %1;\n\tcvt.u32.u8 %0, t;\n\t}" : "=r"(r) : "f"(lo), "f"(hi));
  return r;
}

__device__ __forceinline__ float pow2_of_byte(uint32_t e) {  // 2^(e - 127), e = 255: NaN
  return e == 255u ? __uint_as_float(0x7fc00000u) : __uint_as_float(e ? e << 23 : 1u << 22);
}

// The two values of a byte of codes.
__device__ __forceinline__ float2 from_e2m1x2(uint32_t byte) {
  uint32_t r;
  asm("{\n\t.reg .b8 t;\n\tcvt.u8.u32 t, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, t;\n\t}" : "=r"(r) : "r"(byte));
  return __half22float2(*reinterpret_cast<const __half2*>(&r));
}

constexpr int kQuantWarps = 8;
constexpr int kPer = 16;           // values of a lane: two lanes a block
constexpr int kChunk = 32 * kPer;  // values of a row that a warp takes at a time

// The (row, chunk) pairs of a warp, in order, a grid's warps apart, stepped by its quotient and remainder. What bounds
// these kernels is instructions, not their bytes: 2048 x 14336 halves (74 MB) took 23.8 us (dequantised 19.9) with a 64-bit division
// an item, 22.4 (18.1) without, 14.2 (17.0) with 16 values a lane instead of 8 and maxima of pairs of halves; 14.0 (5.3 TB/s)
// dequantised with the 16 in two pieces.
struct Walk {
  int64_t row, rows_step;
  int chunk, chunk_step;
  __device__ explicit Walk(int chunks) {
    const unsigned n = static_cast<unsigned>(chunks), at = blockIdx.x * kQuantWarps + (threadIdx.x >> 5), step = gridDim.x * kQuantWarps;
    row = at / n;
    chunk = static_cast<int>(at % n);
    rows_step = step / n;
    chunk_step = static_cast<int>(step % n);
  }
  __device__ void next(int chunks) {
    row += rows_step;
    chunk += chunk_step;
    if (chunk >= chunks) {
      chunk -= chunks;
      ++row;
    }
  }
};

// One warp a (row, chunk); rows beyond the matrix up to the tile's end only zero their scales.
template <bool F16, bool VEC>
__global__ void __launch_bounds__(kQuantWarps * 32) quantize_kernel(const Mxfp4Quantize p, int chunks, int64_t rows) {
  const int lane = threadIdx.x & 31;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // a product's weights may start to load
  for (Walk w(chunks); w.row < rows; w.next(chunks)) {
    const int64_t row = w.row, k0 = static_cast<int64_t>(w.chunk) * kChunk + lane * kPer;
    float v[kPer];
    uint32_t amax = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) v[i] = 0.0f;
    if (row < p.rows && k0 < p.K) {
      if (VEC && k0 + kPer <= p.K) {
        const uint4* src = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(p.x) + (row * p.ldx + k0) * (F16 ? 2 : 4));
        uint4 raw[F16 ? 2 : 4];
#pragma unroll
        for (int i = 0; i < (F16 ? 2 : 4); ++i) raw[i] = src[i];
        const uint32_t* u = reinterpret_cast<const uint32_t*>(raw);
        if (F16) {
          __half2 m = __float2half2_rn(0.0f);  // pairs as they are: half the instructions
#pragma unroll
          for (int i = 0; i < kPer / 2; ++i) {
            const __half2 h = *reinterpret_cast<const __half2*>(&u[i]);
            m = __hmax2_nan(m, __habs2(h));
            const float2 f = __half22float2(h);
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
          }
          amax = __float_as_uint(__half2float(__hmax_nan(__low2half(m), __high2half(m)))) & 0x7fffffffu;
        } else {
#pragma unroll
          for (int i = 0; i < kPer; ++i) v[i] = __uint_as_float(u[F16 ? 0 : i]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < kPer; ++i)
          if (k0 + i < p.K) v[i] = load_f(p.x, F16, row * p.ldx + k0 + i);
      }
    }
    if (!(F16 && VEC) || k0 + kPer > p.K) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) amax = max(amax, __float_as_uint(v[i]) & 0x7fffffffu);  // NaN > Inf > finite as bits
    }
    amax = max(amax, __shfl_xor_sync(~0u, amax, 1));
    const uint32_t field = amax >> 23;
    const bool bad = field == 255u;
    const uint32_t e = bad ? 255u : (field > 2u ? field - 2u : 0u);
    const float inv = bad ? 0.0f : __uint_as_float((254u - e) << 23);  // 2^(127 - e); e <= 252 here
    uint32_t c[2] = {0, 0};
    if (!bad) {
#pragma unroll
      for (int i = 0; i < kPer / 2; ++i) c[i >> 2] |= to_e2m1x2(v[2 * i] * inv, v[2 * i + 1] * inv) << (8 * (i & 3));
    }
    const int64_t blk = k0 >> 5;
    if (row < p.rows && blk < p.kb) *reinterpret_cast<uint2*>(p.codes + (row * p.kb + blk) * 16 + (lane & 1) * 8) = make_uint2(c[0], c[1]);
    // the four scale bytes of 8 lanes as one word
    const uint32_t eb = (row < p.rows && blk < p.kb) ? e : 0u;
    uint32_t word = eb << (8 * ((lane >> 1) & 3));
    word |= __shfl_xor_sync(~0u, word, 2);
    word |= __shfl_xor_sync(~0u, word, 4);
    if ((lane & 7) == 0 && (blk >> 2) < ((p.kb + 3) >> 2)) *reinterpret_cast<uint32_t*>(p.scales + scale_offset(row, blk, p.kb)) = word;
  }
}

// The same chunks as two pieces of 8 values a lane, so that a warp writes a whole range at a time.
template <bool F16, bool VEC>
__global__ void __launch_bounds__(kQuantWarps * 32) dequantize_kernel(const Mxfp4Dequantize p, int chunks) {
  constexpr int kPieces = 2, kEach = kPer / kPieces;
  const int lane = threadIdx.x & 31;
  for (Walk at_item(chunks); at_item.row < p.rows; at_item.next(chunks)) {
    const int64_t row = at_item.row, first = static_cast<int64_t>(at_item.chunk) * kChunk + lane * kEach;
    uint32_t w[kPieces];
    float s[kPieces];
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int64_t k0 = first + i * 32 * kEach, blk = k0 >> 5;
      if (k0 >= p.K) continue;
      w[i] = reinterpret_cast<const uint32_t*>(p.codes + (row * p.kb + blk) * 16)[lane & 3];
      s[i] = pow2_of_byte(p.scales[scale_offset(row, blk, p.kb)]);
    }
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int64_t k0 = first + i * 32 * kEach, at = row * p.K + k0;
      if (k0 >= p.K) continue;
      float v[kEach];
#pragma unroll
      for (int j = 0; j < kEach / 2; ++j) {
        const float2 f = from_e2m1x2((w[i] >> (8 * j)) & 255u);
        v[2 * j] = f.x * s[i];
        v[2 * j + 1] = f.y * s[i];
      }
      if (VEC) {  // K is a multiple of 8
        if (F16) {
          uint32_t h[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const __half2 x = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
            h[j] = *reinterpret_cast<const uint32_t*>(&x);
          }
          *reinterpret_cast<uint4*>(static_cast<__half*>(p.out) + at) = make_uint4(h[0], h[1], h[2], h[3]);
        } else {
          float4* dst = reinterpret_cast<float4*>(static_cast<float*>(p.out) + at);
          dst[0] = make_float4(v[0], v[1], v[2], v[3]);
          dst[1] = make_float4(v[4], v[5], v[6], v[7]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
          if (k0 + j >= p.K) break;
          if (F16) static_cast<__half*>(p.out)[at + j] = __float2half_rn(v[j]);
          else static_cast<float*>(p.out)[at + j] = v[j];
        }
      }
    }
  }
}

__global__ void __launch_bounds__(256) tile_scales_kernel(const uint8_t* src, uint8_t* dst, int64_t rows, int64_t kb, int64_t bytes) {
  const int64_t tiles_k = (kb + 3) >> 2;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < bytes; i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int64_t tile = i >> 9, row = (tile / tiles_k) * 128 + ((i >> 2) & 3) * 32 + ((i >> 4) & 31), blk = (tile % tiles_k) * 4 + (i & 3);
    dst[i] = (row < rows && blk < kb) ? src[row * kb + blk] : 0;
  }
}

int grid_for(int64_t blocks, int per_sm) {
  const int64_t most = static_cast<int64_t>(device_sm_count()) * per_sm;
  return static_cast<int>(blocks < most ? (blocks > 0 ? blocks : 1) : most);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace

cudaError_t launch_mxfp4_quantize(const Mxfp4Quantize& p, cudaStream_t s) {
  const int64_t chunks = ceil_div(p.K, kChunk), rows = ceil_div(p.rows, 128) * 128, items = rows * chunks;
  if (items == 0) return cudaSuccess;
  const int grid = grid_for(ceil_div(items, kQuantWarps), 8);
  // 16-byte loads (a ragged end of a row is loaded one by one): the rows start on 16 bytes
  const int64_t es = p.f16 ? 2 : 4;
  const bool vec = aligned16(p.x) && (p.ldx * es) % 16 == 0;
  if (p.f16) {
    if (vec) quantize_kernel<true, true><<<grid, kQuantWarps * 32, 0, s>>>(p, static_cast<int>(chunks), rows);
    else quantize_kernel<true, false><<<grid, kQuantWarps * 32, 0, s>>>(p, static_cast<int>(chunks), rows);
  } else {
    if (vec) quantize_kernel<false, true><<<grid, kQuantWarps * 32, 0, s>>>(p, static_cast<int>(chunks), rows);
    else quantize_kernel<false, false><<<grid, kQuantWarps * 32, 0, s>>>(p, static_cast<int>(chunks), rows);
  }
  return cudaGetLastError();
}

cudaError_t launch_mxfp4_dequantize(const Mxfp4Dequantize& p, cudaStream_t s) {
  const int64_t chunks = ceil_div(p.K, kChunk), items = p.rows * chunks;
  if (items == 0) return cudaSuccess;
  const int grid = grid_for(ceil_div(items, kQuantWarps), 8);
  const bool vec = aligned16(p.out) && p.K % 8 == 0;
  if (p.f16) {
    if (vec) dequantize_kernel<true, true><<<grid, kQuantWarps * 32, 0, s>>>(p, static_cast<int>(chunks));
    else dequantize_kernel<true, false><<<grid, kQuantWarps * 32, 0, s>>>(p, static_cast<int>(chunks));
  } else {
    if (vec) dequantize_kernel<false, true><<<grid, kQuantWarps * 32, 0, s>>>(p, static_cast<int>(chunks));
    else dequantize_kernel<false, false><<<grid, kQuantWarps * 32, 0, s>>>(p, static_cast<int>(chunks));
  }
  return cudaGetLastError();
}

cudaError_t launch_mxfp4_tile_scales(const uint8_t* scales, uint8_t* tiled, int64_t rows, int64_t kb, cudaStream_t s) {
  const int64_t bytes = mxfp4_scale_bytes(rows, kb);
  if (bytes == 0) return cudaSuccess;
  tile_scales_kernel<<<grid_for(ceil_div(bytes, 256), 8), 256, 0, s>>>(scales, tiled, rows, kb, bytes);
  return cudaGetLastError();
}

}  // namespace xrgpu
