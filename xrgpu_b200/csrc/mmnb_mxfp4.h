// Device-pointer problems and launchers of the microscaled 4-bit floating-point operators
// (mmnb_mxfp4.cu, mmnb_mxfp4_gemm_sm100.cu).
//
// Format. A row of K values is cut into blocks of 32 (kb = ceil(K / 32), the last one padded with
// zeros). A block holds 32 codes of 4 bits (sign, 2 exponent bits, 1 mantissa bit: 0, 0.5, 1, 1.5, 2,
// 3, 4, 6), packed low nibble first in 16 bytes, and one scale byte e: value = code * 2^(e - 127), a
// block with e = 255 is NaN. Codes: [rows][kb][16]. Scales are held in tiles of 128 rows by 4 blocks,
// the order in which the tensor cores take them: [ceil(rows/128)][ceil(kb/4)][32][4][4], the byte of
// (row r, block j) at tile (r / 128, j / 4), position [r % 32][(r % 128) / 32][j % 4]; padding is 0.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

namespace xrgpu {

inline int64_t mxfp4_scale_bytes(int64_t rows, int64_t kb) { return (rows + 127) / 128 * ((kb + 3) / 4) * 512; }

struct Mxfp4Quantize {
  int f16;
  int64_t rows, K, kb, ldx;
  const void* x;    // [rows, ldx]
  uint8_t* codes;   // [rows, kb, 16]
  uint8_t* scales;  // tiled
};
cudaError_t launch_mxfp4_quantize(const Mxfp4Quantize& p, cudaStream_t s);

struct Mxfp4Dequantize {
  int f16;
  int64_t rows, K, kb;
  const uint8_t* codes;
  const uint8_t* scales;  // tiled
  void* out;              // [rows, K]
};
cudaError_t launch_mxfp4_dequantize(const Mxfp4Dequantize& p, cudaStream_t s);

// scales [rows, kb] -> tiled
cudaError_t launch_mxfp4_tile_scales(const uint8_t* scales, uint8_t* tiled, int64_t rows, int64_t kb, cudaStream_t s);

struct Mxfp4Matmul {
  int f16;                  // y and bias: 1 float16, 0 float32
  int64_t M, N, K, kb, ldy;
  const uint8_t* a;         // [M, kb, 16]
  const uint8_t* a_scales;  // tiled
  const uint8_t* b;         // [N, kb, 16]
  const uint8_t* b_scales;  // tiled
  const void* bias;         // [N] or nullptr
  void* y;                  // [M, ldy]
  unsigned* err;
};
// early: the kernel before it on the stream writes the activations only and announces its end early, so
// the weights may be loaded while it runs.
cudaError_t launch_mxfp4_matmul(const Mxfp4Matmul& p, bool early, cudaStream_t s);

}  // namespace xrgpu
