// Device-pointer problems and launchers of the 8-bit integer operators (mmnb_int8.cu, mmnb_int8_gemm_sm100.cu) and of
// the router of a mixture of experts (mmnb_moe_route.cu).
//
// A row of values is held as codes int8 [K] and one float32 scale: value = code * scale. Rows of codes start on 16
// bytes (what lies behind a row's K codes is never read).
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

namespace xrgpu {

// n / d for 0 <= n < 2^31 by a multiplication with ceil(2^p / d), p = 31 + ceil(log2 d) (Granlund and Montgomery, 1994): kernels of a
// few microseconds feel the code of a division, which comes from memory before the first load.
struct Divide {
  uint32_t mul;  // 0: d = 1
  int shift;
};
inline Divide divide_by(int d) {
  int l = 0;
  while ((int64_t(1) << l) < d) ++l;
  if (!l) return {0, 0};
  return {static_cast<uint32_t>(((uint64_t(1) << (31 + l)) + d - 1) / d), l - 1};
}
#ifdef __CUDACC__
__device__ __forceinline__ int operator/(int n, const Divide& d) {
  return d.mul ? static_cast<int>(__umulhi(static_cast<uint32_t>(n), d.mul) >> d.shift) : n;
}
#endif

// Row r stands for row order[r] / top_k of `rows` ones (order nullptr: for row r). An entry that fits none counts as a row of
// zeros and is recorded.
struct RowOrder {
  const int32_t* order;
  Divide by_top_k;
  int64_t rows;
  unsigned* err;
};

struct Int8Rows {
  int f16;          // of the values: 1 float16, 0 float32
  int64_t rows, K;
  int64_t ldx, ldc; // row strides of values and codes
  const void* x;
  int8_t* codes;
  float* scales;
  void* out;        // dequantisation: values [rows, K]
  RowOrder from;    // quantisation: which rows of x
};
cudaError_t launch_int8_quantize(const Int8Rows& p, cudaStream_t s);
cudaError_t launch_int8_dequantize(const Int8Rows& p, cudaStream_t s);

// Codes and scales of `rows` rows taken in an order.
struct Int8Gather {
  int64_t rows, K, lds, ldc;  // strides of a and codes
  RowOrder from;
  const int8_t* a;
  const float* a_scales;
  int8_t* codes;
  float* scales;
};
// early: a is what the kernel before it on the stream writes.
cudaError_t launch_int8_gather(const Int8Gather& p, bool early, cudaStream_t s);

// y[r, :] = act(a[r] . b[g]^T * a_scale[r] * b_scale[g, :] + bias[g, :]) for the rows r of group g, offsets[g] <= r <
// offsets[g + 1] (offsets nullptr: one group of all rows).
struct Int8Matmul {
  int f16;       // y: 1 float16, 0 float32
  int bias_f16;
  int act;       // XRGPU_ACT_NONE, _RELU, _SWIGLU (channel pairs)
  int has_limit, zero_rest;
  float alpha, beta, limit;
  int groups;
  int64_t rows, N, K, lda, ldb, ldy;
  const int8_t* a;
  const float* a_scales;
  const int8_t* b;       // [groups * N, ldb]
  const float* b_scales; // [groups, N]
  const void* bias;      // [groups, N] or nullptr
  const int32_t* offsets;
  void* y;
  unsigned* err;
};
// early: the kernel before it on the stream writes a and a_scales only and announces its end early.
cudaError_t launch_int8_matmul(const Int8Matmul& p, bool early, cudaStream_t s);
// The product of a few float rows x [p.rows, ldx], quantised by the same kernel (p.a and p.a_scales are not used), and whether a
// call takes this form.
bool int8_few_rows(const Int8Matmul& p);
cudaError_t launch_int8_few(const Int8Matmul& p, const void* x, bool x_f16, int64_t ldx, cudaStream_t s);

// out[t] = sum_j weights[t, j] y[slots[t, j]], float32 sums in the order of j; slots outside [0, rows) are left out.
struct WeightedRows {
  int f16;                  // out
  int64_t tokens, rows, N, ldy, ldo;
  int top_k;
  const float* y;           // [rows, ldy], ldy a multiple of 4
  const int32_t* slots;     // [tokens, top_k]
  const float* weights;     // [tokens, top_k]
  void* out;
};
cudaError_t launch_weighted_rows(const WeightedRows& p, cudaStream_t s);

// Router: the top_k experts of each token, their weights, and the assignments in the experts' order.
struct MoeRoute {
  int f16;
  int64_t tokens, lds;
  int experts, top_k, normalize;
  const void* scores;   // [tokens, lds]
  int32_t* chosen;      // [tokens, top_k]
  float* weights;       // [tokens, top_k]
  int32_t* order;       // [tokens * top_k]
  int32_t* slots;       // [tokens, top_k]
  int32_t* offsets;     // [experts + 1]
};
uint64_t moe_route_workspace(const MoeRoute& p);
cudaError_t launch_moe_route(const MoeRoute& p, void* ws, cudaStream_t s);

}  // namespace xrgpu
