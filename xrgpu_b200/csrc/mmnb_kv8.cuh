// Device helpers shared by the 8-bit cache kernels.
#pragma once

#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "mmnb_common.cuh"
#include "mmnb_kv8.h"

namespace xrgpu {

struct SeqRows {
  int row0, n, len;  // first row, number of rows, tokens of the sequence (the rows included)
};

// Rows and length of sequence b. Lengths that do not fit are recorded in the error word: rows outside the
// call's give n = 0; a length outside the table's gives n = 0 (append, read) or len = 0 (attention: the rows
// see nothing). More rows than tokens fit attention only, whose first rows then see nothing.
__device__ __forceinline__ SeqRows seq_rows(const Kv8& p, int b, bool attention) {
  SeqRows r;
  if (p.uniform) {
    r.n = p.tokens / p.seqs;
    r.row0 = b * r.n;
  } else {
    r.row0 = p.cu[b];
    r.n = p.cu[b + 1] - r.row0;
  }
  r.len = p.kv_len[b];
  const bool bad_rows = r.row0 < 0 || r.n < 0 || r.n > p.tokens || r.row0 > p.tokens - r.n;
  const bool bad_len = r.len < 0 || static_cast<int64_t>(r.len) > (static_cast<int64_t>(p.max_pages) << p.page_log2) ||
                       (!attention && r.n > r.len);
  if (bad_rows || bad_len) {
    record_device_error(p.err, kErrKv8Length);
    r.len = 0;
    if (bad_rows || !attention) r.row0 = r.n = 0;
  }
  return r;
}

// Page id of page j of sequence b, -1 (recorded) when the table holds none of the pool's.
__device__ __forceinline__ int page_id(const Kv8& p, int b, int j) {
  const int id = p.page_table[static_cast<int64_t>(b) * p.max_pages + j];
  if (id < 0 || id >= p.pages) {
    record_device_error(p.err, kErrKv8Page);
    return -1;
  }
  return id;
}

// First token that the row at position pos sees (a position before the first token is negative, a window may be
// INT_MAX: their difference need not fit an int).
__device__ __forceinline__ int window_from(const Kv8& p, int pos) {
  return p.window > 0 && pos >= p.window ? pos - p.window + 1 : 0;
}

__device__ __forceinline__ float e4m3_value(uint32_t byte) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(byte), __NV_E4M3)));
}

template <bool E4M3>
__device__ __forceinline__ float code_value(uint32_t byte) {
  return E4M3 ? e4m3_value(byte) : static_cast<float>(static_cast<int8_t>(byte));
}

}  // namespace xrgpu
