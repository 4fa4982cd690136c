// Device-pointer problem and launchers of the paged 8-bit key/value cache: append, read back and attention
// (mmnb_kv8.cu, mmnb_kv8_attn.cu).
//
// Cache. Pages [pages][heads][page][D] of 8-bit codes (int8, or float8 e4m3), one float32 scale for each
// (page, head): value = code * scale. Sequence b has kv_len[b] tokens; token j is in page
// page_table[b][j / page], slot j % page. The rows of the call (queries, or new keys and values) are those
// of sequence b from cu_seqlens[b] to cu_seqlens[b + 1], the LAST tokens of the sequence: row
// cu_seqlens[b] + i is position kv_len[b] - n_b + i. Rows behind cu_seqlens[sequences] belong to nobody.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

namespace xrgpu {

// Device error codes: a page id outside the pool; lengths that do not fit the table or the rows.
constexpr unsigned kErrKv8Page = 0x501;
constexpr unsigned kErrKv8Length = 0x502;

struct Kv8 {
  int f16;       // rows: 1 float16, 0 float32
  int e4m3;      // codes: 1 e4m3, 0 int8
  int causal;
  int zero_rest; // attention, read back: rows of no sequence are set to zero
  int few_rows;  // attention: sequences with more rows (tokens x query heads a key/value head) are the prompt kernel's
  int uniform;   // cu_seqlens absent: tokens / sequences rows each
  int tokens, seqs, hq, hkv, D, page, page_log2, pages, max_pages, window;
  int64_t qs, ks, vs, os;  // row strides in elements
  float scale;
  const void* q;   // [tokens, hq, D]
  void* k;         // [tokens, hkv, D]: append reads, read back writes
  void* v;
  void* o;         // [tokens, hq, D]
  uint8_t* k_cache;
  uint8_t* v_cache;
  float* k_scale;  // [pages, hkv]
  float* v_scale;
  const int* page_table;  // [seqs, max_pages]
  const int* cu;          // [seqs + 1] or nullptr
  const int* kv_len;      // [seqs]
  unsigned* err;
};

cudaError_t launch_kv8_append(const Kv8& p, cudaStream_t s);
cudaError_t launch_kv8_read(const Kv8& p, cudaStream_t s);
uint64_t kv8_attention_workspace(const Kv8& p);
cudaError_t launch_kv8_attention(const Kv8& p, void* ws, cudaStream_t s);

}  // namespace xrgpu
