// Attention over the paged 8-bit cache: which kernel a call takes (layout: mmnb_kv8.h).
#include <climits>

#include "mmnb_internal.h"
#include "mmnb_kv8_attn.h"

namespace xrgpu {
namespace {

// Sequences with more rows than this (query tokens x query heads a key/value head) go to the prompt kernel, where a call
// takes it.
constexpr int kFewRows = 64;
// The split kernel's time is its rows, the prompt kernel's its rounds of CTAs (256 rows, all tokens each): it takes a call
// from this many rows a round on. Measured (4096 tokens, 8 key/value heads of 128; us, split / prompt): 1 sequence x 256 rows
// 52 / 115, 4 x 128 83 / 111, 4 x 256 142 / 117, 32 x 32 (two rounds) 148 / 216, 32 x 64 267 / 217, 32 x 256 1001 / 236. Heads of 64
// cost the split kernel half, the prompt kernel nearly the same: 4 x 256 104 / 103, 4 x 512 188 / 103, 32 x 64 192 / 196.
constexpr int64_t kRowsARound = 6500;  // of 128 values

struct Forms {
  bool prompt, few;
};

// The lengths are on the device: the mean number of rows decides. Calls that take the prompt kernel and may hold short
// sequences run both, each of which leaves the other's sequences alone.
Forms choose(Kv8* p) {
  const int64_t rows = ceil_div(p->tokens, p->seqs) * (p->hq / p->hkv), pairs = static_cast<int64_t>(p->seqs) * p->hkv;
  const int64_t rounds = ceil_div(pairs * ceil_div(rows, 256), device_sm_count());
  Forms f;
  f.prompt = p->f16 && rows > kFewRows && pairs * rows * p->D >= rounds * kRowsARound * 128;
  f.few = !f.prompt || !p->uniform;
  p->few_rows = f.prompt ? kFewRows : INT_MAX;
  return f;
}

}  // namespace

uint64_t kv8_attention_workspace(const Kv8& p) {
  Kv8 q = p;
  return choose(&q).few ? kv8_attn_mma_workspace(q) : 0;
}

cudaError_t launch_kv8_attention(const Kv8& p, void* ws, cudaStream_t s) {
  Kv8 q = p;
  const Forms f = choose(&q);
  cudaError_t e = cudaSuccess;
  if (f.prompt) e = launch_kv8_attn_prompt(q, s);
  if (e == cudaSuccess && f.few) e = q.e4m3 ? launch_kv8_attn_mma_e4m3(q, ws, s) : launch_kv8_attn_mma_int8(q, ws, s);
  return e;
}

}  // namespace xrgpu
