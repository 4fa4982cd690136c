// Attention over the paged 8-bit cache: which kernel a call takes (layout: mmnb_kv8.h).
#include <climits>

#include "mmnb_internal.h"
#include "mmnb_kv8_attn.h"

namespace xrgpu {
namespace {

// Sequences with more rows than this (query tokens x query heads a key/value head) go to the prompt kernel.
constexpr int kFewRows = 64;

struct Forms {
  bool prompt, few;
};

// The lengths are on the device: a call whose sequences have few rows on average takes the split kernel for all of
// them (it is right for any), others both kernels, each of which leaves the other's sequences alone.
Forms choose(Kv8* p) {
  const int64_t rows = ceil_div(p->tokens, p->seqs) * (p->hq / p->hkv);
  Forms f;
  f.prompt = p->f16 && rows > kFewRows;
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
