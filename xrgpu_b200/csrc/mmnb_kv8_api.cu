// C entry points of the paged 8-bit key/value cache: argument checks, workspace, launches.
#include <cuda_runtime.h>

#include <climits>
#include <string>

#include "mmnb_internal.h"
#include "mmnb_kv8.h"
#include "xrgpu_mmnb.h"

namespace xrgpu {
namespace {

enum Need { kAppend, kRead, kAttention };

int fail(const std::string& m) { return api_fail(XRGPU_INVALID_ARGUMENT, m); }

bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

int convert(const xrgpu_kv8_problem* c, Need need, Kv8* out) {
  if (!c) return fail("Null problem");
  Kv8 p{};
  if (c->dtype != XRGPU_FLOAT16 && c->dtype != XRGPU_FLOAT32) return fail("T1 must be float32 or float16");
  if (c->cache_dtype != XRGPU_INT8 && c->cache_dtype != XRGPU_FLOAT8_E4M3) return fail("cache codes must be int8 or float8 e4m3");
  p.f16 = c->dtype == XRGPU_FLOAT16;
  p.e4m3 = c->cache_dtype == XRGPU_FLOAT8_E4M3;
  if (c->head_dim != 64 && c->head_dim != 128) return fail("head_dim must be 64 or 128");
  if (c->page != 16 && c->page != 32 && c->page != 64 && c->page != 128) return fail("page must be 16, 32, 64 or 128 tokens");
  if (c->tokens < 0 || c->tokens > INT_MAX || c->sequences < 0 || c->sequences > 65535 || c->pages < 0 || c->pages > INT_MAX ||
      c->max_pages < 0 || c->max_pages > INT_MAX / 128 || c->heads_kv <= 0 || c->heads_kv > 65535)
    return fail("Invalid cache geometry");
  p.tokens = static_cast<int>(c->tokens); p.seqs = static_cast<int>(c->sequences);
  p.hkv = static_cast<int>(c->heads_kv); p.D = static_cast<int>(c->head_dim);
  p.page = static_cast<int>(c->page); p.pages = static_cast<int>(c->pages); p.max_pages = static_cast<int>(c->max_pages);
  while ((1 << p.page_log2) < p.page) ++p.page_log2;
  p.zero_rest = c->zero_rest != 0;
  p.uniform = c->cu_seqlens == nullptr;
  if (p.uniform && p.seqs > 0 && p.tokens % p.seqs) return fail("tokens must be a multiple of sequences without cu_seqlens");
  const int64_t kv_row = c->heads_kv * c->head_dim;
  if (need == kAttention) {
    if (c->heads_q <= 0 || c->heads_q > 65535 || c->heads_q % c->heads_kv) return fail("heads_q must be a multiple of heads_kv");
    if (c->tokens * c->heads_q > INT_MAX) return fail("Invalid cache geometry");
    if (c->window < 0 || c->window > INT_MAX) return fail("window must be >= 0");
    if (c->window > 0 && !c->causal) return fail("a window needs causal attention");
    if (!(c->scale >= -3.4028234e38f && c->scale <= 3.4028234e38f)) return fail("scale must be finite");
    p.hq = static_cast<int>(c->heads_q); p.window = static_cast<int>(c->window); p.causal = c->causal != 0; p.scale = c->scale;
    const int64_t q_row = c->heads_q * c->head_dim;
    p.qs = c->q_stride ? c->q_stride : q_row;
    p.os = c->o_stride ? c->o_stride : q_row;
    if (p.qs < q_row || p.os < q_row) return fail("row strides must cover a row");
  } else {
    p.ks = c->k_stride ? c->k_stride : kv_row;
    p.vs = c->v_stride ? c->v_stride : kv_row;
    if (p.ks < kv_row || p.vs < kv_row) return fail("row strides must cover a row");
  }
  if (p.tokens > 0 && p.seqs > 0) {
    if (need == kAttention ? (!c->q || !c->o) : (!c->k || !c->v)) return fail("null tensor pointer");
    if (!c->kv_len) return fail("null tensor pointer");
    if (p.pages > 0 && p.max_pages > 0 && (!c->k_cache || !c->v_cache || !c->k_scale || !c->v_scale || !c->page_table))
      return fail("null tensor pointer");
    if (!aligned(c->k_cache, 16) || !aligned(c->v_cache, 16)) return fail("the cache must be 16-byte aligned");
  }
  p.q = c->q; p.k = c->k; p.v = c->v; p.o = c->o;
  p.k_cache = c->k_cache; p.v_cache = c->v_cache; p.k_scale = c->k_scale; p.v_scale = c->v_scale;
  p.page_table = c->page_table; p.cu = c->cu_seqlens; p.kv_len = c->kv_len;
  *out = p;
  return XRGPU_OK;
}

int launched(cudaError_t e) {
  if (e != cudaSuccess) return api_fail(XRGPU_RUNTIME_ERROR, std::string("kernel launch failed: ") + cudaGetErrorString(e));
  return XRGPU_OK;
}

// Without sequences every row belongs to none.
cudaError_t zero_rows(const Kv8& p, void* rows, int64_t stride, int heads, cudaStream_t s) {
  const size_t es = p.f16 ? 2 : 4, width = static_cast<size_t>(heads) * p.D * es;
  if (!rows || !p.zero_rest || !p.tokens || p.seqs) return cudaSuccess;
  return cudaMemset2DAsync(rows, static_cast<size_t>(stride) * es, 0, width, p.tokens, s);
}

}  // namespace
}  // namespace xrgpu

extern "C" {

int xrgpu_kv8_append(const xrgpu_kv8_problem* c, void* stream) {
  xrgpu::Kv8 p;
  const int st = xrgpu::convert(c, xrgpu::kAppend, &p);
  if (st) return st;
  p.err = xrgpu::device_error_word();
  return xrgpu::launched(xrgpu::launch_kv8_append(p, static_cast<cudaStream_t>(stream)));
}

int xrgpu_kv8_read(const xrgpu_kv8_problem* c, void* stream) {
  xrgpu::Kv8 p;
  const int st = xrgpu::convert(c, xrgpu::kRead, &p);
  if (st) return st;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e = xrgpu::zero_rows(p, p.k, p.ks, p.hkv, s);
  if (e == cudaSuccess) e = xrgpu::zero_rows(p, p.v, p.vs, p.hkv, s);
  if (e != cudaSuccess) return xrgpu::launched(e);
  p.err = xrgpu::device_error_word();
  return xrgpu::launched(xrgpu::launch_kv8_read(p, s));
}

int xrgpu_kv8_attention_workspace_size(const xrgpu_kv8_problem* c, uint64_t* bytes) {
  xrgpu::Kv8 p;
  const int st = xrgpu::convert(c, xrgpu::kAttention, &p);
  if (st) return st;
  if (bytes) *bytes = p.tokens && p.seqs ? xrgpu::kv8_attention_workspace(p) : 0;
  return XRGPU_OK;
}

int xrgpu_kv8_attention(const xrgpu_kv8_problem* c, void* ws, uint64_t ws_bytes, void* stream) {
  xrgpu::Kv8 p;
  int st = xrgpu::convert(c, xrgpu::kAttention, &p);
  if (st) return st;
  if (!p.tokens || !p.seqs) return xrgpu::launched(xrgpu::zero_rows(p, p.o, p.os, p.hq, static_cast<cudaStream_t>(stream)));
  const uint64_t need = xrgpu::kv8_attention_workspace(p);
  if (need) {
    if (!ws) {
      if ((st = xrgpu::library_workspace(need, &ws))) return st;
    } else if (ws_bytes < need) {
      return xrgpu::fail("workspace too small: need " + std::to_string(need) + " bytes");
    } else if (!xrgpu::aligned(ws, 16)) {
      return xrgpu::fail("workspace must be 16-byte aligned");
    }
  }
  p.err = xrgpu::device_error_word();
  return xrgpu::launched(xrgpu::launch_kv8_attention(p, ws, static_cast<cudaStream_t>(stream)));
}

}  // extern "C"
