// C entry points of the 8-bit integer operators and the router: argument checks, workspace, launches.
#include <cuda_runtime.h>

#include <climits>
#include <string>

#include "mmnb_int8.h"
#include "mmnb_internal.h"
#include "xrgpu_mmnb.h"

namespace xrgpu {
namespace {

int fail(const std::string& m) { return api_fail(XRGPU_INVALID_ARGUMENT, m); }

int launched(cudaError_t e) {
  if (e != cudaSuccess) return api_fail(XRGPU_RUNTIME_ERROR, std::string("kernel launch failed: ") + cudaGetErrorString(e));
  return XRGPU_OK;
}

bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

int t1_code(int32_t dtype, int* f16) {
  if (dtype != XRGPU_FLOAT16 && dtype != XRGPU_FLOAT32) return fail("T1 must be float32 or float16");
  *f16 = dtype == XRGPU_FLOAT16;
  return XRGPU_OK;
}

constexpr int64_t kMaxK = 131071;  // 128 * 128 * K stays within int32
constexpr int64_t kMaxGroups = 1024;
constexpr int64_t kMaxTopK = 32;   // of the router

// Row stride of codes (0: K rounded up to 16).
int code_stride(int64_t given, int64_t K, int64_t* ld) {
  *ld = given ? given : static_cast<int64_t>(align_up(K, 16));
  if (*ld < K || *ld % 16) return fail("rows of codes must lie a multiple of 16 bytes of at least K apart");
  return XRGPU_OK;
}

int rows_of(const xrgpu_int8_tensor* t, Int8Rows* p) {
  if (!t) return fail("Null problem");
  int st = t1_code(t->dtype, &p->f16);
  if (st) return st;
  if (t->rows < 0 || t->rows > INT_MAX || t->K <= 0 || t->K > (int64_t(1) << 30)) return fail("Invalid int8 geometry");
  if ((st = code_stride(t->ldc, t->K, &p->ldc))) return st;
  p->rows = t->rows;
  p->K = t->K;
  if (t->rows == 0) return XRGPU_OK;
  if (!t->codes || !t->scales) return fail("null tensor pointer");
  if (!aligned(t->codes, 16)) return fail("int8 codes must be 16-byte aligned");
  p->codes = t->codes;
  p->scales = t->scales;
  return XRGPU_OK;
}

// Workspace of a product: [codes of its rows][their scales][codes of a][their scales][its results as float32], the parts it needs.
struct Layout {
  uint64_t scales, tokens, token_scales, rows, bytes;
  int64_t ldr;  // row stride of the results
};

// Float rows that are read several times, and many values: quantised once, their codes gathered after that. Else each is quantised
// where it is needed, by one kernel. Measured with the product (16 experts of 512 channels, K 2048; us, each / once, halves and floats): 1024
// tokens by 2 experts (2^22 values) 17.7 / 19.1, 19.2 / 20.0; 2048 by 2 (2^23) 21.8 / 22.8, 24.6 / 24.6; 1024 by 4 (2^23) 22.0 / 21.8, 24.6 /
// 22.6; 4096 by 4 (2^25) 40.7 / 37.6, 51.5 / 40.7.
bool quantise_once(const xrgpu_int8_problem& c) {
  return c.a_dtype != XRGPU_INT8 && c.order && c.rows >= 2 * c.M && c.rows * c.K >= (int64_t(1) << 23);
}
Layout layout(const xrgpu_int8_problem& c, int64_t out_n, bool in_place) {
  Layout l{};
  const uint64_t rows = static_cast<uint64_t>(c.groups ? c.rows : c.M);
  if ((c.a_dtype != XRGPU_INT8 && !in_place) || c.order) {
    l.scales = align_up(rows * align_up(c.K, 16), 256);
    l.tokens = l.rows = l.scales + align_up(rows * 4, 256);
    if (quantise_once(c)) {
      l.token_scales = l.tokens + align_up(static_cast<uint64_t>(c.M) * align_up(c.K, 16), 256);
      l.rows = l.token_scales + align_up(static_cast<uint64_t>(c.M) * 4, 256);
    }
  }
  l.ldr = static_cast<int64_t>(align_up(out_n, 4));
  l.bytes = l.rows + (c.slots ? static_cast<uint64_t>(c.rows) * l.ldr * 4 : 0);
  return l;
}

// Everything but the pointers of tensors.
int check(const xrgpu_int8_problem* c, Int8Matmul* p, Layout* l, bool* in_place) {
  if (!c) return fail("Null problem");
  int st = t1_code(c->dtype, &p->f16);
  if (st) return st;
  if (c->a_dtype != XRGPU_INT8 && c->a_dtype != XRGPU_FLOAT16 && c->a_dtype != XRGPU_FLOAT32)
    return fail("int8 activations must be float32, float16 or int8 codes");
  if (c->M < 0 || c->M > INT_MAX / 2 || c->K <= 0 || c->K > kMaxK || c->N <= 0 || c->N > INT_MAX / 2 || c->groups < 0 ||
      c->groups > kMaxGroups || c->N * (c->groups ? c->groups : 1) > INT_MAX / 2)
    return fail("Invalid int8 geometry");
  if (c->activation != XRGPU_ACT_NONE && c->activation != XRGPU_ACT_RELU && c->activation != XRGPU_ACT_SWIGLU)
    return fail("activation must be none, relu or swiglu");
  if (c->activation == XRGPU_ACT_SWIGLU && c->N % 2) return fail("swiglu needs pairs of channels");
  if (c->activation == XRGPU_ACT_SWIGLU && !(c->alpha - c->alpha == 0.0f && c->beta - c->beta == 0.0f && (!c->has_limit || c->limit >= 0.0f)))
    return fail("swiglu's alpha and beta must be finite, its limit >= 0");
  const int64_t out_n = c->activation == XRGPU_ACT_SWIGLU ? c->N / 2 : c->N;
  if (c->groups) {
    if (c->rows < 0 || c->rows > INT_MAX / 2 || c->tokens < 0 || c->tokens > INT_MAX) return fail("Invalid int8 geometry");
    if ((c->order || c->slots) && (c->top_k < 1 || c->top_k > INT_MAX)) return fail("top_k must be at least 1");
    if (!c->order && c->M != c->rows) return fail("without order a must have the product's rows");
    if (c->rows > 0 && c->M == 0) return fail("order needs rows of a");
    if (c->order && c->M > INT_MAX / c->top_k) return fail("Invalid int8 geometry");
    if (c->slots && c->tokens > INT_MAX / c->top_k) return fail("Invalid int8 geometry");
    if (!c->slots != !c->weights) return fail("slots and weights belong together");
  } else if (c->offsets || c->order || c->slots || c->weights) {
    return fail("a dense product has no offsets, order, slots or weights");
  }
  if (c->a_dtype == XRGPU_INT8) {
    if ((st = code_stride(c->lda, c->K, &p->lda))) return st;
  } else {
    if (c->lda != 0 && c->lda < c->K) return fail("lda must be at least K");
  }
  if ((st = code_stride(c->ldb, c->K, &p->ldb))) return st;
  if (c->ldy != 0 && c->ldy < out_n) return fail("ldy must cover a row of y");
  p->act = c->activation;
  p->has_limit = c->has_limit != 0;
  p->alpha = c->alpha;
  p->beta = c->beta;
  p->limit = c->limit;
  p->bias_f16 = p->f16;
  p->groups = c->groups ? static_cast<int>(c->groups) : 1;
  p->rows = c->groups ? c->rows : c->M;
  p->N = c->N;
  p->K = c->K;
  p->ldy = c->ldy ? c->ldy : out_n;
  p->zero_rest = c->zero_rest != 0;
  p->offsets = c->offsets;
  *in_place = c->a_dtype != XRGPU_INT8 && !c->groups && int8_few_rows(*p);
  *l = layout(*c, out_n, *in_place);
  return XRGPU_OK;
}

int workspace(void** ws, uint64_t given, uint64_t need) {
  if (!need) return XRGPU_OK;
  if (!*ws) return library_workspace(need, ws);
  if (given < need) return fail("workspace too small: need " + std::to_string(need) + " bytes");
  if (!aligned(*ws, 16)) return fail("workspace must be 16-byte aligned");
  return XRGPU_OK;
}

int forward(const xrgpu_int8_problem* c, void* ws, uint64_t ws_bytes, cudaStream_t s) {
  Int8Matmul p{};
  Layout l{};
  bool in_place;
  int st = check(c, &p, &l, &in_place);
  if (st) return st;
  const bool sums = c->slots != nullptr;
  if (sums ? c->tokens == 0 : p.rows == 0) return XRGPU_OK;
  if (!c->y || !c->b || !c->b_scales || (p.rows && !c->a) || (c->groups && !c->offsets)) return fail("null tensor pointer");
  if (c->a_dtype == XRGPU_INT8 && p.rows && !c->a_scales) return fail("null tensor pointer");
  if (!aligned(c->b, 16) || (c->a_dtype == XRGPU_INT8 && !aligned(c->a, 16))) return fail("int8 codes must be 16-byte aligned");
  if ((st = workspace(&ws, ws_bytes, l.bytes))) return st;
  uint8_t* w = static_cast<uint8_t*>(ws);
  p.a = static_cast<const int8_t*>(c->a);
  p.a_scales = c->a_scales;
  p.b = c->b;
  p.b_scales = c->b_scales;
  p.bias = c->bias;
  p.y = c->y;
  p.err = device_error_word();
  if (in_place) return launched(launch_int8_few(p, c->a, c->a_dtype == XRGPU_FLOAT16, c->lda ? c->lda : c->K, s));
  if (p.rows) {
    const RowOrder from{c->order, divide_by(c->order ? static_cast<int>(c->top_k) : 1), c->M, p.err};
    const bool made = c->a_dtype != XRGPU_INT8 || c->order;  // the operand, by a kernel before the product's
    if (made) {
      int8_t* codes = reinterpret_cast<int8_t*>(w);
      float* scales = reinterpret_cast<float*>(w + l.scales);
      const int64_t ld = static_cast<int64_t>(align_up(c->K, 16));
      const bool f16 = c->a_dtype == XRGPU_FLOAT16;
      const int64_t ldx = c->lda ? c->lda : c->K;
      if (quantise_once(*c)) {
        int8_t* tokens = reinterpret_cast<int8_t*>(w + l.tokens);
        float* token_scales = reinterpret_cast<float*>(w + l.token_scales);
        st = launched(launch_int8_quantize({f16, c->M, c->K, ldx, ld, c->a, tokens, token_scales, nullptr, {nullptr, {}, c->M, p.err}}, s));
        if (!st) st = launched(launch_int8_gather({p.rows, c->K, ld, ld, from, tokens, token_scales, codes, scales}, true, s));
      } else if (c->a_dtype != XRGPU_INT8) {
        st = launched(launch_int8_quantize({f16, p.rows, c->K, ldx, ld, c->a, codes, scales, nullptr, from}, s));
      } else {
        st = launched(launch_int8_gather({p.rows, c->K, p.lda, ld, from, p.a, p.a_scales, codes, scales}, false, s));
      }
      if (st) return st;
      p.a = codes;
      p.a_scales = scales;
      p.lda = ld;
    }
    if (sums) {
      p.f16 = 0;
      p.y = w + l.rows;
      p.ldy = l.ldr;
      p.zero_rest = 1;
    }
    if ((st = launched(launch_int8_matmul(p, made, s)))) return st;
  }
  if (!sums) return XRGPU_OK;
  const int64_t out_n = c->activation == XRGPU_ACT_SWIGLU ? c->N / 2 : c->N;
  const WeightedRows r{c->dtype == XRGPU_FLOAT16, c->tokens, p.rows, out_n, l.ldr, c->ldy ? c->ldy : out_n, static_cast<int>(c->top_k),
                       reinterpret_cast<const float*>(w + l.rows), c->slots, c->weights, c->y};
  return launched(launch_weighted_rows(r, s));
}

int route_of(const xrgpu_moe_route_problem* c, MoeRoute* p) {
  if (!c) return fail("Null problem");
  const int st = t1_code(c->dtype, &p->f16);
  if (st) return st;
  if (c->experts < 1 || c->experts > kMaxGroups || c->top_k < 1 || c->top_k > kMaxTopK || c->top_k > c->experts)
    return fail("a router takes up to 1024 experts and a top_k of up to 32 of them");
  if (c->tokens < 0 || c->tokens > INT_MAX || c->tokens * c->top_k > INT_MAX) return fail("Invalid router geometry");
  if (c->lds != 0 && c->lds < c->experts) return fail("row strides must cover a row");
  *p = MoeRoute{p->f16, c->tokens, c->lds ? c->lds : c->experts, static_cast<int>(c->experts), static_cast<int>(c->top_k), c->normalize != 0,
                c->scores, c->chosen, c->weights, c->order, c->slots, c->offsets};
  return XRGPU_OK;
}

}  // namespace
}  // namespace xrgpu

extern "C" {

int xrgpu_int8_quantize(const xrgpu_int8_tensor* t, const void* x, int64_t ldx, void* stream) {
  xrgpu::Int8Rows p{};
  const int st = xrgpu::rows_of(t, &p);
  if (st) return st;
  if (ldx != 0 && ldx < t->K) return xrgpu::fail("ldx must be at least K");
  if (t->rows == 0) return XRGPU_OK;
  if (!x) return xrgpu::fail("null tensor pointer");
  p.x = x;
  p.ldx = ldx ? ldx : t->K;
  p.from.err = xrgpu::device_error_word();
  return xrgpu::launched(xrgpu::launch_int8_quantize(p, static_cast<cudaStream_t>(stream)));
}

int xrgpu_int8_dequantize(const xrgpu_int8_tensor* t, void* out, void* stream) {
  xrgpu::Int8Rows p{};
  const int st = xrgpu::rows_of(t, &p);
  if (st) return st;
  if (t->rows == 0) return XRGPU_OK;
  if (!out) return xrgpu::fail("null tensor pointer");
  p.out = out;
  return xrgpu::launched(xrgpu::launch_int8_dequantize(p, static_cast<cudaStream_t>(stream)));
}

int xrgpu_int8_workspace_size(const xrgpu_int8_problem* c, uint64_t* bytes) {
  xrgpu::Int8Matmul p{};
  xrgpu::Layout l{};
  bool in_place;
  const int st = xrgpu::check(c, &p, &l, &in_place);
  if (st) return st;
  if (bytes) *bytes = l.bytes;
  return XRGPU_OK;
}

int xrgpu_int8_forward(const xrgpu_int8_problem* c, void* ws, uint64_t ws_bytes, void* stream) {
  return xrgpu::forward(c, ws, ws_bytes, static_cast<cudaStream_t>(stream));
}

int xrgpu_moe_route_workspace_size(const xrgpu_moe_route_problem* c, uint64_t* bytes) {
  xrgpu::MoeRoute p{};
  const int st = xrgpu::route_of(c, &p);
  if (st) return st;
  if (bytes) *bytes = p.tokens ? xrgpu::moe_route_workspace(p) : 0;
  return XRGPU_OK;
}

int xrgpu_moe_route(const xrgpu_moe_route_problem* c, void* ws, uint64_t ws_bytes, void* stream) {
  xrgpu::MoeRoute p{};
  int st = xrgpu::route_of(c, &p);
  if (st) return st;
  if (!p.offsets) return xrgpu::fail("null tensor pointer");
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (!p.tokens) return xrgpu::launched(cudaMemsetAsync(p.offsets, 0, static_cast<size_t>(p.experts + 1) * 4, s));
  if (!p.scores || !p.chosen || !p.weights || !p.order || !p.slots) return xrgpu::fail("null tensor pointer");
  if ((st = xrgpu::workspace(&ws, ws_bytes, xrgpu::moe_route_workspace(p)))) return st;
  return xrgpu::launched(xrgpu::launch_moe_route(p, ws, s));
}

}  // extern "C"
