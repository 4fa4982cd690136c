// C entry points of the microscaled 4-bit floating-point operators: argument checks, workspace, launches.
#include <cuda_runtime.h>

#include <climits>
#include <string>

#include "mmnb_internal.h"
#include "mmnb_mxfp4.h"
#include "xrgpu_mmnb.h"

namespace xrgpu {
namespace {

int fail(int status, const std::string& m) { return api_fail(status, m); }

int launched(cudaError_t e) {
  if (e != cudaSuccess) return fail(XRGPU_RUNTIME_ERROR, std::string("kernel launch failed: ") + cudaGetErrorString(e));
  return XRGPU_OK;
}

int t1_code(int32_t dtype, int* f16) {
  if (dtype == XRGPU_FLOAT16) *f16 = 1;
  else if (dtype == XRGPU_FLOAT32) *f16 = 0;
  else return fail(XRGPU_INVALID_ARGUMENT, "T1 must be float32 or float16");
  return XRGPU_OK;
}

bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

int geometry(int64_t rows, int64_t K) {
  if (rows < 0 || K <= 0 || rows > INT_MAX || K > (int64_t(1) << 30)) return fail(XRGPU_INVALID_ARGUMENT, "Invalid mxfp4 geometry");
  return XRGPU_OK;
}

int held(const void* codes, const void* scales) {
  if (!codes || !scales) return fail(XRGPU_INVALID_ARGUMENT, "null tensor pointer");
  if (!aligned(codes, 16) || !aligned(scales, 16)) return fail(XRGPU_INVALID_ARGUMENT, "mxfp4 codes and scales must be 16-byte aligned");
  return XRGPU_OK;
}

// Workspace of a product with float activations: [codes, M * kb * 16][tiled scales].
uint64_t codes_bytes(const xrgpu_mxfp4_problem& c) { return align_up(static_cast<uint64_t>(c.M) * ceil_div(c.K, 32) * 16, 256); }
uint64_t workspace(const xrgpu_mxfp4_problem& c) {
  return c.a_dtype == XRGPU_UINT8 || c.M == 0 ? 0 : codes_bytes(c) + mxfp4_scale_bytes(c.M, ceil_div(c.K, 32));
}

int check(const xrgpu_mxfp4_problem* c, int* f16) {
  if (!c) return fail(XRGPU_INVALID_ARGUMENT, "Null problem");
  int st = t1_code(c->dtype, f16);
  if (st || (st = geometry(c->M, c->K))) return st;
  if (c->N <= 0 || c->N > INT_MAX) return fail(XRGPU_INVALID_ARGUMENT, "Invalid mxfp4 geometry");
  if (c->a_dtype != XRGPU_UINT8 && c->a_dtype != XRGPU_FLOAT16 && c->a_dtype != XRGPU_FLOAT32)
    return fail(XRGPU_INVALID_ARGUMENT, "mxfp4 activations must be float32, float16 or uint8 codes");
  if (c->ldy != 0 && c->ldy < c->N) return fail(XRGPU_INVALID_ARGUMENT, "ldy must be at least N");
  if (c->lda != 0 && c->lda < c->K) return fail(XRGPU_INVALID_ARGUMENT, "lda must be at least K");
  return XRGPU_OK;
}

}  // namespace

int mxfp4_forward(const xrgpu_mxfp4_problem& c, void* ws, uint64_t ws_bytes, cudaStream_t s) {
  int f16 = 0;
  int st = check(&c, &f16);
  if (st) return st;
  if (c.M == 0) return XRGPU_OK;
  if (!c.a || !c.y) return fail(XRGPU_INVALID_ARGUMENT, "null tensor pointer");
  if ((st = held(c.b, c.b_scales))) return st;
  const int64_t kb = ceil_div(c.K, 32);
  const uint8_t* codes = static_cast<const uint8_t*>(c.a);
  const uint8_t* scales = c.a_scales;
  if (c.a_dtype == XRGPU_UINT8) {
    if ((st = held(codes, scales))) return st;
  } else {
    const uint64_t need = workspace(c);
    if (!ws) {
      if ((st = library_workspace(need, &ws))) return st;
    } else if (ws_bytes < need) {
      return fail(XRGPU_INVALID_ARGUMENT, "workspace too small: need " + std::to_string(need) + " bytes");
    } else if (!aligned(ws, 16)) {
      return fail(XRGPU_INVALID_ARGUMENT, "workspace must be 16-byte aligned");
    }
    uint8_t* w = static_cast<uint8_t*>(ws);
    Mxfp4Quantize q{c.a_dtype == XRGPU_FLOAT16, c.M, c.K, kb, c.lda ? c.lda : c.K, c.a, w, w + codes_bytes(c)};
    if ((st = launched(launch_mxfp4_quantize(q, s)))) return st;
    codes = q.codes;
    scales = q.scales;
  }
  Mxfp4Matmul p{f16, c.M, c.N, c.K, kb, c.ldy ? c.ldy : c.N, codes, scales, c.b, c.b_scales, c.bias, c.y, device_error_word()};
  return launched(launch_mxfp4_matmul(p, c.a_dtype != XRGPU_UINT8, s));
}

}  // namespace xrgpu

extern "C" {

int xrgpu_mxfp4_quantize(const xrgpu_mxfp4_tensor* t, const void* x, int64_t ldx, void* stream) {
  if (!t) return xrgpu::fail(XRGPU_INVALID_ARGUMENT, "Null problem");
  int f16 = 0;
  int st = xrgpu::t1_code(t->dtype, &f16);
  if (st || (st = xrgpu::geometry(t->rows, t->K))) return st;
  if (ldx != 0 && ldx < t->K) return xrgpu::fail(XRGPU_INVALID_ARGUMENT, "ldx must be at least K");
  if (t->rows == 0) return XRGPU_OK;
  if (!x) return xrgpu::fail(XRGPU_INVALID_ARGUMENT, "null tensor pointer");
  if ((st = xrgpu::held(t->codes, t->scales))) return st;
  xrgpu::Mxfp4Quantize q{f16, t->rows, t->K, xrgpu::ceil_div(t->K, 32), ldx ? ldx : t->K, x, t->codes, t->scales};
  return xrgpu::launched(xrgpu::launch_mxfp4_quantize(q, static_cast<cudaStream_t>(stream)));
}

int xrgpu_mxfp4_dequantize(const xrgpu_mxfp4_tensor* t, void* out, void* stream) {
  if (!t) return xrgpu::fail(XRGPU_INVALID_ARGUMENT, "Null problem");
  int f16 = 0;
  int st = xrgpu::t1_code(t->dtype, &f16);
  if (st || (st = xrgpu::geometry(t->rows, t->K))) return st;
  if (t->rows == 0) return XRGPU_OK;
  if (!out) return xrgpu::fail(XRGPU_INVALID_ARGUMENT, "null tensor pointer");
  if ((st = xrgpu::held(t->codes, t->scales))) return st;
  xrgpu::Mxfp4Dequantize d{f16, t->rows, t->K, xrgpu::ceil_div(t->K, 32), t->codes, t->scales, out};
  return xrgpu::launched(xrgpu::launch_mxfp4_dequantize(d, static_cast<cudaStream_t>(stream)));
}

int xrgpu_mxfp4_tile_scales(int64_t rows, int64_t blocks, const uint8_t* scales, uint8_t* tiled, void* stream) {
  if (rows < 0 || blocks <= 0 || rows > INT_MAX || blocks > (int64_t(1) << 25)) return xrgpu::fail(XRGPU_INVALID_ARGUMENT, "Invalid mxfp4 geometry");
  if (rows == 0) return XRGPU_OK;
  if (!scales || !tiled) return xrgpu::fail(XRGPU_INVALID_ARGUMENT, "null tensor pointer");
  return xrgpu::launched(xrgpu::launch_mxfp4_tile_scales(scales, tiled, rows, blocks, static_cast<cudaStream_t>(stream)));
}

int xrgpu_mxfp4_scale_bytes(int64_t rows, int64_t K, uint64_t* bytes) {
  const int st = xrgpu::geometry(rows, K);
  if (st) return st;
  if (bytes) *bytes = static_cast<uint64_t>(xrgpu::mxfp4_scale_bytes(rows, xrgpu::ceil_div(K, 32)));
  return XRGPU_OK;
}

int xrgpu_mxfp4_workspace_size(const xrgpu_mxfp4_problem* p, uint64_t* bytes) {
  int f16 = 0;
  const int st = xrgpu::check(p, &f16);
  if (st) return st;
  if (bytes) *bytes = xrgpu::workspace(*p);
  return XRGPU_OK;
}

int xrgpu_mxfp4_forward(const xrgpu_mxfp4_problem* p, void* ws, uint64_t ws_bytes, void* stream) {
  if (!p) return xrgpu::fail(XRGPU_INVALID_ARGUMENT, "Null problem");
  return xrgpu::mxfp4_forward(*p, ws, ws_bytes, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
