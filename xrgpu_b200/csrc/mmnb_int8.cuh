// Quantisation of values to 8-bit codes on the device (format: mmnb_int8.h).
//
// Quantisation of a row: s = max|x| / 127 in float32, code = x / s rounded to nearest, ties to even. The quotient is not
// computed: r = round(x * (1 / s)) is the code or, next to a border, one off it. What is left, x - r s, is exact in one fused step
// (it has no bit below both numbers' last ones and is at most about s / 2), so comparing it with s / 2 decides, and with r's
// last bit a tie. Float32 rows of scales under 2^-60 are brought up by 2^100 first (exact as well); where s has
// only a few bits left (subnormal), x / s may be up to 190, and codes saturate. A row with a NaN or an infinity has scale NaN and codes 0.
#pragma once

#include <cuda_fp16.h>

#include "mmnb_common.cuh"

namespace xrgpu {
namespace {

constexpr float kMagic = 12582912.0f;        // 1.5 * 2^23: t + kMagic rounds t to a whole number
constexpr float kSmallScale = 8.7e-19f;      // about 2^-60

__device__ __forceinline__ uint32_t pack4(const uint32_t* b) { return prmt(prmt(b[0], b[1], 0x0040), prmt(b[2], b[3], 0x0040), 0x5410); }

struct Scale {
  float s, inv, up;  // of values times `up`
};
// A row's scale from the bits of its largest magnitude, and what its codes need; none: all codes are 0.
template <bool F16>
__device__ __forceinline__ float row_scale_of(uint32_t amax, Scale* c, bool* none) {
  const bool bad = amax >= 0x7f800000u;
  const float s = bad ? __uint_as_float(0x7fc00000u) : __fdiv_rn(__uint_as_float(amax), 127.0f);
  *none = bad || s == 0.0f;
  c->up = !F16 && s < kSmallScale ? 0x1p100f : 1.0f;
  c->s = *none ? 1.0f : s * c->up;
  c->inv = __fdiv_rn(1.0f, c->s);
  return s;
}

// Two float32 numbers in a register pair: one instruction for both.
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 unpair(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// Codes of a thread's N values, in the low bytes of b.
template <int N, bool F16>
__device__ __forceinline__ void codes_of(const float (&v)[N], const Scale& c, uint32_t (&b)[N]) {
  const uint64_t inv = pair(c.inv, c.inv), magic = pair(kMagic, kMagic), back = pair(-kMagic, -kMagic), s = pair(-c.s, -c.s), up = pair(c.up, c.up);
  float worst = 0.0f;
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    uint64_t x = pair(v[i], v[i + 1]);
    if (!F16) x = mul2(x, up);
    const uint64_t t = fma2(x, inv, magic);
    const float2 code = unpair(t), left = unpair(fma2(add2(t, back), s, x));
    b[i] = __float_as_uint(code.x);
    b[i + 1] = __float_as_uint(code.y);
    worst = fmaxf(fmaxf(worst, fabsf(left.x)), fabsf(left.y));
  }
  // Hardly ever: a tie or a code one off; small scales, whose quotients may exceed 127 and leave nothing (the last bits of a word that
  // was not clamped are another code: 128 units of 2^-149 by a scale of one came out as -128).
  if (worst >= 0.5f * c.s || (!F16 && c.up != 1.0f)) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float x = F16 ? v[i] : v[i] * c.up, r = __uint_as_float(b[i]) - kMagic, left = fmaf(-r, c.s, x);
      int code = static_cast<int>(r);
      if (fabsf(left) > 0.5f * c.s || (fabsf(left) == 0.5f * c.s && (code & 1))) code += left > 0.0f ? 1 : -1;
      b[i] = static_cast<uint32_t>(max(-127, min(127, code)));
    }
  }
}

// The largest magnitude of values, as the bits of a float32 (NaN > infinity > numbers). Pairs of halves as they are.
template <bool F16>
struct Largest {
  uint32_t m = 0;
  __device__ __forceinline__ void add(uint32_t u) {
    if (F16) {
      const __half2 h = __hmax2_nan(*reinterpret_cast<const __half2*>(&m), __habs2(*reinterpret_cast<const __half2*>(&u)));
      m = *reinterpret_cast<const uint32_t*>(&h);
    } else {
      m = max(m, u & 0x7fffffffu);
    }
  }
  __device__ __forceinline__ uint32_t bits() const {
    if (!F16) return m;
    const __half2 h = *reinterpret_cast<const __half2*>(&m);
    return __float_as_uint(__half2float(__hmax_nan(__low2half(h), __high2half(h)))) & 0x7fffffffu;
  }
};

// 16 bytes of a row from value k0 on, zeros behind K. VEC: rows start on 16 bytes and hold whole units.
template <bool F16, bool VEC>
struct Unit {
  static constexpr int kValues = F16 ? 8 : 4;
  uint32_t u[4];
  __device__ __forceinline__ void load(const void* row, int k0, int K) {
    if (VEC) {
      const uint4 v = k0 < K ? *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(row) + k0 * (F16 ? 2ll : 4ll)) : make_uint4(0, 0, 0, 0);
      u[0] = v.x; u[1] = v.y; u[2] = v.z; u[3] = v.w;
      return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (F16) {
        const uint16_t* h = static_cast<const uint16_t*>(row) + k0;
        const uint32_t lo = k0 + 2 * i < K ? h[2 * i] : 0, hi = k0 + 2 * i + 1 < K ? h[2 * i + 1] : 0;
        u[i] = lo | hi << 16;
      } else {
        u[i] = k0 + i < K ? static_cast<const uint32_t*>(row)[k0 + i] : 0;
      }
    }
  }
  __device__ __forceinline__ void largest(Largest<F16>& l) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) l.add(u[i]);
  }
  // Codes, four a word: kValues / 4 words of `word`.
  __device__ __forceinline__ void codes(const Scale& c, uint32_t* word) const {
    float v[kValues];
    uint32_t b[kValues];
#pragma unroll
    for (int i = 0; i < kValues; ++i) {
      if (F16) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i >> 1]));
        v[i] = (i & 1) ? f.y : f.x;
      } else {
        v[i] = __uint_as_float(u[i & 3]);
      }
    }
    codes_of<kValues, F16>(v, c, b);
    word[0] = pack4(b);
    if (F16) word[1] = pack4(b + (F16 ? 4 : 0));
  }
};

}  // namespace
}  // namespace xrgpu
