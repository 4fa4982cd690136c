// Attention over the paged 8-bit cache for prompts: float16 rows, tcgen05 tensor cores (layout: mmnb_kv8.h).
//
//   o[row, h] = sum_j softmax_j(scale * q . k_j) v_j,   k_j = code * k_scale[page], v_j = code * v_scale[page]
//
// A CTA takes 256 rows of one sequence and key/value head (row r is query token r / G and head r % G of its group of
// G, so the group shares every key and value) as two tiles of 128, and passes once over the tokens they see,
// 64 at a time. Codes are exact float16 numbers: they are widened once a CTA, in registers, on their way
// to shared memory, and the scales stay out of them: k_scale multiplies the scores a page at a time, and
// v_scale joins the exponent of the weights: P' = 2^7 exp2(x + log2(v_scale) - m), m the largest x + log2(v_scale) of
// what the row sees. With m raised only when one exceeds it by 8, P' stays below 2^15, so float16 holds the products of weight
// and value scale to 2^-12 of themselves down to 2^-21 of the row's largest, below that in steps of 2^-31 of it, whatever
// the scales of pages are that other rows see. The normaliser is the float32 sum of P' divided by the same factor, a page
// at a time.
//
// Roles (20 warps, registers moved between them):
//   warps 0-3, 4-7  softmax of tile 0, 1: a thread a row: read S, raise m (and rescale O, rare), write P' over S, at
//                   the end write the row out.
//   warps 8-11, 12-15  widen keys, values: 16-byte loads two steps ahead (page ids three), float16 to the 128-byte swizzle
//                   the tensor cores read (keys K-major, values MN-major: both as they lie, no transposition).
//   warps 16-19     issue the MMAs, one each of tile 0's scores, tile 1's scores, tile 0's values, tile 1's values (one warp
//                   for all spent 40 % of the time on its own waits; the products depend on one another through
//                   barriers only). A warp stays converged and elects the issuing lane, so that descriptors stay in
//                   uniform registers.
// Tensor memory: two S (and P') buffers of 64 columns for each tile at 0 and 128, O at 256 and 384. With two buffers the
// scores of the next step are there when the softmax of this one ends; with one of 128 columns the softmax waited
// for P V, Q K and both signals each step (twice the time).
// Bounds per 128 tokens and 256 rows at D = 128, in cycles: tensor cores 2048, exponentials (16 a cycle) 2048, shared memory
// (Q and K read for each S, V for each O, keys and values written: 320 KB) 2560. Measured 6000, the chain of the softmax
// warps (read S, maximum, exponentials, convert, write P', signal): 2 ragged prompts of up to 4096 rows on as many tokens, 32
// heads on 8 of 128: 443 us, 766 TFLOP/s; 4 x 1024 rows on 4024 tokens 318 us, 742 TFLOP/s (e4m3 305 us; heads of 64 271 and 268
// us: the same chain for half the products).
//
// Every wait is bounded as in mmnb_gemm_sm100.cu.
#include <cuda_runtime.h>

#include "mmnb_kv8_attn.h"
#include "mmnb_kv8.cuh"
#include "mmnb_tcgen05.cuh"

namespace xrgpu {
namespace {

constexpr int kTile = 128;        // rows of a tile
constexpr int kStep = 64;         // tokens of a step
constexpr int kRing = 4;          // steps of keys and of values in shared memory
constexpr int kRows = 2 * kTile;  // rows of a CTA
constexpr int kSoftmaxWarps = 8;
constexpr int kWidenWarps = 4;    // for keys, and as many for values
constexpr int kThreads = (kSoftmaxWarps + 2 * kWidenWarps + 4) * 32;
constexpr int kMmaWarp = kSoftmaxWarps + 2 * kWidenWarps;
constexpr int kChunks = kStep / 16;
// Registers a thread: 20 warps are launched with 96 (as many as an SM sub-partition's five warps can have); the
// warpgroups then trade them.
constexpr int kRegs = 96, kSoftmaxRegs = 112, kWidenRegs = 88, kMmaRegs = 80;
static_assert(256 * kSoftmaxRegs + 256 * kWidenRegs + 128 * kMmaRegs <= kThreads * kRegs, "more registers than the block has");
constexpr float kRaise = 8.0f, kLift = 7.0f;
constexpr float kLog2e = 1.4426950408889634f;
constexpr uint32_t kS = 0, kO = 256;  // tensor memory columns (128 a tile)

constexpr unsigned kErrMma = 0x503, kErrWiden = 0x504, kErrSoftmax = 0x505, kErrDrain = 0x506;

template <int D>
struct Smem {
  static constexpr int kQPanel = kTile * 128, kPanel = kStep * 128;  // 64 float16 of each row
  static constexpr int kQTile = kQPanel * (D / 64), kOperand = kPanel * (D / 64);
  static constexpr int kQ = 0, kK = 2 * kQTile, kV = kK + kRing * kOperand, kEnd = kV + kRing * kOperand;
  static constexpr int kBytes = kEnd + 1024;
};

// What the softmax needs of a step's 16-token chunks: the factor of their scores, log2 and inverse of the values'
// scale, and a bit for each chunk that holds tokens.
struct alignas(16) Meta {
  float kf[kChunks], lv[kChunks], iv[kChunks];
  int oks;
};

struct Bars {
  uint64_t kfull[kRing], kempty[kRing], vfull[kRing], vempty[kRing];
  uint64_t sfull[2][2], pfull[2][2], odone[2][2];  // [tile][step % 2]
  uint64_t done[4];
};

// Values operand: [tokens][64] float16 panels, 64 values of D contiguous (MN-major), 128-byte swizzle: 8-token groups 1024
// bytes apart (stride byte offset), panels kPanel apart (leading byte offset).
template <int D>
__device__ __forceinline__ uint64_t desc_mn(uint32_t saddr) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((saddr >> 4) & 0x3FFFu);
  d |= static_cast<uint64_t>(Smem<D>::kPanel >> 4) << 16;
  d |= static_cast<uint64_t>(1024u >> 4) << 32;
  d |= static_cast<uint64_t>(1u) << 46;
  d |= static_cast<uint64_t>(2u) << 61;
  return d;
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float max3(float a, float b, float c) { return fmaxf(fmaxf(a, b), c); }

// Two float32 operations an instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "add.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}

__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Four codes to two float16x2, in order.
template <bool E4M3>
__device__ __forceinline__ uint2 widen4(uint32_t w) {
  uint2 r;
  if (E4M3) {
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\tcvt.rn.f16x2.e4m3x2 %1, hi;\n\t}"
        : "=r"(r.x), "=r"(r.y) : "r"(w));
  } else {
    w ^= 0x80808080u;  // c + 128 over 1024: the float16 number 1152 + c
    r.x = hsub2_u32(prmt(w, 0x64646464u, 0x4140u), 0x64806480u);
    r.y = hsub2_u32(prmt(w, 0x64646464u, 0x4342u), 0x64806480u);
  }
  return r;
}

__device__ __forceinline__ void sts128(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

template <int N>
__device__ __forceinline__ void regs_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void regs_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

struct Job {
  int b, tile, head, rows;  // rows: of this CTA (<= 256)
  SeqRows r;
  int t0, t1;               // tokens seen by any row
};

template <bool E4M3, int D>
__global__ void __launch_bounds__(kThreads, 1) attn_prompt_kernel(const Kv8 p) {
  using M = Smem<D>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ Bars bars;
  __shared__ Meta meta[2 * kRing];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag, found_b, found_tile;
  const int tid = threadIdx.x, warp = __shfl_sync(~0u, tid >> 5, 0), lane = tid & 31;
  const int G = p.hq / p.hkv, head = blockIdx.x % p.hkv, slot = blockIdx.x / p.hkv;

  // ---- which rows: slot counts the 256-row tiles of the sequences with more than p.few_rows rows; a sequence's
  // last rows, which see most, come first
  if (tid == 0) found_b = -1;
  __syncthreads();
  if (warp == 0) {
    int before = 0;
    for (int b0 = 0; b0 < p.seqs; b0 += 32) {
      const int b = b0 + lane;
      int n = 0;
      if (b < p.seqs) {
        const SeqRows r = seq_rows(p, b, true);
        if (static_cast<int64_t>(r.n) * G > p.few_rows) n = (r.n * G + kRows - 1) / kRows;
      }
      int sum = n;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int o = __shfl_up_sync(~0u, sum, d);
        if (lane >= d) sum += o;
      }
      const int at = slot - before - (sum - n);
      if (at >= 0 && at < n) {
        found_b = b;
        found_tile = n - 1 - at;
      }
      before += __shfl_sync(~0u, sum, 31);
      if (before > slot) break;
    }
  }
  __syncthreads();
  if (found_b < 0) return;
  Job job;
  job.b = found_b;
  job.tile = found_tile;
  job.head = head;
  job.r = seq_rows(p, job.b, true);
  job.rows = min(kRows, job.r.n * G - job.tile * kRows);
  const int pos0 = job.r.len - job.r.n;
  {
    const int first = pos0 + job.tile * kRows / G, last = pos0 + (job.tile * kRows + job.rows - 1) / G;
    job.t1 = p.causal ? min(last + 1, job.r.len) : job.r.len;
    job.t0 = window_from(p, first);
    if (job.t1 < job.t0) job.t1 = job.t0;
  }
  const int j0 = job.t0 / kStep, n_steps = job.t1 > job.t0 ? (job.t1 + kStep - 1) / kStep - j0 : 0;
  const bool two = job.rows > kTile;

  const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
  if (tid == 0) {
    for (int i = 0; i < kRing; ++i) {
      mbar_init(&bars.kfull[i], kWidenWarps);
      mbar_init(&bars.vfull[i], kWidenWarps);
      mbar_init(&bars.kempty[i], two ? 2 : 1);
      mbar_init(&bars.vempty[i], two ? 2 : 1);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&bars.sfull[i >> 1][i & 1], 1);
      mbar_init(&bars.odone[i >> 1][i & 1], 1);
      mbar_init(&bars.pfull[i >> 1][i & 1], 4);
      mbar_init(&bars.done[i], 1);
    }
    abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&tmem_slot);
  const Ctl ctl{&abort_flag, p.err};

  // ---- queries to shared memory (K-major, 128-byte swizzle), negated for a negative scale
  {
    const uint32_t flip = p.scale < 0.0f ? 0x80008000u : 0u;
    const bool vec = (reinterpret_cast<uintptr_t>(p.q) & 15u) == 0 && (p.qs & 7) == 0;
    constexpr int kPer = D / 8;
    for (int e = tid; e < kRows * kPer; e += kThreads) {
      const int r = e / kPer, ch = e % kPer;  // 16-byte chunk ch of row r
      uint32_t v[4] = {0, 0, 0, 0};
      if (r < job.rows) {
        const int rr = job.tile * kRows + r;
        const __half* src = static_cast<const __half*>(p.q) + static_cast<int64_t>(job.r.row0 + rr / G) * p.qs + (head * G + rr % G) * D + ch * 8;
        if (vec) {
          const uint4 u = *reinterpret_cast<const uint4*>(src);
          v[0] = u.x; v[1] = u.y; v[2] = u.z; v[3] = u.w;
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            v[i] = static_cast<uint32_t>(__half_as_ushort(src[2 * i])) | (static_cast<uint32_t>(__half_as_ushort(src[2 * i + 1])) << 16);
        }
      }
      const int row = r & (kTile - 1);
      const uint32_t at = base + M::kQ + (r / kTile) * M::kQTile + (ch >> 3) * M::kQPanel + row * 128 + (((ch & 7) ^ (row & 7)) << 4);
      sts128(at, v[0] ^ flip, v[1] ^ flip, v[2] ^ flip, v[3] ^ flip);
    }
    fence_async_shared();
  }
  __syncthreads();

  if (warp < kSoftmaxWarps) {
    regs_inc<kSoftmaxRegs>();
    // ---------------------------------------------------------------- softmax
    const int a = warp >> 2, q = warp & 3, row = a * kTile + q * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>(32 * q) << 16;
    const uint32_t s_base = tmem + lanes + kS + 128 * a, o_at = tmem + lanes + kO + 128 * a;
    const int rr = job.tile * kRows + min(row, job.rows - 1), pos = pos0 + rr / G;
    const int hi = p.causal ? max(0, min(pos + 1, job.r.len)) : job.r.len, lo = window_from(p, pos);
    float m = -INFINITY, l = 0.0f;
    bool ok = a == 0 || two;
    for (int j = 0; ok && j < n_steps; ++j) {
      const int st = j & 1;
      const uint32_t ph = (j >> 1) & 1, s_at = s_base + kStep * st;
      if (!warp_wait(&bars.sfull[a][st], ph, ctl, kErrSoftmax)) break;
      tc_fence_after();
      const Meta& mt = meta[j & (2 * kRing - 1)];
      const int t0 = (j0 + j) * kStep, lo_r = lo - t0, hi_r = hi - t0, oks = mt.oks;
      uint32_t x[kStep];
      tmem_ld32(s_at, x);
      tmem_ld32(s_at + 32, x + 32);
      tmem_wait_ld();
      tmem_fence_ld(x);
      tmem_fence_ld(x + 32);
      int seen = (1 << kChunks) - 1;  // chunks of which the row sees a token
      if (!__all_sync(~0u, lo_r <= 0 && hi_r >= kStep && oks == (1 << kChunks) - 1)) {
        seen = 0;
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          const int hi_c = (oks >> c) & 1 ? hi_r : 0;
          if (16 * c < hi_c && 16 * c + 16 > lo_r) seen |= 1 << c;
#pragma unroll
          for (int e = 16 * c; e < 16 * c + 16; ++e)
            if (e >= hi_c || e < lo_r) x[e] = 0xff800000u;
        }
      }
      float top = -INFINITY;
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        const float* v = reinterpret_cast<const float*>(x + 16 * c);
        const float t = max3(max3(max3(v[0], v[1], v[2]), max3(v[3], v[4], v[5]), max3(v[6], v[7], v[8])),
                             max3(max3(v[9], v[10], v[11]), max3(v[12], v[13], v[14]), v[15]), -INFINITY);
        top = fmaxf(top, t > -INFINITY ? fmaf(t, mt.kf[c], mt.lv[c]) : -INFINITY);
      }
      const bool raise = top > m + (kRaise + kLift);
      if (__any_sync(~0u, raise)) {
        const float fresh = raise ? top - kLift : m;
        const float f = raise ? (m == -INFINITY ? 0.0f : exp2_approx(m - fresh)) : 1.0f;
        m = fresh;
        l *= f;
        if (j > 0) {  // O may change once the products of the step before are complete
          if (!warp_wait(&bars.odone[a][st ^ 1], ((j - 1) >> 1) & 1, ctl, kErrSoftmax)) break;
          tc_fence_after();
#pragma unroll 1
          for (int i = 0; i < D / 16; ++i) {
            uint32_t o[16];
            tmem_ld16(o_at + 16 * i, o);
            tmem_wait_ld16(o);
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
            tmem_st16(o_at + 16 * i, o);
          }
          tmem_wait_st();
        }
      }
      const float mm = m == -INFINITY ? 0.0f : m;
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        // a page that the row does not see keeps its factors (a NaN) to itself
        const bool sees = (seen >> c) & 1;
        float kf = mt.kf[c], sub = mt.lv[c] - mm, iv = mt.iv[c];
        kf = sees ? kf : 1.0f;
        sub = sees ? sub : 0.0f;
        iv = sees ? iv : 0.0f;
        const float2 kf2 = make_float2(kf, kf), sub2 = make_float2(sub, sub);
        float2 w[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = fma2(make_float2(__uint_as_float(x[16 * c + 2 * e]), __uint_as_float(x[16 * c + 2 * e + 1])), kf2, sub2);
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = make_float2(exp2_approx(w[e].x), exp2_approx(w[e].y));
#pragma unroll
        for (int e = 0; e < 8; ++e) x[8 * c + e] = pack_half2(w[e].x, w[e].y);
        const float2 sum = add2(add2(add2(w[0], w[1]), add2(w[2], w[3])), add2(add2(w[4], w[5]), add2(w[6], w[7])));
        l = fmaf(sum.x + sum.y, iv, l);
      }
      tmem_st32(s_at, *reinterpret_cast<const uint32_t(*)[32]>(x));
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars.pfull[a][st]);
    }
    if (ok && n_steps > 0) ok = warp_wait(&bars.odone[a][(n_steps - 1) & 1], ((n_steps - 1) >> 1) & 1, ctl, kErrSoftmax);
    tc_fence_after();
    if (ok) {
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      __half* dst = static_cast<__half*>(p.o) + static_cast<int64_t>(job.r.row0 + rr / G) * p.os + (head * G + rr % G) * D;
      const bool vec = (reinterpret_cast<uintptr_t>(p.o) & 15u) == 0 && (p.os & 7) == 0;
#pragma unroll 1
      for (int i = 0; i < D / 32; ++i) {
        uint32_t o[32];
        if (n_steps > 0) {
          tmem_ld32(o_at + 32 * i, o);
          tmem_wait_ld();
          tmem_fence_ld(o);
        }
        if (row < job.rows) {
#pragma unroll
          for (int e = 0; e < 32; e += 8) {
            uint32_t h[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
              h[k] = n_steps > 0 && inv != 0.0f ? pack_half2(__uint_as_float(o[e + 2 * k]) * inv, __uint_as_float(o[e + 2 * k + 1]) * inv) : 0u;
            if (vec) {
              *reinterpret_cast<uint4*>(dst + 32 * i + e) = make_uint4(h[0], h[1], h[2], h[3]);
            } else {
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                dst[32 * i + e + 2 * k] = __ushort_as_half(static_cast<unsigned short>(h[k] & 0xffffu));
                dst[32 * i + e + 2 * k + 1] = __ushort_as_half(static_cast<unsigned short>(h[k] >> 16));
              }
            }
          }
        }
      }
    }
  } else if (warp < kMmaWarp) {
    regs_dec<kWidenRegs>();
    // ---------------------------------------------------------------- widen keys or values
    constexpr int kPieces = D / 16;                             // 16-byte pieces a row
    constexpr int kPer = kStep * kPieces / (kWidenWarps * 32);  // pieces a thread
    constexpr int kRowStep = kWidenWarps * 32 / kPieces;
    static_assert(kRowStep % 16 == 0, "a thread's rows lie at the same place of their 16-token chunks");
    const bool keys = warp < kSoftmaxWarps + kWidenWarps;
    // A lane's piece of a row is 16 codes: 16-byte chunks 2 (piece % 4) and + 1 of the row's float16 numbers in panel piece / 4.
    // The lanes of the second panel take the neighbouring row, whose swizzle puts them on the other banks.
    const int ct = tid - (keys ? kSoftmaxWarps : kSoftmaxWarps + kWidenWarps) * 32, piece = ct % kPieces, row0 = (ct / kPieces) ^ (piece >> 2);
    const uint8_t* cache = (keys ? p.k_cache : p.v_cache) + (row0 & 15) * D + piece * 16;
    uint64_t* full = keys ? bars.kfull : bars.vfull;
    uint64_t* empty = keys ? bars.kempty : bars.vempty;
    const int c0 = 2 * (piece & 3);
    const uint32_t line = base + (keys ? M::kK : M::kV) + (piece >> 2) * M::kPanel + row0 * 128;
    const uint32_t at0 = line + ((c0 ^ (row0 & 7)) << 4), at1 = line + (((c0 + 1) ^ (row0 & 7)) << 4);
    // Lane c < kChunks knows chunk c of a step: its page id three steps ahead, two steps ahead where its first token's
    // codes lie (-1: nowhere). The first thread of the keys' warps for each chunk also makes the step's factors: scales two
    // steps ahead, factors one. Chunks in front of what any row sees are nowhere too: their pages may be gone from the table.
    const bool factors = keys && ct < kChunks;
    int id_next = -1, ok_raw = 0, ok_now = 0;
    int64_t chunk_base = -1;
    float ks = 0.0f, vs = 0.0f, kf = 0.0f, lv = 0.0f, iv = 0.0f;
    auto find_page = [&](int j) {
      const int tok = (j0 + j) * kStep + 16 * lane;
      id_next = -1;
      if (j < n_steps && lane < kChunks && tok + 16 > job.t0 && tok < job.t1) id_next = p.page_table[static_cast<int64_t>(job.b) * p.max_pages + (tok >> p.page_log2)];
    };
    auto find = [&](int j) {
      const int tok = (j0 + j) * kStep + 16 * lane;
      const bool wanted = j < n_steps && lane < kChunks && tok + 16 > job.t0 && tok < job.t1, use = wanted && id_next >= 0 && id_next < p.pages;
      if (wanted && !use) record_device_error(p.err, kErrKv8Page);
      const int64_t block = static_cast<int64_t>(id_next) * p.hkv + head;
      chunk_base = use ? ((block << p.page_log2) + (tok & (p.page - 1))) * D : -1;
      if (factors) {
        ok_raw = use;
        ks = vs = 0.0f;
        if (use) {
          ks = p.k_scale[block];
          vs = p.v_scale[block];
        }
      }
    };
    // A k_scale of zero becomes a factor so small that the scores vanish all the same: 0 * infinity never meets a masked
    // score. Value scales below 2^-60 count as 2^-60: with codes of up to 448 either is zero as a float16.
    auto make_factors = [&] {
      const float f = fmaxf(vs, 8.6736174e-19f);
      kf = ks * fabsf(p.scale) * kLog2e;
      if (kf == kf) kf = fmaxf(kf, 1e-30f);
      const bool bad = !(fabsf(vs) <= 3.4028234e38f);
      lv = bad ? __uint_as_float(0x7fc00000u) : __log2f(f);
      iv = bad ? lv : __frcp_rn(f);
      ok_now = ok_raw;
    };
    auto load = [&](int j, uint4 (&to)[kPer]) {
      const int left = job.t1 - (j0 + j) * kStep;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int row = row0 + i * kRowStep;
        const int64_t at = __shfl_sync(~0u, chunk_base, row >> 4);
        to[i] = make_uint4(0, 0, 0, 0);
        if (at >= 0 && row < left) to[i] = *reinterpret_cast<const uint4*>(cache + at);
      }
    };
    auto put = [&](int j, const uint4 (&w)[kPer]) {
      const int st = j & (kRing - 1);
      if (!warp_wait(&empty[st], ((j / kRing) & 1) ^ 1, ctl, kErrWiden)) return false;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const uint2 a = widen4<E4M3>(w[i].x), b = widen4<E4M3>(w[i].y), c = widen4<E4M3>(w[i].z), d = widen4<E4M3>(w[i].w);
        sts128(at0 + st * M::kOperand + i * kRowStep * 128, a.x, a.y, b.x, b.y);
        sts128(at1 + st * M::kOperand + i * kRowStep * 128, c.x, c.y, d.x, d.y);
      }
      if (factors) {
        Meta& mt = meta[j & (2 * kRing - 1)];
        mt.kf[ct] = kf;
        mt.lv[ct] = lv;
        mt.iv[ct] = iv;
        const int oks = __ballot_sync((1u << kChunks) - 1, ok_now);
        if (ct == 0) mt.oks = oks;
      }
      fence_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(&full[st]);
      return true;
    };
    uint4 w0[kPer], w1[kPer];
    find_page(0);
    find(0);
    find_page(1);
    load(0, w0);
    if (factors) make_factors();
    find(1);
    find_page(2);
    load(1, w1);
    // step j: its data in w0 / w1, the factors its own, scales those of j + 1, page ids those of j + 2
    auto turn = [&](int j, uint4 (&w)[kPer]) {
      if (!put(j, w)) return false;
      if (factors) make_factors();
      find(j + 2);
      find_page(j + 3);
      load(j + 2, w);
      return true;
    };
#pragma unroll 1
    for (int j = 0; j < n_steps; j += 2) {
      if (!turn(j, w0)) break;
      if (j + 1 < n_steps && !turn(j + 1, w1)) break;
    }
  } else {
    regs_dec<kMmaRegs>();
  }
  if (warp >= kMmaWarp && (two || !((warp - kMmaWarp) & 1))) {
    // ---------------------------------------------------------------- MMAs (a warp stays converged, so that their operands stay in uniform registers; one lane issues)
    const int a = (warp - kMmaWarp) & 1, issuer = warp - kMmaWarp;
    constexpr uint32_t kF32Out = 1u << 4;
    if (issuer < 2) {  // scores; their buffer held the weights of two steps before
      constexpr uint32_t qk = kF32Out | (static_cast<uint32_t>(kStep >> 3) << 17) | (static_cast<uint32_t>(kTile >> 4) << 24);
      const uint64_t qd = umma_desc_sw128(base + M::kQ + a * M::kQTile), kd = umma_desc_sw128(base + M::kK);
#pragma unroll 1
      for (int j = 0; j < n_steps; ++j) {
        const int st = j & (kRing - 1), b = j & 1;
        if (!warp_wait(&bars.kfull[st], (j / kRing) & 1, ctl, kErrMma) || (j >= 2 && !warp_wait(&bars.odone[a][b], ((j - 2) >> 1) & 1, ctl, kErrMma))) break;
        tc_fence_after();
        if (elect_one()) {
#pragma unroll
          for (int i = 0; i < D / 16; ++i) {
            const uint64_t q_off = static_cast<uint64_t>((i >> 2) * (M::kQPanel >> 4) + 2 * (i & 3)), k_off = static_cast<uint64_t>((i >> 2) * (M::kPanel >> 4) + 2 * (i & 3));
            mma_f16_ss(tmem + kS + 128 * a + kStep * b, qd + q_off, kd + st * (M::kOperand >> 4) + k_off, qk, i > 0);
          }
          mma_commit(&bars.sfull[a][b]);
          mma_commit(&bars.kempty[st]);
        }
        __syncwarp();
      }
    } else {  // values
      constexpr uint32_t pv = kF32Out | (1u << 16) | (static_cast<uint32_t>(D >> 3) << 17) | (static_cast<uint32_t>(kTile >> 4) << 24);
      const uint64_t vd = desc_mn<D>(base + M::kV);
#pragma unroll 1
      for (int j = 0; j < n_steps; ++j) {
        const int st = j & (kRing - 1), b = j & 1;
        if (!warp_wait(&bars.vfull[st], (j / kRing) & 1, ctl, kErrMma) || !warp_wait(&bars.pfull[a][b], (j >> 1) & 1, ctl, kErrMma)) break;
        tc_fence_after();
        if (elect_one()) {
#pragma unroll
          for (int i = 0; i < kStep / 16; ++i)
            mma_f16_ts(tmem + kO + 128 * a, tmem + kS + 128 * a + kStep * b + 8 * i, vd + st * (M::kOperand >> 4) + i * (2048 >> 4), pv, j > 0 || i > 0);
          mma_commit(&bars.odone[a][b]);
          mma_commit(&bars.vempty[st]);
        }
        __syncwarp();
      }
    }
    if (elect_one()) mma_commit(&bars.done[issuer]);  // every MMA that this warp issued has completed once it flips
    __syncwarp();
    drain_wait(&bars.done[issuer], 0, p.err, kErrDrain);
  }

  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
}

template <bool E4M3, int D>
cudaError_t launch(const Kv8& p, cudaStream_t s) {
  // one CTA an SM: it takes all tensor memory
  constexpr int bytes = Smem<D>::kBytes > 120 * 1024 ? Smem<D>::kBytes : 120 * 1024;
  const cudaError_t e = allow_smem<attn_prompt_kernel<E4M3, D>>(bytes);
  if (e != cudaSuccess) return e;
  const int64_t G = p.hq / p.hkv, tiles = p.uniform ? ceil_div(p.tokens / p.seqs * G, kRows) * p.seqs : p.tokens * G / kRows + p.seqs;
  attn_prompt_kernel<E4M3, D><<<static_cast<unsigned>(tiles * p.hkv), kThreads, bytes, s>>>(p);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_kv8_attn_prompt(const Kv8& p, cudaStream_t s) {
  if (p.D == 128) return p.e4m3 ? launch<true, 128>(p, s) : launch<false, 128>(p, s);
  return p.e4m3 ? launch<true, 64>(p, s) : launch<false, 64>(p, s);
}

}  // namespace xrgpu
