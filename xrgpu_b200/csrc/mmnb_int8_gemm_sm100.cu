// Product of 8-bit integer operands with scales for each token and channel, dense or grouped by expert (problem:
// mmnb_int8.h), on tcgen05 tensor cores:
//   y[r, n] = act((sum_k a[r, k] b[n, k]) sa[r] sb[n] + bias[n]), the sum exact in int32.
//
// Orientation. The weights' channels are the MMA's 128-row operand P, the tokens its other one, Q, of any multiple of
// 16 columns up to 256: a group with few rows pays for few columns, weights stream whole, and an accumulator's 32 lanes are
// neighbours of a row of y. A tile is 128 channels of a group by up to tmax of its rows (a group's rows are cut evenly).
//
// Groups. Offsets are on the device: every CTA counts the groups' tiles itself (a scan in shared memory) and takes tiles
// of one line, group by group, the tiles of the same channels next to each other. From the first offset that does not
// fit on there are no groups, and an error is recorded. Rows come in the groups' order: fetching them where the tokens lie was slower by far (16384 x 4096 x
// 4096, 216 us: 483 with 16-byte copies, whose writes need a fence of 2000 cycles a stage before the tensor cores may read
// them; four-row tensor gathers take 60 cycles each, 3800 a stage of 256 rows).
//
// Roles (10 warps): warp 0 loads, warp 1 issues the MMAs, warps 2-9 drain (lane quadrant warp % 4, alternate 16-column chunks).
// Few tiles: K is split over a cluster of up to 8 CTAs whose int32 partial tiles meet in shared memory.
//
// Measured (GPU time of the call, weights from memory): 1 x 4096 x 4096 float rows 7.4 us (16.8 MB, 2.3 TB/s: latency), 16 x 4096 x
// 14336 16.3 us with the rows' quantisation (59 MB, 3.6 TB/s: start and end, then the stream), one token by 8 of 64 experts of
// 4096 x 4096 26.4 us (134 MB, 5.1 TB/s), 64 tokens by 64 experts of 4096 x 2048 with their sums 89.5 us (540 MB, 6.0 TB/s), 2048 x
// 14336 x 4096 86.5 us (2.8 PFLOP/s; tensor cores 78 % of the cycles, at 1.4 GHz under the power limit from the first launch on;
// 99.6 us in calls back to back for seconds), 8192 x 8192 x 8192 372 us, 428 us for seconds (2.6 PFLOP/s at 1.24 GHz).
//
// Every wait is bounded as in mmnb_gemm_sm100.cu.
#include <cuda.h>
#include <cuda_fp16.h>

#include <climits>
#include <type_traits>

#include "mmnb_int8.cuh"
#include "mmnb_int8.h"
#include "mmnb_tcgen05.cuh"

namespace xrgpu {
namespace {

constexpr int kRows = 128;       // channels of a tile
constexpr int kStepBytes = 128;  // codes of a row per stage: one swizzle row
constexpr int kEpilogueWarps = 8;
constexpr int kThreads = (2 + kEpilogueWarps) * 32;
constexpr int kSmemMost = 227 * 1024;
constexpr int kSmemBudget = kSmemMost - 10 * 1024;  // dynamic: less what is declared
constexpr int kMaxStages = 12;
constexpr int kMaxT = 256;
constexpr int kPitch = kRows;    // int32 values a column of a partial tile in shared memory

constexpr unsigned kErrOffsets = 0x701;
constexpr unsigned kErrWaitProducer = 0x711;
constexpr unsigned kErrWaitMma = 0x712;
constexpr unsigned kErrWaitEpilogue = 0x713;
constexpr unsigned kErrDrain = 0x714;

struct Args {
  int n, p_tiles, groups, rows;
  Divide by_p, by_tmax;        // p_tiles, tmax
  int tmax, box, box_log;      // most rows of Q a tile (a multiple of 16); rows of one copy (30: one copy takes all of a tile's)
  int ksteps, ksubs;           // stages along K, 32-value MMA steps along K
  int stages, split, split_log;
  int tmem_cols, acc1;         // acc1: column of the second accumulator
  int early;                   // the weights may be loaded before the previous kernel has finished
  uint32_t stage;              // bytes
  uint32_t tables, scales;     // bytes from the stages' start to the group tables, and to the rows' scales
  int act, has_limit, zero_rest, bias_f16;
  float alpha, beta, limit;
  const int32_t* offsets;
  const float* a_scales;
  const float* b_scales;
  const void* bias;
  void* y;
  int64_t ldy;
  unsigned* err;
};

// D[128 x T] (+)= P (smem, K-major codes) . Q^T in int32.
__device__ __forceinline__ void mma_i8(uint32_t d, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void prefetch_map(const CUtensorMap* m) { asm volatile("prefetch.tensormap [%0];" ::"l"(m) : "memory"); }

// Instruction descriptor: int32 sums of signed 8-bit operands, both K-major, M rows, T columns.
__device__ __forceinline__ uint32_t instruction_desc(int M, int T) {
  return (2u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(T >> 3) << 17) | (static_cast<uint32_t>(M >> 4) << 24);
}

// ------------------------------------------------------------------ tiles
// Tables in shared memory: tile_first [groups + 1] (tiles along the rows before a group), row_first, row_count [groups].
struct Tables {
  int* tile_first;
  int* row_first;
  int* row_count;
};
__device__ __forceinline__ Tables tables_at(uint8_t* at, int groups) {
  int* t = reinterpret_cast<int*>(at);
  return {t, t + groups + 1, t + 2 * groups + 1};
}
inline uint32_t tables_bytes(int groups) { return static_cast<uint32_t>(align_up(static_cast<uint64_t>(3 * groups + 1) * 4, 16)); }

// All threads; ends with a barrier. From the first offset on that decreases or leaves [0, rows] no group has tiles: what comes
// before it is in order, so no two groups share a row. Returns whether all offsets fit.
__device__ __forceinline__ bool make_tables(const Args& a, const Tables& t) {
  __shared__ int chunk_sum[32], chunk_bad[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int base = 32 * warp; base < a.groups; base += kThreads) {
    const int g = base + lane;
    int lo = 0, hi = g < a.groups ? a.rows : 0;
    if (a.offsets && g < a.groups) {
      lo = a.offsets[g];
      hi = a.offsets[g + 1];
    }
    const unsigned bad = __ballot_sync(~0u, lo < 0 || hi < lo || hi > a.rows);
    if (bad && (bad & (2u << lane) - 1)) lo = hi = 0;  // this group, or one before it
    if (g < a.groups) {
      t.row_first[g] = lo;
      t.row_count[g] = hi - lo;
    }
    int s = (hi - lo + a.tmax - 1) / a.by_tmax;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(~0u, s, o);
      if (lane >= o) s += u;
    }
    if (g < a.groups) t.tile_first[g + 1] = s;
    if (lane == 31) {
      chunk_sum[base >> 5] = s;
      chunk_bad[base >> 5] = bad != 0;
      if (bad && blockIdx.x == 0) record_device_error(a.err, kErrOffsets);
    }
  }
  if (threadIdx.x == 0) t.tile_first[0] = 0;
  __syncthreads();
  bool fit = !chunk_bad[0];
  if (a.groups > 32) {
    const int chunks = (a.groups + 31) / 32, sum = lane < chunks ? chunk_sum[lane] : 0;
    const unsigned bad = __ballot_sync(~0u, lane < chunks && chunk_bad[lane]);
    const int last = bad ? __ffs(bad) - 1 : chunks;  // the last chunk that counts
    fit = !bad;
    for (int base = 32 * warp; base < a.groups; base += kThreads) {
      const int chunk = base >> 5, before = __reduce_add_sync(~0u, lane < chunk && lane <= last ? sum : 0);
      if (base + lane < a.groups) t.tile_first[base + lane + 1] = before + (chunk <= last ? t.tile_first[base + lane + 1] : 0);
    }
    __syncthreads();
  }
  return fit;
}

struct Tile {
  int group, pt;   // block of channels
  int row0, rows;  // rows of the product
  int width;       // columns of the MMA: a multiple of GRAIN
};
// Whole warps. Little code, and no division for a group of one tile: what every CTA runs before its first load comes from memory, and
// cost 5000 cycles (1 x 4096 x 4096 7.7 -> 7.2 us without, 333 x 1003 x 4100 13.8 -> 12.8).
template <int GRAIN>
__device__ __forceinline__ Tile tile_at(const Args& a, const Tables& t, int tile) {
  const int q = tile / a.by_p, lane = threadIdx.x & 31;
  // the last group that begins at or before q: among every 32nd, then among 32
  int g = 0;
  if (a.groups > 32) g = 32 * (__popc(__ballot_sync(~0u, 32 * lane < a.groups && t.tile_first[min(32 * lane, a.groups)] <= q)) - 1);
  g += __popc(__ballot_sync(~0u, g + lane < a.groups && t.tile_first[min(g + lane, a.groups)] <= q)) - 1;
  const int first = t.tile_first[g], nt = t.tile_first[g + 1] - first, count = t.row_count[g], local = tile - first * a.p_tiles;
  if (nt == 1) return {g, local, t.row_first[g], count, (count + GRAIN - 1) / GRAIN * GRAIN};
  const int pt = local / nt, qt = local - pt * nt;
  const int even = ((count + nt - 1) / nt + GRAIN - 1) / GRAIN * GRAIN, rows = min(even, count - qt * even);
  return {g, pt, t.row_first[g] + qt * even, rows, (rows + GRAIN - 1) / GRAIN * GRAIN};
}

// ------------------------------------------------------------------ results
template <bool F16>
__device__ __forceinline__ void put(void* y, int64_t at, float v) {
  if (F16) static_cast<__half*>(y)[at] = __float2half_rn(v);
  else static_cast<float*>(y)[at] = v;
}

// (gate, linear) -> gate sigmoid(alpha gate) (linear + beta)
__device__ __forceinline__ float swiglu(const Args& a, float g, float l) {
  if (a.has_limit) {
    g = g > a.limit ? a.limit : g;
    l = l > a.limit ? a.limit : l < -a.limit ? -a.limit : l;
  }
  // the reciprocal within one step; of infinity zero
  float s;
  asm("rcp.approx.f32 %0, %1;" : "=f"(s) : "f"(1.0f + expf(-a.alpha * g)));
  return g * s * (l + a.beta);
}

// Product first with the token's, then with the channel's scale: an int32 and two float32 numbers, each step rounded to 2^-24.
__device__ __forceinline__ float scaled(int acc, float sa, float sb, float bias) { return fmaf(static_cast<float>(acc) * sa, sb, bias); }
// From row scales of 2^96 on the first of these may leave float32 where the result does not: 2^32 is taken from the row's and given to the
// channel's scale, exactly. (A channel's of 2^96 and more stays: any product with it but 0 is out of range.) Such tiles take a loop of
// their own: the same steps for every tile cost 0.6 % of 2048 x 14336 x 4096, so it is 0.2 %.
constexpr float kFarScale = 0x1p96f;
__device__ __forceinline__ float far_row(float sa) { return fabsf(sa) >= kFarScale ? sa * 0x1p-32f : sa; }
__device__ __forceinline__ float far_channel(float sa, float sb) { return fabsf(sa) >= kFarScale && fabsf(sb) < kFarScale ? sb * 0x1p32f : sb; }
__device__ __forceinline__ float relu(float r) { return r < 0.0f ? 0.0f : r; }  // a NaN stays

// Rows of no group (before the first offset, behind the last one that counts) become zero.
template <bool F16>
__device__ __forceinline__ void zero_rest(const Args& a, bool fit, int width) {
  if (!a.zero_rest || !a.offsets) return;
  int lo = a.offsets[0], hi = a.offsets[a.groups];
  if (!fit) {
    const bool none = lo < 0 || lo > a.rows;
    hi = lo = none ? 0 : lo;
    for (int g = 1; !none && g <= a.groups; ++g) {
      const int o = a.offsets[g];
      if (o < hi || o > a.rows) break;
      hi = o;
    }
  }
  for (int r = blockIdx.x; r < lo + a.rows - hi; r += gridDim.x) {
    const int64_t row = r < lo ? r : hi + r - lo;
    for (int n = threadIdx.x; n < width; n += kThreads) put<F16>(a.y, row * a.ldy + n, 0.0f);
  }
}

struct ChannelScale {
  float scale, bias;
  bool far;  // some of the tile's rows have scales of kFarScale and more
};
__device__ __forceinline__ ChannelScale channel_scale(const Args& a, int group, int n) {
  ChannelScale ch{0.0f, 0.0f, false};
  if (n < a.n) {
    const int64_t at = static_cast<int64_t>(group) * a.n + n;
    ch.scale = a.b_scales[at];
    if (a.bias) ch.bias = load_f(a.bias, a.bias_f16, at);
  }
  return ch;
}
// The scales of a tile's rows into the warp's `row_scale`, and the lane's channel's.
__device__ __forceinline__ ChannelScale prepare_scales(const Args& a, const Tile& t, int n, float* row_scale, int lane) {
  ChannelScale ch = channel_scale(a, t.group, n);
  float scale[kMaxT / 32];  // all loads before the first use: one after the other they take 800 cycles each
#pragma unroll
  for (int i = 0; i < kMaxT / 32; ++i) scale[i] = 32 * i + lane < t.rows ? a.a_scales[t.row0 + 32 * i + lane] : 0.0f;
#pragma unroll
  for (int i = 0; i < kMaxT / 32; ++i) {
    if (32 * i < t.width) row_scale[32 * i + lane] = scale[i];
    ch.far |= fabsf(scale[i]) >= kFarScale;
  }
  ch.far = __any_sync(~0u, ch.far);
  __syncwarp();
  return ch;
}

// Results of 16 columns of the lane's channel, as y holds them: float16 two a word, in the order of the columns. With swiglu a lane has
// every other column of its pair of channels: even lanes the even columns, odd lanes the odd ones.
template <bool F16, bool SWIGLU>
constexpr int kWords = (SWIGLU ? 8 : 16) / (F16 ? 2 : 1);

// All lanes of the warp take part; the columns' row scales are at `row_scale`.
template <bool F16, bool SWIGLU>
__device__ __forceinline__ void results(const Args& a, const uint32_t (&v)[16], const ChannelScale& ch, const float* row_scale, int lane, uint32_t (&w)[kWords<F16, SWIGLU>]) {
  float f[16];
  if (!ch.far) {
#pragma unroll
    for (int j = 0; j < 16; ++j) f[j] = scaled(static_cast<int>(v[j]), row_scale[j], ch.scale, ch.bias);
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j) f[j] = scaled(static_cast<int>(v[j]), far_row(row_scale[j]), far_channel(row_scale[j], ch.scale), ch.bias);
  }
  if (SWIGLU) {
    const bool odd = lane & 1;
#pragma unroll
    for (int j = 0; j < 16; j += 2) {
      const float other = __shfl_xor_sync(~0u, odd ? f[j] : f[j + 1], 1);
      f[j / 2] = swiglu(a, odd ? other : f[j], odd ? f[j + 1] : other);
    }
  } else if (a.act == XRGPU_ACT_RELU) {
#pragma unroll
    for (int j = 0; j < 16; ++j) f[j] = relu(f[j]);
  }
#pragma unroll
  for (int j = 0; j < kWords<F16, SWIGLU>; ++j) {
    if (F16) {
      const __half2 h = __floats2half2_rn(f[2 * j], f[(2 * j + 1) & 15]);
      w[j] = *reinterpret_cast<const uint32_t*>(&h);
    } else {
      w[j] = __float_as_uint(f[j]);
    }
  }
}

// They go to rows row0 + col0 + j of y, each by itself, 64 or 128 bytes a warp. (Pairs of channels, joined by shuffles, would make
// half as many stores of as many rows of y each: 11700 cycles for 128 channels by 256 rows, 6400 by single ones; 4000 of these are
// the stores' own.)
template <bool F16, bool SWIGLU>
__device__ __forceinline__ void store_results(const Args& a, const uint32_t (&w)[kWords<F16, SWIGLU>], int row0, int col0, int rows, int n, int lane) {
  using T = typename std::conditional<F16, uint16_t, uint32_t>::type;
  constexpr int kStep = SWIGLU ? 2 : 1;
  if (n >= a.n) return;
  const int odd = SWIGLU ? lane & 1 : 0, left = rows - col0 - odd;
  T* y = static_cast<T*>(a.y) + static_cast<int64_t>(row0 + col0 + odd) * a.ldy + (SWIGLU ? n >> 1 : n);
  auto value = [&](int i) { return static_cast<T>(F16 ? w[i >> 1] >> (16 * (i & 1)) : w[i & (kWords<F16, SWIGLU> - 1)]); };
  if (left > 15) {
#pragma unroll
    for (int j = 0; j < 16; j += kStep, y += kStep * a.ldy) *y = value(j / kStep);
  } else {
#pragma unroll
    for (int j = 0; j < 16; j += kStep, y += kStep * a.ldy)
      if (j < left) *y = value(j / kStep);
  }
}

// 16 columns of a tile's sums, from column `col` on with the rows' scales at `row_scale`, to y.
template <bool F16, bool SWIGLU>
__device__ __forceinline__ void store_chunk(const Args& a, const Tile& t, const uint32_t (&v)[16], int col, int n, const ChannelScale& ch, const float* row_scale, int lane) {
  uint32_t w[kWords<F16, SWIGLU>];
  results<F16, SWIGLU>(a, v, ch, row_scale, lane, w);
  store_results<F16, SWIGLU>(a, w, t.row0, col, t.rows, n, lane);
}

// The warp's chunks of a tile's sums, from tensor memory to y.
template <bool F16, bool SWIGLU>
__device__ __forceinline__ void drain_tile(const Args& a, const Tile& t, uint32_t tmem, int c, int n, const ChannelScale& ch, const float* row_scale, int lane) {
  for (int col = 16 * c; col < t.width; col += 32) {
    uint32_t v[16];
    tmem_ld16(tmem + col, v);
    tmem_wait_ld16(v);
    store_chunk<F16, SWIGLU>(a, t, v, col, n, ch, row_scale + col, lane);
    __syncwarp();
  }
}

// A split tile's sums over the cluster's ranks (128 values of a column lie together at `base` of each): every rank takes its
// share of the columns, a thread the same four channels (`ch`) of each. Little code, once through: 333 x 1003 x 4100 14.3 us with the
// channels' scales loaded a column at a time, 13.8 so, 14.8 with two columns at a time, unrolled. All threads.
template <bool F16, bool SWIGLU>
__device__ __forceinline__ void sum_ranks(const Args& a, const Tile& t, uint32_t base, int rank, const float* row_scale, const ChannelScale (&ch)[4]) {
  constexpr int kLanes = kRows / 4, kColumns = kThreads / kLanes;  // threads a column, columns at a time
  const int share = (t.rows + a.split - 1) >> a.split_log, col0 = rank * share, end = min(t.rows, col0 + share);
  const int row = 4 * (threadIdx.x % kLanes), n = t.pt * kRows + row;
  if (n >= a.n) return;
#pragma unroll 1
  for (int col = col0 + threadIdx.x / kLanes; col < end; col += kColumns) {
    int sum[4] = {0, 0, 0, 0};
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < a.split) {
        const float4 v = ld_cluster_f32x4(map_rank(base + (col * kPitch + row) * 4, k));
        sum[0] += __float_as_int(v.x);
        sum[1] += __float_as_int(v.y);
        sum[2] += __float_as_int(v.z);
        sum[3] += __float_as_int(v.w);
      }
    float f[4];
    const float sa = row_scale[col];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[i] = scaled(sum[i], far_row(sa), far_channel(sa, ch[i].scale), ch[i].bias);
      if (a.act == XRGPU_ACT_RELU) f[i] = relu(f[i]);
    }
    const int64_t at = static_cast<int64_t>(t.row0 + col) * a.ldy;
    if (SWIGLU) {
      put<F16>(a.y, at + (n >> 1), swiglu(a, f[0], f[1]));
      if (n + 2 < a.n) put<F16>(a.y, at + (n >> 1) + 1, swiglu(a, f[2], f[3]));
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (n + i < a.n) put<F16>(a.y, at + n + i, f[i]);
    }
  }
}

// The order of a tile's stages along K: tiles next to each other begin at different ones, so that CTAs side by side do not read the same part of rows
// that lie a power of two apart.
struct Walk {
  int k1, steps, turn;
  __device__ __forceinline__ int at(int ks) const { return ks + turn < k1 ? ks + turn : ks + turn - steps; }
};
__device__ __forceinline__ Walk walk_of(int k0, int k1, int tile) {
  const int steps = k1 - k0;
  return {k1, steps, tile & ((1 << (31 - __clz(steps))) - 1)};
}

// STEPS: 128-byte steps along K of a stage. Two where four such stages fit (narrow tiles), and no more stages than these: fewer waits,
// copies and signals a byte, 256 bytes of a row at a time, and with more loads under way than 128 KB an SM memory is slower. With the
// walk: 64 tokens by 8 of 64 experts of 4096 x 2048 (six stages / five / four / and the walk) 95 / 94 / 91.5 / 89.8 us, 94.5 with 10
// stages of one step; one token by 8 of 64 of 4096 x 4096 29.1 -> 27.5; 16 x 14336 x 4096 15.6 -> 14.5, 64 rows 16.4 -> 15.1.
template <bool F16, bool SWIGLU, int STEPS>
__global__ void __launch_bounds__(kThreads, 1)
    int8_gemm_kernel(const __grid_constant__ CUtensorMap map_p, const __grid_constant__ CUtensorMap map_q, const Args a) {
  extern __shared__ uint8_t smem_raw[];
  const int warp = __shfl_sync(~0u, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int S = a.stages;
  const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
  uint8_t* gbase = smem_raw + (base - raw);
  // a stage: STEPS P tiles of 16 KB, then as many Q tiles of tmax * 128 bytes
  constexpr uint32_t kPartP = kRows * kStepBytes;
  const uint32_t part_q = static_cast<uint32_t>(a.tmax) * kStepBytes;
  __shared__ uint64_t full[kMaxStages], empty[kMaxStages], accfull[2], drained[2], done;
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;

  if (threadIdx.x == kThreads - 32) {  // not warp 0, which reads the offsets
    prefetch_map(&map_p);
    prefetch_map(&map_q);
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&accfull[b], 1);
      mbar_init(&drained[b], kEpilogueWarps);
    }
    mbar_init(&done, 1);
    abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                 ::"r"(smem_u32(&tmem_slot)), "r"(a.tmem_cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  const Tables tables = tables_at(gbase + a.tables, a.groups);
  const int scale_pitch = (a.tmax + 31) & ~31;
  float* const scales = reinterpret_cast<float*>(gbase + a.scales);  // of a tile's rows, a copy a warp: no barrier among them
  tc_fence_before();
  const bool fit = make_tables(a, tables);  // and a barrier
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&tmem_slot);
  const Ctl ctl{&abort_flag, a.err};
  const int rank = a.split > 1 ? static_cast<int>(cluster_rank()) : 0;
  const int tiles = tables.tile_first[a.groups] * a.p_tiles;
  const int first = blockIdx.x >> a.split_log, step = gridDim.x >> a.split_log;
  const int k0 = a.ksteps * rank >> a.split_log, k1 = a.ksteps * (rank + 1) >> a.split_log;

  if (warp == 0) {
    // One lane loads the weights and counts the bytes, copies of token rows are spread over the lanes.
    int g = 0, s = 0;
    uint32_t ph = 0;
    bool ok = true, waited = false;
    for (int tile = first; ok && tile < tiles; tile += step) {
      const Tile t = tile_at<16>(a, tables, tile);
      const int copies = (t.width + (1 << a.box_log) - 1) >> a.box_log;
      const uint32_t bytes = STEPS * (kRows + copies * a.box) * kStepBytes;
      const int p_row = t.group * a.n + t.pt * kRows;
      const Walk walk = walk_of(k0, k1, tile);
      auto load_p = [&](int st, int i_k) {
        const int ks = walk.at(i_k);
        mbar_arrive_expect_tx(&full[st], bytes);
#pragma unroll
        for (int i = 0; i < STEPS; ++i) tma_load_2d(base + st * a.stage + i * kPartP, &map_p, (STEPS * ks + i) * kStepBytes, p_row, &full[st]);
      };
      auto load_q = [&](int st, int i_k) {
        const int ks = walk.at(i_k);
        const uint32_t at = base + st * a.stage + STEPS * kPartP + lane * a.box * kStepBytes;
        if (lane < copies) {
#pragma unroll
          for (int i = 0; i < STEPS; ++i) tma_load_2d(at + i * part_q, &map_q, (STEPS * ks + i) * kStepBytes, t.row0 + lane * a.box, &full[st]);
        }
      };
      // The weights' first stages do not depend on the kernel before this one; the activations do.
      int pre = 0;
      if (!waited) {
        waited = true;
        if (a.early) {
          pre = min(S, k1 - k0);
          if (lane == 0)
            for (int i = 0; i < pre; ++i) load_p(i, k0 + i);
          __syncwarp();
        }
        asm volatile("griddepcontrol.wait;" ::: "memory");
      }
      for (int ks = k0; ks < k1; ++ks, ++g) {
        if (g >= pre) {
          if (!warp_spin(&empty[s], ph ^ 1, ctl, kErrWaitProducer)) {
            ok = false;
            break;
          }
          if (lane == 0) load_p(s, ks);
          __syncwarp();
        }
        load_q(s, ks);
        if (++s == S) {
          s = 0;
          ph ^= 1;
        }
      }
    }
    if (!waited) asm volatile("griddepcontrol.wait;" ::: "memory");
    if (!ok && lane == 0)
      for (int h = (g > S ? g - S : 0); h < g; ++h) drain_wait(&full[h % S], (h / S) & 1, a.err, kErrDrain);
  } else if (warp == 1) {
    // The warp stays converged and elects the issuing lane, so that descriptors stay in uniform registers.
    const uint64_t p_desc = umma_desc_sw128(base), q_desc = umma_desc_sw128(base + STEPS * kPartP);
    int i = 0, s = 0;
    uint32_t ph = 0;
    bool ok = true;
    for (int tile = first; ok && tile < tiles; tile += step, ++i) {
      const uint32_t i_desc = instruction_desc(kRows, tile_at<16>(a, tables, tile).width);
      if (i >= 2 && !warp_spin(&drained[i & 1], ((i - 2) >> 1) & 1, ctl, kErrWaitMma)) break;
      const Walk walk = walk_of(k0, k1, tile);
      tc_fence_after();
      const uint32_t d = tmem + ((i & 1) ? a.acc1 : 0);
      for (int ks = k0; ks < k1; ++ks) {
        if (!warp_spin(&full[s], ph, ctl, kErrWaitMma)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const int subs = a.ksubs - 4 * STEPS * walk.at(ks);
        const uint32_t off = static_cast<uint32_t>(s) * (a.stage >> 4);
        if (elect_one()) {
#pragma unroll
          for (int j = 0; j < 4 * STEPS; ++j) {
            if (j > 0 && j >= subs) break;
            mma_i8(d, p_desc + off + (j / 4) * (kPartP >> 4) + 2 * (j % 4), q_desc + off + (j / 4) * (part_q >> 4) + 2 * (j % 4), i_desc, ks > k0 || j > 0);
          }
          mma_commit(&empty[s]);
        }
        __syncwarp();
        if (++s == S) {
          s = 0;
          ph ^= 1;
        }
      }
      if (ok && elect_one()) mma_commit(&accfull[i & 1]);
      __syncwarp();
    }
    if (elect_one()) mma_commit(&done);  // every MMA of this warp has completed once `done` flips
    __syncwarp();
    drain_wait(&done, 0, a.err, kErrDrain);
  } else {
    const int q = warp & 3, c = (warp - 2) >> 2;
    const uint32_t lane_addr = static_cast<uint32_t>(32 * q) << 16;
    float* const row_scale = scales + (warp - 2) * scale_pitch;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    int i = 0;
    for (int tile = first; tile < tiles; tile += step, ++i) {
      const Tile t = tile_at<16>(a, tables, tile);
      const int b = i & 1, n = t.pt * kRows + 32 * q + lane;
      const ChannelScale ch = prepare_scales(a, t, n, row_scale, lane);
      if (!warp_wait(&accfull[b], (i >> 1) & 1, ctl, kErrWaitEpilogue)) break;
      tc_fence_after();
      const uint32_t acc = tmem + lane_addr + (b ? a.acc1 : 0);
      if (a.split > 1) {
        for (int col = 16 * c; col < t.width; col += 32) {
          uint32_t v[16];
          tmem_ld16(acc + col, v);
          tmem_wait_ld16(v);
#pragma unroll
          for (int j = 0; j < 16; ++j) reinterpret_cast<int*>(gbase)[(col + j) * kPitch + 32 * q + lane] = static_cast<int>(v[j]);
        }
      } else {
        drain_tile<F16, SWIGLU>(a, t, acc, c, n, ch, row_scale, lane);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&drained[b]);
    }
  }

  Tile t{};
  ChannelScale ch[4];  // of the four channels whose sums this thread takes
  if (a.split > 1 && first < tiles) {
    t = tile_at<16>(a, tables, first);
#pragma unroll
    for (int i = 0; i < 4; ++i) ch[i] = channel_scale(a, t.group, t.pt * kRows + 4 * (threadIdx.x % (kRows / 4)) + i);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(a.tmem_cols) : "memory");
  }
  if (a.split > 1) {
    // one tile a cluster: every rank sums its share of the columns over the ranks (128 values of a column lie together)
    cluster_sync();
    if (first < tiles && !*ctl.abort) sum_ranks<F16, SWIGLU>(a, t, base, rank, scales, ch);
    cluster_sync();  // nobody leaves while its partial tile is being read
  }
  zero_rest<F16>(a, fit, SWIGLU ? a.n / 2 : a.n);
}

// ------------------------------------------------------------------ few rows, quantised in place
// A few float rows (decoded tokens) of a dense product, one tile a CTA: the CTA quantises its part of the rows itself, straight into
// the swizzled layout that the MMAs read, while the weights' first stages arrive. No kernel before it, and no trip of the codes
// through memory. Each CTA reads whole rows for their largest magnitudes (ranks that told each other theirs waited 6000 cycles
// for the signal, behind the weights), so this is for few values: a part of 512 a warp and time, four times.
// Roles: warp 0 loads weights, warp 1 issues the MMAs, warps 2-9 quantise, then drain.
constexpr int kFewRows = 16;
constexpr int kFewStep = kFewRows * kStepBytes;  // codes of all rows, a stage's part of K
constexpr int kFewPart = 32 * 16;                // values of a row that a warp takes at a time
constexpr int kFewHeld = 4;                      // of these a warp
constexpr uint32_t kFewStage = kRows * kStepBytes;
constexpr unsigned kErrWaitRanks = 0x715;

struct FewRows {
  const void* x;
  int64_t ldx, K;
  int vec;         // rows of x start on 16 bytes and hold whole units of them
  int parts;       // of a row
  Divide by_parts;
  uint32_t codes, sums;  // bytes from the stages' start to the rows' codes, and to the sums sent by the ranks
};

template <bool XF16, bool VEC>
struct Part {  // 16 values of a lane
  static constexpr int kUnits = XF16 ? 2 : 4;
  Unit<XF16, VEC> u[kUnits];
  __device__ __forceinline__ void load(const FewRows& f, int64_t row, int k0) {
    const uint8_t* x = static_cast<const uint8_t*>(f.x) + row * f.ldx * (XF16 ? 2 : 4);
#pragma unroll
    for (int i = 0; i < kUnits; ++i) u[i].load(x, k0 + i * Unit<XF16, VEC>::kValues, static_cast<int>(f.K));
  }
  __device__ __forceinline__ uint32_t amax() const {
    Largest<XF16> l;
#pragma unroll
    for (int i = 0; i < kUnits; ++i) u[i].largest(l);
    return l.bits();
  }
  __device__ __forceinline__ uint4 codes(const Scale& c, bool none) const {
    uint32_t w[4 + 2];
#pragma unroll
    for (int i = 0; i < kUnits; ++i) u[i].codes(c, w + i * (XF16 ? 2 : 1));
    return none ? make_uint4(0, 0, 0, 0) : make_uint4(w[0], w[1], w[2], w[3]);
  }
};

struct FewShared {
  uint64_t full[kMaxStages], empty[kMaxStages], ready, summed, accfull, done;
  uint32_t largest[kFewRows];             // magnitudes of the rows, as bits
  Scale scale[kEpilogueWarps][kFewRows];  // a copy a warp
  float row_scale[kEpilogueWarps][2 * kFewRows];  // a rank reads 16 from its first row on
  uint32_t tmem_slot;
  int abort_flag;
};

// The eight warps 2-9: the rows' scales, and the codes of the steps k0 .. k1 - 1.
template <bool XF16, bool VEC>
__device__ __forceinline__ void quantise_rows(const Args& a, const FewRows& f, int k0, int k1, FewShared& sh, uint32_t codes) {
  const int warp = (threadIdx.x >> 5) - 2, lane = threadIdx.x & 31;
  const int parts = f.parts, items = a.rows * parts;
  Part<XF16, VEC> held[kFewHeld];
#pragma unroll
  for (int i = 0; i < kFewHeld; ++i) {
    const int item = warp + 8 * i, row = item / f.by_parts;
    if (item < items) held[i].load(f, row, (item - row * parts) * kFewPart + lane * 16);
  }
#pragma unroll
  for (int i = 0; i < kFewHeld; ++i) {
    const int item = warp + 8 * i;
    if (item >= items) break;
    const uint32_t m = __reduce_max_sync(~0u, held[i].amax());
    if (lane == 0) atomicMax(&sh.largest[item / f.by_parts], m);
  }
  __syncwarp();
  asm volatile("bar.sync 1, 256;" ::: "memory");  // these eight warps, none of which leaves before
  if (lane < kFewRows) {
    Scale c;
    bool none;
    sh.row_scale[warp][lane] = row_scale_of<XF16>(sh.largest[lane], &c, &none);
    sh.row_scale[warp][kFewRows + lane] = 0.0f;
    if (none) c.up = 0.0f;  // marks rows whose codes are 0
    sh.scale[warp][lane] = c;
  }
  __syncwarp();
#pragma unroll
  for (int i = 0; i < kFewHeld; ++i) {
    const int item = warp + 8 * i, row = item / f.by_parts, k = (item - row * parts) * kFewPart + lane * 16 - k0 * kStepBytes;
    if (item >= items) break;
    if (k < 0 || k >= (k1 - k0) * kStepBytes) continue;
    const Scale c = sh.scale[warp][row];
    const uint4 w = held[i].codes(c, c.up == 0.0f);
    const uint32_t dst = codes + (k / kStepBytes) * kFewStep + row * kStepBytes + ((((k / 16) & 7) ^ (row & 7)) << 4);
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(w.x), "r"(w.y), "r"(w.z), "r"(w.w) : "memory");
  }
  fence_async_shared();
  __syncwarp();
}

// A split tile's sums: every rank owns `share` of the rows. The warp that read 32 channels of this rank's sums sends each owner
// its part, in the owner's order, waits for the parts of its own rows and adds them up. No rank waits for another to read.
template <bool F16, bool SWIGLU>
__device__ __forceinline__ void exchange_sums(const Args& a, const Tile& t, const uint32_t (&v)[16], uint32_t sums, int rank, int q, int n,
                                              const ChannelScale& ch, FewShared& sh, const float* row_scale, int lane, const Ctl& ctl) {
  const int share = (t.rows + a.split - 1) >> a.split_log;
  int owner = 0, at = 0;
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    if (j >= t.rows) break;
    if (at == share) {
      at = 0;
      ++owner;
    }
    st_cluster_u32(map_rank(sums + ((rank * share + at++) * kRows + 32 * q + lane) * 4, owner), v[j]);  // at [rank][row of the owner][channel]
  }
  const int owners = owner + 1;
  __syncwarp();
  if (lane < owners) arrive_at(&sh.summed, lane);
  if (rank >= owners) return;
  if (!warp_wait(&sh.summed, 0, ctl, kErrWaitRanks) || !__all_sync(~0u, acquire_cluster(&sh.summed, 0))) return;
  const int mine = min(share, t.rows - rank * share);
  uint32_t sum[16] = {};
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    if (j >= mine) break;
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      uint32_t x = 0;
      if (r < a.split) asm volatile("ld.shared.u32 %0, [%1];" : "=r"(x) : "r"(sums + ((r * share + j) * kRows + 32 * q + lane) * 4) : "memory");
      sum[j] += x;
    }
  }
  // this rank's rows, as a tile of their own (scales behind them are those of no row)
  store_chunk<F16, SWIGLU>(a, {0, t.pt, rank * share, mine, kFewRows}, sum, 0, n, ch, row_scale + rank * share, lane);
}

template <bool F16, bool SWIGLU, bool XF16>
__global__ void __launch_bounds__(kThreads, 1) int8_few_kernel(const __grid_constant__ CUtensorMap map_p, const Args a, const FewRows f) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ FewShared sh;
  const int warp = __shfl_sync(~0u, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int S = a.stages;
  const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
  const int rank = a.split > 1 ? static_cast<int>(cluster_rank()) : 0, pt = blockIdx.x >> a.split_log;
  const Tile t{0, pt, 0, a.rows, kFewRows};
  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&sh.full[s], 1);
      mbar_init(&sh.empty[s], 1);
    }
    mbar_init(&sh.ready, kEpilogueWarps);
    mbar_init(&sh.summed, 4 * a.split);
    mbar_init(&sh.accfull, 1);
    mbar_init(&sh.done, 1);
    sh.abort_flag = 0;
    fence_mbar_init();
  }
  if (threadIdx.x < kFewRows) sh.largest[threadIdx.x] = 0;
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem_slot)), "r"(32) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&sh.tmem_slot);
  const Ctl ctl{&sh.abort_flag, a.err};
  const int k0 = a.ksteps * rank >> a.split_log, k1 = a.ksteps * (rank + 1) >> a.split_log, steps = k1 - k0;
  const uint32_t codes = base + f.codes, sums = base + f.sums;
  bool waited = false;  // for the cluster's barrier
  // All ranks' barriers have to be there before the first signal, which comes from the draining warps.
  if (a.split > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");

  if (warp == 0) {
    if (lane == 0) {
      auto load = [&](int i, int s) {
        mbar_arrive_expect_tx(&sh.full[s], kRows * kStepBytes);
        tma_load_2d(base + s * kFewStage, &map_p, (k0 + i) * kStepBytes, pt * kRows, &sh.full[s]);
      };
      int i = 0, s = 0;
      uint32_t ph = 1;
      for (; i < steps; ++i) {
        if (!thread_wait(&sh.empty[s], ph, ctl, kErrWaitProducer)) break;
        load(i, s);
        if (++s == S) {
          s = 0;
          ph ^= 1;
        }
      }
      if (i < steps)
        for (int h = (i > S ? i - S : 0); h < i; ++h) drain_wait(&sh.full[h % S], (h / S) & 1, a.err, kErrDrain);
    }
    __syncwarp();
  } else if (warp == 1) {
    const uint64_t p_desc = umma_desc_sw128(base), q_desc = umma_desc_sw128(codes);
    const uint32_t i_desc = instruction_desc(kRows, kFewRows);
    bool ok = warp_spin(&sh.ready, 0, ctl, kErrWaitMma);
    int s = 0;
    uint32_t ph = 0;
    for (int i = 0; ok && i < steps; ++i) {
      if (!warp_spin(&sh.full[s], ph, ctl, kErrWaitMma)) {
        ok = false;
        break;
      }
      tc_fence_after();
      const int subs = a.ksubs - 4 * (k0 + i);
      const uint32_t p_off = static_cast<uint32_t>(s) * (kFewStage >> 4), q_off = static_cast<uint32_t>(i) * (kFewStep >> 4);
      if (elect_one()) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (j > 0 && j >= subs) break;
          mma_i8(tmem, p_desc + p_off + 2 * j, q_desc + q_off + 2 * j, i_desc, i > 0 || j > 0);
        }
        mma_commit(&sh.empty[s]);
      }
      __syncwarp();
      if (++s == S) {
        s = 0;
        ph ^= 1;
      }
    }
    if (ok && elect_one()) mma_commit(&sh.accfull);
    __syncwarp();
    if (elect_one()) mma_commit(&sh.done);
    __syncwarp();
    drain_wait(&sh.done, 0, a.err, kErrDrain);
  } else {
    const int q = warp & 3, c = (warp - 2) >> 2, n = pt * kRows + 32 * q + lane;
    if (f.vec) quantise_rows<XF16, true>(a, f, k0, k1, sh, codes);
    else quantise_rows<XF16, false>(a, f, k0, k1, sh, codes);
    if (lane == 0) mbar_arrive(&sh.ready);
    __syncwarp();
    if (c == 0) {
      ChannelScale ch = channel_scale(a, 0, n);
      const float* scale = sh.row_scale[warp - 2];
      ch.far = __any_sync(~0u, lane < kFewRows && scale[lane] >= kFarScale);
      if (warp_wait(&sh.accfull, 0, ctl, kErrWaitEpilogue)) {
        tc_fence_after();
        const uint32_t acc = tmem + (static_cast<uint32_t>(32 * q) << 16);
        if (a.split > 1) {
          uint32_t v[16];
          tmem_ld16(acc, v);
          tmem_wait_ld16(v);
          waited = true;
          asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
          exchange_sums<F16, SWIGLU>(a, t, v, sums, rank, q, n, ch, sh, scale, lane, ctl);
        } else {
          drain_tile<F16, SWIGLU>(a, t, acc, 0, n, ch, scale, lane);
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (a.split > 1 && !waited) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(32) : "memory");
  }
  // After a wait that ran out another rank may still send to this one: stay until the others have left, or are here too.
  if (a.split > 1 && *ctl.abort) cluster_sync();
}

// ------------------------------------------------------------------ pairs of CTAs
// For many rows: a cluster of two CTAs on 256 channels by up to 256 rows. Each holds 128 of the channels and half of the rows; the
// first one's MMAs (cta_group::2) read both halves from both shared memories, so that a CTA loads 256 rows a step instead of
// 384 for the same product. Each CTA keeps the sums of its own channels, two accumulators that it drains in turns, under the next
// tile's MMAs. The tiles of a last round that has too few for all pairs are cut into two or four.
// What bounds these products is the clock under the power limit (above), and in cycles the loads from L2, about 49 bytes a cycle and
// SM: a stage, 32 KB a CTA, takes 650 to 700 cycles of the 512 of its MMAs. Tiles of 512 rows (48 KB a stage, 1024 cycles, bound by the
// MMAs) need both accumulators at once, and lost in waiting for the drain what they won: 2048 x 14336 x 4096 86 to 91 us against 86,
// with swiglu 104 against 91. More, smaller copies a stage cost more than the bytes they save (28 cycles a copy; boxes of 64 rows 3 %).
// Signals between the two. Both CTAs' loads complete on the first one's `full`, which expects the bytes of both; the MMAs'
// completion goes to both. The second CTA's epilogue warps meet at its own `drained`, and its warp 1 passes that on with a release at
// cluster scope. What the first CTA waits for it acquires at cluster scope.
constexpr int kStages2 = 6;
constexpr uint32_t kPart2 = kRows * kStepBytes;  // a CTA's channels, or its rows
constexpr uint32_t kStage2 = 2 * kPart2;

__device__ __forceinline__ void mma2_i8(uint32_t d, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// The line of tiles of `pairs` pairs: whole ones, then the pieces of the rest.
struct Line {
  int whole, cut, end;
};
__device__ __forceinline__ Line line_of(int tiles, int pairs) {
  const int rest = tiles % pairs, cut = rest == 0 ? 1 : 4 * rest <= pairs ? 4 : 2 * rest <= pairs ? 2 : 1;
  return {tiles - rest, cut, tiles - rest + rest * cut};
}
__device__ __forceinline__ Tile tile2_at(const Args& a, const Tables& tables, const Line& l, int i) {
  const bool piece = i >= l.whole && l.cut > 1;
  Tile t = tile_at<32>(a, tables, piece ? l.whole + (i - l.whole) / l.cut : i);
  if (piece) {  // possibly an empty one
    const int at = (i - l.whole) % l.cut, rows = ((t.rows + l.cut - 1) / l.cut + 31) / 32 * 32;
    t.row0 += at * rows;
    t.rows = max(0, min(rows, t.rows - at * rows));
    t.width = (t.rows + 31) / 32 * 32;
  }
  return t;
}

template <bool F16, bool SWIGLU>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    int8_gemm2_kernel(const __grid_constant__ CUtensorMap map_p, const __grid_constant__ CUtensorMap map_q, const Args a) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t full[kStages2], empty[kStages2], accfull[2], drained[2], done;
  __shared__ float row_scale[kEpilogueWarps][kMaxT];
  __shared__ uint32_t tmem_slot, fills[2];  // stages that each CTA's loads were issued for (in the first CTA)
  __shared__ int abort_flag;
  const int warp = __shfl_sync(~0u, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
  const int rank = static_cast<int>(cluster_rank());
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages2; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&accfull[b], 1);
      mbar_init(&drained[b], kEpilogueWarps + (rank == 0));  // the first CTA's: and the second CTA
    }
    mbar_init(&done, 1);
    abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  const Tables tables = tables_at(smem_raw + (base - raw) + a.tables, a.groups);
  tc_fence_before();
  const bool fit = make_tables(a, tables);
  cluster_sync();  // both CTAs' barriers are there
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&tmem_slot);
  const Ctl ctl{&abort_flag, a.err};
  const int first = blockIdx.x >> 1, step = gridDim.x >> 1;
  const Line line = line_of(tables.tile_first[a.groups] * a.p_tiles, step);

  if (warp == 0) {
    int g = 0, s = 0;
    uint32_t ph = 0;
    bool ok = true, waited = false;
    for (int tile = first; ok && tile < line.end; tile += step) {
      const Tile t = tile2_at(a, tables, line, tile);
      if (!t.rows) continue;
      const int q_row = t.row0 + rank * (t.width / 2);
      const int p_row = t.group * a.n + (2 * t.pt + rank) * kRows;
      auto load_p = [&](int st, int ks) {
        if (rank == 0) mbar_arrive_expect_tx(&full[st], 2 * kStage2);
        tma2_load_2d(base + st * kStage2, &map_p, ks * kStepBytes, p_row, map_rank(smem_u32(&full[st]), 0));
      };
      // The weights' first stages do not depend on the kernel before this one; the activations do.
      int pre = 0;
      if (!waited) {
        waited = true;
        if (a.early) {
          pre = min(kStages2, a.ksteps);
          if (lane == 0)
            for (int i = 0; i < pre; ++i) load_p(i, i);
          __syncwarp();
        }
        asm volatile("griddepcontrol.wait;" ::: "memory");
      }
      for (int ks = 0; ks < a.ksteps; ++ks, ++g) {
        if (g >= pre) {
          if (!warp_spin(&empty[s], ph ^ 1, ctl, kErrWaitProducer)) {
            ok = false;
            break;
          }
          if (lane == 0) load_p(s, ks);
          __syncwarp();
        }
        if (lane == 0) tma2_load_2d(base + s * kStage2 + kPart2, &map_q, ks * kStepBytes, q_row, map_rank(smem_u32(&full[s]), 0));
        if (++s == kStages2) {
          s = 0;
          ph ^= 1;
        }
      }
    }
    if (!waited) asm volatile("griddepcontrol.wait;" ::: "memory");
    if (lane == 0) st_cluster_u32(map_rank(smem_u32(&fills[rank]), 0), g);
  } else if (warp == 1 && rank == 1) {
    // passes on that this CTA's accumulators have been read
    int i = 0;
    for (int tile = first; tile < line.end; tile += step) {
      if (!tile2_at(a, tables, line, tile).rows) continue;
      if (!warp_spin(&drained[i & 1], (i >> 1) & 1, ctl, kErrWaitMma)) break;
      if (lane == 0) arrive_at(&drained[i & 1], 0);
      __syncwarp();
      ++i;
    }
  } else if (warp == 1) {
    const uint64_t p_desc = umma_desc_sw128(base), q_desc = umma_desc_sw128(base + kPart2);
    int i = 0, s = 0;
    uint32_t ph = 0;
    bool ok = true;
    // both CTAs' loads, or both CTAs' drains
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      return warp_spin(bar, parity, ctl, kErrWaitMma) && __all_sync(~0u, acquire_cluster(bar, parity));
    };
    for (int tile = first; ok && tile < line.end; tile += step) {
      const Tile t = tile2_at(a, tables, line, tile);
      if (!t.rows) continue;
      const uint32_t i_desc = instruction_desc(2 * kRows, t.width);
      if (i >= 2 && !wait(&drained[i & 1], ((i - 2) >> 1) & 1)) break;
      tc_fence_after();
      const uint32_t d = tmem + ((i & 1) ? kMaxT : 0);
      for (int ks = 0; ks < a.ksteps; ++ks) {
        if (!wait(&full[s], ph)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const int subs = a.ksubs - 4 * ks;
        const uint32_t off = static_cast<uint32_t>(s) * (kStage2 >> 4);
        if (elect_one()) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (j > 0 && j >= subs) break;
            mma2_i8(d, p_desc + off + 2 * j, q_desc + off + 2 * j, i_desc, ks > 0 || j > 0);
          }
          mma2_commit(&empty[s]);
        }
        __syncwarp();
        if (++s == kStages2) {
          s = 0;
          ph ^= 1;
        }
      }
      if (ok && elect_one()) mma2_commit(&accfull[i & 1]);
      __syncwarp();
      ++i;
    }
    if (elect_one()) mma2_commit(&done);
    __syncwarp();
    drain_wait(&done, 0, a.err, kErrDrain);
  } else {
    const int q = warp & 3, c = (warp - 2) >> 2;
    const uint32_t lane_addr = static_cast<uint32_t>(32 * q) << 16;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    int i = 0;
    for (int tile = first; tile < line.end; tile += step) {
      const Tile t = tile2_at(a, tables, line, tile);
      if (!t.rows) continue;
      const int b = i & 1, n = (2 * t.pt + rank) * kRows + 32 * q + lane;
      const ChannelScale ch = prepare_scales(a, t, n, row_scale[warp - 2], lane);
      if (!warp_wait(&accfull[b], (i >> 1) & 1, ctl, kErrWaitEpilogue)) break;
      tc_fence_after();
      drain_tile<F16, SWIGLU>(a, t, tmem + lane_addr + (b ? kMaxT : 0), c, n, ch, row_scale[warp - 2], lane);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&drained[b]);
      ++i;
    }
  }

  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && abort_flag) st_cluster_u32(map_rank(smem_u32(&abort_flag), rank ^ 1), 1);
  cluster_sync();  // neither CTA's memory goes while the other may read or signal it
  if (*ctl.abort) {
    // A wait ran out in one of them: tensor copies may be under way. A stage's last fill is awaited (its phase may lack the
    // other CTA's part; then the wait ends by its limit, long after the copies).
    if (rank == 0 && threadIdx.x == 0) {
      const int g = static_cast<int>(max(fills[0], fills[1]));
      for (int s = 0; s < kStages2; ++s) {
        const int n = (g - s + kStages2 - 1) / kStages2;
        if (n > 0) drain_wait(&full[s], (n - 1) & 1, a.err, kErrDrain);
      }
    }
    cluster_sync();
  }
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
  zero_rest<F16>(a, fit, SWIGLU ? a.n / 2 : a.n);
}

// ------------------------------------------------------------------ host side
// Tiles that a call has at the most.
int64_t most_tiles(const Int8Matmul& p, int64_t tmax, int64_t p_rows) {
  const int64_t hit = !p.offsets ? 1 : p.groups < p.rows ? p.groups : p.rows;
  const int64_t along = !p.offsets ? ceil_div(p.rows, tmax) : hit + (p.rows - hit) / tmax;
  return along * ceil_div(p.N, p_rows);
}

struct Launch {
  CUtensorMap p, q;
  int grid, split, steps;
  bool pairs, early;
  size_t smem;
};

template <auto Kernel>
cudaError_t launch_kernel(const Launch& l, const Args& a, cudaStream_t s) {
  cudaError_t e = allow_smem<Kernel>(static_cast<int>(l.smem));
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(l.grid);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = l.smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (l.early) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (!l.pairs && l.split > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = l.split;
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, Kernel, l.p, l.q, a);
}

template <bool F16, bool SWIGLU>
cudaError_t launch(const Launch& l, const Args& a, cudaStream_t s) {
  if (l.pairs) return launch_kernel<int8_gemm2_kernel<F16, SWIGLU>>(l, a, s);
  return l.steps == 2 ? launch_kernel<int8_gemm_kernel<F16, SWIGLU, 2>>(l, a, s) : launch_kernel<int8_gemm_kernel<F16, SWIGLU, 1>>(l, a, s);
}

// Shared memory, stages, split of K and grid of single CTAs.
void single_shape(const Int8Matmul& p, int64_t tiles, int sms, Args& a, Launch& l) {
  // K is split while the CTAs find an SM each, over 8 only for narrow tiles. Measured (us, split 1 / 2 / 4 / 8): 16 x 4096 x 14336
  // 35.4 / 21.9 / 16.1 / 15.7, 16 x 14336 x 4096 (112 tiles) 14.8 / 15.9 / 21.5, 128 x 4096 x 4096 16.1 / 14.5 / 12.0, 333 x 1003 x 4100 in
  // tiles of 128 rows - / 15.1 / 11.2 / 13.2, of 256 - / 17.9 / 13.9 / 20.4.
  const int most = a.tmax <= 32 ? 8 : 4;
  a.split = 1;
  while (a.split < most && tiles * a.split * 2 <= sms && a.ksteps >= 4 * a.split) a.split *= 2, ++a.split_log;
  const uint32_t tables = tables_bytes(p.groups);
  const uint32_t scales = static_cast<uint32_t>(kEpilogueWarps) * ((a.tmax + 31) & ~31) * 4;
  const int budget = kSmemMost - 1024 - 1024 - static_cast<int>(tables + scales);  // what is declared; up to the first 1024-byte boundary
  const uint32_t step = static_cast<uint32_t>(kRows + a.tmax) * kStepBytes;
  l.steps = 8 * step <= static_cast<uint32_t>(budget) ? 2 : 1;  // (figures at the kernel)
  a.ksteps = (a.ksteps + l.steps - 1) / l.steps;
  a.stage = step * l.steps;
  const int steps = static_cast<int>(ceil_div(a.ksteps, a.split));
  const bool one_tile = a.split > 1 || tiles <= sms;
  int stages = budget / static_cast<int>(a.stage);
  const int most_stages = l.steps == 2 ? 4 : kMaxStages;
  if (stages > most_stages) stages = most_stages;
  if (one_tile && stages > steps) stages = steps;
  a.stages = stages;
  size_t smem = static_cast<size_t>(stages) * a.stage;
  const size_t partial = static_cast<size_t>(a.tmax) * kPitch * 4;
  if (a.split > 1 && smem < partial) smem = partial;
  a.tables = static_cast<uint32_t>(smem);
  a.scales = a.tables + tables;
  smem += tables + scales + 1024;
  a.acc1 = one_tile ? 0 : a.tmax;
  a.tmem_cols = 32;
  while (a.tmem_cols < a.acc1 + a.tmax) a.tmem_cols *= 2;
  // CTAs that share an SM share its 512 columns: ask for enough shared memory that no more fit than those feed.
  const size_t least = static_cast<size_t>(227 * 1024) / (512 / a.tmem_cols + 1) + 1024;
  if (smem < least) smem = least;
  l.smem = smem;
  l.split = a.split;
  l.grid = static_cast<int>(a.split > 1 ? tiles * a.split : (tiles < sms ? tiles : sms));
}

// Split of K and stages of the kernel for few float rows; false where it does not take the call: one tile a CTA, rows that its warps
// hold at once.
bool few_shape(const Int8Matmul& p, int sms, Args& a, FewRows& f, Launch& l) {
  if (p.offsets || p.rows > kFewRows || p.rows * ceil_div(p.K, kFewPart) > kEpilogueWarps * kFewHeld) return false;
  const int64_t tiles = ceil_div(p.N, kRows);
  if (tiles > sms) return false;
  a.split = 1;
  while (a.split < 8 && tiles * a.split * 2 <= sms && a.ksteps >= 4 * a.split) a.split *= 2, ++a.split_log;
  const int64_t steps = ceil_div(a.ksteps, a.split), rows = steps * kFewStep;
  // a rank's sums: [ranks][its share of the rows][channels]
  const int64_t sums = a.split > 1 ? a.split * ceil_div(p.rows, a.split) * kRows * 4 : 0;
  int64_t stages = (kSmemBudget - 1024 - rows - sums) / kFewStage;
  if (stages > kMaxStages) stages = kMaxStages;
  if (stages > steps) stages = steps;
  if (stages < steps && stages < 6) return false;  // long rows: their codes leave too little for the weights
  f.parts = static_cast<int>(ceil_div(p.K, kFewPart));
  f.by_parts = divide_by(f.parts);
  a.stages = static_cast<int>(stages);
  a.p_tiles = static_cast<int>(tiles);
  f.codes = static_cast<uint32_t>(stages) * kFewStage;
  f.sums = f.codes + static_cast<uint32_t>(rows);
  l.smem = f.sums + static_cast<size_t>(sums) + 1024;
  l.split = a.split;
  l.grid = static_cast<int>(tiles * a.split);
  return true;
}

template <bool F16, bool SWIGLU, bool XF16>
cudaError_t launch_few(const Launch& l, const Args& a, const FewRows& f, cudaStream_t s) {
  cudaError_t e = allow_smem<int8_few_kernel<F16, SWIGLU, XF16>>(kSmemBudget);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(l.grid);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = l.smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = l.split;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = l.split > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, int8_few_kernel<F16, SWIGLU, XF16>, l.p, a, f);
}

Args arguments(const Int8Matmul& p) {
  Args a{};
  a.n = static_cast<int>(p.N);
  a.groups = p.groups;
  a.rows = static_cast<int>(p.rows);
  a.ksubs = static_cast<int>(ceil_div(p.K, 32));
  a.ksteps = (a.ksubs + 3) / 4;
  a.act = p.act;
  a.has_limit = p.has_limit;
  a.zero_rest = p.zero_rest;
  a.bias_f16 = p.bias_f16;
  a.alpha = p.alpha;
  a.beta = p.beta;
  a.limit = p.limit;
  a.offsets = p.offsets;
  a.a_scales = p.a_scales;
  a.b_scales = p.b_scales;
  a.bias = p.bias;
  a.y = p.y;
  a.ldy = p.ldy;
  a.err = p.err;
  return a;
}

// Rows of a tile of single CTAs at the most: all of a dense product with few of them, else 256, or 128 where one round holds the
// narrower ones too (512 x 4096 x 4096: 16.9 us against 19.4); twice a group's mean, so that most groups take one.
int single_rows(const Int8Matmul& p, int sms) {
  const int64_t mean = ceil_div(p.rows, p.groups), want = p.offsets ? 2 * mean + 8 : mean;
  int64_t t = align_up(want < p.rows ? want : p.rows, 16);
  if (p.offsets) return static_cast<int>(t > kMaxT ? kMaxT : t > 96 ? align_up(t, 64) : t);
  if (t > 128 && most_tiles(p, 128, kRows) <= sms) t = 128;
  return static_cast<int>(t > kMaxT ? kMaxT : t);
}

// Pairs take what fills most of the SMs with tiles of 128 channels by 256 rows, but for short rows only what fills them several
// times. Measured (us, single CTAs / pairs; tiles as counted here): 512 x 4096 x 4096 (64) 14.7 / 17.2, 512 x 6144 x 2048 (96) 13.1 / 13.3, 256 x
// 14336 x 4096 (112) 21.0 / 20.2, 1024 x 4096 x 4096 (128) 18.9 / 18.5, 1500 tokens by 4 of 16 experts of 2048 x 2048 (624) 43.0 / 40.8. Short
// rows: 512 x 8192 x 512 (128) 8.1 / 9.1, 2000 x 4096 x 1024 (256) 14.1 / 14.3, 2560 x 5120 x 768 (400) 17.7 / 17.7, 2560 x 6400 x 1024 (500)
// 23.4 / 21.4. Around the borders, 104 and 370 tiles on 148 SMs, the last round decides and either wins by up to 5 %: 1024 x 3328 x 2048 (104)
// 12.6 / 13.1, 900 x 3400 x 1100 (108) 12.2 / 11.5, 1000 tokens by 4 of 16 experts of 1500 x 768 (372) 23.3 / 24.4, 2000 x 6000 x 1024 (376) 19.0 /
// 18.6, 2304 x 5504 x 768 (387) 17.2 / 17.6.
bool pairs_pay(const Int8Matmul& p, int tmax, int sms) {
  const int64_t tiles = most_tiles(p, kMaxT, kRows);
  return tmax >= 128 && 10 * tiles >= (p.K > 1024 ? 7 : 25) * sms;
}

}  // namespace

bool int8_few_rows(const Int8Matmul& p) {
  Args a = arguments(p);
  FewRows f{};
  Launch l{};
  return few_shape(p, device_sm_count(), a, f, l);
}

cudaError_t launch_int8_few(const Int8Matmul& p, const void* x, bool x_f16, int64_t ldx, cudaStream_t s) {
  Args a = arguments(p);
  FewRows f{x, ldx, p.K, reinterpret_cast<uintptr_t>(x) % 16 == 0 && ldx * (x_f16 ? 2 : 4) % 16 == 0 && p.K % (x_f16 ? 8 : 4) == 0, 0, {}, 0, 0};
  Launch l{};
  if (!few_shape(p, device_sm_count(), a, f, l) || !encode_tensor_map_2d(&l.p, 0, p.b, p.K, p.N, p.ldb, kStepBytes, kRows, true)) return cudaErrorInvalidValue;
  const bool swiglu = p.act == XRGPU_ACT_SWIGLU;
  if (p.f16) {
    if (swiglu) return x_f16 ? launch_few<true, true, true>(l, a, f, s) : launch_few<true, true, false>(l, a, f, s);
    return x_f16 ? launch_few<true, false, true>(l, a, f, s) : launch_few<true, false, false>(l, a, f, s);
  }
  if (swiglu) return x_f16 ? launch_few<false, true, true>(l, a, f, s) : launch_few<false, true, false>(l, a, f, s);
  return x_f16 ? launch_few<false, false, true>(l, a, f, s) : launch_few<false, false, false>(l, a, f, s);
}

cudaError_t launch_int8_matmul(const Int8Matmul& p, bool early, cudaStream_t s) {
  const int sms = device_sm_count();
  Args a = arguments(p);
  a.early = early;

  Launch l{};
  l.early = early;
  a.tmax = single_rows(p, sms);
  l.pairs = pairs_pay(p, a.tmax, sms);
  if (l.pairs) a.tmax = kMaxT;
  a.by_tmax = divide_by(a.tmax);
  const int channels = l.pairs ? 2 * kRows : kRows;
  const int64_t tiles = most_tiles(p, a.tmax, channels);
  if (tiles > INT_MAX / 16) return cudaErrorInvalidValue;
  a.p_tiles = static_cast<int>(ceil_div(p.N, channels));
  a.by_p = divide_by(a.p_tiles);
  if (l.pairs) {
    a.box = kRows;  // one copy a stage, of more rows than a narrow tile needs: a copy takes 28 cycles of its own (64 rows: 89.7 us, 128: 86.8)
    a.split = 1;
    a.stages = kStages2;
    a.tables = kStages2 * kStage2;
    l.smem = a.tables + tables_bytes(p.groups) + 1024;
    l.grid = sms / 2 * 2;
  } else {
    // Rows of one copy: all of a dense tile; of a ragged one, whose last copy may reach into the next group's rows, large ones
    // too (16 rows a copy: 39 cycles each, 620 a stage of 256 rows).
    a.box = !p.offsets ? a.tmax : a.tmax % 64 == 0 ? 64 : 16;
    a.box_log = !p.offsets ? 30 : a.tmax % 64 == 0 ? 6 : 4;
    single_shape(p, tiles, sms, a, l);
  }
  if (!encode_tensor_map_2d(&l.p, 0, p.b, p.K, static_cast<uint64_t>(p.groups) * p.N, p.ldb, kStepBytes, kRows, true) ||
      !encode_tensor_map_2d(&l.q, 0, p.a, p.K, p.rows, p.lda, kStepBytes, a.box, true))
    return cudaErrorInvalidValue;
  if (p.f16) return p.act == XRGPU_ACT_SWIGLU ? launch<true, true>(l, a, s) : launch<true, false>(l, a, s);
  return p.act == XRGPU_ACT_SWIGLU ? launch<false, true>(l, a, s) : launch<false, false>(l, a, s);
}

}  // namespace xrgpu
