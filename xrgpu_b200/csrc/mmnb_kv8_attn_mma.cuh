// Attention over the paged 8-bit cache for few rows (and for float32 rows): one pass over the cache, its
// codes fed to mma.sync as exact float16 numbers, split over the whole GPU along the tokens.
//
//   o[row, h] = sum_j softmax_j(scale * q . k_j) v_j,   k_j = code * k_scale[page], v_j = code * v_scale[page]
//
// Products. A segment is (sequence, key/value head, tile of 8 NT rows); row r of a segment is query token
// r / G and query head r % G of the group of G. Scores are computed transposed, S^T = K Q^T (16 tokens x 8 rows an
// MMA), so that few rows fill the 8 columns and the cache is the 16-row operand; then O^T += V^T P^T. Codes become
// float16 without arithmetic: for float16 rows an int8 code c is taken as the subnormal (c + 128) 2^-24 (exact in
// the MMA), the 128s are taken out by the accumulator's first value: -128 2^-24 sum(q) for the scores, and one
// more MMA with a constant operand, -128 2^-24 sum(p), for the values. e4m3 codes are float16 numbers by
// one conversion. Of float32 rounding, taking out the 128s leaves less than 2^-13 of a value's code. Scales multiply the
// float32 results: the scores of a page by k_scale, each page's O^T by v_scale as it is added to the running one, so pages
// of very different scales lose nothing against one another.
// Weights: 2^7 exp2(x - m) with m the largest score when it was last raised; m is raised only when a score exceeds it by 8,
// so that most steps need one vote instead of a reduction. Weights then lie below 2^15, inside float16, with steps of 2^-24
// far below the largest one. P is rounded to float16 (2^-12 relative, once, like the result); sums are float32, of the
// weights before that rounding. Float32 rows take q and P as pairs of float16 numbers and signed codes: the second one of P
// holds 2^11 times the rest, and its products are summed first and scaled back, so that a weight has 2^-24 of itself, or of
// the largest weight 2^-43 (as the rest itself it lost all bits of weights below 2^-25, of which a long sequence has many).
//
// Order in memory. A step is 32 tokens of keys and values, copied by a warp with 16-byte cp.async into its own ring
// of two or three buffers. 16-byte chunk c of row r lies at c ^ f(r), f(r) = (r & 7) ^ 4 (r & 1) for 128-byte rows (two
// 64-byte rows share a line, see chunk_at): copies and both operand reads touch all banks once.
//
// Balance. The steps of all segments form one sequence; every CTA takes an equal run of it, found from the
// lengths on the device. A segment that lies inside one CTA's run is finished there, one that is cut leaves
// partial results (m, l, O) in the workspace, which combine_kernel joins in the order of the CTAs. Where few short
// segments leave most SMs idle, a cluster of up to 8 CTAs shares each segment instead and joins it through shared
// memory: one launch (one token of one sequence of 2048: 16 -> 10 us).
//
// Bound by the cache's stream, then by the instructions that widen its codes: one token of each of 32 ragged sequences (64 heads on 8
// of 128, int8, 584 MB) 115 us, 5.1 TB/s; 64 sequences of 8192 (32 heads on 8) 190 us, 5.7 TB/s, e4m3 the same, with float32
// rows 232 us (every product twice).
#pragma once

#include <cstdint>

#include "mmnb_kv8.cuh"
#include "mmnb_tcgen05.cuh"
#include "mmnb_kv8_attn.h"

namespace xrgpu {
namespace {

constexpr int kStep = 32;    // tokens a warp takes at a time
constexpr float kRaise = 8.0f;
constexpr float kLift = 7.0f, kDrop = 0.0078125f;  // weights are held times 2^7; 2^-7
constexpr float kRest = 2048.0f;                   // the second half of a weight: 2^11 times what the first one leaves
constexpr float kLog2e = 1.4426950408889634f;

// ------------------------------------------------------------------ small pieces
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unpack_half2(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }
// Two e4m3 codes (low 16 bits) to float16x2.
__device__ __forceinline__ uint32_t e4m3x2_half2(uint32_t v) {
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint32_t e4m3x2_half2_high(uint32_t v) {
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, hi;\n\t}" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint4 lds_v4(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ uint2 lds_v2(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
  return v;
}

// Byte offset of 16-byte chunk c of row r in a tile of D-byte rows.
template <int D>
__device__ __forceinline__ uint32_t chunk_at(int r, int c) {
  if (D == 128) return r * 128 + ((c ^ ((r & 7) ^ ((r & 1) << 2))) << 4);
  return (r >> 1) * 128 + (((((r & 1) << 2) | c) ^ (((r >> 1) & 3) << 1)) << 4);
}

// Four codes of one row (consecutive along D) to two float16x2 registers: int8 pairs are (0, 2), (1, 3), e4m3 pairs
// (0, 1), (2, 3). RAW: int8 codes stay subnormals (c + 128) 2^-24.
template <bool E4M3, bool RAW>
__device__ __forceinline__ void row_pairs(uint32_t w, uint32_t& a, uint32_t& b) {
  if (E4M3) {
    a = e4m3x2_half2(w);
    b = e4m3x2_half2_high(w);
  } else {
    w ^= 0x80808080u;
    a = w & 0x00ff00ffu;
    b = (w >> 8) & 0x00ff00ffu;
    if (!RAW) {
      a = hsub2_u32(a | 0x64006400u, 0x64806480u);
      b = hsub2_u32(b | 0x64006400u, 0x64806480u);
    }
  }
}

// Four codes of each of two tokens' rows to float16x2 registers (token 0, token 1) for each of the four dims.
template <bool E4M3, bool RAW>
__device__ __forceinline__ void token_pairs(uint32_t w0, uint32_t w1, uint32_t (&d)[4]) {
  const uint32_t x = prmt(w0, w1, 0x5140u), y = prmt(w0, w1, 0x7362u);  // bytes t0 d0, t1 d0, t0 d1, t1 d1; d2, d3
  if (E4M3) {
    d[0] = e4m3x2_half2(x);
    d[1] = e4m3x2_half2_high(x);
    d[2] = e4m3x2_half2(y);
    d[3] = e4m3x2_half2_high(y);
  } else {
    const uint32_t xs = x ^ 0x80808080u, ys = y ^ 0x80808080u;
    const uint32_t fill = RAW ? 0u : 0x64646464u;
    d[0] = prmt(xs, fill, 0x4140u);
    d[1] = prmt(xs, fill, 0x4342u);
    d[2] = prmt(ys, fill, 0x4140u);
    d[3] = prmt(ys, fill, 0x4342u);
    if (!RAW) {
#pragma unroll
      for (int i = 0; i < 4; ++i) d[i] = hsub2_u32(d[i], 0x64806480u);
    }
  }
}

// ------------------------------------------------------------------ work: segments and steps
struct SeqWork {
  SeqRows r;
  int tiles, steps, first;  // row tiles, steps of each, first step (32 tokens) that any row sees
};

__device__ __forceinline__ SeqWork seq_work(const Kv8& p, int b, int rows_per_tile) {
  SeqWork w;
  w.r = seq_rows(p, b, true);
  const int G = p.hq / p.hkv;
  w.tiles = static_cast<int64_t>(w.r.n) * G > p.few_rows ? 0 : (w.r.n * G + rows_per_tile - 1) / rows_per_tile;
  w.first = window_from(p, w.r.len - w.r.n) / kStep;
  w.steps = max(1, (w.r.len + kStep - 1) / kStep - w.first);
  return w;
}
__device__ __forceinline__ int64_t seq_total(const Kv8& p, const SeqWork& w) {
  return static_cast<int64_t>(w.tiles) * w.steps * p.hkv;
}

struct Workspace {
  int64_t* start;  // [seqs + 1] first step of each sequence; the total
  float* part;     // [grid][2] partial results: O [rows][D], m [rows], l [rows]
};
__host__ __device__ inline int64_t part_floats(int rows, int D) { return static_cast<int64_t>(rows) * (D + 2); }
__host__ __device__ inline int64_t starts_bytes(int seqs) { return (static_cast<int64_t>(seqs) + 1) * 8 / 256 * 256 + 256; }

// Steps of a CTA's run: an equal share, one a warp at least.
__device__ __forceinline__ int64_t run_length(int64_t total, int grid, int warps) {
  const int64_t q = (total + grid - 1) / grid;
  return q < warps ? warps : q;
}

// ------------------------------------------------------------------ main kernel
template <bool E4M3, int D, int NT, bool F32, bool CL = false>
struct Traits {
  static constexpr int kRows = 8 * NT;
  // One tile of rows leaves registers for 12 warps an SM, whose rings then hold two steps: two CTAs of 6, so that one
  // streams while the other is between segments; 12 together in a cluster. More rows: 8 warps with three steps.
  static constexpr int kWarps = NT == 1 ? (CL ? 12 : 6) : 8, kThreads = kWarps * 32, kStages = NT == 1 ? 2 : 3;
  static constexpr int kCtas = NT == 1 && !CL ? 2 : 1;  // an SM
  static constexpr int kK = D / 16;                   // k steps of the scores
  static constexpr int kMt = D / 16;                  // 16-dim tiles of the output
  static constexpr int kTile = kStep * D;             // bytes of a step's keys (or values)
  static constexpr int kMeta = 32;                    // k_scale[2], v_scale[2], ok[2]
  static constexpr int kStage = 2 * kTile + kMeta;
  static constexpr int kRing = kStages * kStage;
  static constexpr int kQ = NT * kK * 32 * 8 * (F32 ? 2 : 1);
  static constexpr bool kRaw = !E4M3 && !F32;
  static constexpr int kMerge = kRows * D * 4;        // a warp's O in shared memory, over its ring
  static constexpr int kWarpBytes = kRing > kMerge ? kRing : kMerge;
  static constexpr int kJoin = CL ? kRows * (D + 2) * 4 : 0;  // the CTA's (O, m, l), read by its cluster
  static constexpr int kSmem = kWarps * kWarpBytes + kQ + kRows * 16 + kWarps * kRows * 8 + 64 + kJoin;
};

template <bool E4M3, int D, int NT, bool F32, bool CL>
__global__ void __launch_bounds__(Traits<E4M3, D, NT, F32, CL>::kThreads, Traits<E4M3, D, NT, F32, CL>::kCtas) attn_mma_kernel(const Kv8 p, Workspace ws, int split) {
  using C = Traits<E4M3, D, NT, F32, CL>;
  constexpr int kWarps = C::kWarps, kThreads = C::kThreads, kStages = C::kStages;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int64_t scan[kWarps + 1];
  __shared__ int64_t found_at;
  __shared__ int found_b;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, c = lane & 3;
  const int G = p.hq / p.hkv, R = C::kRows;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  const uint32_t ring = smem_u32(smem) + warp * C::kWarpBytes;
  uint8_t* ring_ptr = smem + warp * C::kWarpBytes;
  uint32_t* qfrag = reinterpret_cast<uint32_t*>(smem + kWarps * C::kWarpBytes);
  float* row_fac = reinterpret_cast<float*>(smem + kWarps * C::kWarpBytes + C::kQ);  // [R] score factor
  float* row_cor = row_fac + R;                                                      // [R] -128 2^-24 sum q
  int* row_hi = reinterpret_cast<int*>(row_cor + R);                                 // [R] first token not seen
  int* row_lo = row_hi + R;                                                          // [R] first token seen
  float* warp_m = reinterpret_cast<float*>(row_lo + R);                              // [kWarps][R]
  float* warp_l = warp_m + kWarps * R;
  float* join = reinterpret_cast<float*>(smem + C::kSmem - C::kJoin);                // [R][D], [R] m, [R] l

  // ---- all steps, this CTA's run of them, and the sequence it starts in (kThreads sequences at a time; a second pass
  // finds the start among more)
  auto prefix = [&](int64_t v, int64_t* all) {  // exclusive prefix sum over the threads, and the sum
    int64_t sum = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t o = __shfl_up_sync(~0u, sum, d);
      if (lane >= d) sum += o;
    }
    if (lane == 31) scan[warp] = sum;
    __syncthreads();
    int64_t before = 0, total = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) before += scan[w];
      total += scan[w];
    }
    *all = total;
    return before + sum - v;
  };
  int64_t begin = 0, end = 0;
  int rank = 0;
  if (CL) {
    // cluster `slot` takes a (row tile, head): the slot-th of the tiles of all sequences in order
    rank = static_cast<int>(cluster_rank());
    const int slot = blockIdx.x / split / p.hkv;
    int before = 0;
    if (tid == 0) found_b = -1;
    __syncthreads();
    for (int b0 = 0; b0 < p.seqs; b0 += kThreads) {
      const int b = b0 + tid;
      const int tiles = b < p.seqs ? seq_work(p, b, R).tiles : 0;
      int64_t all;
      const int at = before + static_cast<int>(prefix(tiles, &all));
      if (slot >= at && slot < at + tiles) {
        found_b = b;
        found_at = slot - at;
      }
      before += static_cast<int>(all);
      __syncthreads();
    }
    if (p.zero_rest && blockIdx.x == 0) {  // few rows here: a thread looks for each row's sequence
      for (int row = tid; row < p.tokens; row += kThreads) {
        bool owned = false;
        for (int b = 0; b < p.seqs && !owned; ++b) {
          const SeqRows r = seq_rows(p, b, true);
          owned = row >= r.row0 && row < r.row0 + r.n;
        }
        if (!owned)
          for (int d = 0; d < p.hq * D; ++d) {
            if (F32) static_cast<float*>(p.o)[row * p.os + d] = 0.0f;
            else static_cast<__half*>(p.o)[row * p.os + d] = __half(0.0f);
          }
      }
    }
    if (found_b >= 0) {
      const SeqWork w = seq_work(p, found_b, R);
      const int64_t seg_at = (static_cast<int64_t>(blockIdx.x / split % p.hkv) * w.tiles + found_at) * w.steps;
      begin = seg_at + static_cast<int64_t>(w.steps) * rank / split;
      end = seg_at + static_cast<int64_t>(w.steps) * (rank + 1) / split;
      for (int e = tid; e < R * (D + 2); e += kThreads) join[e] = e >= R * D && e < R * D + R ? -INFINITY : 0.0f;  // of a rank without steps
    }
  } else {
  int64_t total = 0, mine_v = 0, mine_at = 0;
  for (int b0 = 0; b0 < p.seqs; b0 += kThreads) {
    const int b = b0 + tid;
    int64_t all;
    mine_v = b < p.seqs ? seq_total(p, seq_work(p, b, R)) : 0;
    mine_at = total + prefix(mine_v, &all);
    if (blockIdx.x == 0 && b < p.seqs) ws.start[b] = mine_at;
    total += all;
    __syncthreads();
  }
  if (blockIdx.x == 0 && tid == 0) ws.start[p.seqs] = total;
  const int64_t run = run_length(total, gridDim.x, kWarps);
  begin = run * blockIdx.x;
  end = begin + run < total ? begin + run : total;
  if (begin >= end) return;
  if (p.seqs <= kThreads) {
    if (mine_v > 0 && begin >= mine_at && begin < mine_at + mine_v) {
      found_b = tid;
      found_at = mine_at;
    }
    __syncthreads();
  } else {
    int64_t before = 0;
    for (int b0 = 0; b0 < p.seqs; b0 += kThreads) {
      const int b = b0 + tid;
      int64_t all;
      const int64_t v = b < p.seqs ? seq_total(p, seq_work(p, b, R)) : 0, at = before + prefix(v, &all);
      if (v > 0 && begin >= at && begin < at + v) {
        found_b = b;
        found_at = at;
      }
      before += all;
      __syncthreads();
      if (before > begin) break;
    }
  }
  }
  __syncthreads();
  int b = found_b;
  int64_t seq_at = CL ? 0 : found_at;
  SeqWork w = b < 0 ? SeqWork{} : seq_work(p, b, R);

  for (int64_t at = begin; at < end;) {
    while (at >= seq_at + seq_total(p, w)) {  // on to the next sequence that has rows
      seq_at += seq_total(p, w);
      w = seq_work(p, ++b, R);
    }
    const int seg = static_cast<int>((at - seq_at) / w.steps);
    const int64_t seg_at = seq_at + static_cast<int64_t>(seg) * w.steps;
    const int head = seg / w.tiles, tile = seg % w.tiles;
    const int s0 = static_cast<int>(at - seg_at);
    const int s1 = static_cast<int>(end - seg_at < w.steps ? end - seg_at : w.steps);
    const int rows = min(R, w.r.n * G - tile * R);

    // What the first and the last row see (limits grow with the row): steps in which every row sees every token need no mask.
    auto sees_to = [&](int r) {
      const int pos = w.r.len - w.r.n + r / G;
      return max(0, p.causal ? min(pos + 1, w.r.len) : w.r.len);
    };
    auto sees_from = [&](int r) { return window_from(p, w.r.len - w.r.n + r / G); };
    const int row_first = tile * R, row_last = row_first + rows - 1;
    const int all_hi = sees_to(row_first), any_hi = sees_to(row_last), any_lo = sees_from(row_first), all_lo = sees_from(row_last);

    // ---- this warp's steps: s0 + warp, + kWarps, ... Page ids come 16 steps at a time: lane i holds the first page
    // of step i of the batch, lane 16 + i the second one (pages of 16 tokens). A page in front of what the rows see may be
    // gone from the table, and is not looked up.
    const int mine = s1 - s0 > warp ? (s1 - s0 - warp + kWarps - 1) / kWarps : 0;
    const int64_t head_block = static_cast<int64_t>(head) << p.page_log2;
    int ids = -1;
    auto issue = [&](int i) {
      if (i < mine) {
        if ((i & 15) == 0) {
          const int t = (w.first + s0 + warp + (i + (lane & 15)) * kWarps) * kStep + (lane >> 4) * 16;
          ids = -1;
          if (i + (lane & 15) < mine && t < w.r.len && t + (p.page == 16 ? 16 : kStep) > any_lo && (lane < 16 || p.page == 16)) ids = page_id(p, b, t >> p.page_log2);
        }
        const int t0 = (w.first + s0 + warp + i * kWarps) * kStep;
        const int id0 = __shfl_sync(~0u, ids, i & 15);
        const int id1 = p.page == 16 ? __shfl_sync(~0u, ids, 16 + (i & 15)) : id0;
        const uint32_t st = ring + (i % kStages) * C::kStage;
        const int upto = min(any_hi, w.r.len) - t0;  // rows of the step that hold tokens
        constexpr int kPerRow = D / 16, kRowsAt = 32 / kPerRow, kCopies = kStep / kRowsAt;
        const int cr = lane / kPerRow, cc = lane % kPerRow;
        if (p.page != 16 && upto >= kStep && id0 >= 0) {
          // a whole step within one page: 32 rows in a row, at fixed distances on both sides (the swizzle repeats every
          // 8 rows)
          const int64_t off = ((static_cast<int64_t>(id0) * p.hkv << p.page_log2) + head_block + (t0 & (p.page - 1)) + cr) * D + cc * 16;
          const uint8_t* ks = p.k_cache + off;
          const uint8_t* vs = p.v_cache + off;
          const uint32_t even = st + chunk_at<D>(cr, cc), odd = st + chunk_at<D>(cr + kRowsAt, cc) - kRowsAt * D;
#pragma unroll
          for (int j = 0; j < kCopies; ++j) {
            const uint32_t to = ((j * kRowsAt & 7) ? odd : even) + j * kRowsAt * D;
            cp_async16(to, ks + j * kRowsAt * D, 16);
            cp_async16(to + C::kTile, vs + j * kRowsAt * D, 16);
          }
        } else {
#pragma unroll 1
          for (int j = 0; j < kCopies; ++j) {
            const int r = j * kRowsAt + cr;
            const int id = r < 16 ? id0 : id1;
            const bool ok = r < upto && id >= 0;
            const int64_t off = ((static_cast<int64_t>(ok ? id : 0) * p.hkv << p.page_log2) + head_block + ((t0 + r) & (p.page - 1))) * D + cc * 16;
            cp_async16(st + chunk_at<D>(r, cc), p.k_cache + (ok ? off : 0), ok ? 16 : 0);
            cp_async16(st + C::kTile + chunk_at<D>(r, cc), p.v_cache + (ok ? off : 0), ok ? 16 : 0);
          }
        }
        if (lane < 4) {
          const int id = (lane & 1) ? id1 : id0;
          const uint32_t at_m = st + 2 * C::kTile + lane * 4;
          if (id >= 0) cp_async4(at_m, ((lane & 2) ? p.v_scale : p.k_scale) + static_cast<int64_t>(id) * p.hkv + head);
          else *reinterpret_cast<float*>(ring_ptr + (i % kStages) * C::kStage + 2 * C::kTile + lane * 4) = 0.0f;
          if (lane < 2) *reinterpret_cast<int*>(ring_ptr + (i % kStages) * C::kStage + 2 * C::kTile + 16 + lane * 4) = id >= 0;
        }
      }
      cp_commit();
    };
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) issue(i);

    // ---- rows of the segment, while the first steps are under way: queries as operand fragments, limits
    if (tid < R) {
      row_hi[tid] = sees_to(min(row_first + tid, row_last));
      row_lo[tid] = sees_from(min(row_first + tid, row_last));
    }
    for (int r = warp; r < R; r += kWarps) {
      const int rr = tile * R + r;
      const bool real = r < rows;
      const int64_t qat = real ? static_cast<int64_t>(w.r.row0 + rr / G) * p.qs + (head * G + rr % G) * D : 0;
      float sum = 0.0f, unit = 1.0f;
      if (F32) {
        uint32_t a = 0;
        for (int d = lane; d < D; d += 32) a = max(a, real ? __float_as_uint(static_cast<const float*>(p.q)[qat + d]) & 0x7fffffffu : 0u);
        a = __reduce_max_sync(~0u, a);
        // |q / unit| < 2^15: pairs of float16 numbers hold it to 2^-24 of itself and steps of 2^-39 of the row's largest
        unit = __uint_as_float((max(a >> 23, 15u) - 14u) << 23);
      }
      const float inv = F32 ? 1.0f / unit : 1.0f;
      // lane (s, c) of the fragment's row: k step s takes dims 16 (c + 4 (s / 4)) + 4 (s % 4) + 0..3 of lane c
      for (int i = lane; i < C::kK * 4; i += 32) {
        const int s = i >> 2, cc = i & 3, d = 16 * (cc + 4 * (s >> 2)) + 4 * (s & 3);
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = real ? load_f(p.q, !F32, qat + d + e) * inv : 0.0f;
        const int o1 = E4M3 ? 1 : 2, o2 = E4M3 ? 2 : 1;
        const uint32_t h0 = pack_half2(v[0], v[o1]), h1 = pack_half2(v[o2], v[3]);
        uint32_t* at_q = qfrag + (((r >> 3) * C::kK + s) * 32 + (r & 7) * 4 + cc) * 2;
        at_q[0] = h0;
        at_q[1] = h1;
        if (F32) {
          const float2 f0 = unpack_half2(h0), f1 = unpack_half2(h1);
          uint32_t* lo_q = at_q + NT * C::kK * 64;
          lo_q[0] = pack_half2(v[0] - f0.x, v[o1] - f0.y);
          lo_q[1] = pack_half2(v[o2] - f1.x, v[3] - f1.y);
        }
        sum += (v[0] + v[1]) + (v[2] + v[3]);
      }
#pragma unroll
      for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(~0u, sum, d);
      if (lane == 0) {
        row_cor[r] = C::kRaw ? -128.0f / 16777216.0f * sum : 0.0f;
        row_fac[r] = p.scale * kLog2e * unit * (C::kRaw ? 16777216.0f : 1.0f);
      }
    }
    __syncthreads();
    float m[NT][2], l[NT][2], fac[NT][2], cor[NT][2], O[C::kMt][NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        m[n][e] = -INFINITY;
        l[n][e] = 0.0f;
        fac[n][e] = row_fac[n * 8 + 2 * c + e];
        cor[n][e] = row_cor[n * 8 + 2 * c + e];
      }
#pragma unroll
    for (int t = 0; t < C::kMt; ++t)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) O[t][n][e] = 0.0f;
    uint32_t qr[C::kK][2];
    if (NT == 1 && !F32) {
#pragma unroll
      for (int s = 0; s < C::kK; ++s) {
        const uint2 v = reinterpret_cast<const uint2*>(qfrag)[s * 32 + lane];
        qr[s][0] = v.x;
        qr[s][1] = v.y;
      }
    }

    for (int i = 0; i < mine; ++i) {
      issue(i + kStages - 1);
      cp_wait<kStages - 1>();
      __syncwarp();
      const uint32_t st = ring + (i % kStages) * C::kStage;
      const float* meta = reinterpret_cast<const float*>(ring_ptr + (i % kStages) * C::kStage + 2 * C::kTile);
      const int* oks = reinterpret_cast<const int*>(meta + 4);
      const int t0 = (w.first + s0 + warp + i * kWarps) * kStep;

      // scores of 2 x 16 tokens
      float x[2][NT][4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          x[h][n][0] = x[h][n][2] = cor[n][0];
          x[h][n][1] = x[h][n][3] = cor[n][1];
        }
#pragma unroll
        for (int q4 = 0; q4 < C::kK / 4; ++q4) {
          const uint4 k0 = lds_v4(st + chunk_at<D>(16 * h + g, c + 4 * q4)), k1 = lds_v4(st + chunk_at<D>(16 * h + 8 + g, c + 4 * q4));
          const uint32_t w0[4] = {k0.x, k0.y, k0.z, k0.w}, w1[4] = {k1.x, k1.y, k1.z, k1.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int s = 4 * q4 + j;
            uint32_t a0, a1, a2, a3;
            row_pairs<E4M3, C::kRaw>(w0[j], a0, a2);
            row_pairs<E4M3, C::kRaw>(w1[j], a1, a3);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              uint2 qv;
              if (NT == 1 && !F32) qv = make_uint2(qr[s][0], qr[s][1]);
              else qv = reinterpret_cast<const uint2*>(qfrag)[(n * C::kK + s) * 32 + lane];
              mma_16816(x[h][n], a0, a1, a2, a3, qv.x, qv.y);
              if (F32) {
                const uint2 ql = reinterpret_cast<const uint2*>(qfrag)[((NT + n) * C::kK + s) * 32 + lane];
                mma_16816(x[h][n], a0, a1, a2, a3, ql.x, ql.y);
              }
            }
          }
        }
      }
      const float ks0 = meta[0], ks1 = meta[1];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float f0 = fac[n][e] * ks0, f1 = fac[n][e] * ks1;
          x[0][n][e] *= f0;
          x[0][n][e + 2] *= f0;
          x[1][n][e] *= f1;
          x[1][n][e + 2] *= f1;
        }
      if (t0 < all_lo || t0 + kStep > all_hi || !(oks[0] & oks[1])) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int hi = row_hi[n * 8 + 2 * c + e], lo = row_lo[n * 8 + 2 * c + e];
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                const int t = t0 + 16 * h + 8 * k + g;
                if (t >= hi || t < lo || !oks[h]) x[h][n][2 * k + e] = -INFINITY;
              }
          }
      }
      // raise m where a score exceeds it by more than kRaise (or is NaN: it then runs through the weights)
      bool above = false;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float top = m[n][e] + (kRaise + kLift);
          above |= !(x[0][n][e] <= top) | !(x[0][n][e + 2] <= top) | !(x[1][n][e] <= top) | !(x[1][n][e + 2] <= top);
        }
      if (__any_sync(~0u, above)) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float f[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float t = fmaxf(fmaxf(x[0][n][e], x[0][n][e + 2]), fmaxf(x[1][n][e], x[1][n][e + 2]));
            t = fmaxf(t, __shfl_xor_sync(~0u, t, 4));
            t = fmaxf(t, __shfl_xor_sync(~0u, t, 8));
            t = fmaxf(t, __shfl_xor_sync(~0u, t, 16));
            t = fmaxf(t - kLift, m[n][e]);
            f[e] = m[n][e] == t ? 1.0f : exp2_approx(m[n][e] - t);
            m[n][e] = t;
            l[n][e] *= f[e];
          }
#pragma unroll
          for (int k = 0; k < C::kMt; ++k) {
            O[k][n][0] *= f[0];
            O[k][n][1] *= f[1];
            O[k][n][2] *= f[0];
            O[k][n][3] *= f[1];
          }
        }
      }
      // weights, and P^T as B operands
      uint32_t pb[2][NT][2], pl[F32 ? 2 : 1][NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const float m0 = m[n][0] == -INFINITY ? 0.0f : m[n][0], m1 = m[n][1] == -INFINITY ? 0.0f : m[n][1];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const float w0 = exp2_approx(x[h][n][2 * k] - m0), w1 = exp2_approx(x[h][n][2 * k + 1] - m1);
            l[n][0] += w0;
            l[n][1] += w1;
            const uint32_t hw = pack_half2(w0, w1);
            pb[h][n][k] = transpose8(hw);
            if (F32) {
              const float2 f = unpack_half2(hw);
              pl[F32 ? h : 0][n][k] = transpose8(pack_half2((w0 - f.x) * kRest, (w1 - f.y) * kRest));
            }
          }
      }
      // O^T += v_scale (V^T P^T), page by page
      // (with the weights' 2^7 taken out; float32 rows take it out of the products, which leaves v_scale its range)
      const float unit_v = C::kRaw ? 16777216.0f * kDrop : F32 ? 1.0f : kDrop;
      const float vs0 = meta[2] * unit_v, vs1 = meta[3] * unit_v;
      const uint32_t vt = st + C::kTile;
      auto load_v = [&](int t, uint32_t (&v)[D / 32]) {
        if (D == 128) {
          const uint4 u = lds_v4(vt + chunk_at<D>(t, g));
          v[0] = u.x; v[1] = u.y; v[D / 32 - 2] = u.z; v[D / 32 - 1] = u.w;
        } else {
          const uint2 u = lds_v2(vt + chunk_at<D>(t, g >> 1) + 8 * (g & 1));
          v[0] = u.x; v[1] = u.y;
        }
      };
      auto add_values = [&](int h0, int h1, float scale) {
        const bool bad = !(fabsf(scale) <= 3.4028234e38f);
        const float vs = bad ? 0.0f : scale;
        float base[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          base[n][0] = base[n][1] = base[n][2] = base[n][3] = 0.0f;
          if (C::kRaw)  // -128 2^-24 times the sum of the weights
            for (int h = h0; h < h1; ++h) mma_16816(base[n], 0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u, pb[h][n][0], pb[h][n][1]);
        }
        uint32_t v[2][4][D / 32];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (h < h0 || h >= h1) continue;
          load_v(16 * h + 2 * c, v[h][0]);
          load_v(16 * h + 2 * c + 1, v[h][1]);
          load_v(16 * h + 2 * c + 8, v[h][2]);
          load_v(16 * h + 2 * c + 9, v[h][3]);
        }
#pragma unroll
        for (int q = 0; q < D / 32; ++q) {
          float t[2][NT][4];
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) t[0][n][e] = t[1][n][e] = base[n][e];
          uint32_t lo[2][4], hi[2][4];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (h < h0 || h >= h1) continue;
            token_pairs<E4M3, C::kRaw>(v[h][0][q], v[h][1][q], lo[h]);
            token_pairs<E4M3, C::kRaw>(v[h][2][q], v[h][3][q], hi[h]);
          }
          auto products = [&](const uint32_t (&w)[2], int h, int n) {
            mma_16816(t[0][n], lo[h][0], lo[h][1], hi[h][0], hi[h][1], w[0], w[1]);
            mma_16816(t[1][n], lo[h][2], lo[h][3], hi[h][2], hi[h][3], w[0], w[1]);
          };
          if (F32) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              if (h < h0 || h >= h1) continue;
#pragma unroll
              for (int n = 0; n < NT; ++n) products(pl[F32 ? h : 0][n], h, n);
            }
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
              for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) t[k][n][e] *= 1.0f / kRest;
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (h < h0 || h >= h1) continue;
#pragma unroll
            for (int n = 0; n < NT; ++n) products(pb[h][n], h, n);
          }
#pragma unroll
          for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int e = 0; e < 4; ++e) O[2 * q + k][n][e] = fmaf(vs, F32 ? t[k][n][e] * kDrop : t[k][n][e], O[2 * q + k][n][e]);
        }
        if (bad) {  // rows that see none of the page's tokens stay free of its NaN
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int r = n * 8 + 2 * c + e;
              if (row_lo[r] < t0 + 16 * h1 && row_hi[r] > max(t0 + 16 * h0, row_lo[r]))
#pragma unroll
                for (int k = 0; k < C::kMt; ++k) O[k][n][e] = O[k][n][e + 2] = __uint_as_float(0x7fc00000u);
            }
        }
      };
      // a page that no row sees must not reach them, whatever its scale is (0 * NaN)
      if (p.page == 16) {
        if (t0 < any_hi && t0 + 16 > any_lo && oks[0]) add_values(0, 1, vs0);
        if (t0 + 16 < any_hi && t0 + 32 > any_lo && oks[1]) add_values(1, 2, vs1);
      } else if (t0 < any_hi && t0 + kStep > any_lo && oks[0]) {
        add_values(0, 2, vs0);
      }
      __syncwarp();  // the buffer may be filled again
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncwarp();

    // ---- join the warps: O as [rows][D] floats over each warp's ring
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float t = l[n][e];
        t += __shfl_xor_sync(~0u, t, 4);
        t += __shfl_xor_sync(~0u, t, 8);
        t += __shfl_xor_sync(~0u, t, 16);
        if (g == 0) {
          warp_m[warp * R + n * 8 + 2 * c + e] = m[n][e];
          warp_l[warp * R + n * 8 + 2 * c + e] = t * kDrop;
        }
      }
    float* mine_o = reinterpret_cast<float*>(ring_ptr);
    // accumulator tile t: rows g and g + 8 are dims (D / 8) g + 2 t and + 1
#pragma unroll
    for (int t = 0; t < C::kMt; ++t)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          *reinterpret_cast<float2*>(mine_o + (n * 8 + 2 * c + e) * D + (D / 8) * g + 2 * t) = make_float2(O[t][n][e], O[t][n][e + 2]);
    __syncthreads();
    const bool whole = s0 == 0 && s1 == w.steps;
    float* part = ws.part + (static_cast<int64_t>(blockIdx.x) * 2 + (s0 == 0 ? 1 : 0)) * part_floats(R, D);
    for (int e = tid; e < rows * (D / 4); e += kThreads) {
      const int r = e / (D / 4), d = (e % (D / 4)) * 4;
      float mm = -INFINITY, ll = 0.0f;
      for (int k = 0; k < kWarps; ++k) mm = fmaxf(mm, warp_m[k * R + r]);
      float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      for (int k = 0; k < kWarps; ++k) {
        const float mk = warp_m[k * R + r], f = mk == mm ? 1.0f : exp2_approx(mk - mm);
        const float4 v = *reinterpret_cast<const float4*>(smem + k * C::kWarpBytes + (r * D + d) * 4);
        ll = fmaf(f, warp_l[k * R + r], ll);
        o.x = fmaf(f, v.x, o.x);
        o.y = fmaf(f, v.y, o.y);
        o.z = fmaf(f, v.z, o.z);
        o.w = fmaf(f, v.w, o.w);
      }
      if (CL) {
        *reinterpret_cast<float4*>(join + r * D + d) = o;
        if (d == 0) {
          join[R * D + r] = mm;
          join[R * D + R + r] = ll;
        }
      } else if (whole) {
        const float inv = ll == 0.0f ? 0.0f : 1.0f / ll;
        const int rr = tile * R + r;
        const int64_t oat = static_cast<int64_t>(w.r.row0 + rr / G) * p.os + (head * G + rr % G) * D + d;
        if (F32) {
          float* dst = static_cast<float*>(p.o) + oat;
          dst[0] = o.x * inv; dst[1] = o.y * inv; dst[2] = o.z * inv; dst[3] = o.w * inv;
        } else {
          __half* dst = static_cast<__half*>(p.o) + oat;
          dst[0] = __float2half_rn(o.x * inv); dst[1] = __float2half_rn(o.y * inv);
          dst[2] = __float2half_rn(o.z * inv); dst[3] = __float2half_rn(o.w * inv);
        }
      } else {
        *reinterpret_cast<float2*>(part + r * D + d) = make_float2(o.x, o.y);
        *reinterpret_cast<float2*>(part + r * D + d + 2) = make_float2(o.z, o.w);
        if (d == 0) {
          part[R * D + r] = mm;
          part[R * D + R + r] = ll;
        }
      }
    }
    __syncthreads();
    at = seg_at + s1;
  }
  if (CL) {
    cluster_sync();
    if (b >= 0) {
      const int tile = static_cast<int>(found_at), head = blockIdx.x / split % p.hkv, rows = min(R, w.r.n * G - tile * R);
      const uint32_t at = smem_u32(join);
      for (int e = rank * kThreads + tid; e < rows * (D / 4); e += split * kThreads) {
        const int r = e / (D / 4), d = (e % (D / 4)) * 4;
        float mk[8], lk[8], mm = -INFINITY, ll = 0.0f;
        float4 v[8], o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (k < split) {
            const uint32_t there = map_rank(at, k);
            v[k] = ld_cluster_f32x4(there + (r * D + d) * 4);
            mk[k] = ld_cluster_f32(there + (R * D + r) * 4);
            lk[k] = ld_cluster_f32(there + (R * D + R + r) * 4);
          }
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (k < split) mm = fmaxf(mm, mk[k]);
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (k < split) {
            const float f = mk[k] == mm ? 1.0f : exp2_approx(mk[k] - mm);
            ll = fmaf(f, lk[k], ll);
            o.x = fmaf(f, v[k].x, o.x);
            o.y = fmaf(f, v[k].y, o.y);
            o.z = fmaf(f, v[k].z, o.z);
            o.w = fmaf(f, v[k].w, o.w);
          }
        const float inv = ll == 0.0f ? 0.0f : 1.0f / ll;
        const int rr = tile * R + r;
        const int64_t oat = static_cast<int64_t>(w.r.row0 + rr / G) * p.os + (head * G + rr % G) * D + d;
        const float y[4] = {o.x * inv, o.y * inv, o.z * inv, o.w * inv};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (F32) static_cast<float*>(p.o)[oat + i] = y[i];
          else static_cast<__half*>(p.o)[oat + i] = __float2half_rn(y[i]);
        }
      }
    }
    cluster_sync();  // nobody leaves while its part is being read
  }
}

// Joins the partial results of the segments that were cut: a warp a (row, query head).
template <int D, bool F32>
__global__ void __launch_bounds__(256) combine_kernel(const Kv8 p, Workspace ws, int R, int grid, int warps) {
  const int lane = threadIdx.x & 31;
  const int64_t id = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
  const int row = static_cast<int>(id / p.hq), h = static_cast<int>(id % p.hq);
  if (row >= p.tokens) return;
  int b = -1;
  if (p.uniform) {
    b = row / (p.tokens / p.seqs);
  } else {
    for (int b0 = 0; b0 < p.seqs && b < 0; b0 += 32) {
      const bool here = b0 + lane < p.seqs && p.cu[b0 + lane] <= row && row < p.cu[b0 + lane + 1];
      const unsigned m = __ballot_sync(~0u, here);
      if (m) b = b0 + __ffs(m) - 1;
    }
  }
  const SeqWork w = b < 0 ? SeqWork{} : seq_work(p, b, R);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  constexpr int PER = D / 32;
  const int64_t oat = static_cast<int64_t>(row) * p.os + h * D + lane * PER;
  if (w.r.n == 0) {  // a row of no sequence
    if (p.zero_rest)
      for (int e = 0; e < PER; ++e) {
        if (F32) static_cast<float*>(p.o)[oat + e] = 0.0f;
        else static_cast<__half*>(p.o)[oat + e] = __half(0.0f);
      }
    return;
  }
  if (w.tiles == 0) return;
  const int G = p.hq / p.hkv, rr = (row - w.r.row0) * G + h % G, tile = rr / R, r = rr % R;
  const int64_t g0 = ws.start[b] + (static_cast<int64_t>(h / G) * w.tiles + tile) * w.steps, g1 = g0 + w.steps;
  const int64_t run = run_length(ws.start[p.seqs], grid, warps);
  const int c0 = static_cast<int>(g0 / run), c1 = static_cast<int>((g1 - 1) / run);
  if (c0 == c1) return;
  auto part_of = [&](int k) { return ws.part + (static_cast<int64_t>(k) * 2 + (g0 >= run * k ? 1 : 0)) * part_floats(R, D); };
  float mm = -INFINITY;
  for (int k = c0 + lane; k <= c1; k += 32) mm = fmaxf(mm, part_of(k)[R * D + r]);
#pragma unroll
  for (int d = 16; d; d >>= 1) mm = fmaxf(mm, __shfl_xor_sync(~0u, mm, d));
  float o[PER], ll = 0.0f;
#pragma unroll
  for (int e = 0; e < PER; ++e) o[e] = 0.0f;
#pragma unroll 4
  for (int k = c0; k <= c1; ++k) {
    const float* part = part_of(k);
    const float mk = part[R * D + r], f = mk == mm ? 1.0f : exp2_approx(mk - mm);
    ll = fmaf(f, part[R * D + R + r], ll);
#pragma unroll
    for (int e = 0; e < PER; e += 2) {
      const float2 v = *reinterpret_cast<const float2*>(part + r * D + lane * PER + e);
      o[e] = fmaf(f, v.x, o[e]);
      o[e + 1] = fmaf(f, v.y, o[e + 1]);
    }
  }
  const float inv = ll == 0.0f ? 0.0f : 1.0f / ll;
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    if (F32) static_cast<float*>(p.o)[oat + e] = o[e] * inv;
    else static_cast<__half*>(p.o)[oat + e] = __float2half_rn(o[e] * inv);
  }
}

// ------------------------------------------------------------------ host side
// 8-row tiles a segment: as many as an average sequence has rows (or may have here).
inline int row_tiles(const Kv8& p) {
  const int64_t mean = ceil_div(p.tokens, p.seqs) * (p.hq / p.hkv), rows = mean < p.few_rows ? mean : p.few_rows;
  return rows <= 8 ? 1 : 2;  // four tiles spill: 64 x 4 rows of 4 heads a group on 8192 tokens 376 / 245 / 484 us with 1 / 2 / 4
}

// CTAs of a cluster that share a segment, 0: equal runs over all SMs. Clusters take a call whose segments of 8 rows, at
// least two CTAs each, find an SM for every CTA, and whose tables hold at most four steps a warp: there latency counts,
// and segments of more rows would only run fewer CTAs and more code (7 x 5 float32 rows of 5 heads a group: 31 us as
// segments of 32).
inline int cluster_split(const Kv8& p) {
  const int64_t G = p.hq / p.hkv, slots = p.uniform ? ceil_div(p.tokens / p.seqs * G, 8) * p.seqs : p.tokens * G / 8 + p.seqs;
  int split = 8;
  while (split > 1 && slots * p.hkv * split > device_sm_count()) split /= 2;
  const int64_t steps = ceil_div(static_cast<int64_t>(p.max_pages) << p.page_log2, kStep);
  return split > 1 && steps <= 4ll * 12 * split ? split : 0;
}

template <bool E4M3, int D, bool F32>
cudaError_t launch_cluster(const Kv8& p, int split, cudaStream_t s) {
  using C = Traits<E4M3, D, 1, F32, true>;
  static_assert(C::kSmem <= 227 * 1024, "shared memory");
  const cudaError_t e = allow_smem<attn_mma_kernel<E4M3, D, 1, F32, true>>(C::kSmem);
  if (e != cudaSuccess) return e;
  const int64_t G = p.hq / p.hkv, slots = p.uniform ? ceil_div(p.tokens / p.seqs * G, 8) * p.seqs : p.tokens * G / 8 + p.seqs;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(slots * p.hkv * split));
  cfg.blockDim = dim3(C::kThreads);
  cfg.dynamicSmemBytes = C::kSmem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = split;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, attn_mma_kernel<E4M3, D, 1, F32, true>, p, Workspace{}, split);
}

template <bool E4M3, int D, int NT, bool F32>
cudaError_t launch_nt(const Kv8& p, void* ws, cudaStream_t s) {
  using C = Traits<E4M3, D, NT, F32>;
  static_assert((C::kSmem + 1024) * C::kCtas <= 228 * 1024, "shared memory");
  cudaError_t e = allow_smem<attn_mma_kernel<E4M3, D, NT, F32, false>>(C::kSmem);
  if (e != cudaSuccess) return e;
  const int grid = device_sm_count() * C::kCtas;
  Workspace w{static_cast<int64_t*>(ws), reinterpret_cast<float*>(static_cast<char*>(ws) + starts_bytes(p.seqs))};
  attn_mma_kernel<E4M3, D, NT, F32, false><<<grid, C::kThreads, C::kSmem, s>>>(p, w, 1);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>((static_cast<int64_t>(p.tokens) * p.hq + 7) / 8));
  cfg.blockDim = dim3(256);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, combine_kernel<D, F32>, p, w, C::kRows, grid, C::kWarps);
}

template <bool E4M3, int D, bool F32>
cudaError_t launch_rows(const Kv8& p, void* ws, cudaStream_t s) {
  if (const int split = cluster_split(p)) return launch_cluster<E4M3, D, F32>(p, split, s);
  return row_tiles(p) == 1 ? launch_nt<E4M3, D, 1, F32>(p, ws, s) : launch_nt<E4M3, D, 2, F32>(p, ws, s);
}

template <bool E4M3>
cudaError_t launch_code(const Kv8& p, void* ws, cudaStream_t s) {
  if (p.D == 128) return p.f16 ? launch_rows<E4M3, 128, false>(p, ws, s) : launch_rows<E4M3, 128, true>(p, ws, s);
  return p.f16 ? launch_rows<E4M3, 64, false>(p, ws, s) : launch_rows<E4M3, 64, true>(p, ws, s);
}

}  // namespace
}  // namespace xrgpu
