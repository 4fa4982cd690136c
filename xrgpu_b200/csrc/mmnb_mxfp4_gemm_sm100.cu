// Product of two microscaled 4-bit operands on tcgen05 tensor cores (format: mmnb_mxfp4.h):
//   y[m, n] = sum_blocks 2^(ea + eb) sum_32 a w + bias[n].
// The tensor cores take the codes and the scale bytes as they are (block-scaled 4-bit kind, one scale per
// 32 values, float32 accumulators), so nothing is unpacked: a CTA streams code tiles and scale tiles into
// shared memory, copies the scales on into tensor memory and issues the MMAs.
//
// Orientation. An MMA multiplies 128 rows (operand P) by T rows (operand Q). Up to 128 activation rows, P are
// the weights, which stream once, and Q all activations (T the rows rounded up to 16); the K axis is then
// split over a cluster of up to 8 CTAs whose float32 partial tiles meet in shared memory, summed in the
// order of their ranks. For more rows P are the activations, so that a thread's accumulator row is a row of y.
//
// Roles (10 warps): warp 0 loads (one lane: TMA tiles with the 128-byte swizzle, bulk copies of scale
// tiles), warp 1 copies scales to tensor memory and issues the MMAs (one lane), warps 2-9 drain the
// accumulators (lane quadrant warp % 4, alternate 16-column chunks).
//
// Tensor memory: two accumulators of T columns at 0 and acc1, then per stage the scale columns: 4 columns
// (32 lanes x 4 bytes x 4 row groups) for 128 rows x 128 values. Q tiles begin at a row block (one tile, or T a multiple of
// 128), so that their scales begin at a column that is a multiple of 4: other starts are not taken. A stage's columns are rewritten only when
// its shared-memory buffer has come back, that is when the MMAs that read them are done. Only tiles of up to 128 columns
// take turns on a CTA (more rows than that go to pairs of CTAs before they need a second round).
//
// Measured (codes in, GPU time without the launch): 1 x 4096 x 4096 6.3 us (latency), 16 x 14336 x 4096 8.5 us (31 MB, 3.7
// TB/s: latency, then the weights' stream), 2048 x 14336 x 4096 54 us (4.5 PFLOP/s), 8192 x 28672 x 8192 671 us (5.7 PFLOP/s,
// bound by loads from L2; 700 us in calls back to back, at the power limit).
//
// Every wait is bounded as in mmnb_gemm_sm100.cu.
#include <cuda.h>
#include <cuda_fp16.h>

#include <climits>

#include "mmnb_mxfp4.h"
#include "mmnb_tcgen05.cuh"

namespace xrgpu {
namespace {

constexpr int kRows = 128;              // rows of operand P
constexpr int kStepBytes = 128;         // codes of a row per stage: 256 values, one swizzle row
constexpr int kScaleTile = 512;         // scale bytes of 128 rows x 128 values
constexpr int kEpilogueWarps = 8;
constexpr int kThreads = (2 + kEpilogueWarps) * 32;
constexpr int kTmemCols = 512;
constexpr int kSmemBudget = 227 * 1024;
constexpr int kPitch = kRows;           // floats a column of a partial tile in shared memory

constexpr unsigned kErrWaitProducer = 0x601;
constexpr unsigned kErrWaitMma = 0x602;
constexpr unsigned kErrWaitEpilogue = 0x603;
constexpr unsigned kErrDrain = 0x604;

struct Args {
  int p_rows, q_rows;       // valid rows of the operands
  int p_tiles, tiles;       // tiles along P, in all
  int whole;                // pairs: tiles from this one on are halves
  int T, ksteps, k64;       // rows of Q a tile, stages along K, 64-value MMA steps along K
  int stages, split, q_blocks;  // q_blocks: scale row blocks a Q tile spans (1 or 2)
  int acc1;                 // column of the second accumulator
  int tmem_cols, sf_col, sf_stage;
  int early;                // the weights may be loaded before the previous kernel has finished
  uint32_t q_stage, stage;  // bytes
  int64_t tiles_k;          // scale tiles along K
  int sp_blocks, sq_blocks; // row blocks of the scales
  const uint8_t* sp;
  const uint8_t* sq;
  const void* bias;
  void* y;
  int64_t ldy;
  int vec;                  // rows of y start on 16 bytes
  unsigned* err;
};

// D[128 x T] (+)= P (smem, K-major codes) . Q^T, scales in tensor memory.
__device__ __forceinline__ void mma_mxf4(uint32_t d, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t sa,
                                         uint32_t sb, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
      ::"r"(d), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate)
      : "memory");
}

// 32 rows of 16 bytes from shared memory to 4 columns, the same in all four lane quadrants.
__device__ __forceinline__ void scales_to_tmem(uint32_t taddr, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}

// Shared-memory descriptor without swizzle: 8-row groups of 16-byte rows, 128 bytes apart.
__device__ __forceinline__ uint64_t plain_desc(uint32_t saddr) {
  return static_cast<uint64_t>((saddr >> 4) & 0x3FFFu) | (static_cast<uint64_t>(128u >> 4) << 32) | (static_cast<uint64_t>(1u) << 46);
}

// Instruction descriptor: 4-bit floats, both K-major, M = 128, N = T, scales of powers of two, K = 64;
// `half` picks the scale bytes 0-1 (0) or 2-3 (2) of a column.
__device__ __forceinline__ uint32_t instruction_desc(int T, uint32_t half) {
  return (half << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(T >> 3) << 17) | (1u << 23) |
         (static_cast<uint32_t>(kRows >> 4) << 24) | (half << 29);
}

// 16 accumulators of a row of y from column n0 on, plus bias.
template <bool F16>
__device__ __forceinline__ void store_row(const Args& a, int p, int n0, const uint32_t (&v)[16]) {
  float r[16];
#pragma unroll
  for (int j = 0; j < 16; ++j)
    r[j] = __uint_as_float(v[j]) + ((a.bias && n0 + j < a.q_rows) ? load_f(a.bias, F16, n0 + j) : 0.0f);
  if (a.vec && n0 + 16 <= a.q_rows) {
    if (F16) {
      uint32_t h[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const __half2 x = __floats2half2_rn(r[2 * j], r[2 * j + 1]);
        h[j] = *reinterpret_cast<const uint32_t*>(&x);
      }
      uint4* dst = reinterpret_cast<uint4*>(static_cast<__half*>(a.y) + p * a.ldy + n0);
      dst[0] = make_uint4(h[0], h[1], h[2], h[3]);
      dst[1] = make_uint4(h[4], h[5], h[6], h[7]);
    } else {
      float4* dst = reinterpret_cast<float4*>(static_cast<float*>(a.y) + p * a.ldy + n0);
#pragma unroll
      for (int j = 0; j < 4; ++j) dst[j] = make_float4(r[4 * j], r[4 * j + 1], r[4 * j + 2], r[4 * j + 3]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      if (n0 + j >= a.q_rows) break;
      if (F16) static_cast<__half*>(a.y)[p * a.ldy + n0 + j] = __float2half_rn(r[j]);
      else static_cast<float*>(a.y)[p * a.ldy + n0 + j] = r[j];
    }
  }
}

template <bool SWAP, bool F16, int QB>
__global__ void __launch_bounds__(kThreads, 1)
    mxfp4_gemm_kernel(const __grid_constant__ CUtensorMap map_p, const __grid_constant__ CUtensorMap map_q, const Args a) {
  extern __shared__ uint8_t smem_raw[];
  const int warp = __shfl_sync(~0u, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int S = a.stages;
  const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
  uint8_t* gbase = smem_raw + (base - raw);
  // a stage: [P tile 16 KB][Q tile T * 128][P scales 1 KB][Q scales q_blocks * 1 KB]
  __shared__ uint64_t full[12], empty[12], accfull[2], drained[2], done;
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;

  if (threadIdx.x == 0) {
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
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&tmem_slot);
  const Ctl ctl{&abort_flag, a.err};
  const int rank = a.split > 1 ? static_cast<int>(cluster_rank()) : 0;
  const int first = blockIdx.x / a.split, step = gridDim.x / a.split;
  const int k0 = static_cast<int>(static_cast<int64_t>(a.ksteps) * rank / a.split);
  const int k1 = static_cast<int>(static_cast<int64_t>(a.ksteps) * (rank + 1) / a.split);

  if (warp == 0) {
    if (lane == 0) {
      auto load_p = [&](int s, int ks, int pt, int groups) {
        tma_load_2d(base + s * a.stage, &map_p, ks * kStepBytes, pt * kRows, &full[s]);
        bulk_copy_g2s(gbase + s * a.stage + kRows * kStepBytes + a.q_stage, a.sp + (pt * a.tiles_k + 2 * ks) * kScaleTile,
                      groups * kScaleTile, &full[s]);
      };
      auto load_q = [&](int s, int ks, int qt, int groups) {
        tma_load_2d(base + s * a.stage + kRows * kStepBytes, &map_q, ks * kStepBytes, qt * a.T, &full[s]);
        const int rb = qt * a.T / kRows;
        for (int b = 0; b < a.q_blocks && rb + b < a.sq_blocks; ++b)
          bulk_copy_g2s(gbase + s * a.stage + kRows * kStepBytes + a.q_stage + (1 + b) * 2 * kScaleTile,
                        a.sq + (static_cast<int64_t>(rb + b) * a.tiles_k + 2 * ks) * kScaleTile, groups * kScaleTile, &full[s]);
      };
      auto expect = [&](int s, int qt, int groups) {
        const int rb = qt * a.T / kRows, blocks = 1 + min(a.q_blocks, a.sq_blocks - rb);
        mbar_arrive_expect_tx(&full[s], kRows * kStepBytes + a.q_stage + blocks * groups * kScaleTile);
      };
      auto groups_of = [&](int ks) { return min(2, (a.k64 - 4 * ks + 1) >> 1); };
      // The weights' first stages do not depend on the kernel before this one; the activations may.
      const int pt0 = first % a.p_tiles, qt0 = first / a.p_tiles;
      const int pre = (a.early && first < a.tiles) ? min(S, k1 - k0) : 0;
      for (int i = 0; i < pre; ++i) {
        expect(i, qt0, groups_of(k0 + i));
        if (SWAP) load_p(i, k0 + i, pt0, groups_of(k0 + i));
        else load_q(i, k0 + i, qt0, groups_of(k0 + i));
      }
      asm volatile("griddepcontrol.wait;" ::: "memory");
      int g = 0, s = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int tile = first; ok && tile < a.tiles; tile += step) {
        const int pt = tile % a.p_tiles, qt = tile / a.p_tiles;
        for (int ks = k0; ks < k1; ++ks, ++g) {
          const int groups = groups_of(ks);
          if (g < pre) {
            if (SWAP) load_q(s, ks, qt, groups);
            else load_p(s, ks, pt, groups);
          } else {
            if (!thread_wait(&empty[s], ph ^ 1, ctl, kErrWaitProducer)) {
              ok = false;
              break;
            }
            expect(s, qt, groups);
            load_p(s, ks, pt, groups);
            load_q(s, ks, qt, groups);
          }
          if (++s == S) {
            s = 0;
            ph ^= 1;
          }
        }
      }
      if (!ok)
        for (int h = (g > S ? g - S : 0); h < g; ++h) drain_wait(&full[h % S], (h / S) & 1, a.err, kErrDrain);
    }
  } else if (warp == 1) {
    // The warp stays converged and elects the issuing lane, so that descriptors stay in uniform registers: with one
    // lane in a branch of its own each tcgen05 instruction took 100 cycles to issue (a step 1700 instead of 600).
    const uint64_t p_desc = umma_desc_sw128(base), q_desc = umma_desc_sw128(base + kRows * kStepBytes);
    const uint64_t s_desc = plain_desc(base + kRows * kStepBytes + a.q_stage);
    const uint32_t i_desc0 = instruction_desc(a.T, 0u), i_desc1 = instruction_desc(a.T, 2u);
    int i = 0, s = 0;
    uint32_t ph = 0;
    bool ok = true;
    for (int tile = first; ok && tile < a.tiles; tile += step, ++i) {
      if (i >= 2 && !warp_spin(&drained[i & 1], ((i - 2) >> 1) & 1, ctl, kErrWaitMma)) break;
      const uint32_t d = tmem + ((i & 1) ? a.acc1 : 0);
      for (int ks = k0; ks < k1; ++ks) {
        if (!warp_spin(&full[s], ph, ctl, kErrWaitMma)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const int subs = a.k64 - 4 * ks;  // 64-value MMA steps left
        const uint32_t off = static_cast<uint32_t>(s) * (a.stage >> 4);
        const uint32_t sf = tmem + a.sf_col + s * a.sf_stage;
        if (elect_one()) {
          // columns: P group 0, P group 1, Q group 0 (4 a row block), Q group 1
#pragma unroll
          for (int gr = 0; gr < 2; ++gr) {
            if (gr == 1 && subs <= 2) break;
            scales_to_tmem(sf + 4 * gr, s_desc + off + gr * (kScaleTile >> 4));
#pragma unroll
            for (int b = 0; b < QB; ++b)
              scales_to_tmem(sf + 8 + 4 * (gr * QB + b), s_desc + off + ((1 + b) * 2 + gr) * (kScaleTile >> 4));
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (j > 0 && j >= subs) break;
            mma_mxf4(d, p_desc + off + 2 * j, q_desc + off + 2 * j, (j & 1) ? i_desc1 : i_desc0, sf + 4 * (j >> 1),
                     sf + 8 + 4 * (j >> 1) * QB, ks > k0 || j > 0);
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
    if (elect_one()) mma_commit(&done);  // every MMA and copy of this warp has completed once `done` flips
    __syncwarp();
    drain_wait(&done, 0, a.err, kErrDrain);
  } else {
    const int q = warp & 3, c = (warp - 2) >> 2;
    const uint32_t lane_addr = static_cast<uint32_t>(32 * q) << 16;
    int i = 0;
    for (int tile = first; tile < a.tiles; tile += step, ++i) {
      const int pt = tile % a.p_tiles, qt = tile / a.p_tiles, b = i & 1;
      const int p = pt * kRows + 32 * q + lane, q0 = qt * a.T;
      if (!warp_wait(&accfull[b], (i >> 1) & 1, ctl, kErrWaitEpilogue)) break;
      tc_fence_after();
      const float p_bias = (SWAP && a.split == 1 && a.bias && p < a.p_rows) ? load_f(a.bias, F16, p) : 0.0f;
      for (int col = 16 * c; col < a.T; col += 32) {
        uint32_t v[16];
        tmem_ld16(tmem + lane_addr + (b ? a.acc1 : 0) + col, v);
        tmem_wait_ld16(v);
        if (a.split > 1) {
#pragma unroll
          for (int j = 0; j < 16; ++j)
            reinterpret_cast<float*>(gbase)[(col + j) * kPitch + 32 * q + lane] = __uint_as_float(v[j]);
        } else if (SWAP) {
          if (p < a.p_rows) {
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              const int64_t m = q0 + col + j;
              if (m >= a.q_rows) break;
              const float r = __uint_as_float(v[j]) + p_bias;
              if (F16) static_cast<__half*>(a.y)[m * a.ldy + p] = __float2half_rn(r);
              else static_cast<float*>(a.y)[m * a.ldy + p] = r;
            }
          }
        } else if (p < a.p_rows) {
          store_row<F16>(a, p, q0 + col, v);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&drained[b]);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(a.tmem_cols) : "memory");
  }
  if (a.split > 1) {
    // one tile a cluster: every rank sums its share of the columns over the ranks (128 floats of a column lie together),
    // in their order; y's rows run along P for SWAP, else the sums turn round in shared memory
    cluster_sync();
    const int pt = first % a.p_tiles, qt = first / a.p_tiles;
    const int cols = min(a.T, a.q_rows - qt * a.T), share = (cols + a.split - 1) / a.split;
    const int col0 = rank * share, mine = max(0, min(share, cols - col0));
    float* turned = reinterpret_cast<float*>(gbase) + a.T * kPitch;  // [128][share + 1]
    for (int e = threadIdx.x; e < mine * (kRows / 4); e += kThreads) {
      const int col = col0 + e / (kRows / 4), row = 4 * (e % (kRows / 4));
      float4 v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (k < a.split) v[k] = ld_cluster_f32x4(map_rank(base + (col * kPitch + row) * 4, k));
      float r[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (k < a.split) {
          r[0] += v[k].x;
          r[1] += v[k].y;
          r[2] += v[k].z;
          r[3] += v[k].w;
        }
      if (SWAP) {
        const int64_t n = pt * kRows + row, at = static_cast<int64_t>(qt * a.T + col) * a.ldy + n;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (n + i >= a.p_rows) break;
          const float y = a.bias ? r[i] + load_f(a.bias, F16, n + i) : r[i];
          if (F16) static_cast<__half*>(a.y)[at + i] = __float2half_rn(y);
          else static_cast<float*>(a.y)[at + i] = y;
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) turned[(row + i) * (share + 1) + col - col0] = r[i];
      }
    }
    if (!SWAP) {
      __syncthreads();
      const int rows = min(kRows, a.p_rows - pt * kRows);
      for (int e = threadIdx.x; e < rows * mine; e += kThreads) {
        const int row = e / mine, col = e % mine;
        const int64_t n = qt * a.T + col0 + col, at = static_cast<int64_t>(pt * kRows + row) * a.ldy + n;
        const float r = turned[row * (share + 1) + col], y = a.bias ? r + load_f(a.bias, F16, n) : r;
        if (F16) static_cast<__half*>(a.y)[at] = __float2half_rn(y);
        else static_cast<float*>(a.y)[at] = y;
      }
    }
    cluster_sync();  // nobody leaves while its partial tile is being read
  }
}

// ------------------------------------------------------------------ pairs of CTAs
// For many rows: a cluster of two CTAs on one 256 x 256 tile. Each holds its 128 rows of P and half of Q's 256 rows; the
// first one's MMAs (cta_group::2) read both halves from both shared memories, so that a CTA loads 256 rows a step instead
// of 384 for the same product. What bounds it are these loads from L2, 35 KB a CTA and step (12 TB/s in all): 8192 x
// 28672 x 8192 takes 671 us (5.7 PFLOP/s); with the loads left out it was 507.
// Tensor memory: two overlapping accumulators of 256 columns (they and the scales need more than the 512 columns); the
// drain first takes the shared columns into registers, then the next tile may start (without waiting for their stores: 73
// -> 66 us at 2048 x 14336 x 4096 with the launch, before the signals had their present form: 66 -> 61.5). Each CTA keeps the accumulators of its own rows and all scales it needs.
// Signals between the two. Both CTAs' loads complete on the first one's `full` (the scales too are tensor copies: only those
// may signal the pair's other CTA), which expects the bytes of both. The MMAs' completion goes to both. The second CTA's
// epilogue warps meet at its own `drained`, and its warp 1 passes that on with a release at cluster scope. What the
// first CTA waits for it acquires at cluster scope.
__device__ __forceinline__ void mma2_mxf4(uint32_t d, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t sa,
                                          uint32_t sb, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
      ::"r"(d), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void scales2_to_tmem(uint32_t taddr, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
// Arrives on `bar` of both CTAs when the tcgen05 operations issued so far have completed.
__device__ __forceinline__ void mma2_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
               ::"r"(smem_u32(bar)), "h"(static_cast<uint16_t>(3)) : "memory");
}
// Arrives on `bar` of CTA `rank`, after all that this thread has done and observed.
__device__ __forceinline__ void arrive_at(uint64_t* bar, uint32_t rank) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(map_rank(smem_u32(bar), rank)) : "memory");
}
// A probe that acquires at cluster scope what the phase stands for (those of a wait are the CTA's).
__device__ __forceinline__ bool acquire_cluster(uint64_t* bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done) : "r"(smem_u32(bar)), "r"(parity) : "memory");
  return done != 0;
}
// Loads a tile into this CTA's shared memory, its bytes counted by `bar`, the shared::cluster address of a barrier of either CTA.
__device__ __forceinline__ void tma2_load_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void st_cluster_u32(uint32_t addr, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
constexpr int kStages2 = 6;
constexpr uint32_t kStage2 = 2 * kRows * kStepBytes + 6 * kScaleTile;  // P, Q half, P scales, Q scales of both blocks: a CTA's bytes
constexpr int kSfStage2 = 24, kShared2 = kStages2 * kSfStage2;         // scale columns; columns that both accumulators hold
constexpr int kAcc2 = 256 - kShared2, kSfCol2 = 512 - kStages2 * kSfStage2;
static_assert(kShared2 % 16 == 0 && kAcc2 + 256 == kSfCol2, "tensor memory map");

// Tile `t` of a pair: from a.whole on each index is one half (128 rows of Q) of a tile.
struct Tile2 {
  int pt, q0;  // row blocks: pair of P, first of Q
  bool half;
};
__device__ __forceinline__ Tile2 tile2(const Args& a, int t) {
  const bool half = t >= a.whole;
  const int whole = half ? a.whole + ((t - a.whole) >> 1) : t;
  return {whole % a.p_tiles, 2 * (whole / a.p_tiles) + (half ? (t - a.whole) & 1 : 0), half};
}

template <bool F16>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    mxfp4_gemm2_kernel(const __grid_constant__ CUtensorMap map_p, const __grid_constant__ CUtensorMap map_q,
                       const __grid_constant__ CUtensorMap map_sp, const __grid_constant__ CUtensorMap map_sq, const Args a) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t full[kStages2], empty[kStages2], accfull[2], drained[2], done;
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
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(kTmemCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // both CTAs' barriers are there
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&tmem_slot);
  const Ctl ctl{&abort_flag, a.err};
  const int first = blockIdx.x >> 1, step = gridDim.x >> 1;

  if (warp == 0) {
    if (lane == 0) {
      asm volatile("griddepcontrol.wait;" ::: "memory");
      int g = 0, s = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int tile = first; ok && tile < a.tiles; tile += step) {
        const Tile2 t = tile2(a, tile);
        const int pb = 2 * t.pt + rank, q_row = t.q0 * kRows + rank * (t.half ? kRows / 2 : kRows);
        const int sp_tile = static_cast<int>(pb * a.tiles_k), sq_tile = static_cast<int>(t.q0 * a.tiles_k), tiles_k = static_cast<int>(a.tiles_k);
        for (int ks = 0; ks < a.ksteps; ++ks, ++g) {
          if (!thread_wait(&empty[s], ph ^ 1, ctl, kErrWaitProducer)) {
            ok = false;
            break;
          }
          // Every copy counts whole (what lies outside the operands is filled with zeros). A second scale tile behind the
          // last one along K is not used.
          if (rank == 0) mbar_arrive_expect_tx(&full[s], 2 * kStage2);
          const uint32_t at = base + s * kStage2, sc = at + 2 * kRows * kStepBytes, bar = map_rank(smem_u32(&full[s]), 0);
          tma2_load_2d(at, &map_p, ks * kStepBytes, pb * kRows, bar);
          tma2_load_2d(at + kRows * kStepBytes, &map_q, ks * kStepBytes, q_row, bar);  // a half uses the first 64 rows
          tma2_load_2d(sc, &map_sp, 0, sp_tile + 2 * ks, bar);
          tma2_load_2d(sc + 2 * kScaleTile, &map_sq, 0, sq_tile + 2 * ks, bar);
          tma2_load_2d(sc + 4 * kScaleTile, &map_sq, 0, sq_tile + tiles_k + 2 * ks, bar);
          if (++s == kStages2) {
            s = 0;
            ph ^= 1;
          }
        }
      }
      st_cluster_u32(map_rank(smem_u32(&fills[rank]), 0), g);
    }
  } else if (warp == 1 && rank == 1) {
    // passes on that this CTA's accumulators have been read (its epilogue warps have stores under way, which a release of
    // theirs would wait for)
    int i = 0;
    for (int tile = first; tile < a.tiles; tile += step, ++i) {
      if (!warp_spin(&drained[i & 1], (i >> 1) & 1, ctl, kErrWaitMma)) break;
      if (lane == 0) arrive_at(&drained[i & 1], 0);
      __syncwarp();
    }
  } else if (warp == 1) {
    const uint64_t p_desc = umma_desc_sw128(base), q_desc = umma_desc_sw128(base + kRows * kStepBytes);
    const uint64_t s_desc = plain_desc(base + 2 * kRows * kStepBytes);
    const uint32_t wide = static_cast<uint32_t>(kRows >> 4) << 24;  // M = 256
    int i = 0, s = 0;
    uint32_t ph = 0;
    bool ok = true;
    // both CTAs' loads, or both CTAs' drains
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      return warp_spin(bar, parity, ctl, kErrWaitMma) && __all_sync(~0u, acquire_cluster(bar, parity));
    };
    for (int tile = first; ok && tile < a.tiles; tile += step, ++i) {
      if (i > 0 && !wait(&drained[(i - 1) & 1], ((i - 1) >> 1) & 1)) break;
      const uint32_t d = tmem + ((i & 1) ? kAcc2 : 0);
      const int T = tile >= a.whole ? 128 : 256;
      const uint32_t i_desc0 = instruction_desc(T, 0u) + wide, i_desc1 = instruction_desc(T, 2u) + wide;
      for (int ks = 0; ks < a.ksteps; ++ks) {
        if (!wait(&full[s], ph)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const int subs = a.k64 - 4 * ks;
        const uint32_t off = static_cast<uint32_t>(s) * (kStage2 >> 4);
        const uint32_t sf = tmem + kSfCol2 + s * kSfStage2;
        if (elect_one()) {
#pragma unroll
          for (int gr = 0; gr < 2; ++gr) {
            if (gr == 1 && subs <= 2) break;
            scales2_to_tmem(sf + 4 * gr, s_desc + off + gr * (kScaleTile >> 4));
#pragma unroll
            for (int b = 0; b < 2; ++b) scales2_to_tmem(sf + 8 + 4 * (gr * 2 + b), s_desc + off + ((1 + b) * 2 + gr) * (kScaleTile >> 4));
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (j > 0 && j >= subs) break;
            mma2_mxf4(d, p_desc + off + 2 * j, q_desc + off + 2 * j, (j & 1) ? i_desc1 : i_desc0, sf + 4 * (j >> 1), sf + 8 + 8 * (j >> 1), ks > 0 || j > 0);
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
    }
    if (elect_one()) mma2_commit(&done);
    __syncwarp();
    drain_wait(&done, 0, a.err, kErrDrain);
  } else {
    const int q = warp & 3, c = (warp - 2) >> 2;
    const uint32_t lane_addr = static_cast<uint32_t>(32 * q) << 16;
    constexpr int kChunks = 16, kSharedChunks = kShared2 / 16;
    int i = 0;
    for (int tile = first; tile < a.tiles; tile += step, ++i) {
      const Tile2 t = tile2(a, tile);
      const int b = i & 1, p = (2 * t.pt + rank) * kRows + 32 * q + lane, q0 = t.q0 * kRows;
      if (!warp_wait(&accfull[b], (i >> 1) & 1, ctl, kErrWaitEpilogue)) break;
      tc_fence_after();
      // What the next tile's accumulator shares with this one is read before anything is stored: the next tile's MMAs
      // wait for it.
      constexpr int kHeld = (kSharedChunks + 1) / 2;
      const int chunks = t.half ? kChunks / 2 : kChunks;
      auto column = [&](int chunk) { return 16 * (b ? chunk : chunks - 1 - chunk); };
      uint32_t held[kHeld][16];
#pragma unroll
      for (int h = 0; h < kHeld; ++h)
        if (c + 2 * h < chunks) tmem_ld16(tmem + lane_addr + (b ? kAcc2 : 0) + column(c + 2 * h), held[h]);
#pragma unroll
      for (int h = 0; h < kHeld; ++h) tmem_wait_ld16(held[h]);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&drained[b]);
#pragma unroll
      for (int h = 0; h < kHeld; ++h)
        if (p < a.p_rows && c + 2 * h < chunks) store_row<F16>(a, p, q0 + column(c + 2 * h), held[h]);
#pragma unroll 1
      for (int at = c + 2 * kHeld; at < chunks; at += 2) {
        uint32_t v[16];
        tmem_ld16(tmem + lane_addr + (b ? kAcc2 : 0) + column(at), v);
        tmem_wait_ld16(v);
        if (p < a.p_rows) store_row<F16>(a, p, q0 + column(at), v);
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && abort_flag) st_cluster_u32(map_rank(smem_u32(&abort_flag), rank ^ 1), 1);
  cluster_sync();  // neither CTA's memory goes while the other may read or signal it
  if (*ctl.abort) {
    // A wait ran out in one of them: loads may be under way whose other half was never issued. A stage's last fill is
    // made complete, then awaited: the first CTA's bytes alone lack the second's, the second's alone were not expected.
    if (rank == 0 && threadIdx.x == 0) {
      const int g0 = static_cast<int>(fills[0]), g1 = static_cast<int>(fills[1]);
      for (int s = 0; s < kStages2; ++s) {
        const int n0 = (g0 - s + kStages2 - 1) / kStages2, n1 = (g1 - s + kStages2 - 1) / kStages2;
        if (n0 < n1) mbar_arrive_expect_tx(&full[s], kStage2);
        else if (n0 > n1) asm volatile("mbarrier.complete_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(&full[s])), "r"(kStage2) : "memory");
        if (n0 || n1) drain_wait(&full[s], (max(n0, n1) - 1) & 1, a.err, kErrDrain);
      }
    }
    cluster_sync();
  }
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
  }
}

// ------------------------------------------------------------------ host side
struct Shape {
  bool swap;
  int T, split;
};

// Up to 128 activation rows: all of them in one tile. K is split while the CTAs find an SM each (narrow tiles: 1.6
// CTAs an SM, they run side by side); beyond that a split costs more than it gives. Measured (us, split 1 / 2 / 4 / 8):
// 1 x 4096 x 4096 9.4 / 7.6 / 6.4 / 6.9; 16 x 14336 x 4096 10.1 / 8.6 / 13.2 / 18.7; 128 x 4096 x 4096 11.9 / 10.9 / 8.9 / 12.4.
// More rows (here one round of 256 columns, see pairs_pay): tiles of 128 columns where they need no second round either,
// which split like the above: 512 x 4096 x 4096 12.6 (128) / 15.3 (256), 256 x 14336 x 4096 (two rounds) 19.1 / 15.9.
Shape choose(const Mxfp4Matmul& p, int ksteps, int sms) {
  Shape s{p.M <= kRows, 256, 1};
  int64_t tiles, most = sms;
  if (s.swap) {
    s.T = static_cast<int>(align_up(p.M, 16));
    tiles = ceil_div(p.N, kRows);
    if (s.T <= 64) most = sms * 8 / 5;
  } else {
    const int64_t pt = ceil_div(p.M, kRows), narrow = pt * ceil_div(p.N, 128), wide = pt * ceil_div(p.N, 256);
    if (narrow <= sms) s.T = 128;
    tiles = s.T == 128 ? narrow : wide;
  }
  if (s.T <= 128)
    while (s.split < 8 && tiles * s.split * 2 <= most && ksteps >= 4 * s.split) s.split *= 2;
  return s;
}

template <bool SWAP, bool F16, int QB>
cudaError_t launch(const CUtensorMap& mp, const CUtensorMap& mq, const Args& a, int grid, size_t smem, bool early, cudaStream_t s) {
  cudaError_t e = allow_smem<mxfp4_gemm_kernel<SWAP, F16, QB>>(kSmemBudget - 1024);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (early) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (a.split > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = a.split;
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, mxfp4_gemm_kernel<SWAP, F16, QB>, mp, mq, a);
}

// Pairs take what would need a second round of 128 x 256 tiles. Measured (us with the launch, one CTA a tile / pairs):
// 256 x 14336 x 4096 20.5 / 20.5, 1152 x 4096 x 4096 (144 tiles) 18.4 / 22.6, 512 x 4096 x 4096 14.3 / 16.4, but 1024 x 4096 x
// 14336 36.9 / 32.8: many steps along K favour pairs, which the rule leaves out; 2048 x 14336 x 4096 78.8 / 61.5, 4096 x 8192 x 8192 132 / 108, 8192 x 28672 x 8192 852 / 671.
bool pairs_pay(const Mxfp4Matmul& p, int sms) {
  return p.M > kRows && ceil_div(p.M, kRows) * ceil_div(p.N, 256) > sms;
}

template <bool F16>
cudaError_t launch_pairs(const Mxfp4Matmul& p, Args a, bool early, cudaStream_t s) {
  constexpr int smem = kStages2 * kStage2 + 1024;
  cudaError_t e = allow_smem<mxfp4_gemm2_kernel<F16>>(smem);
  if (e != cudaSuccess) return e;
  a.T = 256;
  a.split = 1;
  a.p_rows = static_cast<int>(p.M);
  a.q_rows = static_cast<int>(p.N);
  a.p_tiles = static_cast<int>(ceil_div(p.M, 256));
  const int64_t tiles = a.p_tiles * ceil_div(p.N, 256);
  if (tiles > INT_MAX / 8) return cudaErrorInvalidValue;
  // A last round with few tiles takes them in halves (2048 x 14336 x 4096, 448 tiles on 74 pairs: 69.7 -> 67.6 us with the
  // launch, when it was added).
  const int pairs = device_sm_count() / 2, rest = static_cast<int>(tiles % pairs);
  const bool halve = tiles > pairs && 2 * rest <= pairs;
  a.whole = static_cast<int>(halve ? tiles - rest : tiles);
  a.tiles = static_cast<int>(halve ? tiles + rest : tiles);
  a.tiles_k = ceil_div(p.kb, 4);
  a.sp_blocks = static_cast<int>(ceil_div(p.M, kRows));
  a.sq_blocks = static_cast<int>(ceil_div(p.N, kRows));
  a.sp = p.a_scales;
  a.sq = p.b_scales;
  a.bias = p.bias;
  a.y = p.y;
  a.ldy = p.ldy;
  a.vec = (reinterpret_cast<uintptr_t>(p.y) & 15u) == 0 && (p.ldy * (p.f16 ? 2 : 4)) % 16 == 0;
  a.err = p.err;
  // Scales as rows of a tile's 512 bytes (as 2-byte elements, of which a row of a copy may have 256), two at a time.
  CUtensorMap mp, mq, msp, msq;
  const uint64_t row = static_cast<uint64_t>(p.kb) * 16;
  const int64_t sp_tiles = a.sp_blocks * a.tiles_k, sq_tiles = a.sq_blocks * a.tiles_k;
  if (sp_tiles > INT_MAX / 2 || sq_tiles > INT_MAX / 2 || !encode_tensor_map_2d(&mp, 0, p.a, row, a.p_rows, row, kStepBytes, kRows, true) ||
      !encode_tensor_map_2d(&mq, 0, p.b, row, a.q_rows, row, kStepBytes, kRows, true) ||
      !encode_tensor_map_2d(&msp, 1, a.sp, kScaleTile / 2, sp_tiles, kScaleTile, kScaleTile / 2, 2, false) ||
      !encode_tensor_map_2d(&msq, 1, a.sq, kScaleTile / 2, sq_tiles, kScaleTile, kScaleTile / 2, 2, false))
    return cudaErrorInvalidValue;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(2 * (a.tiles < pairs ? a.tiles : pairs));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = early ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, mxfp4_gemm2_kernel<F16>, mp, mq, msp, msq, a);
}

}  // namespace

cudaError_t launch_mxfp4_matmul(const Mxfp4Matmul& p, bool early, cudaStream_t s) {
  const int sms = device_sm_count();
  Args a{};
  a.k64 = static_cast<int>(ceil_div(p.kb, 2));
  a.ksteps = (a.k64 + 3) / 4;
  if (pairs_pay(p, sms)) return p.f16 ? launch_pairs<true>(p, a, early, s) : launch_pairs<false>(p, a, early, s);
  const Shape sh = choose(p, a.ksteps, sms);
  a.T = sh.T;
  a.split = sh.split;
  a.p_rows = static_cast<int>(sh.swap ? p.N : p.M);
  a.q_rows = static_cast<int>(sh.swap ? p.M : p.N);
  a.p_tiles = static_cast<int>(ceil_div(a.p_rows, kRows));
  const int64_t tiles = static_cast<int64_t>(a.p_tiles) * ceil_div(a.q_rows, a.T);
  if (tiles > INT_MAX / 8) return cudaErrorInvalidValue;
  a.tiles = static_cast<int>(tiles);
  a.q_blocks = a.T > kRows ? 2 : 1;
  a.tiles_k = ceil_div(p.kb, 4);
  a.sp_blocks = a.p_tiles;
  a.sq_blocks = static_cast<int>(ceil_div(a.q_rows, kRows));
  a.sp = sh.swap ? p.b_scales : p.a_scales;
  a.sq = sh.swap ? p.a_scales : p.b_scales;
  a.bias = p.bias;
  a.y = p.y;
  a.ldy = p.ldy;
  a.vec = (reinterpret_cast<uintptr_t>(p.y) & 15u) == 0 && (p.ldy * (p.f16 ? 2 : 4)) % 16 == 0;
  a.err = p.err;
  a.early = early;
  a.q_stage = static_cast<uint32_t>(a.T) * kStepBytes;
  a.stage = kRows * kStepBytes + a.q_stage + (1 + a.q_blocks) * 2 * kScaleTile;
  a.stage = (a.stage + 1023u) & ~1023u;
  a.sf_stage = 8 + 8 * a.q_blocks;
  const int steps = static_cast<int>(ceil_div(a.ksteps, a.split));
  const bool one_tile = a.split > 1 || a.tiles <= sms;
  int stages = (kSmemBudget - 2048) / static_cast<int>(a.stage);
  if (stages > 12) stages = 12;
  if (one_tile && stages > steps) stages = steps;
  if (a.split > 1) {  // all CTAs at once: those that share an SM share its memory
    const int together = static_cast<int>(ceil_div(static_cast<int64_t>(a.tiles) * a.split, sms));
    const int fit = (kSmemBudget / together - 2048) / static_cast<int>(a.stage);
    if (stages > fit && fit >= 2) stages = fit;
  }
  size_t smem = static_cast<size_t>(stages) * a.stage;
  const size_t partial = (static_cast<size_t>(a.T) * kPitch + kRows * (ceil_div(a.T, a.split) + 1)) * 4;
  if (a.split > 1 && smem < partial) smem = partial;
  smem += 1024;
  a.stages = stages;
  // Tensor memory: accumulators, then the stages' scales.
  const int sf = stages * a.sf_stage;
  a.acc1 = one_tile ? 0 : a.T;
  a.sf_col = a.acc1 + a.T;
  a.tmem_cols = 32;
  while (a.tmem_cols < a.sf_col + sf) a.tmem_cols *= 2;
  // CTAs that share an SM share its 512 columns: ask for enough shared memory that no more fit than those feed.
  const size_t least = static_cast<size_t>(kSmemBudget) / (kTmemCols / a.tmem_cols + 1) + 1024;
  if (smem < least) smem = least;
  const int grid = a.split > 1 ? a.tiles * a.split : (a.tiles < sms ? a.tiles : sms);

  CUtensorMap mp, mq;
  const uint64_t row = static_cast<uint64_t>(p.kb) * 16;
  if (!encode_tensor_map_2d(&mp, 0, sh.swap ? p.b : p.a, row, a.p_rows, row, kStepBytes, kRows, true) ||
      !encode_tensor_map_2d(&mq, 0, sh.swap ? p.a : p.b, row, a.q_rows, row, kStepBytes, a.T, true))
    return cudaErrorInvalidValue;
  if (sh.swap) return p.f16 ? launch<true, true, 1>(mp, mq, a, grid, smem, early, s) : launch<true, false, 1>(mp, mq, a, grid, smem, early, s);
  if (a.q_blocks == 1) return p.f16 ? launch<false, true, 1>(mp, mq, a, grid, smem, early, s) : launch<false, false, 1>(mp, mq, a, grid, smem, early, s);
  return p.f16 ? launch<false, true, 2>(mp, mq, a, grid, smem, early, s) : launch<false, false, 2>(mp, mq, a, grid, smem, early, s);
}

}  // namespace xrgpu
