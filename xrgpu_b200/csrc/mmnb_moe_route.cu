// Router of a mixture of experts: each token's top_k experts by score (ties to the lowest index, a NaN counts as -infinity),
// their weights, and the stable order of all assignments (token * top_k + rank) by expert.
//
// Choice: a warp a token. Scores become numbers of 32 bits that order like them: the upper 22 bits of a key of the
// score, then the index counted down, and the largest of the warp is taken out top_k times, from lanes that hold their best four
// sorted. That is exact for float16 (16 bits); for float32 two neighbours of the result that agree in the 22 bits, and a lane
// whose four were all taken while it has more, send the token to the exact form (whole keys, then the lowest index among equals).
// What bounds it is the latency of a token's chain of choices, about 14 instructions each (50 with whole keys): 1.3 instructions a cycle
// of 4, with 32 warps an SM. Four held instead of all: 8192 x 256 16.4 -> 15.5 us, 2000 x 1024 27.9 -> 24.8.
// Weights: exp(s - s_max) over their sum, or over the sum of all experts'.
// Order: a counting sort. Every warp counts its own tokens' experts, the counts are summed over the warps and CTAs before it, and
// each warp writes its assignments in turn from there: no atomics, so the order is always the same. Few tokens: the CTAs of one
// cluster read each other's counts; else a second kernel follows in which every CTA sums the counts of all (from L2).
// Measured (8 experts a token): 64 tokens x 128 experts 5.6 us, 1024 7.9, 32768 20.1; 8192 x 256 of float32 with weights of all 15.0
// (9.5 MB: 1.4 us at the copy rate; the choice takes 9 of them, the order 6).
#include <cuda_fp16.h>

#include "mmnb_common.cuh"
#include "mmnb_int8.h"
#include "mmnb_tcgen05.cuh"

namespace xrgpu {
namespace {

constexpr int kWarps = 32;
constexpr int kThreads = kWarps * 32;
constexpr int kClusterCtas = 8;
// Tokens that a cluster takes, one a warp (128 experts, 8 of them; us, cluster / two kernels: 64 tokens 6.4 / 8.4, 256 7.2 / 8.4, 512 9.3 / 8.4).
constexpr int64_t kClusterTokens = 256;

struct Args {
  MoeRoute p;
  int ctas;
  int per_warp;   // tokens of a warp, in a row
  int32_t* counts;  // [ctas, experts]
  Divide by_width;  // experts up to whole warps
};

// A key that orders like the score; 0 is below every score. -0 equals 0, NaN -infinity.
__device__ __forceinline__ uint32_t key_of(float x) {
  const int u = __float_as_int(x == x ? x + 0.0f : -INFINITY);
  return static_cast<uint32_t>(u ^ ((u >> 31) | static_cast<int>(0x80000000u)));
}
__device__ __forceinline__ float score_of(uint32_t key) {
  return __uint_as_float((key & 0x80000000u) ? key & 0x7fffffffu : ~key);
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  return v;
}

// The chosen experts by whole keys: lane j returns the j-th.
template <int VPL, bool F16>
__device__ __noinline__ int choose_exact(const void* scores, int64_t at0, int E, int k) {
  const int lane = threadIdx.x & 31;
  uint32_t key[VPL], best = 0;
  int at = 0, chosen = 0;
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    key[i] = lane + 32 * i < E ? key_of(load_f(scores, F16, at0 + lane + 32 * i)) : 0u;
    if (key[i] > best) {
      best = key[i];
      at = i;
    }
  }
  for (int j = 0; j < k; ++j) {
    const uint32_t m = __reduce_max_sync(~0u, best);
    const int e = static_cast<int>(__reduce_min_sync(~0u, best == m ? static_cast<unsigned>(lane + 32 * at) : ~0u));
    if (lane == j) chosen = e;
    if (lane == (e & 31)) {
      best = 0;
      at = 0;
#pragma unroll
      for (int i = 0; i < VPL; ++i) {
        if (i == (e >> 5)) key[i] = 0;
        if (key[i] > best) {
          best = key[i];
          at = i;
        }
      }
    }
  }
  return chosen;
}

__device__ __forceinline__ void exchange(uint32_t& a, uint32_t& b) {
  const uint32_t m = max(a, b);
  b = min(a, b);
  a = m;
}
__device__ __forceinline__ void sort_descending(uint32_t (&c)[1]) {}
__device__ __forceinline__ void sort_descending(uint32_t (&c)[2]) { exchange(c[0], c[1]); }
__device__ __forceinline__ void sort_descending(uint32_t (&c)[4]) {
  exchange(c[0], c[1]);
  exchange(c[2], c[3]);
  exchange(c[0], c[2]);
  exchange(c[1], c[3]);
  exchange(c[1], c[2]);
}
// The four largest of `c` and `more`, both in descending order.
__device__ __forceinline__ void keep_four(uint32_t (&c)[4], const uint32_t (&more)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) c[i] = max(c[i], more[3 - i]);  // they rise, then fall, or the other way round
  exchange(c[0], c[2]);
  exchange(c[1], c[3]);
  exchange(c[0], c[1]);
  exchange(c[2], c[3]);
}

// The choice and weights of the warp's tokens, counted into `mine` [experts]. VPL: scores a lane.
template <int VPL, bool F16>
__device__ __forceinline__ void choose(const Args& a, int64_t t0, int64_t t1, int32_t* mine) {
  constexpr int kHeld = VPL < 4 ? VPL : 4;
  const int lane = threadIdx.x & 31, E = a.p.experts, k = a.p.top_k;
  for (int64_t t = t0; t < t1; ++t) {
    float x[VPL];
    uint32_t c[kHeld];
#pragma unroll
    for (int i = 0; i < VPL; ++i) x[i] = lane + 32 * i < E ? load_f(a.p.scores, F16, t * a.p.lds + lane + 32 * i) : 0.0f;
#pragma unroll
    for (int b = 0; b < VPL; b += kHeld) {
      uint32_t more[kHeld];
#pragma unroll
      for (int i = 0; i < kHeld; ++i) {
        const int e = lane + 32 * (b + i);
        more[i] = e < E ? (key_of(x[b + i]) & ~1023u) | (1023u - e) : 0u;
      }
      sort_descending(more);
      if constexpr (VPL > kHeld) {
        if (b > 0) {
          keep_four(c, more);
          continue;
        }
      }
#pragma unroll
      for (int i = 0; i < kHeld; ++i) c[i] = more[i];
    }
    uint32_t pick = 0, last = 0;  // lane j: the j-th
    const int picks = F16 ? k : min(k + 1, E);
    for (int j = 0; j < picks; ++j) {
      const uint32_t m = __reduce_max_sync(~0u, c[0]);
      if (lane == j) pick = m;
      last = m;
      const bool taken = c[0] == m;  // one lane's
#pragma unroll
      for (int i = 0; i + 1 < kHeld; ++i) c[i] = taken ? c[i + 1] : c[i];
      if (taken) c[kHeld - 1] = 0u;
    }
    int chosen = static_cast<int>(1023u - (pick & 1023u));
    bool close = VPL > kHeld && c[0] == 0u && lane + 32 * kHeld < E;  // the lane may hold more of the chosen than it kept
    if (!F16) {
      const uint32_t next = __shfl_down_sync(~0u, pick, 1);
      close |= lane + 1 < k ? (pick ^ next) < 1024u : lane + 1 == k && picks > k && (pick ^ last) < 1024u;
    }
    if ((!F16 || VPL > kHeld) && __any_sync(~0u, close)) chosen = choose_exact<VPL, F16>(a.p.scores, t * a.p.lds, E, k);
    const float score = lane < k ? score_of(key_of(load_f(a.p.scores, F16, t * a.p.lds + chosen))) : 0.0f;
    const float best = __shfl_sync(~0u, score, 0);
    // a token whose scores are all -infinity weighs nothing
    const float w = lane < k && best > -INFINITY ? expf(score - best) : 0.0f;
    float sum = w;
    if (!a.p.normalize) {
      sum = 0.0f;
#pragma unroll
      for (int i = 0; i < VPL; ++i) sum += lane + 32 * i < E && x[i] == x[i] ? expf(x[i] - best) : 0.0f;
    }
    sum = warp_sum(sum);
    if (lane < k) {
      a.p.chosen[t * k + lane] = chosen;
      a.p.weights[t * k + lane] = best > -INFINITY ? w / sum : 0.0f;
      mine[chosen] += 1;  // a token's experts differ
    }
    __syncwarp();
  }
}

// Sum over the threads before, in the order of the threads; *total: of all.
__device__ __forceinline__ int block_scan(int v, int* part, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int s = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(~0u, s, o);
    if (lane >= o) s += u;
  }
  if (lane == 31) part[warp] = s;
  __syncthreads();
  int p = part[lane];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(~0u, p, o);
    if (lane >= o) p += u;
  }
  *total = __shfl_sync(~0u, p, 31);
  const int before = __shfl_sync(~0u, p, max(warp - 1, 0));
  return s - v + (warp ? before : 0);
}

// Places the warp's assignments. hist [kWarps][experts]: the warps' counts; total, before: counts of all CTAs and of those
// before this one for expert threadIdx.x (experts <= kThreads).
__device__ __forceinline__ void place(const Args& a, int64_t t0, int64_t t1, int32_t* hist, int total, int before, bool write_offsets) {
  __shared__ int part[32];
  const int E = a.p.experts, k = a.p.top_k, e = threadIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int all;
  const int first = block_scan(e < E ? total : 0, part, &all);
  if (e < E) {
    if (write_offsets) {
      a.p.offsets[e] = first;
      if (e == E - 1) a.p.offsets[E] = all;
    }
    int at = first + before;
#pragma unroll 8
    for (int w = 0; w < kWarps; ++w) {
      const int c = hist[w * E + e];
      hist[w * E + e] = at;
      at += c;
    }
  }
  __syncthreads();
  int32_t* mine = hist + warp * E;
  for (int64_t t = t0; t < t1; ++t) {
    if (lane < k) {
      const int c = a.p.chosen[t * k + lane], at = mine[c];
      mine[c] = at + 1;
      a.p.slots[t * k + lane] = at;
      a.p.order[at] = static_cast<int32_t>(t * k + lane);
    }
    __syncwarp();
  }
}

struct Range {
  int64_t t0, t1;
};
__device__ __forceinline__ Range tokens_of(const Args& a) {
  const int64_t first = (static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5)) * a.per_warp;
  return {min(first, a.p.tokens), min(first + a.per_warp, a.p.tokens)};
}

// CLUSTER: all CTAs are one cluster, and the kernel does the whole call.
template <int VPL, bool F16, bool CLUSTER>
__global__ void __launch_bounds__(kThreads, 1) choose_kernel(const Args a) {
  extern __shared__ int32_t hist[];
  __shared__ int32_t counts[kThreads];
  const int E = a.p.experts, e = threadIdx.x;
  for (int i = threadIdx.x; i < kWarps * E; i += kThreads) hist[i] = 0;
  __syncthreads();
  const Range r = tokens_of(a);
  choose<VPL, F16>(a, r.t0, r.t1, hist + (threadIdx.x >> 5) * E);
  __syncthreads();
  int count = 0;
  if (e < E) {
#pragma unroll 8
    for (int w = 0; w < kWarps; ++w) count += hist[w * E + e];
  }
  if (!CLUSTER) {
    if (e < E) a.counts[static_cast<int64_t>(blockIdx.x) * E + e] = count;
    return;
  }
  int total = count, before = 0;
  if (a.ctas > 1) {
    counts[e] = count;
    cluster_sync();
    total = 0;
    int c[kClusterCtas];
#pragma unroll
    for (int i = 0; i < kClusterCtas; ++i) c[i] = i < a.ctas ? ld_cluster_s32(map_rank(smem_u32(&counts[e]), i)) : 0;
#pragma unroll
    for (int i = 0; i < kClusterCtas; ++i) {
      total += c[i];
      before += i < static_cast<int>(blockIdx.x) ? c[i] : 0;
    }
    cluster_sync();  // nobody leaves while its counts are being read
  }
  place(a, r.t0, r.t1, hist, total, before, blockIdx.x == 0);
}

__global__ void __launch_bounds__(kThreads, 1) place_kernel(const Args a) {
  extern __shared__ int32_t hist[];
  __shared__ int sums[2][kThreads];
  const int E = a.p.experts, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int i = threadIdx.x; i < kWarps * E; i += kThreads) hist[i] = 0;
  __syncthreads();
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const Range r = tokens_of(a);
  for (int64_t t = r.t0; t < r.t1; ++t) {
    if (lane < a.p.top_k) hist[warp * E + a.p.chosen[t * a.p.top_k + lane]] += 1;
    __syncwarp();
  }
  // Groups of threads take every groups-th CTA's counts, an expert a thread.
  const int width = (E + 31) & ~31, groups = kThreads / a.by_width, g = static_cast<int>(threadIdx.x) / a.by_width, e = threadIdx.x - g * width;
  int total = 0, before = 0;
  if (g < groups && e < E) {
#pragma unroll 16
    for (int c = g; c < a.ctas; c += groups) {
      const int v = a.counts[static_cast<int64_t>(c) * E + e];
      total += v;
      before += c < static_cast<int>(blockIdx.x) ? v : 0;
    }
  }
  sums[0][threadIdx.x] = total;
  sums[1][threadIdx.x] = before;
  __syncthreads();
  total = before = 0;
  if (static_cast<int>(threadIdx.x) < E)
    for (int i = 0; i < groups; ++i) {
      total += sums[0][i * width + threadIdx.x];
      before += sums[1][i * width + threadIdx.x];
    }
  place(a, r.t0, r.t1, hist, total, before, blockIdx.x == 0);
}

// Tokens that one cluster takes: one a warp.
bool one_cluster(const MoeRoute& p) { return p.tokens <= kClusterTokens; }

int per_warp(const MoeRoute& p) {
  const int64_t warps = ceil_div(p.tokens, kWarps), most = one_cluster(p) ? kClusterCtas : device_sm_count();
  return static_cast<int>(ceil_div(p.tokens, kWarps * (warps < most ? warps : most)));
}

template <auto Kernel>
cudaError_t launch_kernel(const Args& a, size_t smem, int cluster, bool early, cudaStream_t s) {
  cudaError_t e = allow_smem<Kernel>(static_cast<int>(smem));
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(a.ctas);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  if (early) {
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
  } else {
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  }
  cfg.attrs = attr;
  cfg.numAttrs = early || cluster > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, Kernel, a);
}

template <int VPL, bool F16>
cudaError_t launch(const Args& a, cudaStream_t s) {
  const size_t smem = static_cast<size_t>(kWarps) * a.p.experts * 4;
  if (one_cluster(a.p)) return launch_kernel<choose_kernel<VPL, F16, true>>(a, smem, a.ctas, false, s);
  const cudaError_t e = launch_kernel<choose_kernel<VPL, F16, false>>(a, smem, 1, false, s);
  return e != cudaSuccess ? e : launch_kernel<place_kernel>(a, smem, 1, true, s);
}
template <int VPL>
cudaError_t launch(const Args& a, cudaStream_t s) {
  return a.p.f16 ? launch<VPL, true>(a, s) : launch<VPL, false>(a, s);
}

}  // namespace

uint64_t moe_route_workspace(const MoeRoute& p) {
  if (one_cluster(p)) return 0;
  return static_cast<uint64_t>(ceil_div(p.tokens, static_cast<int64_t>(kWarps) * per_warp(p))) * p.experts * 4;
}

cudaError_t launch_moe_route(const MoeRoute& p, void* ws, cudaStream_t s) {
  Args a{};
  a.p = p;
  a.per_warp = per_warp(p);
  a.ctas = static_cast<int>(ceil_div(p.tokens, static_cast<int64_t>(kWarps) * a.per_warp));
  a.counts = static_cast<int32_t*>(ws);
  a.by_width = divide_by((p.experts + 31) & ~31);
  if (p.experts <= 32) return launch<1>(a, s);
  if (p.experts <= 64) return launch<2>(a, s);
  if (p.experts <= 128) return launch<4>(a, s);
  if (p.experts <= 256) return launch<8>(a, s);
  if (p.experts <= 512) return launch<16>(a, s);
  return launch<32>(a, s);
}

}  // namespace xrgpu
