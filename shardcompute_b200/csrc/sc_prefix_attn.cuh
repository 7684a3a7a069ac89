// What the attention kernels over paged caches share: rows and keys of a call,
// running softmax references, the joins of partial results, launch helpers.
#pragma once

#include <algorithm>
#include <atomic>

#include "sc_common.cuh"

namespace sc {

constexpr uint64_t PA_WAIT_NS = 2000000000ull;

// Weights on their way through fp16: a row's reference m lies PA_LIFT below a score that was its largest, in powers of
// two, and is raised when one comes to lie PA_LIFT + PA_RAISE above it.  Its weights 2^(c s - m) then reach 2^11 to
// 2^15, half of fp16's range, and keep their 11 bits down to 2^-14.  With a largest weight of 1 to 2^8 in place of that
// thousands of keys 2^-25 below it vanished from the output, though not from the sum that divides it: 16384 keys behind
// one that takes most of the weight and has a value of zero came out 8.6e-2 off, now 1.8e-4 (the output's own rounding).
constexpr float PA_LIFT = 11.f, PA_RAISE = 4.f;

// Where a row's reference m is this far from zero, c s - m in one rounding is no longer small at the largest score: m is
// c s rounded, by up to half of fp32's step there (a weight of 2^16 at m = 2^24, past fp16, and of 2^128 at 2^31).
// There c s is rounded by itself, as it was for m, so that the largest weight is what m was chosen for.
constexpr float PA_FAR = 1048576.f;
__device__ __forceinline__ float far_exponent(float s, float c, float m) {
  const float d = __fsub_rn(__fmul_rn(s, c), m);
  return d > PA_LIFT + PA_RAISE ? PA_LIFT + PA_RAISE : d;  // m - PA_LIFT is rounded as well; a NaN stays
}

// Raised by a kernel whose bounded wait ran out; each source file has its own,
// read by sc_prefix_attn_device_error.
static __device__ int g_prefix_attn_error = 0;
int quant_attn_device_error(int reset);  // that of sc_quant_attn.cu

struct PrefixAttnParams {
  const void* q;       // [T, Hq * HD] in the cache's type (fp16 over codes)
  void* out;           // [T, Hq * HD] in that type
  float* part_o;       // [nslots, T * Hq, HD]: sum of 2^(c (s - m)) v
  float2* part_ml;     // [nslots, T * Hq]: (c m, sum of 2^(c (s - m))); (-inf, 0) where the slot saw no key
  const int32_t *q_start, *kv_lens, *block_table, *prefix_table, *prefix_len;
  int T, B, max_blocks, max_prefix_blocks, n_pages, lg_page, Hq, Hkv, G;
  int pool_rows;       // n_pages * Hkv * page: one past the last row of the pools' tensor maps
  float c;             // scale * log2(e)
  int nslots;          // partial results per row, all kernels of the call together
  int beside;          // many_rows_kernel with TWO: runs beside the one without
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The request's rows [lo, hi) in q, clamped so that no device value leads out of bounds, and its new tokens, which are
// more where q ends before them.
__device__ __forceinline__ void request_rows(const PrefixAttnParams& p, int b, int& lo, int& hi, int& n) {
  const int from = max(p.q_start[b], 0), to = max(p.q_start[b + 1], from);
  lo = min(from, p.T);
  hi = min(to, p.T);
  n = to - from;
}
__device__ __forceinline__ int request_len(const PrefixAttnParams& p, int b) {
  const long long cap = (long long)p.max_blocks << p.lg_page;
  return (int)min((long long)max(p.kv_lens[b], 0), cap);
}
__device__ __forceinline__ int prefix_keys(const PrefixAttnParams& p) {
  if (!p.prefix_len) return 0;
  const long long cap = (long long)p.max_prefix_blocks << p.lg_page;
  return (int)min((long long)max(*p.prefix_len, 0), cap);
}

constexpr int FR_WARPS = 4;     // of a CTA of a few-rows kernel
constexpr int FR_CLUSTER = 8;  // shares of the keys that a cluster joins, at most

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// A value at shared address `a` of the cluster's CTA `rank`.
template <typename V>
__device__ __forceinline__ V ld_peer(uint32_t a, int rank) {
  V v;
  uint32_t at;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(a), "r"(rank));
  if constexpr (sizeof(V) == 16)
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory");
  else
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(at) : "memory");
  return v;
}

// Four outputs: the sums over their weights'.
template <typename T>
__device__ __forceinline__ void store_out(T* dst, const float4& acc, float L) {
  const float inv = L == 0.f ? 0.f : 1.f / L;
  if constexpr (sizeof(T) == 2)
    *reinterpret_cast<uint2*>(dst) = make_uint2(h2_as_u32(__floats2half2_rn(acc.x * inv, acc.y * inv)),
                                                h2_as_u32(__floats2half2_rn(acc.z * inv, acc.w * inv)));
  else
    *reinterpret_cast<float4*>(dst) = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
}

// CTA `rank` of a cluster of `size`: its part of the outputs of a tile of nr rows from the CTAs' results, (m, l) at
// shared address ml_u and o at o_u of each.
template <typename T, int HD>
__device__ __forceinline__ void join_cluster(const PrefixAttnParams& p, uint32_t ml_u, uint32_t o_u, int rank, int size, int nr, int row_lo,
                                             int r0, int h) {
  for (int e = rank * FR_WARPS * 32 + threadIdx.x; e < nr * (HD / 4); e += size * FR_WARPS * 32) {
    const int r = e / (HD / 4), d = (e % (HD / 4)) * 4;
    float2 ml[FR_CLUSTER];
    float4 v[FR_CLUSTER];
    float M = -INFINITY, L = 0.f;
#pragma unroll
    for (int w = 0; w < FR_CLUSTER; ++w) {
      ml[w] = make_float2(-INFINITY, 0.f);
      if (w < size) {
        ml[w] = ld_peer<float2>(ml_u + r * 8, w);
        v[w] = ld_peer<float4>(o_u + (r * HD + d) * 4, w);
      }
      M = fmaxf(M, ml[w].x);
    }
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < FR_CLUSTER; ++w) {
      if (ml[w].x == -INFINITY && ml[w].y == 0.f) continue;
      const float f = ex2(ml[w].x - M);
      acc.x += f * v[w].x;
      acc.y += f * v[w].y;
      acc.z += f * v[w].z;
      acc.w += f * v[w].w;
      L += f * ml[w].y;
    }
    const size_t row = (size_t)(row_lo + (r0 + r) / p.G) * p.Hq + h * p.G + (r0 + r) % p.G;
    store_out(reinterpret_cast<T*>(p.out) + row * HD + d, acc, L);
  }
}

// ---------------------------------------------------------------- join

// One warp per (row, head).  Lane s holds slot s's weight 2^(m_s - M), so the slots' sums are read without waiting for
// one another.  Reads each partial result once, from L2; bound by latency (64 rows, 32 heads of 128, 6 slots: 6.3 MB in
// 5.2 us).
template <typename T, int HD>
__global__ void __launch_bounds__(256) join_slots_kernel(const PrefixAttnParams p) {
  pdl_trigger();
  pdl_wait();
  const int row = blockIdx.x * (blockDim.x / 32) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (row >= p.T * p.Hq) return;
  const int end = p.q_start[p.B];  // on its way together with the weights
  const size_t stride = (size_t)p.T * p.Hq;
  constexpr int V = HD / 32, SETS = 3;  // at most 96 slots
  float2 ml[SETS];
  float M = -INFINITY;
#pragma unroll
  for (int k = 0; k < SETS; ++k) {
    ml[k] = k * 32 + lane < p.nslots ? p.part_ml[(k * 32 + lane) * stride + row] : make_float2(-INFINITY, 0.f);
    M = fmaxf(M, ml[k].x);
  }
  if (row >= min(max(end, 0), p.T) * p.Hq) return;
#pragma unroll
  for (int d = 16; d; d >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, d));
  float acc[V], L = 0.f;
#pragma unroll
  for (int i = 0; i < V; ++i) acc[i] = 0.f;
#pragma unroll
  for (int k = 0; k < SETS; ++k) {
    const float f = ml[k].x == -INFINITY && ml[k].y == 0.f ? 0.f : ex2(ml[k].x - M);  // 0: no key, nothing was written
    L += f * ml[k].y;
    const int n = min(32, p.nslots - k * 32);
#pragma unroll 4
    for (int s = 0; s < n; ++s) {
      const float fs = __shfl_sync(0xffffffffu, f, s);
      if (fs == 0.f) continue;
      const float* src = p.part_o + ((k * 32 + s) * stride + row) * HD + lane * V;
      if constexpr (V == 4) {
        const float4 v = *reinterpret_cast<const float4*>(src);
        acc[0] += fs * v.x; acc[1] += fs * v.y; acc[2] += fs * v.z; acc[3] += fs * v.w;
      } else {
        const float2 v = *reinterpret_cast<const float2*>(src);
        acc[0] += fs * v.x; acc[1] += fs * v.y;
      }
    }
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) L += __shfl_xor_sync(0xffffffffu, L, d);
  const float inv = L == 0.f ? 0.f : 1.f / L;
  T* dst = reinterpret_cast<T*>(p.out) + (size_t)row * HD + lane * V;
#pragma unroll
  for (int i = 0; i < V; ++i) acc[i] *= inv;
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int i = 0; i < V; i += 2) *reinterpret_cast<__half2*>(dst + i) = __floats2half2_rn(acc[i], acc[i + 1]);
  } else if constexpr (V == 4) {
    *reinterpret_cast<float4*>(dst) = make_float4(acc[0], acc[1], acc[2], acc[3]);
  } else {
    *reinterpret_cast<float2*>(dst) = make_float2(acc[0], acc[1]);
  }
}

// ---------------------------------------------------------------- host side

// Shared-memory opt-in of a kernel, once per device.
template <auto KERN>
static cudaError_t opt_in(int smem) {
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  cudaGetDevice(&dev);
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (done.load(std::memory_order_acquire) & bit) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(KERN, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_release);
  return e;
}

struct AttnPlan {
  enum Kind { FEW, SHARED, CHUNKS } kind;
  int splits, row_groups;       // few_rows_kernel
  bool cluster;                 // its shares are joined in a cluster
  int tc_splits, tc_items;      // many_rows_kernel, many_rows_f32_kernel
  int nslots;
};

}  // namespace sc
