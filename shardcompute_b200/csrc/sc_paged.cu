// The bookkeeping of a paged KV cache, on the device: pages reserved for the
// new tokens of a ragged batch, pages given back, and the rotary append into
// the reserved slots.
//
// A cache is a pool of pages [n_pages, Hkv, page, hd]; request b's token i
// lives in page block_table[b][i / page] at offset i % page, and its slot is
// block_table[b][i / page] * page + i % page.  Pages that no request holds
// lie on a stack: free_pages[0 .. free_count).
#include <algorithm>

#include "sc_common.cuh"

namespace sc {

constexpr int PG_THREADS = 1024;
constexpr int PG_BATCH = 4;  // rows or pages a thread has under way
constexpr int PG_MAX_BATCH = 16384;  // a request's scan state is 12 bytes of shared memory: 192 KB

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}

// Inclusive scan over the block of two sums at once (64-bit: lengths that
// are out of range must not wrap into a plausible total).
__device__ __forceinline__ void block_scan2(long long& a, long long& b, long long (*s_w)[2]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long ua = __shfl_up_sync(0xffffffffu, a, o), ub = __shfl_up_sync(0xffffffffu, b, o);
    if (lane >= o) {
      a += ua;
      b += ub;
    }
  }
  if (lane == 31) {
    s_w[warp][0] = a;
    s_w[warp][1] = b;
  }
  __syncthreads();
  long long pa = 0, pb = 0;
  for (int w = 0; w < warp; ++w) {
    pa += s_w[w][0];
    pb += s_w[w][1];
  }
  a += pa;
  b += pb;
  __syncthreads();
}

// First index i in [0, n) with a[i] > x (a is non-decreasing, a[n - 1] > x).
__device__ __forceinline__ int first_above(const int* a, int n, int x) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (a[mid] > x)
      hi = mid;
    else
      lo = mid + 1;
  }
  return lo;
}

struct ReserveParams {
  const int32_t *lens, *new_lens, *prefix_len, *free_pages, *free_count;
  int32_t *block_table, *kv_lens, *q_start, *slots, *positions, *free_out, *status;
  int B, max_blocks, page, n_free, max_tokens;
};

// One cluster.  Every CTA scans all requests (new tokens, new pages) into its
// own shared memory, so each knows every offset and the status without a
// message; then the rows, the pages and the requests are spread over the
// cluster's threads, a row or page finding its request by binary search in
// shared memory.  The one cluster barrier separates the reads of lens and
// free_count from the writes of kv_lens and free_out, which may be the same
// arrays.  Bound by latency: launch, one round trip for the lengths, one for
// the pages.
__global__ void __launch_bounds__(PG_THREADS) paged_reserve_kernel(const ReserveParams p) {
  extern __shared__ int pg_smem[];
  int* s_end = pg_smem;            // new tokens of requests 0..b
  int* s_take = pg_smem + p.B;     // new pages of requests 0..b
  int* s_len = pg_smem + 2 * p.B;  // tokens before this step
  __shared__ long long s_w[PG_THREADS / 32][2];
  __shared__ long long s_tot[2];
  __shared__ int s_bad;
  pdl_trigger();
  pdl_wait();
  if (threadIdx.x == 0) s_bad = 0;
  __syncthreads();
  const int count = *p.free_count;
  const long long cap = (long long)p.max_blocks * p.page;
  long long end0 = 0, take0 = 0;
  for (int b0 = 0; b0 < p.B; b0 += PG_THREADS) {
    const int b = b0 + threadIdx.x;
    long long a = 0, t = 0;
    if (b < p.B) {
      const int len = p.lens[b], add = p.new_lens[b];
      const long long kv = (long long)len + add;
      int bad = 0;
      if (len < 0 || add < 0) bad |= 8;
      if (kv > cap) bad |= 2;
      if (bad) atomicOr(&s_bad, bad);
      if (!(bad & 8)) {
        a = add;
        t = (kv + p.page - 1) / p.page - ((long long)len + p.page - 1) / p.page;
      }
      s_len[b] = len;
    }
    block_scan2(a, t, s_w);
    a += end0;
    t += take0;
    if (b < p.B) {
      s_end[b] = (int)min(a, (long long)INT32_MAX);
      s_take[b] = (int)min(t, (long long)INT32_MAX);
    }
    if (threadIdx.x == PG_THREADS - 1) {
      s_tot[0] = a;
      s_tot[1] = t;
    }
    __syncthreads();
    end0 = s_tot[0];
    take0 = s_tot[1];
    __syncthreads();
  }
  const int prefix = p.prefix_len ? *p.prefix_len : 0;
  int st = s_bad;
  if (take0 > count) st |= 1;
  if (end0 > p.max_tokens) st |= 4;
  if (count < 0 || count > p.n_free) st |= 16;
  cluster_arrive();
  const int nthr = (int)cluster_size() * PG_THREADS, tid = (int)cluster_rank() * PG_THREADS + threadIdx.x;
  if (st == 0) {
    for (int n0 = tid; n0 < (int)take0; n0 += PG_BATCH * nthr) {
      int id[PG_BATCH];
#pragma unroll
      for (int i = 0; i < PG_BATCH; ++i) id[i] = n0 + i * nthr < (int)take0 ? p.free_pages[count - 1 - (n0 + i * nthr)] : 0;
#pragma unroll
      for (int i = 0; i < PG_BATCH; ++i) {
        const int n = n0 + i * nthr;
        if (n >= (int)take0) break;
        const int b = first_above(s_take, p.B, n);
        const int j = (s_len[b] + p.page - 1) / p.page + n - (b ? s_take[b - 1] : 0);
        p.block_table[(size_t)b * p.max_blocks + j] = id[i];
      }
    }
    for (int t0 = tid; t0 < (int)end0; t0 += PG_BATCH * nthr) {
      int at[PG_BATCH], id[PG_BATCH];
#pragma unroll
      for (int i = 0; i < PG_BATCH; ++i) {
        const int t = min(t0 + i * nthr, (int)end0 - 1);
        const int b = first_above(s_end, p.B, t);
        const int len = s_len[b];
        at[i] = len + t - (b ? s_end[b - 1] : 0);
        const int j = at[i] / p.page, have = (len + p.page - 1) / p.page;
        // a block of this step's is on the stack still, an older one in the table
        id[i] = j < have ? p.block_table[(size_t)b * p.max_blocks + j]
                         : p.free_pages[count - 1 - (b ? s_take[b - 1] : 0) - (j - have)];
      }
#pragma unroll
      for (int i = 0; i < PG_BATCH; ++i) {
        const int t = t0 + i * nthr;
        if (t >= (int)end0) break;
        p.slots[t] = id[i] * p.page + at[i] % p.page;
        p.positions[t] = prefix + at[i];
      }
    }
  }
  cluster_wait();
  for (int b = tid; b < p.B; b += nthr) {
    const int add = s_end[b] - (b ? s_end[b - 1] : 0);
    p.kv_lens[b] = s_len[b] + (st == 0 ? add : 0);
    p.q_start[b + 1] = st == 0 ? s_end[b] : 0;
  }
  if (tid == 0) {
    p.q_start[0] = 0;
    *p.free_out = st == 0 ? count - (int)take0 : count;
    *p.status = st;
  }
}

struct TruncateParams {
  const int32_t *lens, *keep, *block_table, *free_count;
  int32_t *free_pages, *lens_out, *free_out, *status;
  int B, max_blocks, page, n_free;
};

// The same shape as the reservation: every CTA scans how many pages each
// request gives back, then a page finds its request and goes to its place
// behind the stack's top.
__global__ void __launch_bounds__(PG_THREADS) paged_truncate_kernel(const TruncateParams p) {
  extern __shared__ int pg_smem[];
  int* s_give = pg_smem;           // pages given back by requests 0..b
  int* s_len = pg_smem + p.B;      // tokens before
  int* s_keep = pg_smem + 2 * p.B; // tokens after
  __shared__ long long s_w[PG_THREADS / 32][2];
  __shared__ long long s_tot;
  __shared__ int s_bad;
  pdl_trigger();
  pdl_wait();
  if (threadIdx.x == 0) s_bad = 0;
  __syncthreads();
  const int count = *p.free_count;
  const long long cap = (long long)p.max_blocks * p.page;
  long long give0 = 0;
  for (int b0 = 0; b0 < p.B; b0 += PG_THREADS) {
    const int b = b0 + threadIdx.x;
    long long g = 0, unused = 0;
    if (b < p.B) {
      const int len = p.lens[b];
      const int kp = min(max(p.keep[b], 0), max(len, 0));
      int bad = 0;
      if (len < 0) bad |= 8;
      if (len > cap) bad |= 2;
      if (bad)
        atomicOr(&s_bad, bad);
      else
        g = ((long long)len + p.page - 1) / p.page - ((long long)kp + p.page - 1) / p.page;
      s_len[b] = len;
      s_keep[b] = kp;
    }
    block_scan2(g, unused, s_w);
    g += give0;
    if (b < p.B) s_give[b] = (int)min(g, (long long)INT32_MAX);
    if (threadIdx.x == PG_THREADS - 1) s_tot = g;
    __syncthreads();
    give0 = s_tot;
    __syncthreads();
  }
  int st = s_bad;
  if (count < 0 || count > p.n_free)
    st |= 16;
  else if (count + give0 > p.n_free)
    st |= 1;
  cluster_arrive();
  const int nthr = (int)cluster_size() * PG_THREADS, tid = (int)cluster_rank() * PG_THREADS + threadIdx.x;
  if (st == 0) {
    for (int n0 = tid; n0 < (int)give0; n0 += PG_BATCH * nthr) {
      int id[PG_BATCH];
#pragma unroll
      for (int i = 0; i < PG_BATCH; ++i) {
        const int n = min(n0 + i * nthr, (int)give0 - 1);
        const int b = first_above(s_give, p.B, n);
        const int j = (s_keep[b] + p.page - 1) / p.page + n - (b ? s_give[b - 1] : 0);
        id[i] = p.block_table[(size_t)b * p.max_blocks + j];
      }
#pragma unroll
      for (int i = 0; i < PG_BATCH; ++i)
        if (n0 + i * nthr < (int)give0) p.free_pages[count + n0 + i * nthr] = id[i];
    }
  }
  cluster_wait();
  for (int b = tid; b < p.B; b += nthr) p.lens_out[b] = st == 0 ? s_keep[b] : s_len[b];
  if (tid == 0) {
    *p.free_out = st == 0 ? count + (int)give0 : count;
    *p.status = st;
  }
}

// Launches one cluster of `ctas` CTAs with programmatic stream serialisation.
template <typename P>
static int launch_cluster(void (*kern)(const P), int ctas, size_t smem, cudaStream_t stream, const P& p, const char* what) {
  if (smem > (48u << 10)) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return check_launch(what, e);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(PG_THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  return check_launch(what, cudaLaunchKernelEx(&cfg, kern, p));
}

// CTAs of the cluster: one per batch of rows a CTA has under way, at most the portable 8.
static int cluster_ctas(int rows) { return std::max(1, std::min(8, (rows + PG_THREADS * PG_BATCH - 1) / (PG_THREADS * PG_BATCH))); }

// ---------------------------------------------------------------- append

template <typename T>
__device__ __forceinline__ void ld4(const T* p, float (&v)[4]);
template <>
__device__ __forceinline__ void ld4<float>(const float* p, float (&v)[4]) {
  const float4 a = *reinterpret_cast<const float4*>(p);
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
}
template <>
__device__ __forceinline__ void ld4<__half>(const __half* p, float (&v)[4]) {
  const uint2 a = *reinterpret_cast<const uint2*>(p);
  const float2 x = __half22float2(u32_as_h2(a.x)), y = __half22float2(u32_as_h2(a.y));
  v[0] = x.x; v[1] = x.y; v[2] = y.x; v[3] = y.y;
}
__device__ __forceinline__ void st4(float* p, const float (&v)[4]) {
  *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
}
__device__ __forceinline__ void st4(__half* p, const float (&v)[4]) {
  *reinterpret_cast<uint2*>(p) =
      make_uint2(h2_as_u32(__floats2half2_rn(v[0], v[1])), h2_as_u32(__floats2half2_rn(v[2], v[3])));
}

struct AppendParams {
  const void* qkv;
  const int32_t *rows_end, *slots, *positions;  // rows_end: one past the last row that is used
  const float *cos_tab, *sin_tab;
  void *q_out, *k_pages, *v_pages;
  int rows, Hq, Hkv, hd, max_pos, n_pages, page;
};

// A thread takes eight values of a row: four pairs (d, d + hd/2) of a q or k
// head, rotated, or eight values of a v head.  q, k and v are rounded once, to
// the cache's type; the products of the rotation are not fused, as in
// rope_append_kernel.  Moves its bytes once; bound by HBM for many rows, by
// the launch and two dependent loads for few.
template <typename ST, typename CT>
__global__ void __launch_bounds__(256) paged_append_kernel(const AppendParams p) {
  pdl_trigger();
  pdl_wait();
  const int per_row = (p.Hq + 2 * p.Hkv) * (p.hd / 8);
  const size_t it = (size_t)blockIdx.x * blockDim.x + threadIdx.x;
  const int row = (int)(it / per_row), e = (int)(it % per_row);
  if (row >= min(p.rows, *p.rows_end)) return;
  const int per_head = p.hd / 8, half = p.hd / 2;
  const int h = e / per_head, d = (e % per_head) * 4;
  const ST* src = reinterpret_cast<const ST*>(p.qkv) + ((size_t)row * (p.Hq + 2 * p.Hkv) + h) * p.hd;
  const int pos = p.positions[row], slot = p.slots[row];
  const bool pos_ok = pos >= 0 && pos < p.max_pos;
  const bool ok = pos_ok && slot >= 0 && slot / p.page < p.n_pages;
  const int id = slot / p.page, off = slot % p.page;
  float a[4], b[4];
  if (h >= p.Hq + p.Hkv) {
    if (!ok) return;
    ld4<ST>(src + 2 * d, a);
    ld4<ST>(src + 2 * d + 4, b);
    CT* dst = reinterpret_cast<CT*>(p.v_pages) + (((size_t)id * p.Hkv + (h - p.Hq - p.Hkv)) * p.page + off) * p.hd;
    st4(dst + 2 * d, a);
    st4(dst + 2 * d + 4, b);
    return;
  }
  if (h >= p.Hq && !ok) return;
  ld4<ST>(src + d, a);
  ld4<ST>(src + d + half, b);
  float c[4] = {1.f, 1.f, 1.f, 1.f}, s[4] = {0.f, 0.f, 0.f, 0.f}, x[4], y[4];
  if (pos_ok) {
    ld4<float>(p.cos_tab + (size_t)pos * half + d, c);
    ld4<float>(p.sin_tab + (size_t)pos * half + d, s);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[i] = __fadd_rn(__fmul_rn(a[i], c[i]), __fmul_rn(-b[i], s[i]));
    y[i] = __fadd_rn(__fmul_rn(b[i], c[i]), __fmul_rn(a[i], s[i]));
  }
  CT* dst = h < p.Hq ? reinterpret_cast<CT*>(p.q_out) + ((size_t)row * p.Hq + h) * p.hd
                     : reinterpret_cast<CT*>(p.k_pages) + (((size_t)id * p.Hkv + (h - p.Hq)) * p.page + off) * p.hd;
  st4(dst + d, x);
  st4(dst + d + half, y);
}

}  // namespace sc

extern "C" {

int sc_paged_reserve(const int32_t* lens, const int32_t* new_lens, int B, const int32_t* prefix_len,
                     int32_t* block_table, int max_blocks, const int32_t* free_pages, int n_free,
                     const int32_t* free_count, int page_size, int max_tokens, int32_t* kv_lens, int32_t* q_start,
                     int32_t* slots, int32_t* positions, int32_t* free_count_out, int32_t* status,
                     cudaStream_t stream) {
  using namespace sc;
  SC_REQUIRE(lens && new_lens && block_table && free_pages && free_count && kv_lens && q_start && slots && positions &&
                 free_count_out && status,
             SC_ERR_ARG, "paged_reserve: null pointer");
  SC_REQUIRE(B >= 1 && B <= PG_MAX_BATCH, SC_ERR_SHAPE, "paged_reserve: 1..%d requests (got %d)", PG_MAX_BATCH, B);
  SC_REQUIRE(max_blocks >= 1 && n_free >= 1 && max_tokens >= 1, SC_ERR_SHAPE, "paged_reserve: empty shape");
  SC_REQUIRE(page_size >= 1 && (long long)n_free * page_size <= INT32_MAX && (long long)max_blocks * page_size <= INT32_MAX,
             SC_ERR_SHAPE, "paged_reserve: slots past 32 bits (%d pages of %d, %d blocks)", n_free, page_size, max_blocks);
  const ReserveParams p = {lens,        new_lens, prefix_len, free_pages, free_count, block_table, kv_lens, q_start, slots,
                           positions,   free_count_out, status, B, max_blocks, page_size, n_free, max_tokens};
  return launch_cluster(paged_reserve_kernel, cluster_ctas(std::max(max_tokens, B)), (size_t)B * 12, stream, p, "paged_reserve");
}

int sc_paged_truncate(const int32_t* lens, const int32_t* keep, int B, const int32_t* block_table, int max_blocks,
                      int32_t* free_pages, int n_free, const int32_t* free_count, int page_size, int32_t* lens_out,
                      int32_t* free_count_out, int32_t* status, cudaStream_t stream) {
  using namespace sc;
  SC_REQUIRE(lens && keep && block_table && free_pages && free_count && lens_out && free_count_out && status, SC_ERR_ARG,
             "paged_truncate: null pointer");
  SC_REQUIRE(B >= 1 && B <= PG_MAX_BATCH, SC_ERR_SHAPE, "paged_truncate: 1..%d requests (got %d)", PG_MAX_BATCH, B);
  SC_REQUIRE(max_blocks >= 1 && n_free >= 1, SC_ERR_SHAPE, "paged_truncate: empty shape");
  SC_REQUIRE(page_size >= 1 && (long long)n_free * page_size <= INT32_MAX && (long long)max_blocks * page_size <= INT32_MAX,
             SC_ERR_SHAPE, "paged_truncate: slots past 32 bits (%d pages of %d, %d blocks)", n_free, page_size, max_blocks);
  const TruncateParams p = {lens, keep, block_table, free_count, free_pages, lens_out, free_count_out, status, B,
                            max_blocks, page_size, n_free};
  return launch_cluster(paged_truncate_kernel, cluster_ctas(std::min(n_free, 16 * B)), (size_t)B * 12, stream, p,
                        "paged_truncate");
}

int sc_paged_rope_append(const void* qkv, int qkv_dtype, int rows, const int32_t* rows_end, const int32_t* slots,
                         const int32_t* positions, const float* cos_tab, const float* sin_tab, int max_pos, int Hq,
                         int Hkv, int hd, void* q_out, void* k_pages, void* v_pages, int cache_dtype, int n_pages,
                         int page_size, cudaStream_t stream) {
  using namespace sc;
  SC_REQUIRE(qkv && rows_end && slots && positions && cos_tab && sin_tab && q_out && k_pages && v_pages, SC_ERR_ARG,
             "paged_rope_append: null pointer");
  SC_REQUIRE(rows >= 1 && Hq >= 1 && Hkv >= 1 && n_pages >= 1 && page_size >= 1 && max_pos >= 1, SC_ERR_SHAPE,
             "paged_rope_append: empty shape");
  SC_REQUIRE(hd >= 8 && hd % 8 == 0, SC_ERR_SHAPE, "paged_rope_append: head_dim %d is not a multiple of 8", hd);
  SC_REQUIRE((long long)n_pages * page_size <= INT32_MAX, SC_ERR_SHAPE, "paged_rope_append: slots past 32 bits");
  SC_REQUIRE((qkv_dtype == SC_F16 || qkv_dtype == SC_F32) && (cache_dtype == SC_F16 || cache_dtype == SC_F32), SC_ERR_ARG,
             "paged_rope_append: dtype");
  SC_REQUIRE((((uintptr_t)qkv | (uintptr_t)q_out | (uintptr_t)k_pages | (uintptr_t)v_pages | (uintptr_t)cos_tab |
               (uintptr_t)sin_tab) & 15) == 0,
             SC_ERR_ARG, "paged_rope_append: tensors must start on 16-byte boundaries");
  const size_t blocks = ((size_t)rows * (Hq + 2 * Hkv) * (hd / 8) + 255) / 256;
  SC_REQUIRE(blocks <= INT32_MAX, SC_ERR_SHAPE, "paged_rope_append: %d rows are too many for one launch", rows);
  const AppendParams p = {qkv, rows_end, slots, positions, cos_tab, sin_tab, q_out, k_pages, v_pages,
                          rows, Hq, Hkv, hd, max_pos, n_pages, page_size};
  auto kern = qkv_dtype == SC_F32 ? (cache_dtype == SC_F32 ? paged_append_kernel<float, float> : paged_append_kernel<float, __half>)
                                  : (cache_dtype == SC_F32 ? paged_append_kernel<__half, float> : paged_append_kernel<__half, __half>);
  ::sc::launch(kern, dim3((unsigned)blocks), dim3(256), 0, stream, p);
  return check_launch("paged_rope_append");
}

}  // extern "C"
