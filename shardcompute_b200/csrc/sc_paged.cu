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
// Consecutive rows or pages of a thread.  Reservation: one while the cluster's threads last (8 requests, 8 rows: 8 4.3 us,
// 1 3.0 us), else eight (1500 requests, 38000 rows: 4 11.4 us, 8 9.4 us).  Truncation, whose pages lie in many requests'
// tables (1024 requests, 7000 pages): 8 8.8 us, 4 5.4 us, 2 5.1 us.
constexpr int PG_RUN = 8, PG_RUN_BACK = 2;
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
  long long pa = lane < warp ? s_w[lane][0] : 0, pb = lane < warp ? s_w[lane][1] : 0;
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    pa += __shfl_xor_sync(0xffffffffu, pa, o);
    pb += __shfl_xor_sync(0xffffffffu, pb, o);
  }
  a += pa;
  b += pb;
  __syncthreads();
}

// x / d for 0 <= x < 2^31 by a product: m = floor(2^(31 + l) / d) + 1 with l = ceil(log2 d) is off by less than
// 2^-(31 + l) relative to 1 / d, too little to reach the next whole number.
struct PageDiv {
  unsigned long long m;
  int d, sh;
  __device__ __forceinline__ int div(int x) const { return (int)(((unsigned long long)(unsigned)x * m) >> sh); }
  __device__ __forceinline__ int up(int x) const { return x > 0 ? div(x - 1) + 1 : 0; }
};
static PageDiv page_div(int d) {
  int l = 0;
  while ((1ll << l) < d) ++l;
  return {(1ull << (31 + l)) / (unsigned)d + 1, d, 31 + l};
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
  int B, max_blocks, n_free, max_tokens;
  PageDiv page;
};

// One cluster.  Every CTA scans all requests (new tokens, new pages) into its
// own shared memory, so each knows every offset and the status without a
// message; then the rows, the pages and the requests are spread over the
// cluster's threads, a run of rows or pages a thread, which finds the
// first one's request by binary search in shared memory and walks on.  The one cluster barrier separates the reads of lens and
// free_count from the writes of kv_lens and free_out, which may be the same
// arrays.  Bound by latency: launch, one round trip for the lengths, one for
// the pages.
template <int RUN>
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
  const int count = *p.free_count, prefix = p.prefix_len ? *p.prefix_len : 0;
  const long long cap = (long long)p.max_blocks * p.page.d;
  // a thread takes consecutive requests: its own sums, one scan of those, then the sums up to each request
  const int each = (p.B + blockDim.x - 1) / blockDim.x, b_lo = min(p.B, (int)threadIdx.x * each), b_hi = min(p.B, b_lo + each);
  long long end0 = 0, take0 = 0;
  int bad = 0;
  for (int b = b_lo; b < b_hi; ++b) {
    const int len = p.lens[b], add = p.new_lens[b];
    const long long kv = (long long)len + add;
    int a = 0, t = 0;
    if (len < 0 || add < 0) {
      bad |= 8;
    } else {
      a = add;
      // past 32 bits only where it does not fit the table either
      t = kv <= INT32_MAX ? p.page.up((int)kv) - p.page.up(len) : (int)((kv - len) / p.page.d);
    }
    if (kv > cap) bad |= 2;
    s_len[b] = len;
    s_end[b] = a;
    s_take[b] = t;
    end0 += a;
    take0 += t;
  }
  if (bad) atomicOr(&s_bad, bad);
  long long ea = end0, ta = take0;
  block_scan2(ea, ta, s_w);
  if (threadIdx.x == blockDim.x - 1) {
    s_tot[0] = ea;
    s_tot[1] = ta;
  }
  ea -= end0;
  ta -= take0;
  for (int b = b_lo; b < b_hi; ++b) {
    ea += s_end[b];
    ta += s_take[b];
    s_end[b] = (int)min(ea, (long long)INT32_MAX);
    s_take[b] = (int)min(ta, (long long)INT32_MAX);
  }
  __syncthreads();
  end0 = s_tot[0];
  take0 = s_tot[1];
  int st = s_bad;
  if (take0 > count) st |= 1;
  if (end0 > p.max_tokens) st |= 4;
  if (count < 0 || count > p.n_free) st |= 16;
  cluster_arrive();
  const int nthr = (int)cluster_size() * blockDim.x, tid = (int)cluster_rank() * blockDim.x + threadIdx.x;
  const bool wide = (((uintptr_t)p.slots | (uintptr_t)p.positions) & 15) == 0;
  if (st == 0) {
    // the pages by the threads from the cluster's other end: few are needed, and the rows' are busy
    for (int n0 = (nthr - 1 - tid) * RUN; n0 < (int)take0; n0 += RUN * nthr) {
      int b = first_above(s_take, p.B, n0);
#pragma unroll
      for (int i = 0; i < RUN; ++i) {
        const int n = n0 + i;
        if (n >= (int)take0) break;
        while (s_take[b] <= n) ++b;
        const int j = p.page.up(s_len[b]) + n - (b ? s_take[b - 1] : 0);
        p.block_table[(size_t)b * p.max_blocks + j] = p.free_pages[count - 1 - n];
      }
    }
    for (int t0 = tid * RUN; t0 < (int)end0; t0 += RUN * nthr) {
      int b = first_above(s_end, p.B, t0);
      int at[RUN], off[RUN], id[RUN];
#pragma unroll
      for (int i = 0; i < RUN; ++i) {
        const int t = min(t0 + i, (int)end0 - 1);
        while (s_end[b] <= t) ++b;
        const int len = s_len[b];
        at[i] = len + t - (b ? s_end[b - 1] : 0);
        const int j = p.page.div(at[i]), have = p.page.up(len);
        off[i] = at[i] - j * p.page.d;
        // a block of this step's is on the stack still, an older one in the table
        id[i] = j < have ? p.block_table[(size_t)b * p.max_blocks + j]
                         : p.free_pages[count - 1 - (b ? s_take[b - 1] : 0) - (j - have)];
      }
      if (RUN >= 4 && wide && t0 + RUN <= (int)end0) {
#pragma unroll
        for (int i = 0; i + 3 < RUN; i += 4) {
          *reinterpret_cast<int4*>(p.slots + t0 + i) = make_int4(id[i] * p.page.d + off[i], id[i + 1] * p.page.d + off[i + 1],
                                                                 id[i + 2] * p.page.d + off[i + 2], id[i + 3] * p.page.d + off[i + 3]);
          *reinterpret_cast<int4*>(p.positions + t0 + i) =
              make_int4(prefix + at[i], prefix + at[i + 1], prefix + at[i + 2], prefix + at[i + 3]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < RUN; ++i) {
          if (t0 + i >= (int)end0) break;
          p.slots[t0 + i] = id[i] * p.page.d + off[i];
          p.positions[t0 + i] = prefix + at[i];
        }
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
  int B, max_blocks, n_free;
  PageDiv page;
};

// The same shape as the reservation: every CTA scans how many pages each
// request gives back, then a page finds its request and goes to its place
// behind the stack's top.  Bound by latency as that is (1024 requests 4.7 us).
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
  const long long cap = (long long)p.max_blocks * p.page.d;
  const int each = (p.B + blockDim.x - 1) / blockDim.x, b_lo = min(p.B, (int)threadIdx.x * each), b_hi = min(p.B, b_lo + each);
  long long give0 = 0, unused = 0;
  int bad = 0;
  for (int b = b_lo; b < b_hi; ++b) {
    const int len = p.lens[b];
    const int kp = min(max(p.keep[b], 0), max(len, 0));
    int g = 0;
    if (len < 0)
      bad |= 8;
    else if (len > cap)
      bad |= 2;
    else
      g = p.page.up(len) - p.page.up(kp);
    s_len[b] = len;
    s_keep[b] = kp;
    s_give[b] = g;
    give0 += g;
  }
  if (bad) atomicOr(&s_bad, bad);
  long long ga = give0;
  block_scan2(ga, unused, s_w);
  if (threadIdx.x == blockDim.x - 1) s_tot = ga;
  ga -= give0;
  for (int b = b_lo; b < b_hi; ++b) {
    ga += s_give[b];
    s_give[b] = (int)min(ga, (long long)INT32_MAX);
  }
  __syncthreads();
  give0 = s_tot;
  int st = s_bad;
  if (count < 0 || count > p.n_free)
    st |= 16;
  else if (count + give0 > p.n_free)
    st |= 1;
  cluster_arrive();
  const int nthr = (int)cluster_size() * blockDim.x, tid = (int)cluster_rank() * blockDim.x + threadIdx.x;
  if (st == 0) {
    for (int n0 = tid * PG_RUN_BACK; n0 < (int)give0; n0 += PG_RUN_BACK * nthr) {
      int b = first_above(s_give, p.B, n0), id[PG_RUN_BACK];
#pragma unroll
      for (int i = 0; i < PG_RUN_BACK; ++i) {
        const int n = min(n0 + i, (int)give0 - 1);
        while (s_give[b] <= n) ++b;
        id[i] = p.block_table[(size_t)b * p.max_blocks + p.page.up(s_keep[b]) + n - (b ? s_give[b - 1] : 0)];
      }
#pragma unroll
      for (int i = 0; i < PG_RUN_BACK; ++i)
        if (n0 + i < (int)give0) p.free_pages[count + n0 + i] = id[i];
    }
  }
  cluster_wait();
  for (int b = tid; b < p.B; b += nthr) p.lens_out[b] = st == 0 ? s_keep[b] : s_len[b];
  if (tid == 0) {
    *p.free_out = st == 0 ? count + (int)give0 : count;
    *p.status = st;
  }
}

// Launches one cluster with programmatic stream serialisation, for `items` rows or pages at most: CTAs of up to 1024
// threads, up to the portable 8.
template <typename P>
static int launch_cluster(void (*kern)(const P), int items, int run, size_t smem, cudaStream_t stream, const P& p, const char* what) {
  if (smem > (48u << 10)) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return check_launch(what, e);
  }
  const long long threads = ((long long)items + run - 1) / run;
  const int ctas = (int)std::max(1ll, std::min(8ll, (threads + PG_THREADS - 1) / PG_THREADS));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3((unsigned)std::max(128ll, std::min((long long)PG_THREADS, (std::max(threads, (long long)p.B) + 31) / 32 * 32)));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchAttribute& cl = attr[pdl_enabled() ? 1 : 0];
  cl.id = cudaLaunchAttributeClusterDimension;
  cl.val.clusterDim.x = ctas;
  cl.val.clusterDim.y = cl.val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = (pdl_enabled() ? 1 : 0) + (ctas > 1 ? 1 : 0);  // a CTA alone is a cluster without being told
  return check_launch(what, cudaLaunchKernelEx(&cfg, kern, p));
}

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
  int row0, items, Hq, Hkv, hd, max_pos, n_pages;
  PageDiv page, per_row, per_head;  // items of a row, of a head
};

constexpr int AP_ITEMS = 2;  // of a thread

// An item is eight values of a row: four pairs (d, d + hd/2) of a q or k
// head, rotated, or eight values of a v head.  q, k and v are rounded once, to
// the cache's type; the products of the rotation are not fused, as in
// rope_append_kernel.  Moves its bytes once; bound by HBM for many rows, by
// the launch and two dependent loads for few (8150 rows of 40 heads of 64, fp32:
// 169 MB in 30.8 us, 5.5 TB/s).
template <typename ST, typename CT>
__global__ void __launch_bounds__(256) paged_append_kernel(const AppendParams p) {
  pdl_trigger();
  pdl_wait();
  const int end = *p.rows_end;
  const int half = p.hd / 2;
  int row[AP_ITEMS], h[AP_ITEMS], d[AP_ITEMS], pos[AP_ITEMS], slot[AP_ITEMS];
  bool live[AP_ITEMS];
  float a[AP_ITEMS][4], b[AP_ITEMS][4], c[AP_ITEMS][4], s[AP_ITEMS][4];
#pragma unroll
  for (int i = 0; i < AP_ITEMS; ++i) {
    const int it = (blockIdx.x * AP_ITEMS + i) * 256 + threadIdx.x;
    live[i] = it < p.items;
    const int r = live[i] ? p.per_row.div(it) : 0, e = it - r * p.per_row.d;
    row[i] = p.row0 + r;
    live[i] = live[i] && row[i] < end;
    h[i] = live[i] ? p.per_head.div(e) : 0;
    d[i] = (e - h[i] * p.per_head.d) * 4;
    pos[i] = slot[i] = -1;
    if (live[i]) {
      pos[i] = p.positions[row[i]];
      slot[i] = p.slots[row[i]];
      const ST* src = reinterpret_cast<const ST*>(p.qkv) + ((size_t)row[i] * (p.Hq + 2 * p.Hkv) + h[i]) * p.hd;
      const bool v = h[i] >= p.Hq + p.Hkv;  // a v head: eight values in a row, from 2 d
      ld4<ST>(src + (v ? 2 * d[i] : d[i]), a[i]);
      ld4<ST>(src + (v ? 2 * d[i] + 4 : d[i] + half), b[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < AP_ITEMS; ++i) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      c[i][k] = 1.f;
      s[i][k] = 0.f;
    }
    if (live[i] && h[i] < p.Hq + p.Hkv && pos[i] >= 0 && pos[i] < p.max_pos) {
      ld4<float>(p.cos_tab + (size_t)pos[i] * half + d[i], c[i]);
      ld4<float>(p.sin_tab + (size_t)pos[i] * half + d[i], s[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < AP_ITEMS; ++i) {
    if (!live[i]) continue;
    const int id = slot[i] >= 0 ? p.page.div(slot[i]) : p.n_pages, off = slot[i] - id * p.page.d;
    const bool ok = pos[i] >= 0 && pos[i] < p.max_pos && id < p.n_pages;
    if (h[i] >= p.Hq && !ok) continue;
    if (h[i] >= p.Hq + p.Hkv) {
      CT* dst = reinterpret_cast<CT*>(p.v_pages) + (((size_t)id * p.Hkv + (h[i] - p.Hq - p.Hkv)) * p.page.d + off) * p.hd;
      st4(dst + 2 * d[i], a[i]);
      st4(dst + 2 * d[i] + 4, b[i]);
      continue;
    }
    float x[4], y[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      x[k] = __fadd_rn(__fmul_rn(a[i][k], c[i][k]), __fmul_rn(-b[i][k], s[i][k]));
      y[k] = __fadd_rn(__fmul_rn(b[i][k], c[i][k]), __fmul_rn(a[i][k], s[i][k]));
    }
    CT* dst = h[i] < p.Hq ? reinterpret_cast<CT*>(p.q_out) + ((size_t)row[i] * p.Hq + h[i]) * p.hd
                          : reinterpret_cast<CT*>(p.k_pages) + (((size_t)id * p.Hkv + (h[i] - p.Hq)) * p.page.d + off) * p.hd;
    st4(dst + d[i], x);
    st4(dst + d[i] + half, y);
  }
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
                           positions,   free_count_out, status, B, max_blocks, n_free, max_tokens, page_div(page_size)};
  const bool thin = max_tokens <= 8 * PG_THREADS;
  return launch_cluster(thin ? paged_reserve_kernel<1> : paged_reserve_kernel<PG_RUN>, max_tokens, thin ? 1 : PG_RUN, (size_t)B * 12, stream,
                        p, "paged_reserve");
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
                            max_blocks, n_free, page_div(page_size)};
  return launch_cluster(paged_truncate_kernel, std::min(n_free, 16 * B), PG_RUN_BACK, (size_t)B * 12, stream, p,
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
  SC_REQUIRE(((long long)Hq + 2 * Hkv) * (hd / 8) <= (1 << 24), SC_ERR_SHAPE, "paged_rope_append: rows of %d heads are too wide", Hq + 2 * Hkv);
  const int per_row = (Hq + 2 * Hkv) * (hd / 8), most = (1 << 30) / per_row;  // rows of a launch: items stay below 2^30
  for (int row0 = 0; row0 < rows; row0 += std::min(most, rows - row0)) {
    const int n = std::min(most, rows - row0);
    const AppendParams p = {qkv,   rows_end,    slots, positions, cos_tab, sin_tab, q_out,   k_pages,
                            v_pages, row0, n * per_row, Hq,    Hkv,       hd,      max_pos, n_pages, page_div(page_size),
                            page_div(per_row), page_div(hd / 8)};
    auto kern = qkv_dtype == SC_F32 ? (cache_dtype == SC_F32 ? paged_append_kernel<float, float> : paged_append_kernel<float, __half>)
                                    : (cache_dtype == SC_F32 ? paged_append_kernel<__half, float> : paged_append_kernel<__half, __half>);
    ::sc::launch(kern, dim3((unsigned)((p.items + 256 * AP_ITEMS - 1) / (256 * AP_ITEMS))), dim3(256), 0, stream, p);
    const int st = check_launch("paged_rope_append");
    if (st != SC_OK) return st;
  }
  return SC_OK;
}

}  // extern "C"
