// Attention of a ragged batch over a paged cache whose requests share a
// prefix: row i of request b (n new tokens, len tokens with them) sees the
// prefix's keys [0, P) and its own tokens [0, len - n + i].
//
//   o = sum_j exp(scale q.k_j - m) v_j / sum_j exp(scale q.k_j - m)
//
// over the keys it sees; m is any bound of the exponents, so a key range can
// be summed apart (o, l, m) and joined later.  A row that sees no key is zero.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include <cuda.h>
#include <cudaTypedefs.h>

#include "sc_tc.cuh"

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

// Raised by a kernel whose bounded wait ran out; read by
// sc_prefix_attn_device_error.
__device__ int g_prefix_attn_error = 0;

struct PrefixAttnParams {
  const void* q;       // [T, Hq * HD] in the cache's type
  void* out;           // [T, Hq * HD] in the cache's type
  float* part_o;       // [nslots, T * Hq, HD]: sum of 2^(c (s - m)) v
  float2* part_ml;     // [nslots, T * Hq]: (c m, sum of 2^(c (s - m))); (-inf, 0) where the slot saw no key
  const int32_t *q_start, *kv_lens, *block_table, *prefix_table, *prefix_len;
  int T, B, max_blocks, max_prefix_blocks, n_pages, lg_page, Hq, Hkv, G;
  int pool_rows;       // n_pages * Hkv * page: one past the last row of the pools' tensor maps
  float c;             // scale * log2(e)
  int nslots;          // partial results per row, all kernels of the call together
};

struct PoolMaps {
  CUtensorMap k, v;
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

// Copy of a box of pool rows, from 128-byte column `chunk` on, into shared memory, completing on `bar`.
__device__ __forceinline__ void tma3d_at(uint32_t dst, const CUtensorMap* map, int row, int chunk, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::
          "r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(row), "r"(chunk), "r"(smem_u32(bar))
      : "memory");
}
// ---------------------------------------------------------------- few rows

// Kernel for few rows per request.  A CTA takes a request, a kv head, a share
// of the keys and every row_groups-th tile of rows; its warps take tiles of 16 (fp32: 8) keys in turn, each with its own
// ring of tiles in shared memory (a TMA copy per 16 or 8 keys, which never
// straddle a page) and its own running (m, l, o), so no barrier
// stands in the loop.  The warps' results are joined at the end, and with
// CLUSTER those of the CTAs that share a request's keys, each CTA a part of the
// outputs from all the CTAs' shared memory: no partial results in memory, no
// kernel after this one (four requests behind 500 tokens 12.3 -> 7.6 us).
// Few keys: bound by latency, three dependent loads before the first tile and
// the joins.  Many: by the stream of keys, 64 requests of up to 1500 tokens, 8 kv
// heads of 128, with the join 42 us in fp16 and 76 us in fp32 (4.8 and 4.7 TB/s).
//
// fp16: mma m16n8k16 over up to 16 rows (the request's tokens x the group's
// heads).  P is rounded to fp16 for the second product, 2^11 to 2^15 high
// (PA_LIFT): 2^-11 of each weight, on the order of the output's own rounding,
// down to weights of 2^-25 of the row's largest, and steps of 2^-35 of that
// below, where fp16 has no more bits.
// fp32: every operand is split into two tf32 parts (split_tf32); up to 8 rows
// lie in the 16-row fragment as [hi; lo], so two tf32 products (with K's hi
// and its lo) give all four terms.  The tensor cores cut their sums off, always
// towards zero, so a tile's products are added to o outside of them (in them,
// 16000 keys left out 2.4e-6 of o).  A value that is not finite gives NaN.
constexpr int FR_WARPS = 4;
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

template <typename T, int HD>
struct FewRows {
  static constexpr bool F16 = sizeof(T) == 2;
  static constexpr int RT = F16 ? 16 : 8;               // rows per tile
  static constexpr int KT = F16 ? 16 : 8;               // keys per tile
  static constexpr int NJ = KT / 8;                     // 8-key blocks of the product
  static constexpr int NB = HD * (int)sizeof(T) / 128;  // 128-byte chunks per key
  static constexpr int SUB = KT * 128;                  // bytes of a chunk of a tile
  static constexpr int TILE = NB * SUB;                 // bytes of a K or V tile
  static constexpr int STAGE = 2 * TILE;
  static constexpr int NST = HD == 128 ? 3 : 6;         // stages per warp: 96 KB a CTA, two CTAs an SM
  static constexpr int SMEM = FR_WARPS * NST * STAGE + 1024;
  static constexpr float LIFT = F16 ? PA_LIFT : 0.f, RAISE = F16 ? PA_RAISE : 8.f;  // tf32 has fp32's range
};

__device__ __forceinline__ void ldsm4(uint32_t a, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a));
}
__device__ __forceinline__ void ldsm4_t(uint32_t a, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a));
}
// D(16x8, fp32) += A(16x8, tf32) * B(8x8, tf32); the operands' low 13 bits are not used.
__device__ __forceinline__ void mma_1688(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// x = hi + lo: hi is x rounded to tf32's 11 bits, lo the exact rest, of which the products use 11 bits too (what
// they drop is below 2^-21 of x, on either side of zero).  An x that is not finite has a lo that is NaN.
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo) {
  hi = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
  lo = __float_as_uint(x - __uint_as_float(hi));
}

// Whether one of 16 bytes' values (fp16 or fp32) has all bits of its exponent set.
template <typename T>
__device__ __forceinline__ bool not_finite(const uint4& v) {
  constexpr uint32_t mask = sizeof(T) == 2 ? 0x7c007c00u : 0x7f800000u, one = sizeof(T) == 2 ? 0x04000400u : 0x00800000u,
                     top = sizeof(T) == 2 ? 0x80008000u : 0x80000000u;
  return ((((v.x & mask) + one) | ((v.y & mask) + one) | ((v.z & mask) + one) | ((v.w & mask) + one)) & top) != 0;
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

template <typename T, int HD, bool CLUSTER>
__global__ void __launch_bounds__(FR_WARPS * 32)
few_rows_kernel(const PrefixAttnParams p, const __grid_constant__ PoolMaps maps, int with_prefix, int splits, int row_groups,
                int slot0) {
  using C = FewRows<T, HD>;
  constexpr int RT = C::RT, NST = C::NST, KT = C::KT, NJ = C::NJ, SUB = C::SUB;
  extern __shared__ __align__(1024) unsigned char fr_smem[];
  __shared__ __align__(8) uint64_t full[FR_WARPS][NST];
  __shared__ float s_m[FR_WARPS][RT], s_l[FR_WARPS][RT];
  __shared__ float2 s_ml[CLUSTER ? RT : 1];
  __shared__ int s_abort;
  unsigned char* base = fr_smem + ((1024 - (smem_u32(fr_smem) & 1023)) & 1023);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int q4 = lane & 3, r8 = lane >> 2;
  const int split = blockIdx.x % splits, group = blockIdx.x / splits, h = blockIdx.y, b = blockIdx.z;
  if (threadIdx.x == 0) {
    for (int w = 0; w < FR_WARPS; ++w)
      for (int s = 0; s < NST; ++s) mbar_init(&full[w][s], 1);
    s_abort = 0;
    fence_mbar_init();
  }
  __syncthreads();
  pdl_trigger();
  // Without the prefix this kernel follows many_rows_kernel, whose CTAs all are past their own wait by the time
  // this one starts: what both read is there, and they run side by side.  One CTA, the last to be placed, waits for
  // that kernel before it ends, so that the join, which waits for this one, has both results.
  if (with_prefix) pdl_wait();
  const int P = with_prefix ? prefix_keys(p) : 0, np = (P + KT - 1) / KT;
  const int t0 = split * FR_WARPS + warp, step = splits * FR_WARPS;
  // the pool rows of this warp's tiles first .. first + 31, one per lane; -1: no such page
  auto rows_of = [&](int first) {
    const long long t = t0 + (long long)step * (first + lane);
    const bool pre = t < np;
    const long long key = (pre ? t : t - np) * KT;
    const int blk = (int)min(key >> p.lg_page, (long long)INT32_MAX);
    if (blk >= (pre ? p.max_prefix_blocks : p.max_blocks)) return -1;
    const int id = pre ? p.prefix_table[blk] : p.block_table[(size_t)b * p.max_blocks + blk];
    if (id < 0 || id >= p.n_pages) return -1;
    return ((id * p.Hkv + h) << p.lg_page) + ((int)key & ((1 << p.lg_page) - 1));
  };
  const int rows0 = rows_of(0);
  int row_lo, row_hi, n;
  request_rows(p, b, row_lo, row_hi, n);
  const int rows_b = (row_hi - row_lo) * p.G, len = request_len(p, b);
  unsigned char* ring = base + (size_t)warp * NST * C::STAGE;
  const uint32_t ring_u = smem_u32(ring);
  uint32_t issued = 0, used = 0;  // tiles of this warp's ring, over all row tiles

  for (int r0 = group * RT; r0 < rows_b; r0 += row_groups * RT) {
    const int nr = min(RT, rows_b - r0);
    // own keys that the tile's last row sees
    const int own = max(0, min(len, len - n + (r0 + nr - 1) / p.G + 1));
    const int nt = np + (own + KT - 1) / KT;
    // This warp's tiles are t0 + step i, whatever the lengths are: without a prefix the first page ids are asked for
    // before the lengths are there.
    const int cnt = max(0, (nt - t0 + step - 1) / step);

    int rows = rows0;
    uint32_t absent = 0;  // stages whose tile has no page
    auto issue = [&](int i) {
      if (i && (i & 31) == 0) rows = rows_of(i);
      const int r = __shfl_sync(0xffffffffu, rows, i & 31);
      const int s = issued % NST;
      absent = (absent & ~(1u << s)) | ((r < 0 ? 1u : 0u) << s);
      if (lane == 0) mbar_arrive_expect_tx(&full[warp][s], C::STAGE);
      __syncwarp();
      if (lane < 2)
        tma3d_at(ring_u + s * C::STAGE + lane * C::TILE, lane ? &maps.v : &maps.k, r < 0 ? p.pool_rows : r, 0,
                 &full[warp][s]);  // past the end: zeros
      ++issued;
    };
    for (int i = 0; i < min(NST, cnt); ++i) issue(i);

    // ---- q fragments
    uint32_t qa[C::F16 ? HD / 16 : HD / 8][4];
    auto q_row = [&](int r) {  // tile row -> its q, null past the last
      if (r >= nr) return (const T*)nullptr;
      const int tok = row_lo + (r0 + r) / p.G, g = (r0 + r) % p.G;
      return reinterpret_cast<const T*>(p.q) + ((size_t)tok * p.Hq + h * p.G + g) * HD;
    };
    if constexpr (C::F16) {
      const T *qx = q_row(r8), *qy = q_row(r8 + 8);
#pragma unroll
      for (int ks = 0; ks < HD / 16; ++ks) {
        const int d = ks * 16 + q4 * 2;
        qa[ks][0] = qx ? *reinterpret_cast<const uint32_t*>(qx + d) : 0u;
        qa[ks][1] = qy ? *reinterpret_cast<const uint32_t*>(qy + d) : 0u;
        qa[ks][2] = qx ? *reinterpret_cast<const uint32_t*>(qx + d + 8) : 0u;
        qa[ks][3] = qy ? *reinterpret_cast<const uint32_t*>(qy + d + 8) : 0u;
      }
    } else {
      const T* qx = q_row(r8);
#pragma unroll
      for (int dd = 0; dd < HD / 32; ++dd)
#pragma unroll
        for (int s = 0; s < 2; ++s) {  // chunk 2 q4 + s of the 32 values: two steps of k
          float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
          if (qx) v = *reinterpret_cast<const float4*>(qx + dd * 32 + (2 * q4 + s) * 4);
          const int ks = dd * 4 + s * 2;
          split_tf32(v.x, qa[ks][0], qa[ks][1]);
          split_tf32(v.y, qa[ks][2], qa[ks][3]);
          split_tf32(v.z, qa[ks + 1][0], qa[ks + 1][1]);
          split_tf32(v.w, qa[ks + 1][2], qa[ks + 1][3]);
        }
    }
    // own keys that the first row sees, and each of this thread's rows (rows past the last: as the last)
    const int see_first = max(0, min(len, len - n + r0 / p.G + 1));
    const int see0 = r8 < nr ? max(0, len - n + (r0 + r8) / p.G + 1) : own;
    const int see1 = r8 + 8 < nr ? max(0, len - n + (r0 + r8 + 8) / p.G + 1) : own;

    const uint32_t k_lane = (((lane >> 4) << 3) + (lane & 7)) * 128 + ((((lane >> 3) & 1) ^ (lane & 7)) << 4);
    const uint32_t v_lane = ((((lane >> 3) & 1) << 3) + (lane & 7)) * 128 + (((lane >> 4) ^ (lane & 7)) << 4);
    constexpr int NO = HD / 8;
    float o[NO][4];
#pragma unroll
    for (int i = 0; i < NO; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
    bool far = false;  // of some row of this warp's

    for (int i = 0; i < cnt; ++i, ++used) {
      const int s = used % NST;
      if (!mbar_wait_warp(&full[warp][s], (used / NST) & 1u, &s_abort, PA_WAIT_NS)) break;
      const uint32_t ks_u = ring_u + s * C::STAGE, vs_u = ks_u + C::TILE;
      const int t = t0 + step * i;
      const bool gone = (absent >> s) & 1u;
      const int first = (t < np ? t : t - np) * KT;
      const bool part = gone || (t < np ? P : see_first) - first < KT;  // not every row sees every key
      float sc[NJ][4];
#pragma unroll
      for (int j = 0; j < NJ; ++j) sc[j][0] = sc[j][1] = sc[j][2] = sc[j][3] = 0.f;
      if constexpr (C::F16) {
        // lane l: row l & 7 of key block l >> 4, 16-byte piece 2 ks + (l >> 3 & 1), swizzled by its row
        const uint32_t ra = ks_u + k_lane;
#pragma unroll
        for (int ks = 0; ks < HD / 16; ++ks) {
          uint32_t kb[4];
          ldsm4((ra ^ ((2 * ks & 7) << 4)) + (ks >> 2) * SUB, kb);
          mma_16816(sc[0], qa[ks][0], qa[ks][1], qa[ks][2], qa[ks][3], kb[0], kb[1]);
          mma_16816(sc[NJ - 1], qa[ks][0], qa[ks][1], qa[ks][2], qa[ks][3], kb[2], kb[3]);
        }
      } else {
        const uint32_t ra = ks_u + r8 * 128;
        float cr[4] = {0.f, 0.f, 0.f, 0.f};  // K's low parts, apart: a shorter chain of sums
#pragma unroll
        for (int dd = 0; dd < HD / 32; ++dd)
#pragma unroll
          for (int c2 = 0; c2 < 2; ++c2) {
            const float4 v = lds_f4(ra + dd * SUB + (((2 * q4 + c2) ^ r8) << 4));
            uint32_t hi[4], lo[4];
            split_tf32(v.x, hi[0], lo[0]);
            split_tf32(v.y, hi[1], lo[1]);
            split_tf32(v.z, hi[2], lo[2]);
            split_tf32(v.w, hi[3], lo[3]);
            const int ks = dd * 4 + c2 * 2;
            mma_1688(cr, qa[ks], lo[0], lo[1]);
            mma_1688(sc[0], qa[ks], hi[0], hi[1]);
            mma_1688(cr, qa[ks + 1], lo[2], lo[3]);
            mma_1688(sc[0], qa[ks + 1], hi[2], hi[3]);
          }
        // rows 8..15 of the fragment: q's low parts
        sc[0][0] += (sc[0][2] + cr[0]) + cr[2];
        sc[0][1] += (sc[0][3] + cr[1]) + cr[3];
      }
      if (part) {
        const int lim0 = gone ? 0 : (t < np ? P : see0) - first, lim1 = gone ? 0 : (t < np ? P : see1) - first;
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int key = j * 8 + q4 * 2 + e;
            if (key >= lim0) sc[j][e] = -INFINITY;
            if (C::F16 && key >= lim1) sc[j][2 + e] = -INFINITY;
          }
      }
      // ---- running softmax.  A row's m, the same in its four lanes, is raised (and o rescaled) only when a weight
      // passes 2^(LIFT + RAISE): the lanes seldom have to agree on a maximum.
      float x0 = fmaxf(sc[0][0], sc[0][1]), x1 = fmaxf(sc[0][2], sc[0][3]);
      if (NJ == 2) {
        x0 = fmaxf(x0, fmaxf(sc[NJ - 1][0], sc[NJ - 1][1]));
        x1 = fmaxf(x1, fmaxf(sc[NJ - 1][2], sc[NJ - 1][3]));
      }
      x0 = __fadd_rn(__fmul_rn(x0, p.c), -C::LIFT);
      x1 = C::F16 ? __fadd_rn(__fmul_rn(x1, p.c), -C::LIFT) : -INFINITY;
      if (__any_sync(0xffffffffu, x0 > m0 + C::RAISE || x1 > m1 + C::RAISE)) {
#pragma unroll
        for (int d = 1; d <= 2; d <<= 1) {
          x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, d));
          x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, d));
        }
        x0 = fmaxf(m0, x0);
        x1 = fmaxf(m1, x1);
        const float f0 = m0 == -INFINITY ? 0.f : ex2(m0 - x0), f1 = m1 == -INFINITY ? 0.f : ex2(m1 - x1);
        l0 *= f0;
        l1 *= f1;
#pragma unroll
        for (int k = 0; k < NO; ++k) {
          o[k][0] *= f0;
          o[k][1] *= f0;
          o[k][2] *= C::F16 ? f1 : f0;
          o[k][3] *= C::F16 ? f1 : f0;
        }
        m0 = x0;
        m1 = x1;
        far = __any_sync(0xffffffffu, (fabsf(m0) >= PA_FAR && m0 != -INFINITY) || (fabsf(m1) >= PA_FAR && m1 != -INFINITY));
      }
      float n0 = m0 == -INFINITY ? 0.f : m0, n1 = m1 == -INFINITY ? 0.f : m1, c = p.c;
      if (far) {
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[j][e] = far_exponent(sc[j][e], c, e < 2 ? n0 : n1);
        n0 = n1 = 0.f;
        c = 1.f;
      }
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        sc[j][0] = ex2(fmaf(sc[j][0], c, -n0));
        sc[j][1] = ex2(fmaf(sc[j][1], c, -n0));
        l0 += sc[j][0] + sc[j][1];
        if (C::F16) {
          sc[j][2] = ex2(fmaf(sc[j][2], c, -n1));
          sc[j][3] = ex2(fmaf(sc[j][3], c, -n1));
          l1 += sc[j][2] + sc[j][3];
        }
      }
      // ---- o += P V.  Slots behind the last key may hold anything: their V counts as zero.
      const int lim = gone ? 0 : min(KT, (t < np ? P : own) - first);  // keys that any row sees
      // whether V holds an infinity or NaN at a key that some of the rows see and some do not
      auto hidden_not_finite = [&](uint32_t v, int end) {
        const int from = t < np ? end : max(0, see_first - first);
        bool bad = false;
        for (int e = lane; e < (end - from) * C::NB * 8; e += 32) {
          const int k = from + e / (C::NB * 8), c = e % (C::NB * 8);
          bad |= not_finite<T>(lds_v4(v + (c >> 3) * SUB + k * 128 + ((c & 7) << 4)));
        }
        return __any_sync(0xffffffffu, bad) != 0;
      };
      if constexpr (C::F16) {
        const uint32_t a0 = h2_as_u32(__floats2half2_rn(sc[0][0], sc[0][1])), a1 = h2_as_u32(__floats2half2_rn(sc[0][2], sc[0][3]));
        const uint32_t a2 = h2_as_u32(__floats2half2_rn(sc[NJ - 1][0], sc[NJ - 1][1])),
                       a3 = h2_as_u32(__floats2half2_rn(sc[NJ - 1][2], sc[NJ - 1][3]));
        const uint32_t ra = vs_u + v_lane;
        auto product = [&](uint32_t k0, uint32_t k1) {
#pragma unroll
          for (int nb = 0; nb < HD / 16; ++nb) {
            uint32_t vb[4];
            ldsm4_t((ra ^ ((2 * nb & 7) << 4)) + (nb >> 2) * SUB, vb);
            mma_16816(o[2 * nb], a0, a1, a2, a3, vb[0] & k0, vb[1] & k1);
            mma_16816(o[2 * nb + 1], a0, a1, a2, a3, vb[2] & k0, vb[3] & k1);
          }
        };
        if (!part) {
          product(0xffffffffu, 0xffffffffu);
        } else if (hidden_not_finite(vs_u, lim)) {
          // a row's weight of zero must not meet the infinity or NaN of a token that it does not see
          const int lim0 = see0 - first, lim1 = see1 - first;
#pragma unroll 1
          for (int k = 0; k < lim; ++k) {
            const float y0 = k & 1 ? (k & 8 ? sc[NJ - 1][1] : sc[0][1]) : (k & 8 ? sc[NJ - 1][0] : sc[0][0]);
            const float y1 = k & 1 ? (k & 8 ? sc[NJ - 1][3] : sc[0][3]) : (k & 8 ? sc[NJ - 1][2] : sc[0][2]);
            const int from = (lane & ~3) | ((k & 7) >> 1);
            const float p0 = __shfl_sync(0xffffffffu, y0, from), p1 = __shfl_sync(0xffffffffu, y1, from);
#pragma unroll
            for (int nb = 0; nb < NO; ++nb) {
              const float2 v = __half22float2(u32_as_h2(lds_u32(vs_u + (nb >> 3) * SUB + k * 128 + (((nb & 7) ^ (k & 7)) << 4) + q4 * 4)));
              if (k < lim0) {
                o[nb][0] += p0 * v.x;
                o[nb][1] += p0 * v.y;
              }
              if (k < lim1) {
                o[nb][2] += p1 * v.x;
                o[nb][3] += p1 * v.y;
              }
            }
          }
        } else {
          const int key = q4 * 2;
          product((key < lim ? 0xffffu : 0u) | (key + 1 < lim ? 0xffff0000u : 0u),
                  (key + 8 < lim ? 0xffffu : 0u) | (key + 9 < lim ? 0xffff0000u : 0u));
        }
      } else if (part && hidden_not_finite(vs_u, lim)) {
        const int lim0 = see0 - first;
#pragma unroll 1
        for (int k = 0; k < lim; ++k) {
          const float p0 = __shfl_sync(0xffffffffu, k & 1 ? sc[0][1] : sc[0][0], (lane & ~3) | (k >> 1));
          if (k >= lim0) continue;
#pragma unroll
          for (int dd = 0; dd < HD / 32; ++dd) {
            const float4 va = lds_f4(vs_u + dd * SUB + k * 128 + (((2 * q4) ^ (k & 7)) << 4));
            const float4 vb = lds_f4(vs_u + dd * SUB + k * 128 + (((2 * q4 + 1) ^ (k & 7)) << 4));
            const float xa[4] = {va.x, va.y, va.z, va.w}, xb[4] = {vb.x, vb.y, vb.z, vb.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              o[dd * 4 + e][0] += p0 * xa[e];
              o[dd * 4 + e][1] += p0 * xb[e];
            }
          }
        }
      } else {
        uint32_t pa[4];
        split_tf32(sc[0][0], pa[0], pa[1]);
        split_tf32(sc[0][1], pa[2], pa[3]);
        const int key = 2 * q4;  // slots q4 and q4 + 4 of k: keys 2 q4 and 2 q4 + 1
        const bool u0 = !part || key < lim, u1 = !part || key + 1 < lim;
#pragma unroll
        for (int dd = 0; dd < HD / 32; ++dd) {
          const uint32_t sub = vs_u + dd * SUB;
          float4 va = lds_f4(sub + key * 128 + ((r8 ^ key) << 4));
          float4 vb = lds_f4(sub + (key + 1) * 128 + ((r8 ^ (key + 1)) << 4));
          if (!u0) va = make_float4(0.f, 0.f, 0.f, 0.f);
          if (!u1) vb = make_float4(0.f, 0.f, 0.f, 0.f);
          const float xa[4] = {va.x, va.y, va.z, va.w}, xb[4] = {vb.x, vb.y, vb.z, vb.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            uint32_t h0, e0, h1, e1;
            split_tf32(xa[e], h0, e0);
            split_tf32(xb[e], h1, e1);
            float y[4] = {0.f, 0.f, 0.f, 0.f};
            mma_1688(y, pa, e0, e1);
            mma_1688(y, pa, h0, h1);
#pragma unroll
            for (int k = 0; k < 4; ++k) o[dd * 4 + e][k] += y[k];
          }
        }
      }
      __syncwarp();
      if (i + NST < cnt) issue(i + NST);
    }
    // ---- join the warps
    const bool failed = __syncthreads_or(issued != used);  // a wait ran out (also: every ring is free)
    if (failed) {
      if (CLUSTER)  // the others' barriers: two for this tile of rows and for each that follows
        for (int r = r0; r < rows_b; r += row_groups * RT) {
          cluster_sync();
          cluster_sync();
        }
      break;
    }
#pragma unroll
    for (int d = 1; d <= 2; d <<= 1) {
      l0 += __shfl_xor_sync(0xffffffffu, l0, d);
      l1 += __shfl_xor_sync(0xffffffffu, l1, d);
    }
    float* so = reinterpret_cast<float*>(ring);  // [RT][HD], this warp's ring
    if (q4 == 0) {
      s_m[warp][r8] = m0;
      s_l[warp][r8] = l0;
      if (C::F16) {
        s_m[warp][(r8 + 8) % RT] = m1;
        s_l[warp][(r8 + 8) % RT] = l1;
      }
    }
    if constexpr (C::F16) {
#pragma unroll
      for (int k = 0; k < NO; ++k) {
        *reinterpret_cast<float2*>(so + r8 * HD + k * 8 + q4 * 2) = make_float2(o[k][0], o[k][1]);
        *reinterpret_cast<float2*>(so + (r8 + 8) * HD + k * 8 + q4 * 2) = make_float2(o[k][2], o[k][3]);
      }
    } else {
#pragma unroll
      for (int dd = 0; dd < HD / 32; ++dd) {  // block e's columns 2 q4 and 2 q4 + 1 are values 8 q4 + e and 8 q4 + 4 + e
        float* dst = so + r8 * HD + dd * 32 + q4 * 8;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          dst[e] = o[dd * 4 + e][0] + o[dd * 4 + e][2];
          dst[4 + e] = o[dd * 4 + e][1] + o[dd * 4 + e][3];
        }
      }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < nr * (HD / 4); e += FR_WARPS * 32) {
      const int r = e / (HD / 4), d = (e % (HD / 4)) * 4;
      float M = -INFINITY;
#pragma unroll
      for (int w = 0; w < FR_WARPS; ++w) M = fmaxf(M, s_m[w][r]);
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      float L = 0.f;
#pragma unroll
      for (int w = 0; w < FR_WARPS; ++w) {
        if (s_m[w][r] == -INFINITY && s_l[w][r] == 0.f) continue;
        const float f = ex2(s_m[w][r] - M);
        const float4 v = *reinterpret_cast<const float4*>(base + (size_t)w * NST * C::STAGE + ((size_t)r * HD + d) * 4);
        acc.x += f * v.x;
        acc.y += f * v.y;
        acc.z += f * v.z;
        acc.w += f * v.w;
        L += f * s_l[w][r];
      }
      const int tok = row_lo + (r0 + r) / p.G, g = (r0 + r) % p.G;
      const size_t row = (size_t)tok * p.Hq + h * p.G + g;
      if (CLUSTER) {
        *reinterpret_cast<float4*>(base + ((size_t)(RT + r) * HD + d) * 4) = acc;  // behind warp 0's result
        if (d == 0) s_ml[CLUSTER ? r : 0] = make_float2(M, L);
      } else if (p.nslots == 1) {
        store_out<T>(reinterpret_cast<T*>(p.out) + row * HD + d, acc, L);
      } else {
        const size_t at = (size_t)(slot0 + split) * p.T * p.Hq + row;
        *reinterpret_cast<float4*>(p.part_o + at * HD + d) = acc;
        if (d == 0) p.part_ml[at] = make_float2(M, L);
      }
    }
    if (CLUSTER) {  // join the CTAs, each a part of the outputs
      __syncthreads();
      cluster_sync();
      join_cluster<T, HD>(p, smem_u32(s_ml), smem_u32(base) + RT * HD * 4, split, splits, nr, row_lo, r0, h);
      __syncthreads();
      cluster_sync();  // before a result is written over, or its CTA exits
    }
    // the rings hold the joined results: written by threads, next by copies
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncthreads();
  }
  // copies in flight land before the CTA may exit (after a wait that ran out)
  if (lane == 0)
    for (; used < issued; ++used) {
      int ignore = 0;
      mbar_wait_bounded(&full[warp][used % NST], (used / NST) & 1u, &ignore, PA_WAIT_NS);
    }
  if (threadIdx.x == 0 && s_abort) atomicExch(&g_prefix_attn_error, 1);
  if (!with_prefix && blockIdx.x == gridDim.x - 1 && blockIdx.y == gridDim.y - 1 && blockIdx.z == gridDim.z - 1) pdl_wait();
}

// ---------------------------------------------------------------- many rows, fp16

// Kernel for many rows of queries over the same keys, on the tensor cores
// (tcgen05): the shared prefix under the rows of all requests, or one
// request's prompt chunk.  A CTA takes two tiles of 128 rows (a row: a token
// and a head of the group), a kv head and a share of the keys:
//   warp 0     TMA producer: K and V tiles of 128 keys through one ring, a
//              copy per page and 64-wide column, issued by a lane each
//   warps 1, 2 MMA issuers of tile 0 and of tile 1: S = Q K^T into TMEM, then
//              O += P V with P read from TMEM, each half of P as it is ready
//   warp 3     zeroes V's slots behind the last key, which may hold anything
//              (0 x NaN is NaN), before the MMA issuers use the tile
//   warps 4-7, 8-11: softmax of tile 0 and of tile 1, a thread per row, which
//              holds its 128 scores in registers: their maximum, P = exp2(c s
//              - m) in fp16 over S's own columns, its sum in fp32, and in the
//              end O / l or a partial result
// The tiles take turns: while one is in the softmax, the other is in the
// tensor cores.  The reference a row is scaled by is raised, and O rescaled,
// only when a weight passes 2^15 (PA_LIFT); l is summed in fp32.
// TMEM: S0 | S1 (128 columns each, P in the first 64), O0 | O1 (HD each).
// Bound by the softmax's chain: 12 chunks of 120 to 700 tokens behind a prefix of
// 2050, 32 heads of 128, 295 us in a graph, 722 TFLOP/s, 44 % of the tensor
// cores' cycles (call after call, with the clock down under the power cap, 316 us).
constexpr int TC_M = 128, TC_N = 128;   // rows and keys of a tile
constexpr int TC_THREADS = 12 * 32;
constexpr int TC_REGS_CTL = 88, TC_REGS_SM = 208;  // 128 x 88 + 256 x 208: what the block starts with, 384 x 168
constexpr int TC_HAND = 3;  // quarter of a tile before which its softmax lets the other one start

template <int HD>
struct ManyRows {
  static constexpr int NCH = HD / 64;               // 64-wide columns
  static constexpr int TILE = TC_N * HD * 2;        // bytes of a Q, K or V tile
  static constexpr int NBUF = HD == 128 ? 5 : 8;    // K and V tiles in the ring
  static constexpr int SMEM = 2 * TILE + NBUF * TILE + 1024;
};

__device__ __forceinline__ bool pa_wait(uint64_t* bar, uint32_t parity, volatile int* abort) {
  return mbar_wait_bounded(bar, parity, abort, PA_WAIT_NS);
}

// The same for one thread on the critical path: polls, and looks at the clock now and then.
__device__ __forceinline__ bool pa_spin(uint64_t* bar, uint32_t parity, volatile int* abort) {
  for (int i = 0; i < 64; ++i)
    if (mbar_test_wait(bar, parity)) return true;
  return pa_wait(bar, parity, abort);
}

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]),
               "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const float (&v)[32]) {
  uint32_t a[16], b[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    a[i] = __float_as_uint(v[i]);
    b[i] = __float_as_uint(v[16 + i]);
  }
  tmem_st16(taddr, a);
  tmem_st16(taddr + 16, b);
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// 32 columns, not waited for: tmem_wait_ld, then tmem_ready of each block before its values are used.
__device__ __forceinline__ void tmem_ld32_async(uint32_t taddr, float* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
        "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]),
        "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]),
        "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_ready(float* v) {  // no use of v[0..31] moves above this
#pragma unroll
  for (int i = 0; i < 32; i += 8)
    asm volatile("" : "+f"(v[i]), "+f"(v[i + 1]), "+f"(v[i + 2]), "+f"(v[i + 3]), "+f"(v[i + 4]), "+f"(v[i + 5]), "+f"(v[i + 6]), "+f"(v[i + 7]));
}
__device__ __forceinline__ void tmem_ld32_wait(uint32_t taddr, float* v) {
  tmem_ld32_async(taddr, v);
  tmem_wait_ld();
  tmem_ready(v);
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// two fp32 in one instruction
__device__ __forceinline__ uint64_t pack2(float x, float y) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(x), "f"(y));
  return d;
}
__device__ __forceinline__ void unpack2(uint64_t d, float& x, float& y) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(d));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// A warp's 32 rows of RB bytes, a row in each lane's registers (`get(c)`: its c-th 16 bytes), to global rows of `stride`
// bytes: through shared memory (`sm`, 32 RB bytes of this warp's own), so that a row's lanes write next to each other.
// Written straight from the registers, the 128 rows of a tile took 4300 clocks.
template <int RB, typename F>
__device__ __forceinline__ void flush_rows(uint32_t sm, F get, char* dst, size_t stride, size_t row, bool valid) {
  constexpr int LPR = RB / 16, RPI = 32 / LPR;  // lanes per row, rows per store
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int c = 0; c < LPR; ++c) {
    const uint4 v = get(c);
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(sm + lane * RB + ((c ^ (lane & (LPR - 1))) << 4)), "r"(v.x), "r"(v.y),
                 "r"(v.z), "r"(v.w)
                 : "memory");
  }
  __syncwarp();
  const int c = lane % LPR;
#pragma unroll
  for (int j = 0; j < 32 / RPI; ++j) {
    const int r = j * RPI + lane / LPR;
    const size_t to = __shfl_sync(0xffffffffu, (unsigned long long)row, r);
    const bool ok = __shfl_sync(0xffffffffu, (int)valid, r);
    const uint4 v = lds_v4(sm + r * RB + ((c ^ (r & (LPR - 1))) << 4));
    if (ok) *reinterpret_cast<uint4*>(dst + to * stride + c * 16) = v;
  }
  __syncwarp();
}
__device__ __forceinline__ uint4 f4_as_u4(const float* v) {
  return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
}

// The rows and keys of a CTA of the many-rows kernels: `item`-th block of ROWS rows (of the whole batch where PACKED,
// else of one request, items counted over the requests), every splits-th of its tiles of KEYS keys.
struct RowShare {
  int b, r0;               // request; first row, counted in the request (in the batch where PACKED)
  int row_lo, rows;        // the request's first token in q, its rows
  int n, len, P, np, own;  // its new tokens, its tokens; prefix keys, prefix tiles; own keys that the last row sees
  int all;                 // own keys that every row sees
  int t0, step, cnt;       // tiles: t0 + step i
  bool work;
};

template <bool PACKED, int ROWS, int KEYS, int THREADS>
__device__ __forceinline__ RowShare row_share(const PrefixAttnParams& p, int item, int split, int splits, int& s_req, int& s_row0,
                                              int* s_sum) {
  RowShare w;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int row_hi;
  if (PACKED) {
    w.b = 0;
    w.row_lo = 0;
    w.n = row_hi = min(max(p.q_start[p.B], 0), p.T);
    w.r0 = item * ROWS;
    w.work = true;
  } else {
    // s_req, s_row0: the request that holds the item, found by a scan of the requests' items
    int before = 0;
    for (int b0 = 0; b0 < p.B; b0 += THREADS) {
      const int bb = b0 + threadIdx.x;
      int lo, hi, n, cnt = 0;
      if (bb < p.B) {
        request_rows(p, bb, lo, hi, n);
        cnt = (int)(((long long)(hi - lo) * p.G + ROWS - 1) / ROWS);
      }
      int sum = cnt;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, sum, d);
        if (lane >= d) sum += u;
      }
      if (lane == 31) s_sum[warp] = sum;
      __syncthreads();
      int at = before;
      for (int i = 0; i < THREADS / 32; ++i) {
        if (i < warp) at += s_sum[i];
        before += s_sum[i];
      }
      at += sum - cnt;
      if (item >= at && item < at + cnt) {
        s_req = bb;
        s_row0 = (item - at) * ROWS;
      }
      __syncthreads();
      if (s_req >= 0) break;
    }
    w.work = s_req >= 0;
    w.b = max(s_req, 0);
    w.r0 = s_row0;
    request_rows(p, w.b, w.row_lo, row_hi, w.n);
  }
  w.rows = (row_hi - w.row_lo) * p.G;  // fits: T * Hq does
  w.work = w.work && w.r0 < w.rows;
  w.len = PACKED ? 0 : request_len(p, w.b);
  w.P = prefix_keys(p);
  w.np = (w.P + KEYS - 1) / KEYS;
  const int last = min(w.r0 + ROWS, w.rows) - 1;
  w.own = PACKED || !w.work ? 0 : max(0, min(w.len, w.len - w.n + last / p.G + 1));
  w.all = PACKED || !w.work ? 0 : max(0, min(w.len, w.len - w.n + w.r0 / p.G + 1));
  // every splits-th tile, so that the first one does not depend on the lengths
  w.t0 = split;
  w.step = splits;
  w.cnt = w.work ? max(0, (w.np + (w.own + KEYS - 1) / KEYS - split + splits - 1) / splits) : 0;
  return w;
}

// PACKED: rows of all requests, keys of the prefix.  Otherwise: rows of one
// request, keys of the prefix and its own.
template <int HD, bool PACKED>
__global__ void __launch_bounds__(TC_THREADS, 1)
many_rows_kernel(const PrefixAttnParams p, const __grid_constant__ PoolMaps maps, int splits, int slot0) {
  using C = ManyRows<HD>;
  constexpr int NBUF = C::NBUF;
  extern __shared__ __align__(1024) unsigned char mr_smem[];
  __shared__ __align__(8) uint64_t full[NBUF], empty[NBUF], q_full[2], s_full[2], p_full[2][2], o_full[2], v_clean[NBUF], drained[2], turn[2][4];
  __shared__ uint32_t s_tmem, s_absent[16];
  __shared__ int s_abort, s_req, s_row0, s_sum[TC_THREADS / 32];
  __shared__ int s_any_bad, s_bad[3][PACKED ? 1 : HD];  // per column the first hidden key with inf, -inf, NaN
  unsigned char* base = mr_smem + ((1024 - (smem_u32(mr_smem) & 1023)) & 1023);
  const uint32_t q_u = smem_u32(base), ring_u = q_u + 2 * C::TILE;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int split = blockIdx.x % splits, item = blockIdx.x / splits, h = blockIdx.y;
  if (threadIdx.x == 0) {
    for (int i = 0; i < NBUF; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 3);  // the MMA issuers (warp 3 for the second where it has no rows), and warp 3
      mbar_init(&v_clean[i], 1);
    }
    for (int x = 0; x < 2; ++x) {
      mbar_init(&q_full[x], TC_M);
      mbar_init(&s_full[x], 1);
      mbar_init(&p_full[x][0], 4);
      mbar_init(&p_full[x][1], 4);
      mbar_init(&o_full[x], 1);
      mbar_init(&drained[x], 1);
      for (int i = 0; i < 4; ++i) mbar_init(&turn[x][i], 1);
    }
    s_abort = 0;
    s_req = -1;
    s_row0 = 0;
    s_any_bad = 0;
    fence_mbar_init();
  }
  if (!PACKED)
    for (int i = threadIdx.x; i < 3 * HD; i += TC_THREADS) s_bad[i / HD][PACKED ? 0 : i % HD] = INT32_MAX;
  if (warp == 1) tmem_alloc_cols(&s_tmem, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_wait();
  pdl_trigger();  // after the wait: few_rows_kernel relies on it
  volatile int* abort = &s_abort;
  const uint32_t tmem = s_tmem;

  const RowShare w = row_share<PACKED, 2 * TC_M, TC_N, TC_THREADS>(p, item, split, splits, s_req, s_row0, s_sum);
  const int b = w.b, r0 = w.r0, row_lo = w.row_lo, rows = w.rows, n = w.n, len = w.len, P = w.P, np = w.np, own = w.own;
  const int cnt = w.cnt;
  const bool work = w.work;
  const int nx = work && r0 + TC_M < rows ? 2 : 1;  // row tiles in use
  auto tile_of = [&](int i) { return w.t0 + w.step * i; };
  // keys of tile t that exist
  auto keys_of = [&](int t) { return t < np ? P - t * TC_N : own - (t - np) * TC_N; };
  if (warp < 4)
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(TC_REGS_CTL));
  else
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(TC_REGS_SM));
  if (warp == 0) {
    // ================================ TMA producer ================================
    // copies: a page's rows (128 at most) of a 64-wide column, one per lane
    const int lg_box = min(p.lg_page, 7), sub = lane / C::NCH, ch = lane % C::NCH;
    auto pool_row = [&](int t) {  // this lane's first row of tile t in the pools; -1: no such page
      const bool pre = PACKED || t < np;
      const long long key = (long long)(pre ? t : t - np) * TC_N + (sub << lg_box);
      const int blk = (int)min(key >> p.lg_page, (long long)INT32_MAX);
      if (blk >= (pre ? p.max_prefix_blocks : p.max_blocks)) return -1;
      const int id = pre ? p.prefix_table[blk] : p.block_table[(size_t)b * p.max_blocks + blk];
      return id >= 0 && id < p.n_pages ? ((id * p.Hkv + h) << p.lg_page) + (int)(key & ((1 << p.lg_page) - 1)) : -1;
    };
    const int copies = (TC_N >> lg_box) * C::NCH;
    uint32_t it = 0;
    bool ok = true;
    int next = pool_row(tile_of(0));
    for (int i = 0; i < cnt && ok; ++i) {
      const int keys = keys_of(tile_of(i));
      const int row = sub << lg_box < keys ? next : -1;
      if (i + 1 < cnt) next = pool_row(tile_of(i + 1));
      uint32_t gone = 0;  // keys of this tile that have no page, a bit per 16
#pragma unroll
      for (int k = 0; k < TC_N / 16; ++k) gone |= (__shfl_sync(0xffffffffu, row, ((k * 16) >> lg_box) * C::NCH) < 0 ? 1u : 0u) << k;
      if (lane == 0) s_absent[i & 15] = gone;
#pragma unroll
      for (int kv = 0; kv < 2; ++kv, ++it) {
        const int s = it % NBUF;
        ok = __all_sync(0xffffffffu, pa_wait(&empty[s], ((it / NBUF) & 1u) ^ 1u, abort));
        if (!ok) break;
        if (lane == 0) mbar_arrive_expect_tx(&full[s], C::TILE);
        __syncwarp();
        if (lane < copies)
          tma3d_at(ring_u + s * C::TILE + ch * (TC_N * 128) + (sub << lg_box) * 128, kv ? &maps.v : &maps.k,
                   row < 0 ? p.pool_rows : row, ch, &full[s]);
      }
    }
    // copies in flight land before the CTA may exit
    if (lane == 0) {
      int ignore = 0;
      for (uint32_t k = it > NBUF ? it - NBUF : 0; k < it; ++k) pa_wait(&full[k % NBUF], (k / NBUF) & 1u, &ignore);
    }
  } else if (warp <= 2) {
    // ================================ MMA issuers ================================
    const int x = warp - 1;
    if (lane == 0 && x < nx && cnt > 0) {
      constexpr uint32_t idesc_s = (1u << 4) | ((TC_N >> 3) << 17) | ((TC_M >> 4) << 24);
      constexpr uint32_t idesc_o = (1u << 4) | (1u << 16) | ((HD >> 3) << 17) | ((TC_M >> 4) << 24);  // V: contiguous along N
      const uint32_t ts = tmem + x * TC_N, to = tmem + 2 * TC_N + x * HD;
      const uint64_t dq = umma_desc_sw128(q_u + x * C::TILE), dk = umma_desc_sw128(ring_u), dv = umma_desc_sw128_mn(ring_u, TC_N * 128);
      auto at = [](uint32_t it) { return (uint64_t)((it % NBUF) * (C::TILE >> 4)); };  // a ring tile, in descriptor units
      auto wait_full = [&](uint32_t it) { return pa_spin(&full[it % NBUF], (it / NBUF) & 1u, abort); };
      auto issue_s = [&](uint32_t it) {  // S = Q K^T
        const uint64_t k = dk + at(it);
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk) {
          const uint32_t off = ((kk >> 2) * (TC_N * 128) + (kk & 3) * 32) >> 4;
          umma_f16(ts, dq + off, k + off, idesc_s, kk != 0);
        }
        tc_commit(&s_full[x]);
        tc_commit(&empty[it % NBUF]);
      };
      bool ok = pa_spin(&q_full[x], 0, abort) && wait_full(0);
      if (ok) {
        tc_fence_after();
        issue_s(0);
      }
      for (int i = 0; i < cnt && ok; ++i) {
        const uint32_t vi = 2 * i + 1, ki = 2 * i + 2;
        ok = pa_spin(&v_clean[vi % NBUF], (vi / NBUF) & 1u, abort);
        const uint64_t v = dv + at(vi);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          ok = ok && pa_spin(&p_full[x][half], i & 1, abort);
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int kk = half * (TC_N / 32); kk < (half + 1) * (TC_N / 32); ++kk)
            umma_f16_ta(to, ts + kk * 8, v + kk * (2048 >> 4), idesc_o, (i | kk) != 0);
        }
        if (!ok) break;
        tc_commit(&empty[vi % NBUF]);
        if (i + 1 == cnt) {
          tc_commit(&o_full[x]);
        } else {
          ok = wait_full(ki);
          if (ok) issue_s(ki);
        }
      }
    }
  } else if (warp == 3) {
    // ================================ V looked over ================================
    // Every tile passes here before the MMA issuers take it, and is freed as by them: a barrier's parity says which of
    // two phases is over, not which of many.
    for (uint32_t it = 0; it < 2u * cnt; ++it) {
      const int s = it % NBUF, t = tile_of((int)(it / 2)), keys = min(TC_N, keys_of(t));
      if (!__all_sync(0xffffffffu, pa_wait(&full[s], (it / NBUF) & 1u, abort))) break;
      const uint32_t v = ring_u + s * C::TILE;
      // keys from here on are hidden from some row
      const int shown = PACKED || t < np ? keys : max(0, min(keys, w.all - (t - np) * TC_N));
      if ((it & 1) && shown < TC_N) {
        for (int e = lane; e < (keys - shown) * 8 * C::NCH; e += 32) {
          const int r = shown + e / (8 * C::NCH), c = e % (8 * C::NCH);
          const uint32_t at = v + (c >> 3) * (TC_N * 128) + r * 128 + ((c & 7) << 4);
          const uint4 u = lds_v4(at);
          if (!not_finite<__half>(u)) continue;
          // it is zero for the products; at the end the rows that see it become what it makes of them
          uint32_t y[4] = {u.x, u.y, u.z, u.w};
          for (int k = 0; k < 8; ++k) {
            const uint32_t half = (y[k >> 1] >> ((k & 1) * 16)) & 0xffffu;
            if ((half & 0x7c00u) != 0x7c00u) continue;
            const int col = (c >> 3) * 64 + ((c & 7) ^ (r & 7)) * 8 + k;
            atomicMin(&s_bad[half == 0x7c00u ? 0 : half == 0xfc00u ? 1 : 2][col], (t - np) * TC_N + r);
            y[k >> 1] &= k & 1 ? 0x0000ffffu : 0xffff0000u;
            s_any_bad = 1;
          }
          asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(y[0]), "r"(y[1]), "r"(y[2]), "r"(y[3]) : "memory");
        }
        // the slots behind the last key may hold anything
        for (int e = lane; e < (TC_N - keys) * 8 * C::NCH; e += 32) {
          const int r = keys + e / (8 * C::NCH), c = e % (8 * C::NCH);
          asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(v + (c >> 3) * (TC_N * 128) + r * 128 + ((c & 7) << 4)), "r"(0)
                       : "memory");
        }
        fence_async_smem();
        __threadfence_block();
        __syncwarp();
      }
      if (lane == 0) {
        mbar_arrive(&v_clean[s]);
        mbar_arrive(&empty[s]);
        if (nx == 1) mbar_arrive(&empty[s]);
      }
    }
  } else if (warp >= 4) {
    // ================================ softmax ================================
    const int x = (warp - 4) >> 2;               // row tile
    const int lanes = (warp & 3) * 32;           // TMEM lanes this warp may access
    const int r = r0 + x * TC_M + lanes + lane;  // this thread's row
    const uint32_t st = tmem + ((uint32_t)lanes << 16) + x * TC_N, ot = tmem + ((uint32_t)lanes << 16) + 2 * TC_N + x * HD;
    const bool valid = r < rows;
    const int see = PACKED ? 0 : (valid ? max(0, min(len, len - n + r / p.G + 1)) : own);
    const float c = p.c;
    float m = -INFINITY, l = 0.f;
    bool far = false;
    if (x < nx && cnt > 0) {
      // ---- Q: this warp's 32 rows, 16 bytes a lane, into the K-major swizzled tile
      constexpr int LPR = HD / 8;  // 16-byte pieces of a row
      const uint32_t qt = q_u + x * C::TILE;
      uint4 qv[LPR];
#pragma unroll
      for (int e = 0; e < LPR; ++e) {
        const int gr = r0 + x * TC_M + lanes + (e * 32 + lane) / LPR, pc = (e * 32 + lane) % LPR;
        qv[e] = make_uint4(0u, 0u, 0u, 0u);
        if (gr < rows) {
          const size_t at = ((size_t)(row_lo + gr / p.G) * p.Hq + h * p.G + gr % p.G) * HD + pc * 8;
          qv[e] = *reinterpret_cast<const uint4*>(reinterpret_cast<const __half*>(p.q) + at);
        }
      }
#pragma unroll
      for (int e = 0; e < LPR; ++e) {
        const int rr = lanes + (e * 32 + lane) / LPR, pc = (e * 32 + lane) % LPR;
        asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(qt + (pc >> 3) * (TC_M * 128) + sw128(rr, pc & 7)), "r"(qv[e].x),
                     "r"(qv[e].y), "r"(qv[e].z), "r"(qv[e].w)
                     : "memory");
      }
      fence_async_smem();
      mbar_arrive(&q_full[x]);

      bool ok = true;
      for (int i = 0; i < cnt; ++i) {
        ok = __all_sync(0xffffffffu, pa_wait(&s_full[x], i & 1, abort));
        if (!ok) break;
        tc_fence_after();
        const int t = tile_of(i);
        const uint32_t gone = s_absent[i & 15];
        const int lim = (t < np ? P : see) - (t < np ? t : t - np) * TC_N;  // keys of the tile this row sees
        const bool part = __any_sync(0xffffffffu, lim < TC_N) || gone != 0;
        auto seen = [&](int k) { return k < lim && !((gone >> (k / 16)) & 1u); };
        float v[TC_N];
#pragma unroll
        for (int q = 0; q < TC_N; q += 32) tmem_ld32_async(st + q, v + q);
        tmem_wait_ld();
#pragma unroll
        for (int q = 0; q < TC_N; q += 32) tmem_ready(v + q);
        if (part) {
#pragma unroll
          for (int k = 0; k < TC_N; ++k) v[k] = seen(k) ? v[k] : -INFINITY;
        }
        auto row_max = [&]() {
          float a0 = fmaxf(v[0], v[1]), a1 = fmaxf(v[2], v[3]), a2 = fmaxf(v[4], v[5]), a3 = fmaxf(v[6], v[7]);
#pragma unroll
          for (int k = 8; k < TC_N; k += 8) {
            a0 = max3(a0, v[k], v[k + 1]);
            a1 = max3(a1, v[k + 2], v[k + 3]);
            a2 = max3(a2, v[k + 4], v[k + 5]);
            a3 = max3(a3, v[k + 6], v[k + 7]);
          }
          return __fadd_rn(__fmul_rn(fmaxf(fmaxf(a0, a1), fmaxf(a2, a3)), c), -PA_LIFT);
        };
        auto raise = [&](float mx) {
          const float mn = fmaxf(m, mx);
          const float f = m == -INFINITY ? 0.f : ex2(m - mn);
          m = mn;
          far = __any_sync(0xffffffffu, fabsf(m) >= PA_FAR && m != -INFINITY);
          l *= f;
          if (i > 0) {  // S is there: so is the last product into O
#pragma unroll
            for (int q = 0; q < HD / 32; ++q) {
              float u[32];
              tmem_ld32_wait(ot + q * 32, u);
#pragma unroll
              for (int k = 0; k < 32; ++k) u[k] *= f;
              tmem_st32(ot + q * 32, u);
            }
          }
        };
        uint64_t l2[2];
        uint32_t pw[16];
        auto quarter = [&](int q, auto is_far) {  // P of 32 keys
          const float mm = m == -INFINITY ? 0.f : m;
          const uint64_t c2 = pack2(c, c), m2 = pack2(-mm, -mm);
#pragma unroll
          for (int k = 0; k < 32; k += 2) {
            float e0, e1;
            if constexpr (is_far) {
              e0 = far_exponent(v[q * 32 + k], c, mm);
              e1 = far_exponent(v[q * 32 + k + 1], c, mm);
            } else {
              unpack2(fma2(pack2(v[q * 32 + k], v[q * 32 + k + 1]), c2, m2), e0, e1);
            }
            e0 = ex2(e0);
            e1 = ex2(e1);
            l2[(k >> 1) & 1] = add2(l2[(k >> 1) & 1], pack2(e0, e1));
            pw[k / 2] = h2_as_u32(__floats2half2_rn(e0, e1));
          }
        };
        const float mx = row_max();
        if (__any_sync(0xffffffffu, mx > m + PA_RAISE)) raise(mx);  // also from -inf
        // The two warps of a scheduler take turns here, or both tiles fall into step: both in the softmax, then both
        // in the tensor cores.
        if (nx == 2 && (x == 1 || i > 0)) {
          ok = __all_sync(0xffffffffu, pa_wait(&turn[x][warp & 3], (x == 1 ? i : i - 1) & 1, abort));
          if (!ok) break;
        }
        l2[0] = l2[1] = pack2(0.f, 0.f);
        auto weights = [&](auto is_far) {
          quarter(0, is_far);
          tmem_st16(st, pw);  // over columns of S that have been read
#pragma unroll
          for (int q = 1; q < TC_N / 32; ++q) {
            if (q == TC_HAND && nx == 2 && lane == 0) mbar_arrive(&turn[x ^ 1][warp & 3]);
            quarter(q, is_far);
            tmem_st16(st + q * 16, pw);
            if (q & 1) {
              tmem_wait_st();
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(&p_full[x][q >> 1]);
            }
          }
        };
        if (far)
          weights(std::true_type{});
        else
          weights(std::false_type{});
        float l0, l1;
        unpack2(add2(l2[0], l2[1]), l0, l1);
        l += l0 + l1;
      }
      // ---- O / l, or the partial result
      ok = ok && __all_sync(0xffffffffu, pa_wait(&o_full[x], 0, abort));
      tc_fence_after();
      if (ok) {
        const size_t row = valid ? (size_t)(row_lo + r / p.G) * p.Hq + h * p.G + r % p.G : 0;
        const size_t at = (size_t)(slot0 + split) * p.T * p.Hq + row;
        const float inv = l == 0.f ? 0.f : 1.f / l;
        if (valid && p.nslots > 1) p.part_ml[at] = make_float2(m, l);
        const uint32_t sm = q_u + x * C::TILE + lanes * (HD * 2);  // in the tile's Q, which is done with
        auto unhide = [&](float* v, int col, int count) {  // what is not finite, for the rows that see it
          if constexpr (!PACKED) {
            if (!s_any_bad) return;
#pragma unroll
            for (int k = 0; k < count; ++k) {
              const bool up = see > s_bad[0][col + k], down = see > s_bad[1][col + k];
              if (see > s_bad[2][col + k] || (up && down))
                v[k] = NAN;
              else if (up || down)
                v[k] += up ? INFINITY : -INFINITY;
            }
          }
        };
        if (!__any_sync(0xffffffffu, valid)) {
          // rows behind the last
        } else if (p.nslots > 1) {
#pragma unroll
          for (int q = 0; q < HD; q += HD / 2) {
            float v[HD / 2];
#pragma unroll
            for (int k = 0; k < HD / 2; k += 32) {
              tmem_ld32_wait(ot + q + k, v + k);
              unhide(v + k, q + k, 32);
            }
            flush_rows<HD * 2>(sm, [&](int c) { return f4_as_u4(v + c * 4); }, reinterpret_cast<char*>(p.part_o + (at - row) * HD + q),
                               HD * sizeof(float), row, valid);
          }
        } else {
          uint32_t o2[HD / 2];
#pragma unroll
          for (int k = 0; k < HD; k += 32) {
            float v[32];
            tmem_ld32_wait(ot + k, v);
            unhide(v, k, 32);
#pragma unroll
            for (int j = 0; j < 16; ++j) o2[k / 2 + j] = h2_as_u32(__floats2half2_rn(v[2 * j] * inv, v[2 * j + 1] * inv));
          }
          flush_rows<HD * 2>(sm, [&](int c) { return make_uint4(o2[4 * c], o2[4 * c + 1], o2[4 * c + 2], o2[4 * c + 3]); },
                             reinterpret_cast<char*>(p.out), HD * sizeof(__half), row, valid);
        }
      }
    } else if (x < nx && work && valid) {  // no keys in this share
      const size_t row = (size_t)(row_lo + r / p.G) * p.Hq + h * p.G + r % p.G;
      if (p.nslots > 1) {
        p.part_ml[(size_t)(slot0 + split) * p.T * p.Hq + row] = make_float2(-INFINITY, 0.f);
      } else {
        for (int d = 0; d < HD; d += 8)
          *reinterpret_cast<uint4*>(reinterpret_cast<__half*>(p.out) + row * HD + d) = make_uint4(0u, 0u, 0u, 0u);
      }
    }
  }
  // after a wait that ran out: the products in flight have ended before the TMEM is freed
  tc_fence_before();
  const bool failed = __syncthreads_or(*abort);
  tc_fence_after();
  if (failed && (warp == 1 || warp == 2) && lane == 0) {
    int ignore = 0;
    tc_commit(&drained[warp - 1]);
    pa_wait(&drained[warp - 1], 0, &ignore);
  }
  __syncthreads();
  if (warp == 1) {
    tmem_dealloc_cols(tmem, 512);
    tmem_relinquish();
  }
  if (threadIdx.x == 0 && failed) atomicExch(&g_prefix_attn_error, 1);
}

// ---------------------------------------------------------------- many rows, fp32

// The many-rows kernel for fp32.  Every operand x is carried as three bf16
// parts, x0 = bf16(x), x1 = bf16(x - x0), x2 = bf16(x - x0 - x1): 8 bits each,
// so that all 24 are there, and bf16 has fp32's range.  A product of two
// operands is the six products of parts that count: x0 y0, x0 y1, x1 y0, x0 y2,
// x1 y1, x2 y0; what is left out is 2^-25 of it at most.  (Two fp16 parts and
// three products carried 22 bits of values from 2^-14 to 65504 only, and of
// weights down to 2^-14: values of 1e-9 came out 8e-3 off, 1e5 as NaN.)
//   S = Q K^T: in two fp32 accumulators, (q0 + q1) k0 and the rest, for K's
//     parts lie one behind the other and [k0 | k1] is one product of twice the
//     width.
//   O = P V: in one, small products first.
// The tensor cores cut their fp32 sums off, always towards zero.  Over a long
// row that adds up (3.5e-8 of O per 16 keys, 3.6e-5 after 16500), so every
// tile's products are added to a sum of their own, in fp32 and rounded to
// nearest: 3.6e-7 of O at any length.  A value that is not finite, or rounds
// past bf16's largest, gives NaN.  One tile of 128 rows, tiles of 64 keys:
//   warp 0       TMA producer: raw fp32 K and V through a ring, 8 KB a stage
//   warp 1       MMA issuer; S of the next tile goes ahead of O = P V of this one
//   warps 4-11   softmax, two threads per row with half the tile's keys each,
//                which tell each other the maxima they find (P's parts over
//                S's columns)
//   warps 12-19  split Q, then each raw stage, into the parts; V's slots
//                behind the last key, which may hold anything, become zero
// TMEM: two buffers of S (two accumulators of 64 columns each), the products, their sum.
// Bound by the chain from a raw tile to its product, which the 227 KB leave no
// room to double: 2.9 us a tile (the two fp16 parts took 2.4), 39 % of the tensor
// cores' cycles; 12 chunks of 120 to 700 tokens behind 2050, 32 heads of 128,
// 1210 us, 176 TFLOP/s (1060 of bf16 products; two fp16 parts 1116 us).  The
// warps' parts run side by side and share the instruction cache: with the splits
// and products unrolled at every place, 128 KB of code, the same took 1.7 times as
// long.
constexpr int TF_N = 64;              // keys of a tile
constexpr int TF_BOX = 8;             // keys of a copy
constexpr int TF_THREADS = 20 * 32;
constexpr int TF_CONV = 8;            // warps that split
constexpr float TF_RAISE = 8.f;       // a row's reference is raised when a weight passes 2^8

template <int HD>
struct ManyRowsF32 {
  static constexpr int NCH = HD / 64;               // 64-wide bf16 columns
  static constexpr int QT = TC_M * HD * 2;          // bytes of one part of Q
  static constexpr int CH = TF_N * 128;             // bytes of a 64-wide column of one part of a tile
  static constexpr int PT = NCH * CH;               // bytes of one part of a K or V tile
  static constexpr int LPK = HD / 8;                // lanes that split a key, 8 values each
  static constexpr int KPW = 32 / LPK;              // keys of a warp at a time
  static constexpr int KEYS = TF_CONV * KPW;        // keys of a raw stage, which the warps split in one go
  static constexpr int STEPS = TF_N / KEYS;         // stages of a tile
  static constexpr int BOX = TF_BOX * HD * 4;       // bytes of one copy
  static constexpr int COPIES = KEYS / TF_BOX;      // copies of a stage
  static constexpr int RAW = COPIES * BOX;          // bytes of a stage
  static constexpr int NRAW = HD == 128 ? 4 : 12;
  static constexpr int SMEM = 3 * QT + 6 * PT + NRAW * RAW;  // to the last byte of 227 KB with the static part
};

// two fp32 -> bf16, packed, x in the low half
__device__ __forceinline__ uint32_t bf16_pair(float x, float y) {
  uint32_t d;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(y), "f"(x));
  return d;
}
// two fp32 -> their three bf16 parts, packed; the differences are exact
__device__ __forceinline__ void split_bf16(float x, float y, uint32_t& p0, uint32_t& p1, uint32_t& p2) {
  const uint64_t minus = pack2(-1.f, -1.f);
  uint64_t rest = pack2(x, y);
  p0 = bf16_pair(x, y);
  rest = fma2(pack2(__uint_as_float(p0 << 16), __uint_as_float(p0 & 0xffff0000u)), minus, rest);
  unpack2(rest, x, y);
  p1 = bf16_pair(x, y);
  rest = fma2(pack2(__uint_as_float(p1 << 16), __uint_as_float(p1 & 0xffff0000u)), minus, rest);
  unpack2(rest, x, y);
  p2 = bf16_pair(x, y);
}
// eight fp32 -> 16 bytes of each part, at shared address `at` and `part` bytes further each
__device__ __forceinline__ void split_bf16x8(const float4& a, const float4& b, uint32_t at, uint32_t part) {
  uint32_t y[3][4];
  split_bf16(a.x, a.y, y[0][0], y[1][0], y[2][0]);
  split_bf16(a.z, a.w, y[0][1], y[1][1], y[2][1]);
  split_bf16(b.x, b.y, y[0][2], y[1][2], y[2][2]);
  split_bf16(b.z, b.w, y[0][3], y[1][3], y[2][3]);
#pragma unroll
  for (int i = 0; i < 3; ++i)
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at + i * part), "r"(y[i][0]), "r"(y[i][1]), "r"(y[i][2]), "r"(y[i][3])
                 : "memory");
}

template <int HD, bool PACKED>
__global__ void __launch_bounds__(TF_THREADS, 1)
many_rows_f32_kernel(const PrefixAttnParams p, const __grid_constant__ PoolMaps maps, int splits, int slot0) {
  using C = ManyRowsF32<HD>;
  constexpr int NRAW = C::NRAW, CH = C::CH;
  extern __shared__ __align__(1024) unsigned char mf_smem[];
  __shared__ __align__(8) uint64_t raw_full[NRAW], raw_empty[NRAW], q_full, k_full, v_full, s_full[2], p_full[2], max_full[4], pv_done, o_full, drained;
  __shared__ uint32_t s_tmem, s_absent[16];
  __shared__ int s_abort, s_req, s_row0, s_sum[TF_THREADS / 32];
  __shared__ float s_max[2][2][TC_M];  // by tile's parity, by half
  __shared__ int s_any_bad, s_bad[PACKED ? 1 : HD];  // per column the first hidden key with an infinity or NaN
  const uint32_t q_u = smem_u32(mf_smem), k_u = q_u + 3 * C::QT, v_u = k_u + 3 * C::PT, raw_u = v_u + 3 * C::PT;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int split = blockIdx.x % splits, item = blockIdx.x / splits, h = blockIdx.y;
  if (q_u & 1023) {  // the tiles' swizzle counts on the declared alignment
    pdl_wait();  // few_rows_kernel relies on it here as well
    if (threadIdx.x == 0) atomicExch(&g_prefix_attn_error, 1);
    return;
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < NRAW; ++i) {
      mbar_init(&raw_full[i], 1);
      mbar_init(&raw_empty[i], TF_CONV);
    }
    mbar_init(&q_full, TF_CONV);
    mbar_init(&k_full, TF_CONV);
    mbar_init(&v_full, TF_CONV);
    mbar_init(&s_full[0], 1);
    mbar_init(&s_full[1], 1);
    mbar_init(&p_full[0], 8);  // by buffer of S: P of the next tile may be there before this one's is taken
    mbar_init(&p_full[1], 8);
    for (int i = 0; i < 4; ++i) mbar_init(&max_full[i], 2);  // the two warps of 32 rows
    mbar_init(&pv_done, 1);
    mbar_init(&o_full, 1);
    mbar_init(&drained, 1);
    s_abort = 0;
    s_req = -1;
    s_row0 = 0;
    s_any_bad = 0;
    fence_mbar_init();
  }
  if (!PACKED && threadIdx.x < HD) s_bad[PACKED ? 0 : threadIdx.x] = INT32_MAX;
  if (warp == 1) tmem_alloc_cols(&s_tmem, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_wait();
  pdl_trigger();  // after the wait: few_rows_kernel relies on it
  volatile int* abort = &s_abort;
  const uint32_t tmem = s_tmem;  // S: buffer j at 128 j, its cross part 64 further; the products at 256, their sum at 384
  const RowShare w = row_share<PACKED, TC_M, TF_N, TF_THREADS>(p, item, split, splits, s_req, s_row0, s_sum);
  const int np = w.np, cnt = w.cnt;
  auto keys_of = [&](int t) { return t < np ? w.P - t * TF_N : w.own - (t - np) * TF_N; };
  // K tiles run one ahead of V tiles through the ring: K0 K1 V0 K2 V1 ...

  if (warp == 0) {
    // ================================ TMA producer ================================
    auto rows_of = [&](int i) {  // the pool rows of tile i, one per copy
      const int t = w.t0 + w.step * i;
      int at = -1;
      if (lane < TF_N / TF_BOX && lane * TF_BOX < keys_of(t)) {
        const int key = (t < np ? t : t - np) * TF_N + lane * TF_BOX, blk = key >> p.lg_page;
        const int id = t < np ? p.prefix_table[blk] : p.block_table[(size_t)w.b * p.max_blocks + blk];
        if (id >= 0 && id < p.n_pages) at = ((id * p.Hkv + h) << p.lg_page) + (key & ((1 << p.lg_page) - 1));
      }
      const uint32_t gone = __ballot_sync(0xffffffffu, at < 0) & ((1u << (TF_N / TF_BOX)) - 1);
      if (lane == 0) s_absent[i & 15] = gone;  // a bit per copy
      return at;
    };
    uint32_t it = 0;
    auto copy = [&](const CUtensorMap* map, int rows) {
#pragma unroll
      for (int j = 0; j < C::STEPS; ++j, ++it) {
        const int s = it % NRAW, at = __shfl_sync(0xffffffffu, rows, j * C::COPIES + lane % C::COPIES);
        if (!__all_sync(0xffffffffu, pa_wait(&raw_empty[s], ((it / NRAW) & 1u) ^ 1u, abort))) return false;
        if (lane == 0) mbar_arrive_expect_tx(&raw_full[s], C::RAW);
        __syncwarp();
        if (lane < C::COPIES) tma3d_at(raw_u + s * C::RAW + lane * C::BOX, map, at < 0 ? p.pool_rows : at, 0, &raw_full[s]);
      }
      return true;
    };
    bool ok = true;
    int row = -1, before = -1;
#pragma unroll 1
    for (int i = 0; i <= cnt && ok && cnt; ++i) {  // K of tile i, then V of tile i - 1
      before = row;
      if (i < cnt) {
        row = rows_of(i);
        ok = copy(&maps.k, row);
      }
      if (i > 0 && ok) ok = copy(&maps.v, before);
    }
    if (lane == 0) {  // copies in flight land before the CTA may exit
      int ignore = 0;
      for (uint32_t k = it > NRAW ? it - NRAW : 0; k < it; ++k) pa_wait(&raw_full[k % NRAW], (k / NRAW) & 1u, &ignore);
    }
  } else if (warp == 1) {
    // ================================ MMA issuer ================================
    if (lane == 0 && cnt > 0) {
      constexpr uint32_t mn = (1u << 4) | (1u << 7) | (1u << 10) | ((TC_M >> 4) << 24);  // bf16 by bf16 into fp32
      constexpr uint32_t idesc_s2 = mn | ((2 * TF_N >> 3) << 17), idesc_s = mn | ((TF_N >> 3) << 17);
      constexpr uint32_t idesc_o = mn | (1u << 16) | ((HD >> 3) << 17);
      const uint64_t q0 = umma_desc_sw128(q_u), q1 = umma_desc_sw128(q_u + C::QT), q2 = umma_desc_sw128(q_u + 2 * C::QT);
      const uint64_t kd = umma_desc_sw128(k_u);
      const uint64_t vd = umma_desc_sw128_mn(v_u, CH);
      const uint32_t to = tmem + 256;
      bool ok = pa_spin(&q_full, 0, abort);
#pragma unroll 1
      for (int i = -1; i < cnt && ok; ++i) {
        if (i + 1 < cnt) {  // S of the next tile; its buffer held P of tile i - 1, whose product comes before this one
          if (!(ok = pa_spin(&k_full, (i + 1) & 1, abort))) break;
          tc_fence_after();
          const uint32_t ts = tmem + ((i + 1) & 1) * 128;
#pragma unroll
          for (int kk = 0; kk < HD / 16; ++kk) {
            // K: 64-wide column, in it the 64 rows of each part
            const uint32_t qo = ((kk >> 2) * (TC_M * 128) + (kk & 3) * 32) >> 4, ko = ((kk >> 2) * 3 * CH + (kk & 3) * 32) >> 4;
            umma_f16(ts, q0 + qo, kd + ko, idesc_s2, kk != 0);  // q0 k0 | q0 k1
            umma_f16(ts, q1 + qo, kd + ko, idesc_s2, 1u);       // q1 k0 | q1 k1
            umma_f16(ts + 64, q2 + qo, kd + ko, idesc_s, 1u);   // q2 k0
            umma_f16(ts + 64, q0 + qo, kd + ko + (2 * CH >> 4), idesc_s, 1u);  // q0 k2
          }
          tc_commit(&s_full[(i + 1) & 1]);
        }
        if (i < 0) continue;
        ok = pa_spin(&v_full, i & 1, abort) && pa_spin(&p_full[i & 1], (i >> 1) & 1, abort);
        if (!ok) break;
        tc_fence_after();
        const uint32_t pt = tmem + (i & 1) * 128;  // P's parts, 32 columns each
        auto product = [&](int a, int b, int kk, uint32_t accumulate) {  // part a of P by part b of V
          umma_f16_ta(to, pt + a * 32 + kk * 8, vd + ((b * C::PT + kk * 2048) >> 4), idesc_o, accumulate);
        };
#pragma unroll
        for (int kk = 0; kk < TF_N / 16; ++kk) {
          product(2, 0, kk, kk != 0);
          product(1, 1, kk, 1u);
          product(0, 2, kk, 1u);
          product(1, 0, kk, 1u);
          product(0, 1, kk, 1u);
        }
#pragma unroll
        for (int kk = 0; kk < TF_N / 16; ++kk) product(0, 0, kk, 1u);
        tc_commit(&pv_done);
        if (i + 1 == cnt) tc_commit(&o_full);
      }
    }
  } else if (warp >= 12) {
    // ================================ split Q, K and V ================================
    constexpr int LPK = C::LPK, KPW = C::KPW, STEPS = C::STEPS;
    const int cw = warp - 12, g = lane % LPK, sub = lane / LPK;
    const bool odd = (g >> 2) & 1;
    uint32_t it = 0;
    // Slots from `keys` on become zero, and what is not finite (or not in bf16) from `shown` on: rows that do not
    // see those keys have weights of zero for them, the others become NaN at the end.  key0: the tile's first own key.
    auto convert = [&](bool is_v, int keys, int shown, int key0) {
      const uint32_t to = is_v ? v_u + (g >> 3) * CH : k_u + (g >> 3) * 3 * CH, part = is_v ? C::PT : CH;
#pragma unroll 1
      for (int j = 0; j < STEPS; ++j, ++it) {
        const int s = it % NRAW;
        if (!__all_sync(0xffffffffu, pa_wait(&raw_full[s], (it / NRAW) & 1u, abort))) return false;
        const int in = cw * KPW + sub, r = in % TF_BOX, key = j * C::KEYS + in;  // key of the stage, of the tile
        // 8 values: pieces 2 (g % 4) and 2 (g % 4) + 1 of 128-byte chunk g / 4; odd chunks in the other order, so that
        // eight lanes read all the banks
        const uint32_t at = raw_u + s * C::RAW + (in / TF_BOX) * C::BOX + (g >> 2) * (TF_BOX * 128) + r * 128;
        const int p0 = 2 * (g & 3) + odd;
        float4 a = lds_f4(at + ((p0 ^ (r & 7)) << 4)), b = lds_f4(at + (((p0 ^ 1) ^ (r & 7)) << 4));
        if (key >= keys) a = b = make_float4(0.f, 0.f, 0.f, 0.f);
        if (!PACKED && key >= shown) {
          float* y[8] = {&a.x, &a.y, &a.z, &a.w, &b.x, &b.y, &b.z, &b.w};
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            if (fabsf(*y[k]) < __uint_as_float(0x7f7f8000u)) continue;  // what bf16 rounds to a number
            *y[k] = 0.f;
            atomicMin(&s_bad[PACKED ? 0 : g * 8 + ((k < 4) != odd ? k & 3 : 4 + (k & 3))], key0 + key);
            s_any_bad = 1;
          }
        }
        split_bf16x8(odd ? b : a, odd ? a : b, to + sw128(key, g & 7), part);
        __syncwarp();  // the stage's values are in registers
        if (lane == 0) mbar_arrive(&raw_empty[s]);
      }
      fence_async_smem();
      if (!PACKED) __threadfence_block();
      __syncwarp();
      return true;
    };
    if (cnt > 0) {
      constexpr int QS = TC_M / (TF_CONV * KPW);  // this warp's share of Q's rows
#pragma unroll 1
      for (int j0 = 0; j0 < QS; j0 += 4) {
        float4 a[4], b[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int gr = w.r0 + ((j0 + j) * TF_CONV + cw) * KPW + sub;
          a[j] = b[j] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (gr < w.rows) {
            const float4* src = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p.q) +
                                                                ((size_t)(w.row_lo + gr / p.G) * p.Hq + h * p.G + gr % p.G) * HD + g * 8);
            a[j] = src[0];
            b[j] = src[1];
          }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          split_bf16x8(a[j], b[j], q_u + (g >> 3) * (TC_M * 128) + sw128(((j0 + j) * TF_CONV + cw) * KPW + sub, g & 7), C::QT);
        }
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_full);
    }
    bool ok = true;
#pragma unroll 1
    for (int n = 0; n < 2 * cnt && ok; ++n) {  // K0 K1 V0 K2 V1 ...
      const bool is_v = n == 2 * cnt - 1 || (n > 0 && !(n & 1));
      const int i = is_v ? (n - 1) >> 1 : (n + 1) >> 1, t = w.t0 + w.step * i, key0 = (t - np) * TF_N;
      // K goes where S of the tile before is done with, V where the product of the tile before is
      if (i > 0) ok = __all_sync(0xffffffffu, is_v ? pa_wait(&pv_done, (i - 1) & 1, abort) : pa_wait(&s_full[(i - 1) & 1], ((i - 1) >> 1) & 1, abort));
      ok = ok && convert(is_v, is_v ? keys_of(t) : TF_N, PACKED || !is_v || t < np ? TF_N : w.all - key0, key0);
      if (ok && lane == 0) mbar_arrive(is_v ? &v_full : &k_full);
    }
  } else if (warp >= 4) {
    // ================================ softmax ================================
    const int half = (warp - 4) >> 2;  // keys 32 half .. 32 half + 31 of every tile; half of O's columns
    const int lanes = (warp & 3) * 32;
    const int r = w.r0 + lanes + lane;  // this thread's row
    const uint32_t tl = tmem + ((uint32_t)lanes << 16), ot = tl + 256 + half * (HD / 2), sum = ot + 128;
    const bool valid = w.work && r < w.rows;
    const int see = PACKED ? 0 : (valid ? max(0, min(w.len, w.len - w.n + r / p.G + 1)) : w.own);
    const float c = p.c;
    float m = -INFINITY, l = 0.f;
    const size_t row = valid ? (size_t)(w.row_lo + r / p.G) * p.Hq + h * p.G + r % p.G : 0;
    const size_t at = (size_t)(slot0 + split) * p.T * p.Hq + row;
    bool far = false;
    if (cnt > 0) {
      bool ok = true;
      for (int i = 0; i < cnt; ++i) {
        ok = __all_sync(0xffffffffu, pa_wait(&s_full[i & 1], (i >> 1) & 1, abort));
        if (!ok) break;
        tc_fence_after();
        const uint32_t st = tl + (i & 1) * 128 + half * 32;
        const int t = w.t0 + w.step * i;
        const uint32_t gone = (s_absent[i & 15] >> (half * (32 / TF_BOX))) & ((1u << (32 / TF_BOX)) - 1);
        // of this thread's keys, those that its row sees
        const int lim = (t < np ? w.P : see) - (t < np ? t : t - np) * TF_N - half * 32;
        float v[32], x[32];
        tmem_ld32_async(st, v);
        tmem_ld32_async(st + 64, x);
        tmem_wait_ld();
        tmem_ready(v);
        tmem_ready(x);
#pragma unroll
        for (int k = 0; k < 32; k += 2) unpack2(add2(pack2(v[k], v[k + 1]), pack2(x[k], x[k + 1])), v[k], v[k + 1]);
        if (__any_sync(0xffffffffu, lim < 32) || gone != 0) {
#pragma unroll
          for (int k = 0; k < 32; ++k) v[k] = k < lim && !((gone >> (k / TF_BOX)) & 1u) ? v[k] : -INFINITY;
        }
        float a0 = fmaxf(v[0], v[1]), a1 = fmaxf(v[2], v[3]);
#pragma unroll
        for (int k = 4; k < 32; k += 4) {
          a0 = max3(a0, v[k], v[k + 1]);
          a1 = max3(a1, v[k + 2], v[k + 3]);
        }
        float mx = fmaxf(a0, a1) * c;
        s_max[i & 1][half][lanes + lane] = mx;
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&max_full[warp & 3]);
        ok = __all_sync(0xffffffffu, pa_wait(&max_full[warp & 3], i & 1, abort));  // both have read S, too: P goes over it
        if (!ok) break;
        tc_fence_after();
        mx = fmaxf(mx, s_max[i & 1][half ^ 1][lanes + lane]);
        const bool up = __any_sync(0xffffffffu, mx > m + TF_RAISE);  // also from -inf; the other half comes to the same
        float f = 1.f;
        if (up) {
          const float mn = fmaxf(m, mx);
          f = m == -INFINITY ? 0.f : ex2(m - mn);
          m = mn;
          far = __any_sync(0xffffffffu, fabsf(m) >= PA_FAR && m != -INFINITY);
          l *= f;
        }
        const float mm = m == -INFINITY ? 0.f : m;
        uint64_t l2 = pack2(0.f, 0.f);
        const uint32_t pt = tl + (i & 1) * 128 + half * 16;
        auto weights = [&](auto is_far) {
          const uint64_t c2 = pack2(c, c), m2 = pack2(-mm, -mm);
#pragma unroll
          for (int q = 0; q < 32; q += 16) {
            uint32_t p0[8], p1[8], p2[8];
#pragma unroll
            for (int k = 0; k < 16; k += 2) {
              float e0, e1;
              if constexpr (is_far) {
                e0 = far_exponent(v[q + k], c, mm);
                e1 = far_exponent(v[q + k + 1], c, mm);
              } else {
                unpack2(fma2(pack2(v[q + k], v[q + k + 1]), c2, m2), e0, e1);
              }
              e0 = ex2(e0);
              e1 = ex2(e1);
              l2 = add2(l2, pack2(e0, e1));
              split_bf16(e0, e1, p0[k / 2], p1[k / 2], p2[k / 2]);
            }
            tmem_st8(pt + q / 2, p0);
            tmem_st8(pt + 32 + q / 2, p1);
            tmem_st8(pt + 64 + q / 2, p2);
          }
        };
        if (far)
          weights(std::true_type{});
        else
          weights(std::false_type{});
        if (i > 0) {  // the last tile's products, made while this tile's P was, go to the sum
          ok = __all_sync(0xffffffffu, pa_wait(&pv_done, (i - 1) & 1, abort));
          if (!ok) break;
          tc_fence_after();
#pragma unroll 1
          for (int q = 0; q < HD / 2; q += 32) {
            float u[32];
            tmem_ld32_wait(ot + q, u);
            if (i > 1) {
              float y[32];
              tmem_ld32_wait(sum + q, y);
#pragma unroll
              for (int k = 0; k < 32; ++k) u[k] += y[k];
            }
#pragma unroll
            for (int k = 0; k < 32; ++k) u[k] *= f;
            tmem_st32(sum + q, u);
          }
        }
        float l0, l1;
        unpack2(l2, l0, l1);
        l += l0 + l1;
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[i & 1]);
      }
      ok = ok && __all_sync(0xffffffffu, pa_wait(&o_full, 0, abort));
      tc_fence_after();
      if (ok) {
        s_max[cnt & 1][half][lanes + lane] = l;
        __syncwarp();
        if (lane == 0) mbar_arrive(&max_full[warp & 3]);
        ok = __all_sync(0xffffffffu, pa_wait(&max_full[warp & 3], cnt & 1, abort));
        l += s_max[cnt & 1][half ^ 1][lanes + lane];
        const float inv = l == 0.f ? 0.f : 1.f / l;
        if (valid && p.nslots > 1 && half == 0) p.part_ml[at] = make_float2(m, l);
        float* dst = (p.nslots > 1 ? p.part_o + (at - row) * HD : reinterpret_cast<float*>(p.out)) + half * (HD / 2);
        const float f = p.nslots > 1 ? 1.f : inv;
        float v[HD / 2];
#pragma unroll
        for (int q = 0; q < HD / 2; q += 32) {
          tmem_ld32_wait(ot + q, v + q);
          if (cnt > 1) {
            float x[32];
            tmem_ld32_wait(sum + q, x);
#pragma unroll
            for (int k = 0; k < 32; ++k) v[q + k] += x[k];
          }
#pragma unroll
          for (int k = 0; k < 32; ++k) v[q + k] *= f;
          if (!PACKED && s_any_bad) {
#pragma unroll
            for (int k = 0; k < 32; ++k)
              if (see > s_bad[PACKED ? 0 : half * (HD / 2) + q + k]) v[q + k] = NAN;
          }
        }
        // through Q's tiles, which are done with
        flush_rows<HD * 2>(q_u + (warp - 4) * 32 * HD * 2, [&](int c) { return f4_as_u4(v + c * 4); }, reinterpret_cast<char*>(dst),
                           HD * sizeof(float), row, valid);
      }
    } else if (valid && half == 0) {  // no keys in this share
      if (p.nslots > 1) {
        p.part_ml[at] = make_float2(-INFINITY, 0.f);
      } else {
        for (int d = 0; d < HD; d += 4)
          *reinterpret_cast<float4*>(reinterpret_cast<float*>(p.out) + row * HD + d) = make_float4(0.f, 0.f, 0.f, 0.f);
      }
    }
  }
  // after a wait that ran out: the products in flight have ended before the TMEM is freed
  tc_fence_before();
  const bool failed = __syncthreads_or(*abort);
  tc_fence_after();
  if (failed && threadIdx.x == 32) {
    int ignore = 0;
    tc_commit(&drained);
    pa_wait(&drained, 0, &ignore);
  }
  __syncthreads();
  if (warp == 1) {
    tmem_dealloc_cols(tmem, 512);
    tmem_relinquish();
  }
  if (threadIdx.x == 0 && failed) atomicExch(&g_prefix_attn_error, 1);
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

// A pool [rows, hd] as (128-byte chunk, row, chunk index), box (chunk, box_rows, box_chunks), 128-byte swizzle: a
// copy lies in shared memory as box_chunks sub-tiles of box_rows rows of 128 bytes.
static bool pool_map(CUtensorMap* m, const void* pool, size_t rows, int hd, bool f16, int box_rows, int box_chunks) {
  static const PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      ptr = nullptr;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
  }();
  if (!fn) return false;
  const int es = f16 ? 2 : 4, chunk = 128 / es;
  cuuint64_t dims[3] = {(cuuint64_t)chunk, (cuuint64_t)rows, (cuuint64_t)(hd / chunk)};
  cuuint64_t strides[2] = {(cuuint64_t)hd * es, 128};
  cuuint32_t box[3] = {(cuuint32_t)chunk, (cuuint32_t)box_rows, (cuuint32_t)box_chunks}, step[3] = {1, 1, 1};
  return fn(m, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, const_cast<void*>(pool), dims,
            strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

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

// How a call is cut.  The host knows the rows T and the requests B, not which request has how many, nor how many
// keys there are, only how many the tables hold.
//   few rows      few_rows_kernel over the prefix and the requests' own keys, its shares joined in a cluster if they are short
//   shared        a many-rows kernel, PACKED, over the prefix, few_rows_kernel over the own keys
//   chunks        a many-rows kernel over both, a request's rows at a time
struct AttnPlan {
  enum Kind { FEW, SHARED, CHUNKS } kind;
  int splits, row_groups;       // few_rows_kernel
  bool cluster;                 // its shares are joined in a cluster
  int tc_splits, tc_items;      // many_rows_kernel, many_rows_f32_kernel
  int nslots;
};

static AttnPlan plan_attn(int T, int B, int Hkv, int G, int hd, bool f16, long long own_keys, long long prefix_keys, int sms) {
  AttnPlan a{};
  const int per_cta = f16 ? 2 * TC_M : TC_M, tile = f16 ? TC_N : TF_N;
  const long long rows = (long long)T * G, items = (rows + per_cta - 1) / per_cta;
  const auto ceil_div = [](long long x, long long y) { return (x + y - 1) / y; };
  const int rt = f16 ? 16 : 8;
  const long long groups = ceil_div(rows, (long long)B * rt), slots = 2ll * sms;  // few_rows_kernel: two CTAs an SM
  // The few-rows kernel streams a request's keys, the prefix's too, once per tile of 16 (8) rows.  While that is little it
  // beats the others: up to so many keys a CTA slot, in clusters of eight at most.  us in a graph, fp16, few | shared: 8 kv
  // heads of 128, 1050 keys a slot 17.6 | 21.2 and 17.6 | 20.2, 1300 19.1 | 19.7, 2100 28.1 | 23.8; 4 of 64, 1050 13.8 |
  // 16.1, 2050 21.2 | 18.8; few | chunks: 210 13.3 | 16.5, 410 13.4 | 21.3 and 18.6 | 24.8, 520 19.0 | 17.9 and 14.0 | 13.6,
  // 1250 31.2 | 20.9.  fp32, few | shared: 142 12.6 | 16.0 and 8.4 | 11.0, 266 16.4 | 19.2, 277 17.9 | 15.6 and 13.2 | 12.4, 392
  // 21.5 | 23.8 and 15.1 | 14.6, 490 36.2 | 19.1; few | chunks: 104 9.2 | 11.2, 121 11.1 | 16.1, 182 12.9 | 19.1, 225 18.2 |
  // 18.2 and 13.3 | 12.1, 242 18.5 | 19.0 and 14.7 | 12.0, 303 19.4 | 17.0 and 15.0 | 12.0.
  const double load = (double)(own_keys + prefix_keys) * std::max(slots / FR_CLUSTER, (long long)B * Hkv * groups) / slots;
  const bool many = rows >= 64ll * B, shares = prefix_keys > 0 && B > 1;
  if (load <= (many ? (f16 ? 450 : 220) : (f16 ? 1100 : 320)) || !(many || shares))
    a.kind = AttnPlan::FEW;
  // A chunk fills its last tile of rows for itself alone, where SHARED packs all requests' rows: worth a second kernel while
  // a request has less than a tile and the prefix is most of what it sees (behind 2000 tokens, shared | chunks: 8 requests of
  // 80 rows 29.3 | 43.9, of 160 21.1 | 27.6, of 240 55.8 | 40.1; behind 300 with 200 own, fp32, of 150 57.1 | 37.7).
  else if (!many || (shares && rows < 192ll * B && prefix_keys >= 4 * own_keys))
    a.kind = AttnPlan::SHARED;
  else
    a.kind = AttnPlan::CHUNKS;
  if (a.kind != AttnPlan::FEW) {
    // Shares of the keys until there is a CTA for every SM; with the own keys' kernel beside it, for this kernel's part
    // of the SMs only.  That part goes by the two kernels' work, as far as the host knows it: a tile takes an SM 2.1 us
    // (256 rows, 128 keys, fp16) or 2.9 us (128 rows, 64 keys, fp32), and own keys, taken for half of what the tables
    // hold, stream at 44 KB a us and SM.  Measured over the splits 3, 4, 6, 8, 10, 14: 64 requests behind 8197 tokens,
    // fp16, 61, 53, 55, 58, 60, 64 us (the rule takes 4); 32 behind 4099, fp32, 82, 68, 51, 45, 45, 48 us (it takes 8).
    long long part = 1000;
    const long long tiles = ceil_div(prefix_keys + (a.kind == AttnPlan::CHUNKS ? own_keys : 0), tile);
    if (a.kind == AttnPlan::SHARED) {
      const double many = (double)items * Hkv * tiles * (f16 ? 2.1 : 2.9);
      const double few = (double)B * own_keys / 2 * Hkv * hd * (f16 ? 4 : 8) / 44e3;
      part = (long long)(1000 * many / (many + few));
    }
    a.tc_items = (int)(a.kind == AttnPlan::CHUNKS ? items + B : items);
    a.tc_splits = (int)std::max(1ll, std::min({(sms * part / 1000 + items * Hkv / 2) / (items * Hkv), sms / (items * Hkv), tiles, 32ll}));
    // No more shares than their longest one needs: eight tiles in five shares take two each, as in four.  A second share
    // brings the join: not for less than three tiles (us, chunks, one share | as many as there are SMs for; fp16: 3 requests
    // of 150 tokens, 2 tiles 14.3 | 21.6; 8 of 60 behind 300, 4 tiles in two shares 18.5 | 25.9; one of 150 behind 300, 4 in
    // four 20.4 | 17.9; fp32: 8 of 20, 2 tiles 15.7 | 19.9).
    a.tc_splits = (int)ceil_div(tiles, ceil_div(tiles, a.tc_splits));
    if (a.kind == AttnPlan::CHUNKS && tiles - ceil_div(tiles, a.tc_splits) < 3) a.tc_splits = 1;
    // The tensor cores' cut-off sums lose 1.1e-9 of O per key; with fp16 that is left, up to 131072 keys a share (1.4e-4, the
    // output's own error is 1.8e-4).  A table with room for more is cut.
    if (f16) a.tc_splits = std::max(a.tc_splits, (int)std::min(32ll, ceil_div(tiles, 131072 / TC_N)));
    a.nslots = a.tc_splits;
  }
  if (a.kind != AttnPlan::CHUNKS) {
    const long long keys = own_keys + (a.kind == AttnPlan::FEW ? prefix_keys : 0);
    // (row tiles are counted for the mean request: twice as many CTAs, so that one of twice the rows does not take twice as long)
    const long long want = ceil_div(4ll * sms, (long long)B * Hkv);
    a.row_groups = (int)std::max(1ll, std::min(want, groups > 1 ? 2 * groups : 1));
    // Shares of 64 keys or more.  Of as many as all run at once, while there are few keys for each place of a CTA; what the
    // few-rows kernel alone computes is then joined within a cluster.  Past that four CTAs per SM, which even out requests of
    // different lengths, or for one request use the whole machine, and their results are joined by a kernel more.
    // Measured with lengths spread evenly up to the longest (us in a graph, all at once | four, no prefix; fp16: 64 requests,
    // 8 kv heads of 128, 870 keys a place 19.1 | 23.5, 2600 40.9 | 40.4, 6900 99.7 | 94.1; 16, 4 of 64, 1000 12.6 | 17.8, 3000
    // 28.2 | 26.9; fp32: 4, 8 of 128, 500 25.8 | 29.8, 1500 54.8 | 46.1; 64, 860 37.2 | 38.0, 2600 87.0 | 74.3).
    const long long most = ceil_div(keys, 64);
    const long long once = std::max(1ll, std::min({slots / ((long long)B * Hkv * a.row_groups), most, a.kind == AttnPlan::FEW ? (long long)FR_CLUSTER : 64ll}));
    const bool few_keys = (double)keys * std::max(ceil_div(slots, once), (long long)B * Hkv * a.row_groups) <= slots * (f16 ? 1536 : 512);
    a.splits = (int)(few_keys ? once : std::max(1ll, std::min({ceil_div(want, a.row_groups), most, 64ll})));
    a.cluster = few_keys && a.kind == AttnPlan::FEW && a.splits > 1;
    a.nslots += a.cluster ? 1 : a.splits;
  }
  return a;
}

template <auto KERN>
static int run_many_rows(int smem, int threads, const PrefixAttnParams& p, const PoolMaps& maps, const AttnPlan& a, cudaStream_t stream) {
  const cudaError_t e = opt_in<KERN>(smem);
  if (e != cudaSuccess) return check_launch("prefix_attn", e);
  launch(KERN, dim3((unsigned)(a.tc_splits * a.tc_items), p.Hkv), dim3(threads), smem, stream, p, maps, a.tc_splits, 0);
  return check_launch("prefix_attn_many_rows");
}

template <typename T, int HD, bool CLUSTER>
static int run_few_rows(const PrefixAttnParams& p, const PoolMaps& maps, const AttnPlan& a, cudaStream_t stream) {
  constexpr auto kern = few_rows_kernel<T, HD, CLUSTER>;
  constexpr int smem = FewRows<T, HD>::SMEM;
  const cudaError_t e = opt_in<kern>(smem);
  if (e != cudaSuccess) return check_launch("prefix_attn", e);
  launch_clusters(CLUSTER ? a.splits : 1, kern, dim3(a.splits * a.row_groups, p.Hkv, p.B), dim3(FR_WARPS * 32), smem, stream, p, maps,
                  a.kind == AttnPlan::FEW ? 1 : 0, a.splits, a.row_groups, a.kind == AttnPlan::SHARED ? a.tc_splits : 0);
  return check_launch("prefix_attn_few_rows");
}

template <typename T, int HD>
static int run_attn(const PrefixAttnParams& p, const void* k, const void* v, const AttnPlan& a, cudaStream_t stream) {
  using C = FewRows<T, HD>;
  int st = SC_OK;
  static_assert(C::F16 || C::KT == TF_BOX, "both fp32 kernels copy boxes of eight keys");
  PoolMaps maps;
  const auto encode = [&](int box, int chunks) {
    return pool_map(&maps.k, k, p.pool_rows, HD, C::F16, box, chunks) && pool_map(&maps.v, v, p.pool_rows, HD, C::F16, box, chunks);
  };
  const bool tiles = C::F16 && a.kind != AttnPlan::FEW;  // many_rows_kernel: a page's rows of a 64-wide column at a time
  SC_REQUIRE(tiles ? encode(std::min(TC_N, 1 << p.lg_page), 1) : encode(C::KT, C::NB), SC_ERR_CUDA,
             "prefix_attn: tensor map of the pages refused");
  if (a.kind != AttnPlan::FEW) {
    const bool packed = a.kind == AttnPlan::SHARED;
    if constexpr (C::F16)
      st = packed ? run_many_rows<many_rows_kernel<HD, true>>(ManyRows<HD>::SMEM, TC_THREADS, p, maps, a, stream)
                  : run_many_rows<many_rows_kernel<HD, false>>(ManyRows<HD>::SMEM, TC_THREADS, p, maps, a, stream);
    else
      st = packed ? run_many_rows<many_rows_f32_kernel<HD, true>>(ManyRowsF32<HD>::SMEM, TF_THREADS, p, maps, a, stream)
                  : run_many_rows<many_rows_f32_kernel<HD, false>>(ManyRowsF32<HD>::SMEM, TF_THREADS, p, maps, a, stream);
    if (st != SC_OK) return st;
  }
  if (a.kind != AttnPlan::CHUNKS) {
    SC_REQUIRE(!tiles || encode(C::KT, C::NB), SC_ERR_CUDA, "prefix_attn: tensor map of the pages refused");
    st = a.cluster ? run_few_rows<T, HD, true>(p, maps, a, stream) : run_few_rows<T, HD, false>(p, maps, a, stream);
    if (st != SC_OK) return st;
  }
  if (p.nslots == 1) return SC_OK;
  launch(join_slots_kernel<T, HD>, dim3((unsigned)(((size_t)p.T * p.Hq + 7) / 8)), dim3(256), 0, stream, p);
  return check_launch("prefix_attn_join");
}

}  // namespace sc

extern "C" {

int sc_prefix_attn_device_error(int reset) {
  int v = 0;
  cudaMemcpyFromSymbol(&v, sc::g_prefix_attn_error, sizeof(int));
  if (reset) {
    const int z = 0;
    cudaMemcpyToSymbol(sc::g_prefix_attn_error, &z, sizeof(int));
  }
  return v;
}

size_t sc_prefix_attn_workspace_bytes(int T, int B, int Hq, int Hkv, int hd, int max_blocks, int max_prefix_blocks,
                                      int page_size, int dtype) {
  if (T < 1 || B < 1 || Hq < 1 || Hkv < 1 || hd < 1 || max_blocks < 0 || max_prefix_blocks < 0 || page_size < 1) return 0;
  if (Hq % Hkv) return 0;
  const sc::AttnPlan a = sc::plan_attn(T, B, Hkv, Hq / Hkv, hd, dtype == SC_F16, (long long)max_blocks * page_size,
                                       (long long)max_prefix_blocks * page_size, sc::sm_count());
  return a.nslots <= 1 ? 0 : (size_t)a.nslots * T * Hq * (hd + 2) * sizeof(float);
}

int sc_prefix_attn(const void* q, const void* k_pages, const void* v_pages, int dtype, int T, const int32_t* q_start,
                   const int32_t* kv_lens, const int32_t* block_table, int B, int max_blocks,
                   const int32_t* prefix_table, const int32_t* prefix_len, int max_prefix_blocks, int Hq, int Hkv,
                   int hd, int n_pages, int page_size, float scale, void* out, void* workspace, size_t workspace_bytes,
                   cudaStream_t stream) {
  using namespace sc;
  SC_REQUIRE(q && k_pages && v_pages && q_start && kv_lens && block_table && out, SC_ERR_ARG, "prefix_attn: null pointer");
  SC_REQUIRE(!prefix_len || (prefix_table && max_prefix_blocks >= 1), SC_ERR_ARG, "prefix_attn: a prefix needs its table");
  SC_REQUIRE(dtype == SC_F16 || dtype == SC_F32, SC_ERR_ARG, "prefix_attn: dtype");
  SC_REQUIRE(hd == 64 || hd == 128, SC_ERR_UNSUPPORTED, "prefix_attn: head_dim %d unsupported (64, 128)", hd);
  SC_REQUIRE(page_size >= 16 && page_size <= 32768 && (page_size & (page_size - 1)) == 0, SC_ERR_UNSUPPORTED,
             "prefix_attn: page size %d unsupported (a power of two from 16)", page_size);
  SC_REQUIRE(T >= 1 && B >= 1 && B <= 65535 && max_blocks >= 1 && n_pages >= 1, SC_ERR_SHAPE, "prefix_attn: bad T/B/max_blocks");
  SC_REQUIRE(Hkv >= 1 && Hkv <= 65535 && Hq >= Hkv && Hq % Hkv == 0, SC_ERR_SHAPE, "prefix_attn: Hq=%d not a multiple of Hkv=%d", Hq, Hkv);
  SC_REQUIRE((long long)n_pages * Hkv * page_size < INT32_MAX && (long long)T * Hq <= (1 << 30) &&
                 (long long)max_blocks * page_size <= INT32_MAX && (long long)max_prefix_blocks * page_size <= INT32_MAX,
             SC_ERR_SHAPE, "prefix_attn: rows past 32 bits");
  const float c = scale * 1.4426950408889634f;  // log2(e)
  SC_REQUIRE(scale > 0.f && c < INFINITY, SC_ERR_ARG, "prefix_attn: scale must be positive and below 2.3e38");
  SC_REQUIRE((((uintptr_t)q | (uintptr_t)k_pages | (uintptr_t)v_pages | (uintptr_t)out) & 15) == 0, SC_ERR_ARG,
             "prefix_attn: tensors must start on 16-byte boundaries");
  if (!prefix_len) max_prefix_blocks = 0;
  const AttnPlan a = plan_attn(T, B, Hkv, Hq / Hkv, hd, dtype == SC_F16, (long long)max_blocks * page_size,
                               (long long)max_prefix_blocks * page_size, sm_count());
  const size_t need = sc_prefix_attn_workspace_bytes(T, B, Hq, Hkv, hd, max_blocks, max_prefix_blocks, page_size, dtype);
  SC_REQUIRE(workspace_bytes >= need && (need == 0 || workspace), SC_ERR_WORKSPACE,
             "prefix_attn: workspace of %zu bytes needed (got %zu)", need, workspace_bytes);
  SC_REQUIRE(((uintptr_t)workspace & 15) == 0, SC_ERR_ARG, "prefix_attn: the workspace must start on a 16-byte boundary");
  PrefixAttnParams p{};
  p.q = q;
  p.out = out;
  p.part_o = static_cast<float*>(workspace);
  p.part_ml = reinterpret_cast<float2*>(p.part_o + (size_t)a.nslots * T * Hq * hd);
  p.q_start = q_start;
  p.kv_lens = kv_lens;
  p.block_table = block_table;
  p.prefix_table = prefix_table;
  p.prefix_len = prefix_len;
  p.T = T;
  p.B = B;
  p.max_blocks = max_blocks;
  p.max_prefix_blocks = max_prefix_blocks;
  p.n_pages = n_pages;
  p.lg_page = __builtin_ctz(page_size);
  p.Hq = Hq;
  p.Hkv = Hkv;
  p.G = Hq / Hkv;
  p.pool_rows = n_pages * Hkv * page_size;
  p.c = c;
  p.nslots = a.nslots;
  if (dtype == SC_F16)
    return hd == 128 ? run_attn<__half, 128>(p, k_pages, v_pages, a, stream) : run_attn<__half, 64>(p, k_pages, v_pages, a, stream);
  return hd == 128 ? run_attn<float, 128>(p, k_pages, v_pages, a, stream) : run_attn<float, 64>(p, k_pages, v_pages, a, stream);
}

}  // extern "C"
