// Attention of a ragged batch over a paged cache whose requests share a
// prefix: row i of request b (n new tokens, len tokens with them) sees the
// prefix's keys [0, P) and its own tokens [0, len - n + i].
//
//   o = sum_j exp(scale q.k_j - m) v_j / sum_j exp(scale q.k_j - m)
//
// over the keys it sees; m is any bound of the exponents, so a key range can
// be summed apart (o, l, m) and joined later.  A row that sees no key is zero.
#include <cudaTypedefs.h>

#include "sc_many_rows.cuh"

namespace sc {

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

// How a call is cut.  The host knows the rows T and the requests B, not which request has how many, nor how many
// keys there are, only how many the tables hold.
//   few rows      few_rows_kernel over the prefix and the requests' own keys, its shares joined in a cluster if they are short
//   shared        a many-rows kernel, PACKED, over the prefix, few_rows_kernel over the own keys
//   chunks        a many-rows kernel over both, a request's rows at a time
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
      st = packed ? run_many_rows<many_rows_kernel<HD, true, PoolMaps>>(ManyRows<HD>::SMEM, TC_THREADS, p, maps, a, stream)
                  : run_many_rows<many_rows_kernel<HD, false, PoolMaps>>(ManyRows<HD>::SMEM, TC_THREADS, p, maps, a, stream);
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
  return v | sc::quant_attn_device_error(reset);
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
