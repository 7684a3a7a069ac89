// Attention of a ragged batch behind a shared prefix (sc_prefix_attn.cu) over
// pages in 8 or 4 bits: a token's k and v of a head are s c + b by groups of
// dims (sc_quant.cuh), and the codes c go into the products as they are:
//   q.k = sum_g s_g (q_g.c_g) + b_g (sum of q over g)
//   o_g = sum_j (p_j s_jg) c_jg + sum_j p_j b_jg
#include "sc_prefix_attn.cuh"
#include "sc_quant.cuh"

namespace sc {

// ---------------------------------------------------------------- few rows

// A CTA takes a request, a kv head, a share of the keys and every row_groups-th
// tile of rows; its warps take blocks of 16 tokens in turn, each with a ring of
// blocks of its own (one bulk copy each) and a running (m, l, o) of its own.
//
// mma.sync m16n8k16 with the tokens (S = K Q^T), then the dims (O = V^T P^T) as
// its 16 rows, the queries as its 8 columns: a decoded token of four heads
// fills half of them, where queries as rows would fill a quarter.  A register
// of K's or V's operand is one AND of a word of codes (fp16 subnormals), so a
// value costs 0.6 instructions; scales and biases are applied in fp32, to S
// per group and to the weights before their product.  S passes to the second
// product's operand through movmatrix.
//
// q is scaled per row by a power of two so that its largest value is in
// [2^11, 2^12): exact, and the 1/16 that the codes at 2^-20 need loses nothing.
// The weights p s are rounded to fp16, 2^11 to 2^15 high at the row's largest p s
// (PA_LIFT over c s + log2 of the token's largest scale): 2^-11 of each, the
// output's own rounding, down to 2^-25 of that largest.
template <typename QB, int NT>
struct FewRowsQuant {
  static constexpr int RT = 8 * NT;            // rows of a tile
  static constexpr int WORDS = QB::KSH / 4;    // of codes in a thread's share of a token
  static constexpr int PER = 32 / QB::BITS;    // codes of a word
  static constexpr int KSTEPS = QB::HD / 16, MT = QB::HD / 16;
  static constexpr int NST = QB::BYTES > 3000 ? 4 : QB::BYTES > 1600 ? 5 : 8;
  static constexpr int OUT = 2 * RT * QB::HD * 4;  // a warp's result, and the CTA's behind it
  static constexpr int RING = NST * QB::BYTES > OUT ? NST * QB::BYTES : OUT;
  static constexpr int SMEM = FR_WARPS * RING + 128;
  static constexpr int CTAS = NT == 1 ? 4 : 3;  // of an SM
};

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ float min_keep_nan(float a, float b) {
  float d;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
// N words from shared memory.
template <int N>
__device__ __forceinline__ void lds_words(uint32_t a, uint32_t (&w)[N]) {
  if constexpr (N == 1) {
    w[0] = lds_u32(a);
  } else if constexpr (N == 2) {
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(a));
  } else {
    const uint4 v = lds_v4(a);
    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
  }
}
// A thread's share of a token's K (of a pair's V): `at` is its first piece, `other` its second where it has two.
template <int N>
__device__ __forceinline__ void lds_share(uint32_t at, uint32_t other, uint32_t (&w)[N]) {
  if constexpr (N == 8) {
    uint32_t x[4], y[4];
    lds_words<4>(at, x);
    lds_words<4>(other, y);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = x[i];
      w[4 + i] = y[i];
    }
  } else {
    lds_words<N>(at, w);
  }
}

template <typename QB, int NT, bool CLUSTER>
__global__ void __launch_bounds__(FR_WARPS * 32, FewRowsQuant<QB, NT>::CTAS)
few_rows_quant_kernel(const PrefixAttnParams p, const uint8_t* pages, int with_prefix, int splits, int row_groups, int slot0) {
  using C = FewRowsQuant<QB, NT>;
  constexpr int RT = C::RT, NST = C::NST, KT = 16, HD = QB::HD, NG = QB::NG, GS = QB::GS, WORDS = C::WORDS, PER = C::PER;
  extern __shared__ __align__(128) unsigned char fq_smem[];
  __shared__ __align__(8) uint64_t full[FR_WARPS][NST];
  __shared__ float s_m[FR_WARPS][RT], s_l[FR_WARPS][RT];
  __shared__ float2 s_ml[CLUSTER ? RT : 1];
  __shared__ int s_abort;
  unsigned char* base = fq_smem;
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
  // Without the prefix this kernel runs beside the prefix's, as few_rows_kernel does (sc_prefix_attn.cu).
  if (with_prefix) pdl_wait();
  const int P = with_prefix ? prefix_keys(p) : 0, np = (P + KT - 1) / KT;
  const int t0 = split * FR_WARPS + warp, step = splits * FR_WARPS;
  // the pool's blocks of this warp's tiles first .. first + 31, one per lane; -1: no such page
  auto blocks_of = [&](int first) {
    const long long t = t0 + (long long)step * (first + lane);
    const bool pre = t < np;
    const long long key = (pre ? t : t - np) * KT;
    const int blk = (int)min(key >> p.lg_page, (long long)INT32_MAX);
    if (blk >= (pre ? p.max_prefix_blocks : p.max_blocks)) return -1;
    const int id = pre ? p.prefix_table[blk] : p.block_table[(size_t)b * p.max_blocks + blk];
    if (id < 0 || id >= p.n_pages) return -1;
    return ((id * p.Hkv + h) << (p.lg_page - 4)) + (((int)key & ((1 << p.lg_page) - 1)) >> 4);
  };
  const int blocks0 = blocks_of(0);
  int row_lo, row_hi, n;
  request_rows(p, b, row_lo, row_hi, n);
  const int rows_b = (row_hi - row_lo) * p.G, len = request_len(p, b);
  unsigned char* ring = base + (size_t)warp * C::RING;
  const uint32_t ring_u = smem_u32(ring);
  uint32_t issued = 0, used = 0;  // tiles of this warp's ring, over all row tiles

  for (int r0 = group * RT; r0 < rows_b; r0 += row_groups * RT) {
    const int nr = min(RT, rows_b - r0);
    // own keys that the tile's last row sees
    const int own = max(0, min(len, len - n + (r0 + nr - 1) / p.G + 1));
    const int nt = np + (own + KT - 1) / KT;
    const int cnt = max(0, (nt - t0 + step - 1) / step);

    int blocks = blocks0;
    uint32_t absent = 0;  // stages whose tile has no page
    auto issue = [&](int i) {
      if (i && (i & 31) == 0) blocks = blocks_of(i);
      const int blk = __shfl_sync(0xffffffffu, blocks, i & 31);
      const int s = issued % NST;
      absent = (absent & ~(1u << s)) | ((blk < 0 ? 1u : 0u) << s);
      if (lane == 0) {
        if (blk < 0) {
          mbar_arrive(&full[warp][s]);
        } else {
          mbar_arrive_expect_tx(&full[warp][s], QB::BYTES);
          bulk_load(ring + s * QB::BYTES, pages + (size_t)blk * QB::BYTES, QB::BYTES, &full[warp][s]);
        }
      }
      __syncwarp();
      ++issued;
    };
    for (int i = 0; i < min(NST, cnt); ++i) issue(i);

    // ---- q fragments: this lane's column of a tile of 8 rows, its dims those of its share of K
    uint32_t qb[NT][C::KSTEPS][2];
    float qsum[NT][NG][2], cq[NT][2];  // of the columns 2 q4 and 2 q4 + 1
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const int r = j * 8 + r8;
      const __half* src = nullptr;
      if (r < nr) src = reinterpret_cast<const __half*>(p.q) + ((size_t)(row_lo + (r0 + r) / p.G) * p.Hq + h * p.G + (r0 + r) % p.G) * HD;
      float x[WORDS][PER], big = 0.f, sum[NG];
#pragma unroll
      for (int g = 0; g < NG; ++g) sum[g] = 0.f;
#pragma unroll
      for (int w = 0; w < WORDS; ++w) {
        constexpr int SH = GS / 4;
        const int d = w * PER / SH * GS + q4 * SH + w * PER % SH;
        uint32_t u[PER / 2];
#pragma unroll
        for (int k = 0; k < PER / 2; ++k) u[k] = 0u;
        if (src) {
          if constexpr (PER == 8) {
            const uint4 v = *reinterpret_cast<const uint4*>(src + d);
            u[0] = v.x; u[1] = v.y; u[2] = v.z; u[3] = v.w;
          } else {
            const uint2 v = *reinterpret_cast<const uint2*>(src + d);
            u[0] = v.x; u[1] = v.y;
          }
        }
#pragma unroll
        for (int k = 0; k < PER / 2; ++k) {
          const float2 f = __half22float2(u32_as_h2(u[k]));
          x[w][2 * k] = f.x;
          x[w][2 * k + 1] = f.y;
          big = fmaxf(big, fmaxf(fabsf(f.x), fabsf(f.y)));
          sum[w * PER / SH] += f.x + f.y;
        }
      }
#pragma unroll
      for (int d = 1; d <= 2; d <<= 1) {
        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, d));
#pragma unroll
        for (int g = 0; g < NG; ++g) sum[g] += __shfl_xor_sync(0xffffffffu, sum[g], d);
      }
      // 2^k: the row's largest value to [2^11, 2^12) (an infinity, or no value at all: 1)
      const int e = (int)(__float_as_uint(big) >> 23) - 127, k = big > 0.f && e < 128 ? 11 - e : 0;
      const float up = __uint_as_float((uint32_t)(127 + k) << 23), down = __uint_as_float((uint32_t)(127 + 24 - k) << 23);
#pragma unroll
      for (int w = 0; w < WORDS; ++w) {
        auto pair = [&](int a, int c, float f) { return h2_as_u32(__floats2half2_rn(x[w][a] * f, x[w][c] * f)); };
        if constexpr (PER == 8) {
          qb[j][2 * w][0] = pair(0, 4, up);
          qb[j][2 * w][1] = pair(2, 6, up);
          qb[j][2 * w + 1][0] = pair(1, 5, up * 0.0625f);
          qb[j][2 * w + 1][1] = pair(3, 7, up * 0.0625f);
        } else {
          qb[j][w][0] = pair(0, 2, up);
          qb[j][w][1] = pair(1, 3, up);
        }
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int from = (2 * q4 + c) * 4;
        const float back = __shfl_sync(0xffffffffu, down, from);  // 2^(24 - k)
        cq[j][c] = p.c * back;
#pragma unroll
        for (int g = 0; g < NG; ++g) qsum[j][g][c] = __shfl_sync(0xffffffffu, sum[g], from) / back;
      }
    }
    // own keys that the first row sees, and each of this thread's columns (rows past the last: as the last)
    const int see_first = max(0, min(len, len - n + r0 / p.G + 1));
    int see[NT][2];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int r = j * 8 + 2 * q4 + c;
        see[j][c] = r < nr ? max(0, len - n + (r0 + r) / p.G + 1) : own;
      }

    float o[C::MT][NT][4], bias[NT][NG][2], m[NT][2], l[NT][2];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
#pragma unroll
      for (int i = 0; i < C::MT; ++i) o[i][j][0] = o[i][j][1] = o[i][j][2] = o[i][j][3] = 0.f;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        m[j][c] = -INFINITY;
        l[j][c] = 0.f;
#pragma unroll
        for (int g = 0; g < NG; ++g) bias[j][g][c] = 0.f;
      }
    }
    const uint32_t k_lane = QB::KSH == 32 ? r8 * QB::ROW + ((r8 & 1) << 6) + q4 * 16 : r8 * QB::ROW + q4 * QB::KSH;
    const uint32_t v_lane = QB::V + q4 * 2 * QB::ROW + QB::piece_v(q4, r8, 0);
    const uint32_t meta_lane = r8 * 4 * NG;

    for (int i = 0; i < cnt; ++i, ++used) {
      const int s = used % NST;
      if (!mbar_wait_warp(&full[warp][s], (used / NST) & 1u, &s_abort, PA_WAIT_NS)) break;
      const int t = t0 + step * i;
      if ((absent >> s) & 1u) {  // nothing to see
        __syncwarp();
        if (i + NST < cnt) issue(i + NST);
        continue;
      }
      const uint32_t tile = ring_u + s * QB::BYTES;
      const int first = (t < np ? t : t - np) * KT;
      const bool part = (t < np ? P : see_first) - first < KT;  // not every row sees every key
      // ---- S = K Q^T
      float sc[NT][4];
#pragma unroll
      for (int j = 0; j < NT; ++j) sc[j][0] = sc[j][1] = sc[j][2] = sc[j][3] = 0.f;
      {
        uint32_t ka[WORDS], kb[WORDS], ma[NG], mb[NG];  // tokens r8 and r8 + 8
        lds_share<WORDS>(tile + k_lane, tile + (k_lane ^ 64), ka);
        lds_share<WORDS>(tile + k_lane + 8 * QB::ROW, tile + (k_lane ^ 64) + 8 * QB::ROW, kb);
        lds_words<NG>(tile + QB::KM + meta_lane, ma);
        lds_words<NG>(tile + QB::KM + meta_lane + 32 * NG, mb);
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          float y[NT][4];
#pragma unroll
          for (int j = 0; j < NT; ++j) y[j][0] = y[j][1] = y[j][2] = y[j][3] = 0.f;
#pragma unroll
          for (int w = g * WORDS / NG; w < (g + 1) * WORDS / NG; ++w) {
            const uint32_t a = ka[w], c = kb[w];
#pragma unroll
            for (int j = 0; j < NT; ++j) {
              if constexpr (PER == 8) {
                mma_16816(y[j], a & 0x000f000fu, c & 0x000f000fu, (a >> 8) & 0x000f000fu, (c >> 8) & 0x000f000fu, qb[j][2 * w][0], qb[j][2 * w][1]);
                mma_16816(y[j], a & 0x00f000f0u, c & 0x00f000f0u, (a >> 8) & 0x00f000f0u, (c >> 8) & 0x00f000f0u, qb[j][2 * w + 1][0],
                          qb[j][2 * w + 1][1]);
              } else {
                mma_16816(y[j], a & 0x00ff00ffu, c & 0x00ff00ffu, (a >> 8) & 0x00ff00ffu, (c >> 8) & 0x00ff00ffu, qb[j][w][0], qb[j][w][1]);
              }
            }
          }
          const float2 x0 = __half22float2(u32_as_h2(ma[g])), x1 = __half22float2(u32_as_h2(mb[g]));
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            sc[j][0] = fmaf(x0.x, y[j][0], fmaf(x0.y, qsum[j][g][0], sc[j][0]));
            sc[j][1] = fmaf(x0.x, y[j][1], fmaf(x0.y, qsum[j][g][1], sc[j][1]));
            sc[j][2] = fmaf(x1.x, y[j][2], fmaf(x1.y, qsum[j][g][0], sc[j][2]));
            sc[j][3] = fmaf(x1.x, y[j][3], fmaf(x1.y, qsum[j][g][1], sc[j][3]));
          }
        }
      }
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[j][e] *= cq[j][e & 1];
      uint32_t hidden = 0;  // bit 4 j + e
      if (part) {
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (r8 + (e >> 1) * 8 >= (t < np ? P : see[j][e & 1]) - first) {
              hidden |= 1u << (4 * j + e);
              sc[j][e] = -INFINITY;
            }
      }
      // ---- V's scales and biases; log2 of a bound of the largest scale
      float2 v0[NG], v1[NG];
      float lg[2], cap[2];
      {
        uint32_t ma[NG], mb[NG];
        lds_words<NG>(tile + QB::VM + meta_lane, ma);
        lds_words<NG>(tile + QB::VM + meta_lane + 32 * NG, mb);
        float big0 = 0x1p-24f, big1 = 0x1p-24f;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          v0[g] = __half22float2(u32_as_h2(ma[g]));
          v1[g] = __half22float2(u32_as_h2(mb[g]));
          big0 = fmaxf(big0, v0[g].x);
          big1 = fmaxf(big1, v1[g].x);
        }
        lg[0] = (float)((int)(__float_as_uint(big0) >> 23) - 126);
        lg[1] = (float)((int)(__float_as_uint(big1) >> 23) - 126);
        cap[0] = PA_LIFT + PA_RAISE - lg[0];
        cap[1] = PA_LIFT + PA_RAISE - lg[1];
      }
      // ---- running softmax: a column's m, the same in its eight lanes, is raised (and o rescaled) only when some p s may pass
      // 2^(PA_LIFT + PA_RAISE)
      float x[NT][2];
      bool up = false;
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          x[j][c] = fmaxf(sc[j][c] + lg[0], sc[j][2 + c] + lg[1]) - PA_LIFT;
          up |= x[j][c] > m[j][c] + PA_RAISE;
        }
      if (__any_sync(0xffffffffu, up)) {
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
#pragma unroll
            for (int d = 4; d <= 16; d <<= 1) x[j][c] = fmaxf(x[j][c], __shfl_xor_sync(0xffffffffu, x[j][c], d));
            const float mn = fmaxf(m[j][c], x[j][c]), f = m[j][c] == -INFINITY ? 0.f : ex2(m[j][c] - mn);
            m[j][c] = mn;
            l[j][c] *= f;
#pragma unroll
            for (int g = 0; g < NG; ++g) bias[j][g][c] *= f;
#pragma unroll
            for (int k = 0; k < C::MT; ++k) {
              o[k][j][c] *= f;
              o[k][j][2 + c] *= f;
            }
          }
      }
      // (the difference is rounded apart from c s, and the exponent kept to what m was chosen for: m far from zero is itself
      // rounded by more than a little)
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float mm = m[j][e & 1] == -INFINITY ? 0.f : m[j][e & 1];
          sc[j][e] = ex2(min_keep_nan(sc[j][e] - mm, cap[e >> 1]));
          l[j][e & 1] += sc[j][e];
        }
      // ---- O += V^T (P s)^T, and the biases' part
      uint32_t va[WORDS], vb[WORDS];  // pairs of tokens q4 and q4 + 4
      lds_share<WORDS>(tile + v_lane, tile + v_lane + 128, va);
      lds_share<WORDS>(tile + v_lane + 8 * QB::ROW, tile + v_lane + 8 * QB::ROW + 128, vb);
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        uint32_t pb[NT][2];
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          float ps[4], pz[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            ps[e] = sc[j][e] * (e < 2 ? v0[g].x : v1[g].x);
            pz[e] = sc[j][e] * (e < 2 ? v0[g].y : v1[g].y);
          }
          if (part) {  // what is hidden may be an infinity or NaN
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (hidden >> (4 * j + e) & 1u) ps[e] = pz[e] = 0.f;
          }
          bias[j][g][0] += pz[0] + pz[2];
          bias[j][g][1] += pz[1] + pz[3];
          pb[j][0] = transpose8x8(h2_as_u32(__floats2half2_rn(ps[0], ps[1])));
          pb[j][1] = transpose8x8(h2_as_u32(__floats2half2_rn(ps[2], ps[3])));
        }
#pragma unroll
        for (int w = g * WORDS / NG; w < (g + 1) * WORDS / NG; ++w) {
          const uint32_t a = va[w], c = vb[w];
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            if constexpr (PER == 8) {
              mma_16816(o[2 * w][j], a & 0x000f000fu, (a >> 8) & 0x000f000fu, c & 0x000f000fu, (c >> 8) & 0x000f000fu, pb[j][0], pb[j][1]);
              mma_16816(o[2 * w + 1][j], a & 0x00f000f0u, (a >> 8) & 0x00f000f0u, c & 0x00f000f0u, (c >> 8) & 0x00f000f0u, pb[j][0], pb[j][1]);
            } else {
              mma_16816(o[w][j], a & 0x00ff00ffu, (a >> 8) & 0x00ff00ffu, c & 0x00ff00ffu, (c >> 8) & 0x00ff00ffu, pb[j][0], pb[j][1]);
            }
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
    float* so = reinterpret_cast<float*>(ring);  // [RT][HD], this warp's ring
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int d = 4; d <= 16; d <<= 1) {
          l[j][c] += __shfl_xor_sync(0xffffffffu, l[j][c], d);
#pragma unroll
          for (int g = 0; g < NG; ++g) bias[j][g][c] += __shfl_xor_sync(0xffffffffu, bias[j][g][c], d);
        }
        const int r = j * 8 + 2 * q4 + c;
        if (r8 == 0) {
          s_m[warp][r] = m[j][c];
          s_l[warp][r] = l[j][c];
        }
#pragma unroll
        for (int k = 0; k < C::MT; ++k)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            // the place in this thread's eighth of the groups of tile k's rows r8 (e = 0) and r8 + 8
            const int at = PER == 8 ? (k >> 1) * 4 + 2 * e + (k & 1) : 2 * k + e, g = at / (GS / 8);
            so[r * HD + g * GS + r8 * (GS / 8) + at % (GS / 8)] =
                fmaf(o[k][j][2 * e + c], PER == 8 && (k & 1) ? 0x1p20f : 0x1p24f, bias[j][g][c]);
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
        const float4 v = *reinterpret_cast<const float4*>(base + (size_t)w * C::RING + ((size_t)r * HD + d) * 4);
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
        store_out<__half>(reinterpret_cast<__half*>(p.out) + row * HD + d, acc, L);
      } else {
        const size_t at = (size_t)(slot0 + split) * p.T * p.Hq + row;
        *reinterpret_cast<float4*>(p.part_o + at * HD + d) = acc;
        if (d == 0) p.part_ml[at] = make_float2(M, L);
      }
    }
    if (CLUSTER) {  // join the CTAs, each a part of the outputs
      __syncthreads();
      cluster_sync();
      join_cluster<__half, HD>(p, smem_u32(s_ml), smem_u32(base) + RT * HD * 4, split, splits, nr, row_lo, r0, h);
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

// ---------------------------------------------------------------- host side

int quant_attn_device_error(int reset) {
  int v = 0;
  cudaMemcpyFromSymbol(&v, g_prefix_attn_error, sizeof(int));
  if (reset) {
    const int z = 0;
    cudaMemcpyToSymbol(g_prefix_attn_error, &z, sizeof(int));
  }
  return v;
}

static AttnPlan plan_quant_attn(int T, int B, int Hkv, int G, long long own_keys, long long prefix_keys, int sms) {
  AttnPlan a{};
  const long long rows = (long long)T * G;
  const auto ceil_div = [](long long x, long long y) { return (x + y - 1) / y; };
  const long long groups = ceil_div(rows, (long long)B * 8), slots = 4ll * sms;
  a.kind = AttnPlan::FEW;
  const long long keys = own_keys + prefix_keys;
  const long long want = ceil_div(8ll * sms, (long long)B * Hkv);
  a.row_groups = (int)std::max(1ll, std::min(want, groups > 1 ? 2 * groups : 1));
  const long long most = ceil_div(keys, 64);
  const long long once = std::max(1ll, std::min({slots / ((long long)B * Hkv * a.row_groups), most, (long long)FR_CLUSTER}));
  const bool few_keys = (double)keys * std::max(ceil_div(slots, once), (long long)B * Hkv * a.row_groups) <= slots * 1536.0;
  a.splits = (int)(few_keys ? once : std::max(1ll, std::min({ceil_div(want, a.row_groups), most, 64ll})));
  a.cluster = few_keys && a.splits > 1;
  a.nslots = a.cluster ? 1 : a.splits;
  return a;
}

template <typename QB, int NT, bool CLUSTER>
static int run_few_rows_quant(const PrefixAttnParams& p, const uint8_t* pages, const AttnPlan& a, cudaStream_t stream) {
  constexpr auto kern = few_rows_quant_kernel<QB, NT, CLUSTER>;
  constexpr int smem = FewRowsQuant<QB, NT>::SMEM;
  const cudaError_t e = opt_in<kern>(smem);
  if (e != cudaSuccess) return check_launch("prefix_attn_q", e);
  launch_clusters(CLUSTER ? a.splits : 1, kern, dim3(a.splits * a.row_groups, p.Hkv, p.B), dim3(FR_WARPS * 32), smem, stream, p, pages,
                  a.kind == AttnPlan::FEW ? 1 : 0, a.splits, a.row_groups, a.kind == AttnPlan::SHARED ? a.tc_splits : 0);
  return check_launch("prefix_attn_q");
}

template <typename QB>
static int run_quant_attn(const PrefixAttnParams& p, const uint8_t* pages, const AttnPlan& a, cudaStream_t stream) {
  const bool two = (long long)p.T * p.G > 8ll * p.B;
  int st;
  if (two)
    st = a.cluster ? run_few_rows_quant<QB, 2, true>(p, pages, a, stream) : run_few_rows_quant<QB, 2, false>(p, pages, a, stream);
  else
    st = a.cluster ? run_few_rows_quant<QB, 1, true>(p, pages, a, stream) : run_few_rows_quant<QB, 1, false>(p, pages, a, stream);
  if (st != SC_OK || p.nslots == 1) return st;
  launch(join_slots_kernel<__half, QB::HD>, dim3((unsigned)(((size_t)p.T * p.Hq + 7) / 8)), dim3(256), 0, stream, p);
  return check_launch("prefix_attn_q_join");
}

}  // namespace sc

extern "C" {

size_t sc_prefix_attn_q_workspace_bytes(int T, int B, int Hq, int Hkv, int hd, int max_blocks, int max_prefix_blocks,
                                        int page_size) {
  if (T < 1 || B < 1 || Hq < 1 || Hkv < 1 || hd < 1 || max_blocks < 0 || max_prefix_blocks < 0 || page_size < 1) return 0;
  if (Hq % Hkv) return 0;
  const sc::AttnPlan a = sc::plan_quant_attn(T, B, Hkv, Hq / Hkv, (long long)max_blocks * page_size, (long long)max_prefix_blocks * page_size,
                                             sc::sm_count());
  return a.nslots <= 1 ? 0 : (size_t)a.nslots * T * Hq * (hd + 2) * sizeof(float);
}

int sc_prefix_attn_q(const void* q, const void* pages, int bits, int group, int T, const int32_t* q_start,
                     const int32_t* kv_lens, const int32_t* block_table, int B, int max_blocks,
                     const int32_t* prefix_table, const int32_t* prefix_len, int max_prefix_blocks, int Hq, int Hkv,
                     int hd, int n_pages, int page_size, float scale, void* out, void* workspace,
                     size_t workspace_bytes, cudaStream_t stream) {
  using namespace sc;
  SC_REQUIRE(q && pages && q_start && kv_lens && block_table && out, SC_ERR_ARG, "prefix_attn_q: null pointer");
  SC_REQUIRE(!prefix_len || (prefix_table && max_prefix_blocks >= 1), SC_ERR_ARG, "prefix_attn_q: a prefix needs its table");
  SC_REQUIRE(quant_kind_ok(hd, bits, group), SC_ERR_UNSUPPORTED,
             "prefix_attn_q: head_dim %d in %d bits by groups of %d unsupported (64 or 128; 4 or 8; 32 or 64)", hd, bits, group);
  SC_REQUIRE(page_size >= 16 && page_size <= 32768 && (page_size & (page_size - 1)) == 0, SC_ERR_UNSUPPORTED,
             "prefix_attn_q: page size %d unsupported (a power of two from 16)", page_size);
  SC_REQUIRE(T >= 1 && B >= 1 && B <= 65535 && max_blocks >= 1 && n_pages >= 1, SC_ERR_SHAPE, "prefix_attn_q: bad T/B/max_blocks");
  SC_REQUIRE(Hkv >= 1 && Hkv <= 65535 && Hq >= Hkv && Hq % Hkv == 0, SC_ERR_SHAPE, "prefix_attn_q: Hq=%d not a multiple of Hkv=%d", Hq, Hkv);
  SC_REQUIRE((long long)n_pages * Hkv * page_size < INT32_MAX && (long long)T * Hq <= (1 << 30) &&
                 (long long)max_blocks * page_size <= INT32_MAX && (long long)max_prefix_blocks * page_size <= INT32_MAX,
             SC_ERR_SHAPE, "prefix_attn_q: rows past 32 bits");
  const float c = scale * 1.4426950408889634f;  // log2(e); 2^28 of it with q's own scaling
  SC_REQUIRE(scale > 0.f && c < 0x1p96f, SC_ERR_ARG, "prefix_attn_q: scale must be positive and below 5e28");
  SC_REQUIRE((((uintptr_t)q | (uintptr_t)pages | (uintptr_t)out) & 15) == 0, SC_ERR_ARG,
             "prefix_attn_q: tensors must start on 16-byte boundaries");
  if (!prefix_len) max_prefix_blocks = 0;
  const AttnPlan a = plan_quant_attn(T, B, Hkv, Hq / Hkv, (long long)max_blocks * page_size, (long long)max_prefix_blocks * page_size, sm_count());
  const size_t need = sc_prefix_attn_q_workspace_bytes(T, B, Hq, Hkv, hd, max_blocks, max_prefix_blocks, page_size);
  SC_REQUIRE(workspace_bytes >= need && (need == 0 || workspace), SC_ERR_WORKSPACE,
             "prefix_attn_q: workspace of %zu bytes needed (got %zu)", need, workspace_bytes);
  SC_REQUIRE(((uintptr_t)workspace & 15) == 0, SC_ERR_ARG, "prefix_attn_q: the workspace must start on a 16-byte boundary");
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
  p.c = c;
  p.nslots = a.nslots;
  return with_quant_block(hd, bits, group, [&](auto block) {
    return run_quant_attn<decltype(block)>(p, static_cast<const uint8_t*>(pages), a, stream);
  });
}

}  // extern "C"
