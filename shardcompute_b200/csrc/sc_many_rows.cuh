// The many-rows attention kernel in fp16 (sc_prefix_attn.cu), on the tensor
// cores, and what it shares with the one in fp32.
#pragma once

#include <type_traits>

#include <cuda.h>

#include "sc_prefix_attn.cuh"
#include "sc_quant.cuh"
#include "sc_tc.cuh"

namespace sc {

// Where the keys come from: pools of values by TMA, or (QuantSource) blocks of codes.
struct PoolMaps {
  CUtensorMap k, v;
};
template <typename QB>
struct QuantSource {
  const uint8_t* pages;
};

// Copy of a box of pool rows, from 128-byte column `chunk` on, into shared memory, completing on `bar`.
__device__ __forceinline__ void tma3d_at(uint32_t dst, const CUtensorMap* map, int row, int chunk, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::
          "r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(row), "r"(chunk), "r"(smem_u32(bar))
      : "memory");
}

// Whether one of 16 bytes' values (fp16 or fp32) has all bits of its exponent set.
template <typename T>
__device__ __forceinline__ bool not_finite(const uint4& v) {
  constexpr uint32_t mask = sizeof(T) == 2 ? 0x7c007c00u : 0x7f800000u, one = sizeof(T) == 2 ? 0x04000400u : 0x00800000u,
                     top = sizeof(T) == 2 ? 0x80008000u : 0x80000000u;
  return ((((v.x & mask) + one) | ((v.y & mask) + one) | ((v.z & mask) + one) | ((v.w & mask) + one)) & top) != 0;
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
//   warps 12-15, over codes (sc_quant_attn.cu): the producer's copies are blocks
//              of codes, K and V of 64 tokens a stage; these warps write the values
//              s c + b, rounded to fp16 once (K for rows of few keys in two terms, a
//              tile of the ring each), into the ring that TMA fills otherwise.
//              Their loops are rolled: unrolled, the SM's instruction cache no longer
//              held what its warps run (the chunks below, 4 bits, 336 us; 300 so)
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
constexpr int TC_THREADS_QUANT = 16 * 32;
constexpr int TC_REGS_CTL_QUANT = 56, TC_REGS_SM_QUANT = 200;  // 256 x 56 + 256 x 200 = 512 x 128
// Over codes: rows that all see this many keys take k rounded once to fp16, as a cache in fp16 would hold it; the others as the sum of two
// fp16 terms (QuantValues::two_terms).  The rounding's errors, 2^-12 of each k, are independent of one another and even out over many keys;
// over few they do not: the output's error against float64, over that of the output's own rounding, rows that see 32, 128, 512, 1024, 2048
// keys, heads of 64, channels that stand out: 2.0, 1.9, 1.5, 1.35, 1.2 with one term, 1.35, 1.26, 1.12, 1.09, 1.05 with two (v and the weights
// are rounded in both).  The second term costs half as many products again: 12 prompts of up to 700 tokens alone, heads of 128, 4 bits, 105
// -> 126 us; the two kernels side by side 304 -> 310 us for 12 chunks behind 2050, 243 -> 269 for a prompt of 4000.
constexpr int TC_TWO_TERMS = 1024;
constexpr int TC_HAND = 3;  // quarter of a tile before which its softmax lets the other one start

template <int HD, typename Src = PoolMaps>
struct ManyRows {
  static constexpr bool QUANT = false;
  static constexpr int THREADS = TC_THREADS, REGS_CTL = TC_REGS_CTL, REGS_SM = TC_REGS_SM;
  static constexpr int TILE = TC_N * HD * 2;        // bytes of a Q, K or V tile
  static constexpr int NBUF = HD == 128 ? 5 : 8;    // K and V tiles in the ring
  static constexpr int NRAW = 1, RAW = 0;
  static constexpr int SMEM = 2 * TILE + NBUF * TILE + 1024;
};
template <int HD, typename QB>
struct ManyRows<HD, QuantSource<QB>> {
  static constexpr bool QUANT = true;
  static constexpr int THREADS = TC_THREADS_QUANT, REGS_CTL = TC_REGS_CTL_QUANT, REGS_SM = TC_REGS_SM_QUANT;
  static constexpr int TILE = TC_N * HD * 2;
  static constexpr int NBUF = HD == 128 ? (QB::BITS == 4 ? 4 : 3) : 8;
  static constexpr int RB = 4;  // blocks of 16 tokens to a stage of codes
  static constexpr int RAW = RB * QB::BYTES, NRAW = 3, STAGES = 8 / RB;  // stages of a tile
  static constexpr int SMEM = 2 * TILE + NBUF * TILE + NRAW * RAW + 1024;
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

// The producer over codes (a warp): blocks of 16 tokens, one copy each by a lane.
template <int HD, bool PACKED, typename Src>
__device__ __forceinline__ void quant_producer(const PrefixAttnParams& p, const Src& src, const RowShare& w, int b, int h, unsigned char* raw,
                                               uint64_t* raw_full, uint64_t* raw_empty, uint32_t* s_absent, volatile int* abort) {
  using C = ManyRows<HD, Src>;
  constexpr int RB = C::RB, BYTES = C::RAW / RB, NRAW = C::NRAW;
  const int lane = threadIdx.x & 31, blk8 = lane & 7;
  auto block_of = [&](int t) {  // this lane's block of tile t in the pool; -1: no such page
    const bool pre = PACKED || t < w.np;
    const long long key = (long long)(pre ? t : t - w.np) * TC_N + blk8 * 16;
    const int blk = (int)min(key >> p.lg_page, (long long)INT32_MAX);
    if (blk >= (pre ? p.max_prefix_blocks : p.max_blocks)) return -1;
    const int id = pre ? p.prefix_table[blk] : p.block_table[(size_t)b * p.max_blocks + blk];
    return id >= 0 && id < p.n_pages ? ((id * p.Hkv + h) << (p.lg_page - 4)) + (int)((key & ((1 << p.lg_page) - 1)) >> 4) : -1;
  };
  uint32_t it = 0;
  bool ok = true;
  int next = block_of(w.t0);
  for (int i = 0; i < w.cnt && ok; ++i) {
    const int t = w.t0 + w.step * i, keys = t < w.np ? w.P - t * TC_N : w.own - (t - w.np) * TC_N;
    const int block = blk8 * 16 < keys ? next : -1;
    if (i + 1 < w.cnt) next = block_of(t + w.step);
    const uint32_t gone = __ballot_sync(0xffffffffu, block < 0) & 0xffu;
    if (lane == 0) s_absent[i & 15] = gone;
#pragma unroll
    for (int st = 0; st < C::STAGES; ++st, ++it) {
      const int s = it % NRAW, there = RB - __popc((gone >> (RB * st)) & ((1u << RB) - 1u));
      ok = __all_sync(0xffffffffu, pa_wait(&raw_empty[s], ((it / NRAW) & 1u) ^ 1u, abort));
      if (!ok) break;
      if (lane == 0) {
        if (there)
          mbar_arrive_expect_tx(&raw_full[s], there * BYTES);
        else
          mbar_arrive(&raw_full[s]);
      }
      __syncwarp();
      if (lane < 8 && lane / RB == st && block >= 0)
        bulk_load(raw + s * C::RAW + lane % RB * BYTES, src.pages + (size_t)block * BYTES, BYTES, &raw_full[s]);
    }
  }
  // copies in flight land before the CTA may exit
  if (lane == 0) {
    int ignore = 0;
    for (uint32_t k = it > NRAW ? it - NRAW : 0; k < it; ++k) pa_wait(&raw_full[k % NRAW], (k / NRAW) & 1u, &ignore);
  }
}

__device__ __forceinline__ void sts_v4(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
__device__ __forceinline__ void sts_v2(uint32_t a, uint32_t x, uint32_t y) {
  asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(a), "r"(x), "r"(y) : "memory");
}

// The values of a stage's codes, RB blocks, by four warps: a thread takes RB/2 shares of K (a quarter of a token's) and as many
// of V (an eighth of a pair of tokens').
template <int HD, typename QB, int RB>
struct QuantValues {
  static constexpr int WORDS = QB::KSH / 4, GS = QB::GS, NG = QB::NG;
  static __device__ __forceinline__ void load(uint32_t at, uint32_t other, uint32_t (&w)[WORDS]) {
    if constexpr (WORDS == 2) {
      asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(at));
    } else {
#pragma unroll
      for (int i = 0; i < WORDS; i += 4) {
        const uint4 v = lds_v4(i ? other : at);
        w[i] = v.x; w[i + 1] = v.y; w[i + 2] = v.z; w[i + 3] = v.w;
      }
    }
  }
  // K at `raw` to the tile's rows from row0 on.
  static __device__ __forceinline__ void keys(uint32_t raw, uint32_t tile, int row0) {
    const int tid = threadIdx.x & 127;
#pragma unroll 1
    for (int u = 0; u < RB / 2; ++u) {
      const int token = u * 32 + (tid >> 2), t = tid & 3, tok = token & 15, row = row0 + token;
      const uint32_t block = raw + (token >> 4) * QB::BYTES, at = block + tok * QB::ROW + QB::piece_k(tok, t, 0);
      uint32_t w[WORDS], sb[NG];
      load(at, block + tok * QB::ROW + (QB::piece_k(tok, t, 0) ^ 64), w);
#pragma unroll
      for (int g = 0; g < NG; ++g) sb[g] = lds_u32(block + QB::KM + (tok * NG + g) * 4);
#pragma unroll
      for (int c = 0; c < HD / 32; ++c) {  // eight dims
        const int l = c * 8, g = l / (GS / 4), d = g * GS + t * (GS / 4) + l % (GS / 4);
        const __half2 s = __low2half2(u32_as_h2(sb[g])), b = __high2half2(u32_as_h2(sb[g]));
        uint32_t y[4];
        if constexpr (QB::BITS == 4) {
          __half2 x[4];
          unpack_u4(w[c], x);
#pragma unroll
          for (int k = 0; k < 4; ++k) x[k] = hfma2_rn(x[k], s, b);
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            y[k] = __byte_perm(h2_as_u32(x[2 * k]), h2_as_u32(x[2 * k + 1]), 0x5410);
            y[2 + k] = __byte_perm(h2_as_u32(x[2 * k]), h2_as_u32(x[2 * k + 1]), 0x7632);
          }
        } else {
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            __half2 x[2];
            unpack_u8(w[2 * c + k], x);
            x[0] = hfma2_rn(x[0], s, b);
            x[1] = hfma2_rn(x[1], s, b);
            y[2 * k] = __byte_perm(h2_as_u32(x[0]), h2_as_u32(x[1]), 0x5410);
            y[2 * k + 1] = __byte_perm(h2_as_u32(x[0]), h2_as_u32(x[1]), 0x7632);
          }
        }
        sts_v4(tile + (d >> 6) * (TC_N * 128) + sw128(row, (d >> 3) & 7), y[0], y[1], y[2], y[3]);
      }
    }
  }
  // (s, b) of a group taken apart for its codes' distances d = c - MID from their middle: x.x = (s1, b1), x.y = (s2, b2), with
  // s c + b = (s1 d + b1) + (s2 d + b2).  With b' = b + MID s, the middle's value:
  //   s1 the s of 11 - BITS significant bits, b1 the multiple of its last one next to b': s1 d + b1 has 11 bits, so fp16 holds it exactly
  //     (4 bits: s2 d + b2 too; 8 bits: to 2^-15 of MID s);
  //   where b' is too large beside s for that, s1 = 0: b' alone, and s d to fp16's 2^-12;
  //   next to fp16's limits s2 = 0, one term, as an fp16 cache would hold the value.
  static __device__ __forceinline__ uint2 two_terms(uint32_t sb) {
    constexpr float MID = QB::BITS == 4 ? 8.f : 128.f;
    constexpr uint32_t DROP = QB::BITS == 4 ? 17 : 21, UP = QB::BITS == 4 ? 4 : 8;
    const float2 x = __half22float2(u32_as_h2(sb));
    const float mid = fmaf(MID, x.x, x.y);
    const uint32_t u = __float_as_uint(x.x), e = u & 0xff800000u;
    const float grid = __uint_as_float(e + ((17u + UP - 4u) << 23) + 0x400000u);  // 1.5 2^23 of the last bits of s1
    const bool far = fabsf(mid) > __uint_as_float(e + (UP << 23)), end = fabsf(mid) + (MID + 1.f) * x.x >= 32768.f;
    const float s1 = end ? x.x : far ? 0.f : __uint_as_float((u + (1u << (DROP - 1))) & ~((1u << DROP) - 1u));
    const __half b1 = __float2half_rz(end || far ? mid : __fsub_rn(__fadd_rn(mid, grid), grid));  // (rz: a sum next to the limit stays below it)
    const float b2 = end ? 0.f : mid - __half2float(b1);
    return make_uint2(h2_as_u32(__halves2half2(__float2half_rn(s1), b1)), h2_as_u32(__floats2half2_rn(end ? 0.f : x.x - s1, b2)));
  }
  // Codes of a word less MID: four (two) half2 in the order of unpack_u4 (unpack_u8), exact.
  static __device__ __forceinline__ void distances(uint32_t w, __half2 (&x)[QB::BITS == 4 ? 4 : 2]) {
    if constexpr (QB::BITS == 4) {
      const __half2 low = u32_as_h2(0x64086408u), k16th = u32_as_h2(0x2c002c00u), high = u32_as_h2(0xd480d480u);  // 1032, 1/16, -72
      const uint32_t w8 = w >> 8;
      x[0] = __hsub2(u32_as_h2((w & 0x000f000fu) | 0x64006400u), low);
      x[1] = hfma2_rn(u32_as_h2((w & 0x00f000f0u) | 0x64006400u), k16th, high);
      x[2] = __hsub2(u32_as_h2((w8 & 0x000f000fu) | 0x64006400u), low);
      x[3] = hfma2_rn(u32_as_h2((w8 & 0x00f000f0u) | 0x64006400u), k16th, high);
    } else {
      const __half2 low = u32_as_h2(0x64806480u);  // 1152
      x[0] = __hsub2(u32_as_h2((w & 0x00ff00ffu) | 0x64006400u), low);
      x[1] = __hsub2(u32_as_h2(((w >> 8) & 0x00ff00ffu) | 0x64006400u), low);
    }
  }
  // K as two terms, each to its tile.  A warp's eight tokens of a step have 8 NG groups, of which each lane takes one apart.
  static __device__ __forceinline__ void keys_two(uint32_t raw, uint32_t tile, uint32_t tile2, int row0) {
    const int tid = threadIdx.x & 127, lane = threadIdx.x & 31;
#pragma unroll 1
    for (int u = 0; u < RB / 2; ++u) {
      const int token = u * 32 + (tid >> 2), t = tid & 3, tok = token & 15, row = row0 + token;
      const uint32_t block = raw + (token >> 4) * QB::BYTES, at = block + tok * QB::ROW + QB::piece_k(tok, t, 0);
      uint32_t w[WORDS];
      load(at, block + tok * QB::ROW + (QB::piece_k(tok, t, 0) ^ 64), w);
      const int mine = (token & ~7) + (lane & 7);  // eight tokens in a row: of one block
      const uint2 terms = two_terms(lds_u32(block + QB::KM + ((mine & 15) * NG + (lane >> 3) % NG) * 4));
      uint32_t sb1 = 0u, sb2 = 0u;
#pragma unroll
      for (int c = 0; c < HD / 32; ++c) {  // eight dims
        const int l = c * 8, g = l / (GS / 4), d = g * GS + t * (GS / 4) + l % (GS / 4);
        if (l % (GS / 4) == 0) {
          sb1 = __shfl_sync(0xffffffffu, terms.x, g * 8 + (lane >> 2));
          sb2 = __shfl_sync(0xffffffffu, terms.y, g * 8 + (lane >> 2));
        }
        __half2 x[4];  // dims i and i + 4 (8 bits: 0 and 2, 1 and 3, and four on)
        if constexpr (QB::BITS == 4) {
          distances(w[c], x);
        } else {
          __half2 lo[2], hi[2];
          distances(w[2 * c], lo);
          distances(w[2 * c + 1], hi);
          x[0] = lo[0]; x[1] = lo[1]; x[2] = hi[0]; x[3] = hi[1];
        }
        const uint32_t to = (d >> 6) * (TC_N * 128) + sw128(row, (d >> 3) & 7);
#pragma unroll
        for (int term = 0; term < 2; ++term) {
          const __half2 s = __low2half2(u32_as_h2(term ? sb2 : sb1)), b = __high2half2(u32_as_h2(term ? sb2 : sb1));
          uint32_t z[4], y[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) z[k] = h2_as_u32(hfma2_rn(x[k], s, b));
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            // 4 bits: dims 0 1 | 2 3 | 4 5 | 6 7 of pairs (0, 4) .. (3, 7); 8 bits: of (0, 2), (1, 3), (4, 6), (5, 7)
            y[QB::BITS == 4 ? k : 2 * k] = __byte_perm(z[2 * k], z[2 * k + 1], 0x5410);
            y[QB::BITS == 4 ? 2 + k : 2 * k + 1] = __byte_perm(z[2 * k], z[2 * k + 1], 0x7632);
          }
          sts_v4((term ? tile2 : tile) + to, y[0], y[1], y[2], y[3]);
        }
      }
    }
  }
  // V; blocks whose bit in `gone` is set are zero.
  static __device__ __forceinline__ void values(uint32_t raw, uint32_t tile, int row0, uint32_t gone) {
    const int tid = threadIdx.x & 127;
#pragma unroll 1
    for (int u = 0; u < RB / 2; ++u) {
      const int pair = u * 16 + (tid >> 3), t = tid & 7, pr = pair & 7, row = row0 + 2 * pair;
      const uint32_t block = raw + (pair >> 3) * QB::BYTES, at = block + QB::V + pr * 2 * QB::ROW + QB::piece_v(pr, t, 0);
      const uint32_t keep = (gone >> (pair >> 3)) & 1u ? 0u : 0xffffffffu;
      uint32_t w[WORDS];
      load(at, at + 128, w);
      constexpr int Q = GS / 8 / 4;  // quads of dims that a thread has of a group
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const uint32_t even = lds_u32(block + QB::VM + (2 * pr * NG + g) * 4), odd = lds_u32(block + QB::VM + ((2 * pr + 1) * NG + g) * 4);
        const __half2 s = u32_as_h2(__byte_perm(even, odd, 0x5410)), b = u32_as_h2(__byte_perm(even, odd, 0x7632));
        uint32_t e[2 * Q], o[2 * Q];
#pragma unroll
        for (int k = 0; k < Q; ++k) {
          __half2 x[4];  // dim i of both tokens
          if constexpr (QB::BITS == 4) {
            unpack_u4(w[g * Q + k], x);
          } else {
            __half2 lo[2], hi[2];
            unpack_u8(w[2 * (g * Q + k)], lo);
            unpack_u8(w[2 * (g * Q + k) + 1], hi);
            x[0] = lo[0]; x[1] = lo[1]; x[2] = hi[0]; x[3] = hi[1];
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) x[i] = hfma2_rn(x[i], s, b);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            e[2 * k + i] = __byte_perm(h2_as_u32(x[2 * i]), h2_as_u32(x[2 * i + 1]), 0x5410) & keep;
            o[2 * k + i] = __byte_perm(h2_as_u32(x[2 * i]), h2_as_u32(x[2 * i + 1]), 0x7632) & keep;
          }
        }
        const int d = g * GS + t * (GS / 8);
        const uint32_t to = tile + (d >> 6) * (TC_N * 128) + ((d & 7) << 1);
        if constexpr (Q == 2) {
          sts_v4(to + sw128(row, (d >> 3) & 7), e[0], e[1], e[2], e[3]);
          sts_v4(to + sw128(row + 1, (d >> 3) & 7), o[0], o[1], o[2], o[3]);
        } else {
          sts_v2(to + sw128(row, (d >> 3) & 7), e[0], e[1]);
          sts_v2(to + sw128(row + 1, (d >> 3) & 7), o[0], o[1]);
        }
      }
    }
  }
};

template <int HD, typename Src>
struct QuantBlockOf;
template <int HD, typename QB>
struct QuantBlockOf<HD, QuantSource<QB>> {
  using type = QB;
};

template <int HD, typename Src>
__device__ __forceinline__ void quant_writer(int cnt, uint32_t ring_u, uint32_t raw_u, uint64_t* full, uint64_t* empty, uint64_t* raw_full,
                                             uint64_t* raw_empty, const uint32_t* s_absent, volatile int* abort) {
  using C = ManyRows<HD, Src>;
  using V = QuantValues<HD, typename QuantBlockOf<HD, Src>::type, C::RB>;
  constexpr int NBUF = C::NBUF, NRAW = C::NRAW;
  const int lane = threadIdx.x & 31;
  auto wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, pa_wait(bar, parity, abort)); };
  uint32_t it = 0;
  for (int i = 0; i < cnt; ++i) {
    const uint32_t ki = 2 * i, vi = 2 * i + 1;
    const uint32_t kt = ring_u + (ki % NBUF) * C::TILE, vt = ring_u + (vi % NBUF) * C::TILE;
    if (!wait(&empty[ki % NBUF], ((ki / NBUF) & 1u) ^ 1u)) return;
#pragma unroll 1
    for (int st = 0; st < C::STAGES; ++st, ++it) {
      const int s = it % NRAW, row0 = st * C::RB * 16;
      if (!wait(&raw_full[s], (it / NRAW) & 1u)) return;
      V::keys(raw_u + s * C::RAW, kt, row0);
      if (st == C::STAGES - 1) {
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&full[ki % NBUF]);
      }
      if (st == 0 && !wait(&empty[vi % NBUF], ((vi / NBUF) & 1u) ^ 1u)) return;
      V::values(raw_u + s * C::RAW, vt, row0, s_absent[i & 15] >> (C::RB * st));
      fence_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&raw_empty[s]);
        if (st == C::STAGES - 1) mbar_arrive(&full[vi % NBUF]);
      }
    }
  }
}

// K as two terms, all of a tile's K ahead of its V, whose place may be free only when the products of the tile before are done: S waits for
// K, and three tiles may be the whole ring.
template <int HD, typename Src>
__device__ __forceinline__ void quant_writer_two(int cnt, uint32_t ring_u, uint32_t raw_u, uint64_t* full, uint64_t* empty, uint64_t* raw_full,
                                                 uint64_t* raw_empty, const uint32_t* s_absent, volatile int* abort) {
  using C = ManyRows<HD, Src>;
  using V = QuantValues<HD, typename QuantBlockOf<HD, Src>::type, C::RB>;
  constexpr int NBUF = C::NBUF, NRAW = C::NRAW;
  const int lane = threadIdx.x & 31;
  auto wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, pa_wait(bar, parity, abort)); };
  auto place = [&](uint32_t t) { return wait(&empty[t % NBUF], ((t / NBUF) & 1u) ^ 1u); };
  for (int i = 0; i < cnt; ++i) {
    const uint32_t ki = 3 * i, li = ki + 1, vi = ki + 2, it = C::STAGES * i;
    const uint32_t kt = ring_u + (ki % NBUF) * C::TILE, lt = ring_u + (li % NBUF) * C::TILE, vt = ring_u + (vi % NBUF) * C::TILE;
    if (!place(ki) || !place(li)) return;
#pragma unroll 1
    for (int st = 0; st < C::STAGES; ++st) {
      const int s = (it + st) % NRAW;
      if (!wait(&raw_full[s], ((it + st) / NRAW) & 1u)) return;
      V::keys_two(raw_u + s * C::RAW, kt, lt, st * C::RB * 16);
    }
    fence_async_smem();
    __syncwarp();
    if (lane == 0) {
      mbar_arrive(&full[ki % NBUF]);
      mbar_arrive(&full[li % NBUF]);
    }
    if (!place(vi)) return;
#pragma unroll 1
    for (int st = 0; st < C::STAGES; ++st) {
      const int s = (it + st) % NRAW;
      V::values(raw_u + s * C::RAW, vt, st * C::RB * 16, s_absent[i & 15] >> (C::RB * st));
      fence_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&raw_empty[s]);
        if (st == C::STAGES - 1) mbar_arrive(&full[vi % NBUF]);
      }
    }
  }
}

// PACKED: rows of all requests, keys of the prefix.  Otherwise: rows of one
// request, keys of the prefix and its own.  Over codes rows of which some sees
// fewer than TC_TWO_TERMS keys are those of the kernel with TWO, k in two terms, the others those of the one
// without, which it runs beside (p.beside: no wait for that one until the end).
template <int HD, bool PACKED, typename Src, bool TWO = false>
__global__ void __launch_bounds__(ManyRows<HD, Src>::THREADS, 1)
many_rows_kernel(const PrefixAttnParams p, const __grid_constant__ Src src, int splits, int slot0) {
  using C = ManyRows<HD, Src>;
  constexpr int NBUF = C::NBUF, NCH = HD / 64, TPK = TWO ? 3 : 2;  // NCH: 64-wide columns; TPK: ring tiles to a tile of keys, K (or its two terms) and V
  extern __shared__ __align__(1024) unsigned char mr_smem[];
  __shared__ __align__(8) uint64_t full[NBUF], empty[NBUF], q_full[2], s_full[2], p_full[2][2], o_full[2], v_clean[NBUF], drained[2], turn[2][4];
  __shared__ uint32_t s_tmem, s_absent[16];
  __shared__ int s_abort, s_req, s_row0, s_sum[C::THREADS / 32];
  __shared__ __align__(8) uint64_t raw_full[C::NRAW], raw_empty[C::NRAW];  // over codes
  __shared__ int s_any_bad, s_bad[3][PACKED ? 1 : HD];  // per column the first hidden key with inf, -inf, NaN
  unsigned char* base = mr_smem + ((1024 - (smem_u32(mr_smem) & 1023)) & 1023);
  const uint32_t q_u = smem_u32(base), ring_u = q_u + 2 * C::TILE;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int split = blockIdx.x % splits, item = blockIdx.x / splits, h = blockIdx.y;
  if (threadIdx.x == 0) {
    for (int i = 0; i < NBUF; ++i) {
      mbar_init(&full[i], C::QUANT ? 4 : 1);
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
    if constexpr (C::QUANT)
      for (int i = 0; i < C::NRAW; ++i) {
        mbar_init(&raw_full[i], 1);
        mbar_init(&raw_empty[i], 4);
      }
    s_abort = 0;
    s_req = -1;
    s_row0 = 0;
    s_any_bad = 0;
    fence_mbar_init();
  }
  if (!PACKED)
    for (int i = threadIdx.x; i < 3 * HD; i += C::THREADS) s_bad[i / HD][PACKED ? 0 : i % HD] = INT32_MAX;
  if (warp == 1) tmem_alloc_cols(&s_tmem, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const bool beside = TWO && p.beside;
  if (!beside) pdl_wait();
  pdl_trigger();  // after the wait: few_rows_kernel relies on it
  volatile int* abort = &s_abort;
  const uint32_t tmem = s_tmem;

  RowShare w = row_share<PACKED, 2 * TC_M, TC_N, C::THREADS>(p, item, split, splits, s_req, s_row0, s_sum);
  if (C::QUANT && PACKED && w.P < TC_TWO_TERMS) w.P = w.np = w.cnt = 0;  // few_rows_quant_kernel's
  const bool last_cta = blockIdx.x == gridDim.x - 1 && blockIdx.y == gridDim.y - 1;
  if (C::QUANT && !PACKED && (w.P < TC_TWO_TERMS && w.all < TC_TWO_TERMS - w.P) != TWO) {  // the other kernel's
    if (warp == 1) {
      tmem_dealloc_cols(tmem, 512);
      tmem_relinquish();
    }
    if (beside && last_cta) pdl_wait();
    return;
  }
  const int b = w.b, r0 = w.r0, row_lo = w.row_lo, rows = w.rows, n = w.n, len = w.len, P = w.P, np = w.np, own = w.own;
  const int cnt = w.cnt;
  const bool work = w.work;
  const int nx = work && r0 + TC_M < rows ? 2 : 1;  // row tiles in use
  auto tile_of = [&](int i) { return w.t0 + w.step * i; };
  // keys of tile t that exist
  auto keys_of = [&](int t) { return t < np ? P - t * TC_N : own - (t - np) * TC_N; };
  if (warp < 4 || (C::QUANT && warp >= 12))
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::REGS_CTL));
  else
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::REGS_SM));
  if (C::QUANT && warp == 0) {
    if constexpr (C::QUANT) quant_producer<HD, PACKED, Src>(p, src, w, b, h, base + (2 + NBUF) * C::TILE, raw_full, raw_empty, s_absent, abort);
  } else if (C::QUANT && warp >= 12) {
    if constexpr (C::QUANT)
      if constexpr (TWO)
        quant_writer_two<HD, Src>(w.cnt, ring_u, ring_u + NBUF * C::TILE, full, empty, raw_full, raw_empty, s_absent, abort);
      else
        quant_writer<HD, Src>(w.cnt, ring_u, ring_u + NBUF * C::TILE, full, empty, raw_full, raw_empty, s_absent, abort);
  } else if (warp == 0) {
   if constexpr (!C::QUANT) {
    // ================================ TMA producer ================================
    // copies: a page's rows (128 at most) of a 64-wide column, one per lane
    const int lg_box = min(p.lg_page, 7), sub = lane / NCH, ch = lane % NCH;
    auto pool_row = [&](int t) {  // this lane's first row of tile t in the pools; -1: no such page
      const bool pre = PACKED || t < np;
      const long long key = (long long)(pre ? t : t - np) * TC_N + (sub << lg_box);
      const int blk = (int)min(key >> p.lg_page, (long long)INT32_MAX);
      if (blk >= (pre ? p.max_prefix_blocks : p.max_blocks)) return -1;
      const int id = pre ? p.prefix_table[blk] : p.block_table[(size_t)b * p.max_blocks + blk];
      return id >= 0 && id < p.n_pages ? ((id * p.Hkv + h) << p.lg_page) + (int)(key & ((1 << p.lg_page) - 1)) : -1;
    };
    const int copies = (TC_N >> lg_box) * NCH;
    uint32_t it = 0;
    bool ok = true;
    int next = pool_row(tile_of(0));
    for (int i = 0; i < cnt && ok; ++i) {
      const int keys = keys_of(tile_of(i));
      const int row = sub << lg_box < keys ? next : -1;
      if (i + 1 < cnt) next = pool_row(tile_of(i + 1));
      uint32_t gone = 0;  // keys of this tile that have no page, a bit per 16
#pragma unroll
      for (int k = 0; k < TC_N / 16; ++k) gone |= (__shfl_sync(0xffffffffu, row, ((k * 16) >> lg_box) * NCH) < 0 ? 1u : 0u) << k;
      if (lane == 0) s_absent[i & 15] = gone;
#pragma unroll
      for (int kv = 0; kv < 2; ++kv, ++it) {
        const int s = it % NBUF;
        ok = __all_sync(0xffffffffu, pa_wait(&empty[s], ((it / NBUF) & 1u) ^ 1u, abort));
        if (!ok) break;
        if (lane == 0) mbar_arrive_expect_tx(&full[s], C::TILE);
        __syncwarp();
        if (lane < copies)
          tma3d_at(ring_u + s * C::TILE + ch * (TC_N * 128) + (sub << lg_box) * 128, kv ? &src.v : &src.k,
                   row < 0 ? p.pool_rows : row, ch, &full[s]);
      }
    }
    // copies in flight land before the CTA may exit
    if (lane == 0) {
      int ignore = 0;
      for (uint32_t k = it > NBUF ? it - NBUF : 0; k < it; ++k) pa_wait(&full[k % NBUF], (k / NBUF) & 1u, &ignore);
    }
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
      auto wait_full = [&](uint32_t it) {
        return pa_spin(&full[it % NBUF], (it / NBUF) & 1u, abort) && (!TWO || pa_spin(&full[(it + 1) % NBUF], ((it + 1) / NBUF) & 1u, abort));
      };
      auto issue_s = [&](uint32_t it) {  // S = Q K^T
        const uint64_t k = dk + at(it);
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk) {
          const uint32_t off = ((kk >> 2) * (TC_N * 128) + (kk & 3) * 32) >> 4;
          umma_f16(ts, dq + off, k + off, idesc_s, kk != 0);
        }
        if constexpr (TWO) {
          const uint64_t k2 = dk + at(it + 1);
#pragma unroll
          for (int kk = 0; kk < HD / 16; ++kk) {
            const uint32_t off = ((kk >> 2) * (TC_N * 128) + (kk & 3) * 32) >> 4;
            umma_f16(ts, dq + off, k2 + off, idesc_s, 1);
          }
          tc_commit(&empty[(it + 1) % NBUF]);
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
        const uint32_t vi = TPK * i + TPK - 1, ki = vi + 1;
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
    for (uint32_t it = 0; it < (uint32_t)TPK * cnt; ++it) {
      const int s = it % NBUF, t = tile_of((int)(it / TPK)), keys = min(TC_N, keys_of(t));
      if (!__all_sync(0xffffffffu, pa_wait(&full[s], (it / NBUF) & 1u, abort))) break;
      const uint32_t v = ring_u + s * C::TILE;
      // keys from here on are hidden from some row
      const int shown = PACKED || t < np ? keys : max(0, min(keys, w.all - (t - np) * TC_N));
      if (it % TPK == TPK - 1 && shown < TC_N) {
        for (int e = lane; e < (keys - shown) * 8 * NCH; e += 32) {
          const int r = shown + e / (8 * NCH), c = e % (8 * NCH);
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
        for (int e = lane; e < (TC_N - keys) * 8 * NCH; e += 32) {
          const int r = keys + e / (8 * NCH), c = e % (8 * NCH);
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
  if (beside && last_cta) pdl_wait();
}

}  // namespace sc
