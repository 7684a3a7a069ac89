// Attention of a ragged batch behind a shared prefix (sc_prefix_attn.cu) over
// pages in 8 or 4 bits: a token's k and v of a head are s c + b by groups of
// dims (sc_quant.cuh), and the codes c go into the products as they are:
//   q.k = sum_g s_g (q_g.c_g) + b_g (sum of q over g)
//   o_g = sum_j (p_j s_jg) c_jg + sum_j p_j b_jg
#include "sc_many_rows.cuh"

namespace sc {

// ---------------------------------------------------------------- few rows

// For few rows per request.  A CTA takes a request, a kv head, a tile of rows and
// a share of the keys; its four warps take steps of 32 tokens (two blocks, a bulk copy
// each) in turn, each with a ring of blocks and a running (m, l, o) of its own, so no
// barrier stands in the loop.  Short shares are joined in a cluster, as in
// few_rows_kernel (sc_prefix_attn.cu); long ones are pieces of a line on which all units
// follow one another (StreamArgs), so that every CTA has as much to do whatever the
// lengths are, and a kernel joins what lies in several pieces.
//
// mma.sync m16n8k16 with the tokens (S = K Q^T), then the dims (O = V^T P^T) as
// its 16 rows, the queries as its 8 columns: a decoded token of four heads
// fills half of them, where queries as rows would fill a quarter, and tcgen05's 128 rows
// of queries a thirtieth.  A register of an operand is a shift and an AND of a word of codes
// (fp16 subnormals), of V an AND alone, so a value costs 0.7 instructions; scales and biases are applied in
// fp32, to S per group and to the weights before their product.  S passes to the second
// product's operand through movmatrix; of V's nibbles the pair n0 + 16 n1 goes in beside
// n0, which saves the masks of n1.
//
// q is scaled per row by a power of two so that its largest value is in
// [2^11, 2^12): exact, but for what is below 2^-36 of that largest.  K's codes are moved up to the top of the subnormals (4 bits: code
// 2^-18, 8 bits: 2^-22), since the tensor cores cut their sums below what an operand's exponent allows, and a subnormal's is that
// of 2^-14: a product with q is then off as one of fp32 with the largest code would be.  As they lie (2^-24, 2^-20) q.c beside a dim of
// q 2000 times the rest was up to 16 steps of fp32 off (of 16 times that dim), now 0.4; the shifts take 2 us of the 44 below, and codes
// made whole (1024 + c, less 1024), which keep the exponents of small codes too, 6 us.
// q's fragments lie in shared memory: in registers they kept a fifth CTA from the SM.
// The weights p s are rounded to fp16, 2^11 to 2^15 high at the row's largest p s
// (PA_LIFT over c s + log2 of the token's largest scale): 2^-11 of each, the
// output's own rounding, down to 2^-25 of that largest.  Their error meets c - MID, not c,
// since what is added back of MID is MID times the rounded weights' sum: about zero, codes
// and bias are two large numbers of different signs (3.2e-4 of the output for one key, now
// 2.1e-4, 2.07e-4 of it the output's rounding).
//
// Two requests of 140000 tokens together, 8 kv heads of 128, 4 bits: 161 MB in 44 us with the
// join; twice the tokens take 29 us more (5.6 TB/s), so 15 us are starts (lengths, page ids,
// first blocks, one after another) and ends.  Four requests behind 700 tokens 7.5 us, latency.
template <typename QB, int NT, bool CLUSTER>
struct FewRowsQuant {
  static constexpr int RT = 8 * NT;            // rows of a tile
  static constexpr int WORDS = QB::KSH / 4;    // of codes in a thread's share of a token
  static constexpr int PER = 32 / QB::BITS;    // codes of a word
  static constexpr float MID = QB::BITS == 4 ? 8.f : 128.f;
  static constexpr int UNIT = QB::BITS == 4 ? 18 : 22;  // a code of K is taken as 2^-UNIT of itself
  static constexpr int KSTEPS = QB::HD / 16, MT = QB::HD / 16;
  // Blocks of 16 tokens to a step: two, which share the step's fixed costs; one of the largest blocks, so that four CTAs fit an SM
  // in place of three (16 heads of 128, 8 bits, groups of 32, 32 requests of up to 3500 tokens: 66 -> 52 us).  In groups of 64 so on the line
  // alone, whose requests are long (of up to 3500 tokens 48 -> 43 us, 64 of them 101 -> 88, five CTAs 91; 128 behind a prefix of 8197 with up to
  // 300 of their own 77 -> 68): in clusters, up to 1000 tokens, it took 22 us in place of 19.
  static constexpr int NBK = QB::BYTES > 4500 || (!CLUSTER && NT == 1 && QB::BYTES > 4300) ? 1 : 2, KEYS = 16 * NBK;
  static constexpr int STAGE = NBK * QB::BYTES;
  static constexpr int NST = NBK == 1 ? 2 : STAGE > 4000 ? 2 : STAGE > 2400 ? 3 : 4;
  static constexpr int OUT = 2 * RT * QB::HD * 4;  // a warp's result, and the CTA's behind it
  static constexpr int RING = NST * STAGE > OUT ? NST * STAGE : OUT;
  static constexpr int QBYTES = NT * KSTEPS * 256;  // q's fragments
  static constexpr int SMEM = FR_WARPS * RING + QBYTES;
  // CTAs of an SM, by shared memory and by registers, of which they leave too few in some instances: 4 bits, heads of 128, groups of 64, 92 bytes
  // are spilled on the line and 112 in clusters; groups of 32, 124 and, tiles of 16 rows in clusters, 220; 8 bits, groups of 64, 120 with
  // such tiles on the line.
  static constexpr int CTAS = NT == 1 ? (SMEM > 56000 ? 3 : SMEM > 44000 || QB::NG == 4 || QB::BYTES > 4300 ? 4 : 5) : QB::NG == 4 || SMEM > 75000 ? 2 : 3;
  static constexpr int CTAS_CLUSTER = NT == 1 ? (CTAS < 4 ? CTAS : QB::NG == 4 ? 3 : 4) : 2;
};

// Work of the CTAs where a grid of requests would leave them uneven: the (request, kv head, tile of rows) follow one another on
// a line, each as long as its tiles of keys and FQ_UNIT more, and each CTA takes a piece of `quantum`.  What a piece holds of
// a unit that reaches past it goes to one of the CTA's two places for partial results (first unit, last unit).
struct StreamArgs {
  long long* offsets;  // [B + 1]: where each request's units begin, and the quantum behind them: written by CTA 0, for the join
  float* o;            // [2 CTAs, RT, HD]
  float2* ml;          // [2 CTAs, RT]
  int ctas;
};
constexpr int FQ_UNIT = 128;   // keys that a unit's start and end are worth
constexpr int FQ_LEAST = 256;  // keys of a piece, at least

// A request's tiles of keys (all that some row of it sees, at most), its tiles of rows.
struct StreamRequest {
  int row_lo, rows, n, len, nt, tiles;
  long long units;
};
template <int RT, int KEYS>
__device__ __forceinline__ StreamRequest stream_request(const PrefixAttnParams& p, int b, int np) {
  StreamRequest r;
  int hi;
  request_rows(p, b, r.row_lo, hi, r.n);
  r.rows = (hi - r.row_lo) * p.G;
  r.len = request_len(p, b);
  r.nt = np + (int)(((long long)r.len + KEYS - 1) / KEYS);
  r.tiles = (r.rows + RT - 1) / RT;
  r.units = (long long)r.tiles * p.Hkv * (r.nt + FQ_UNIT / KEYS);
  return r;
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
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

// Keys of the prefix that the few-rows kernel takes.  PREFIX_SHORT: those of a prefix too short for the many-rows kernel, which then leaves
// it alone: for its precision (TC_TWO_TERMS), and since a table may hold far more than it does.
enum { PREFIX_NONE, PREFIX_ALL, PREFIX_SHORT };
__device__ __forceinline__ int few_rows_prefix(const PrefixAttnParams& p, int with_prefix) {
  const int P = with_prefix == PREFIX_NONE ? 0 : prefix_keys(p);
  return with_prefix == PREFIX_SHORT && P >= TC_TWO_TERMS ? 0 : P;
}

template <typename QB, int NT, bool CLUSTER>
__global__ void __launch_bounds__(FR_WARPS * 32, CLUSTER ? FewRowsQuant<QB, NT, CLUSTER>::CTAS_CLUSTER : FewRowsQuant<QB, NT, CLUSTER>::CTAS)
few_rows_quant_kernel(const PrefixAttnParams p, const uint8_t* pages, int with_prefix, int splits, int row_groups, int slot0,
                      const StreamArgs stream) {
  using C = FewRowsQuant<QB, NT, CLUSTER>;
  constexpr int RT = C::RT, NST = C::NST, KT = C::KEYS, NBK = C::NBK, HD = QB::HD, NG = QB::NG, GS = QB::GS, WORDS = C::WORDS, PER = C::PER, UNIT = C::UNIT;
  extern __shared__ __align__(128) unsigned char fq_smem[];
  __shared__ __align__(8) uint64_t full[FR_WARPS][NST];
  __shared__ float s_m[FR_WARPS][RT], s_l[FR_WARPS][RT];
  __shared__ float s_cq[RT], s_qsum[NG][RT];
  __shared__ float2 s_ml[CLUSTER ? RT : 1];
  __shared__ long long s_sum[FR_WARPS], s_at;
  __shared__ int s_abort, s_b;
  unsigned char* base = fq_smem + C::QBYTES;
  const uint32_t q_u = smem_u32(fq_smem);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int q4 = lane & 3, r8 = lane >> 2;
  if (threadIdx.x == 0) {
    for (int w = 0; w < FR_WARPS; ++w)
      for (int s = 0; s < NST; ++s) mbar_init(&full[w][s], 1);
    s_abort = s_b = 0;
    s_at = 0;
    fence_mbar_init();
  }
  __syncthreads();
  // Without the prefix this kernel runs beside the prefix's, as few_rows_kernel does (sc_prefix_attn.cu).
  if (with_prefix == PREFIX_ALL) pdl_wait();
  pdl_trigger();  // after the wait: the join relies on it
  const int P = few_rows_prefix(p, with_prefix), np = (int)(((long long)P + KT - 1) / KT);
  unsigned char* ring = base + (size_t)warp * C::RING;
  const uint32_t ring_u = smem_u32(ring);
  int s_in = 0, s_out = 0;            // the stage that the next tile goes to, that it comes from
  uint32_t phase = 0, in_flight = 0;  // of s_out's barrier; tiles asked for and not yet waited for

  // The pool's blocks of tiles t0 + step (first .. first + 32 / NBK - 1) of request b and head h, NBK lanes a tile; -1: no such page.
  auto blocks_of = [&](int b, int h, int t0, int step, int first) {
    const long long t = t0 + (long long)step * (first + lane / NBK);
    const bool pre = t < np;
    const long long key = (pre ? t : t - np) * KT + lane % NBK * 16;
    const int blk = (int)min(key >> p.lg_page, (long long)INT32_MAX);
    if (blk >= (pre ? p.max_prefix_blocks : p.max_blocks)) return -1;
    const int id = pre ? p.prefix_table[blk] : p.block_table[(size_t)b * p.max_blocks + blk];
    if (id < 0 || id >= p.n_pages) return -1;
    return ((id * p.Hkv + h) << (p.lg_page - 4)) + (int)((key & ((1 << p.lg_page) - 1)) >> 4);
  };

  // Rows r0 .. r0 + nr of request b under this warp's tiles t0 + step i, i < cnt; `own`: own keys that the last of the rows sees.
  // The warps' results go to their rings, (m, l) to s_m and s_l.  False after a wait that ran out.
  auto attend = [&](int b, int h, int row_lo, int n, int len, int r0, int nr, int own, int t0, int step, int cnt, int blocks) {
    constexpr uint32_t ALL = (1u << NBK) - 1;
    uint32_t absent = 0;  // blocks without a page, NBK bits per stage
    auto issue = [&](int i) {
      if (i && i % (32 / NBK) == 0) blocks = blocks_of(b, h, t0, step, i);
      const int blk = __shfl_sync(0xffffffffu, blocks, NBK * (i % (32 / NBK)) + lane % NBK);
      const uint32_t there = __ballot_sync(0xffffffffu, blk >= 0) & ALL;
      absent = (absent & ~(ALL << (NBK * s_in))) | ((there ^ ALL) << (NBK * s_in));
      if (lane == 0) {
        if (there)
          mbar_arrive_expect_tx(&full[warp][s_in], (there == 3u ? 2 : 1) * QB::BYTES);
        else
          mbar_arrive(&full[warp][s_in]);
      }
      __syncwarp();
      if (lane < NBK && blk >= 0)
        bulk_load(ring + s_in * C::STAGE + lane * QB::BYTES, pages + (size_t)blk * QB::BYTES, QB::BYTES, &full[warp][s_in]);
      s_in = s_in + 1 == NST ? 0 : s_in + 1;
      ++in_flight;
    };
    // ---- q's fragments, by all warps: eight dims of a row a lane, those of a word (8 bits: two) of a thread's share of K; asked for
    // ahead of the copies, which wait for the page ids
    constexpr int LPR = HD / 8, SH = GS / 4, QR = FR_WARPS * 256 / HD, PASSES = (RT + QR - 1) / QR;
    const int qc = threadIdx.x % LPR, t = qc & 3, w = qc >> 2;
    uint4 qv[PASSES];
#pragma unroll
    for (int k = 0; k < PASSES; ++k) {
      const int r = k * QR + (int)threadIdx.x / LPR, tok = (r0 + r) / p.G;
      qv[k] = make_uint4(0u, 0u, 0u, 0u);
      if (r < nr)
        qv[k] = *reinterpret_cast<const uint4*>(reinterpret_cast<const __half*>(p.q) + ((size_t)(row_lo + tok) * p.Hq + h * p.G + (r0 + r - tok * p.G)) * HD +
                                                w * 8 / SH * GS + t * SH + w * 8 % SH);
    }
    for (int i = 0; i < min(NST, cnt); ++i) issue(i);
#pragma unroll
    for (int k1 = 0; k1 < PASSES; ++k1) {
      const int r = k1 * QR + (int)threadIdx.x / LPR;
      const uint4 u = qv[k1];
      float x[8];
      const uint32_t uu[4] = {u.x, u.y, u.z, u.w};
      float big = 0.f, sum = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 f = __half22float2(u32_as_h2(uu[k]));
        x[2 * k] = f.x;
        x[2 * k + 1] = f.y;
        big = fmaxf(big, fmaxf(fabsf(f.x), fabsf(f.y)));
        sum += f.x + f.y;
      }
#pragma unroll
      for (int z = 1; z < LPR; z <<= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, z));
#pragma unroll
      for (int z = 1; z < SH / 2; z <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, z);  // four shares, SH / 8 words of each
      // 2^k: the row's largest value to [2^11, 2^12) (an infinity, or no value at all: 1)
      const int e = (int)(__float_as_uint(big) >> 23) - 127, k = big > 0.f && e < 128 ? 11 - e : 0;
      const float up = __uint_as_float((uint32_t)(127 + k) << 23), back = __uint_as_float((uint32_t)(127 + UNIT - k) << 23);
      auto pair = [&](int a, int b2) { return h2_as_u32(__floats2half2_rn(x[a] * up, x[b2] * up)); };
      // the fragment of two steps of k, 16 bytes a lane
      const uint32_t to = q_u + (((r >> 3) * (C::KSTEPS / 2) + w) * 32 + (r & 7) * 4 + t) * 16;
      if (r >= RT) continue;  // heads of 64 and eight rows: half of the threads
      if constexpr (PER == 8)
        asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(to), "r"(pair(0, 4)), "r"(pair(2, 6)), "r"(pair(1, 5)),
                     "r"(pair(3, 7)) : "memory");
      else
        asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(to), "r"(pair(0, 2)), "r"(pair(1, 3)), "r"(pair(4, 6)),
                     "r"(pair(5, 7)) : "memory");
      if (qc == 0) s_cq[r] = fmaxf(p.c * back, 0x1p-149f);  // not zero: -inf times it stays -inf
      if (w * 8 % SH == 0 && t == 0) s_qsum[w * 8 / SH][r] = sum / back;
    }
    __syncthreads();
    float qsum[NT][NG][2], cq[NT][2];  // of the columns 2 q4 and 2 q4 + 1
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        cq[j][c] = s_cq[j * 8 + 2 * q4 + c];
#pragma unroll
        for (int g = 0; g < NG; ++g) qsum[j][g][c] = s_qsum[g][j * 8 + 2 * q4 + c];
      }
    // own keys that the first row sees
    const int see_first = max(0, min(len, len - n + r0 / p.G + 1));

    float o[C::MT][NT][4], z[NG][NT][4], bias[NT][NG][2], m[NT][2], l[NT][2];
    bool far = false;  // m of some column
#pragma unroll
    for (int j = 0; j < NT; ++j) {
#pragma unroll
      for (int i = 0; i < C::MT; ++i) o[i][j][0] = o[i][j][1] = o[i][j][2] = o[i][j][3] = 0.f;
#pragma unroll
      for (int g = 0; g < NG; ++g) z[g][j][0] = z[g][j][1] = z[g][j][2] = z[g][j][3] = 0.f;
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

    for (int i = 0; i < cnt; ++i) {
      if (!mbar_wait_warp(&full[warp][s_out], phase, &s_abort, PA_WAIT_NS)) return false;
      const uint32_t tile = ring_u + s_out * C::STAGE;
      const uint32_t gone = (absent >> (NBK * s_out)) & ALL;
      --in_flight;
      if (++s_out == NST) {
        s_out = 0;
        phase ^= 1u;
      }
      const int t = t0 + step * i;
      const int first = (t < np ? t : t - np) * KT;
      const bool part = gone || (t < np ? P : see_first) - first < KT;  // not every row sees every key
      // ---- S = K Q^T: tokens r8, r8 + 8 of each block by columns 2 q4, 2 q4 + 1
      float sc[NT][4 * NBK];
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4 * NBK; ++e) sc[j][e] = 0.f;
      {
        uint32_t ka[NBK][WORDS], kb[NBK][WORDS];
#pragma unroll
        for (int k = 0; k < NBK; ++k) {
          const uint32_t block = tile + k * QB::BYTES;
          lds_share<WORDS>(block + k_lane, block + (k_lane ^ 64), ka[k]);
          lds_share<WORDS>(block + k_lane + 8 * QB::ROW, block + (k_lane ^ 64) + 8 * QB::ROW, kb[k]);
        }
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          float y[NT][4 * NBK];
#pragma unroll
          for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 4 * NBK; ++e) y[j][e] = 0.f;
#pragma unroll
          for (int w = g * C::KSTEPS / 2 / NG; w < (g + 1) * C::KSTEPS / 2 / NG; ++w)  // two steps of k
#pragma unroll
            for (int j = 0; j < NT; ++j) {
              const uint4 q = lds_v4(q_u + ((j * (C::KSTEPS / 2) + w) * 32 + lane) * 16);
#pragma unroll
              for (int k = 0; k < NBK; ++k) {
                float(&z)[4] = *reinterpret_cast<float(*)[4]>(&y[j][4 * k]);
                if constexpr (PER == 8) {
                  const uint32_t a = ka[k][w], c = kb[k][w], M = 0x03c003c0u;  // code 2^-18
                  mma_16816(z, (a << 6) & M, (c << 6) & M, (a >> 2) & M, (c >> 2) & M, q.x, q.y);
                  mma_16816(z, (a << 2) & M, (c << 2) & M, (a >> 6) & M, (c >> 6) & M, q.z, q.w);
                } else {
#pragma unroll
                  for (int i = 0; i < 2; ++i) {
                    const uint32_t a = ka[k][2 * w + i], c = kb[k][2 * w + i], M = 0x03fc03fcu;  // code 2^-22
                    mma_16816(z, (a << 2) & M, (c << 2) & M, (a >> 6) & M, (c >> 6) & M, i ? q.z : q.x, i ? q.w : q.y);
                  }
                }
              }
            }
#pragma unroll
          for (int k = 0; k < NBK; ++k) {
            const float2 x0 = __half22float2(u32_as_h2(lds_u32(tile + k * QB::BYTES + QB::KM + meta_lane + 4 * g)));
            const float2 x1 = __half22float2(u32_as_h2(lds_u32(tile + k * QB::BYTES + QB::KM + meta_lane + 32 * NG + 4 * g)));
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                sc[j][4 * k + c] = fmaf(x0.x, y[j][4 * k + c], fmaf(x0.y, qsum[j][g][c], sc[j][4 * k + c]));
                sc[j][4 * k + 2 + c] = fmaf(x1.x, y[j][4 * k + 2 + c], fmaf(x1.y, qsum[j][g][c], sc[j][4 * k + 2 + c]));
              }
          }
        }
      }
      uint32_t hidden = 0;  // bit 4 NBK j + e
      if (part) {
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int r = j * 8 + 2 * q4 + c;  // rows past the last see what the last does
            const int lim = (t < np ? P : r < nr ? max(0, min(len, len - n + (r0 + r) / p.G + 1)) : own) - first;
#pragma unroll
            for (int e = c; e < 4 * NBK; e += 2)
              if (r8 + (e >> 1) * 8 >= lim || (gone >> (e >> 2)) & 1u) {
                hidden |= 1u << (4 * NBK * j + e);
                sc[j][e] = -INFINITY;
              }
          }
      }
      // ---- V's scales and biases; log2 of a bound of each token's largest scale.  A group that stands for NaN, by its bias, has no part
      // in it: an infinite scale would press the weights of every key to nothing, for the other groups too.
      uint32_t mv[2 * NBK][NG];
      float lg[2 * NBK];
#pragma unroll
      for (int k = 0; k < 2 * NBK; ++k) {
        lds_words<NG>(tile + (k >> 1) * QB::BYTES + QB::VM + meta_lane + (k & 1) * 32 * NG, mv[k]);
        float big = 0x1p-24f;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          const float2 sb = __half22float2(u32_as_h2(mv[k][g]));
          big = fmaxf(big, fmaf(sb.y, 0.f, sb.x));  // NaN: the other one
        }
        lg[k] = (float)((int)(__float_as_uint(fminf(big, 65504.f)) >> 23) - 126);
      }
      // ---- running softmax: a column's m, the same in its eight lanes, is raised (and o rescaled) only when some p s may pass
      // 2^(PA_LIFT + PA_RAISE)
      float x[NT][2];
      bool up = false;
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          x[j][c] = fmaxf(fmaf(sc[j][c], cq[j][c], lg[0]), fmaf(sc[j][2 + c], cq[j][c], lg[1]));
          if constexpr (NBK == 2)
            x[j][c] = fmaxf(x[j][c], fmaxf(fmaf(sc[j][4 * NBK - 4 + c], cq[j][c], lg[2 * NBK - 2]), fmaf(sc[j][4 * NBK - 2 + c], cq[j][c], lg[2 * NBK - 1])));
          up |= x[j][c] > m[j][c] + (PA_LIFT + PA_RAISE);
        }
      if (__any_sync(0xffffffffu, up)) {
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
#pragma unroll
            for (int d = 4; d <= 16; d <<= 1) x[j][c] = fmaxf(x[j][c], __shfl_xor_sync(0xffffffffu, x[j][c], d));
            // (a column that did not pass keeps its m: what the others see has no influence on it, not even on its roundings)
            const float mn = x[j][c] > m[j][c] + (PA_LIFT + PA_RAISE) ? x[j][c] - PA_LIFT : m[j][c], f = m[j][c] == -INFINITY ? 0.f : ex2(m[j][c] - mn);
            m[j][c] = mn;
            l[j][c] *= f;
#pragma unroll
            for (int g = 0; g < NG; ++g) bias[j][g][c] *= f;
#pragma unroll
            for (int k = 0; k < C::MT; ++k) {
              o[k][j][c] *= f;
              o[k][j][2 + c] *= f;
            }
            z[0][j][c] *= f;
            if constexpr (NG > 1) z[NG - 1][j][c] *= f;
            if constexpr (NG > 2) {
              z[1][j][c] *= f;
              z[2][j][c] *= f;
            }
          }
        bool any = false;
#pragma unroll
        for (int j = 0; j < NT; ++j) any |= (fabsf(m[j][0]) >= PA_FAR && m[j][0] != -INFINITY) || (fabsf(m[j][1]) >= PA_FAR && m[j][1] != -INFINITY);
        far = __any_sync(0xffffffffu, any);
      }
      // p = 2^(c s - m).  Where m is far from zero it is itself rounded by more than a little: there the difference is rounded apart
      // from c s, and the exponent kept to what m was chosen for.
      auto weights = [&](auto is_far) {
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int e = 0; e < 4 * NBK; ++e) {
            const float mm = m[j][e & 1] == -INFINITY ? 0.f : m[j][e & 1];
            float d = fmaf(sc[j][e], cq[j][e & 1], -mm);
            if constexpr (is_far)
              if (fabsf(mm) >= PA_FAR) d = min_keep_nan(__fsub_rn(__fmul_rn(sc[j][e], cq[j][e & 1]), mm), PA_LIFT + PA_RAISE - lg[e >> 1]);
            sc[j][e] = ex2(d);
            l[j][e & 1] += sc[j][e];
          }
      };
      if (far)
        weights(std::true_type{});
      else
        weights(std::false_type{});
      // ---- O += V^T (P s)^T, and the biases' part
#pragma unroll
      for (int k = 0; k < NBK; ++k) {
        const uint32_t block = tile + k * QB::BYTES + v_lane;
        uint32_t va[WORDS], vb[WORDS];  // pairs of tokens q4 and q4 + 4
        lds_share<WORDS>(block, block + 128, va);
        lds_share<WORDS>(block + 8 * QB::ROW, block + 8 * QB::ROW + 128, vb);
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          float2 v0 = __half22float2(u32_as_h2(mv[2 * k][g])), v1 = __half22float2(u32_as_h2(mv[2 * k + 1][g]));
          v0.y = fmaf(v0.x, C::MID, v0.y);
          v1.y = fmaf(v1.x, C::MID, v1.y);
          uint32_t pb[NT][2];
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            float ps[4];
            if (part) {  // what is hidden may be an infinity or NaN
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const bool out = hidden >> (4 * (NBK * j + k) + e) & 1u;
                ps[e] = out ? 0.f : sc[j][4 * k + e] * (e < 2 ? v0.x : v1.x);
                bias[j][g][e & 1] += out ? 0.f : sc[j][4 * k + e] * (e < 2 ? v0.y : v1.y);
              }
            } else {
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                ps[e] = sc[j][4 * k + e] * (e < 2 ? v0.x : v1.x);
                bias[j][g][e & 1] = fmaf(sc[j][4 * k + e], e < 2 ? v0.y : v1.y, bias[j][g][e & 1]);
              }
            }
            pb[j][0] = transpose8x8(h2_as_u32(__floats2half2_rn(ps[0], ps[1])));
            pb[j][1] = transpose8x8(h2_as_u32(__floats2half2_rn(ps[2], ps[3])));
            // (1, not 2^-24 as in the codes: the tensor cores cut their sums off 24 bits below what the largest product's exponents
            // allow, and a subnormal counts as 2^-14 there: of 2^-24 ten bits are left, 2.8e-4 of the output; of the codes 16 and more)
            mma_16816(z[g][j], 0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u, pb[j][0], pb[j][1]);
          }
#pragma unroll
          for (int w = g * WORDS / NG; w < (g + 1) * WORDS / NG; ++w) {
            const uint32_t a = va[w], c = vb[w];
#pragma unroll
            for (int j = 0; j < NT; ++j) {
              if constexpr (PER == 8) {
                const uint32_t a0 = a & 0x00ff00ffu, a1 = __byte_perm(a, 0u, 0x4341), c0 = c & 0x00ff00ffu, c1 = __byte_perm(c, 0u, 0x4341);
                mma_16816(o[2 * w][j], a0 & 0x000f000fu, a1 & 0x000f000fu, c0 & 0x000f000fu, c1 & 0x000f000fu, pb[j][0], pb[j][1]);
                mma_16816(o[2 * w + 1][j], a0, a1, c0, c1, pb[j][0], pb[j][1]);  // n0 + 16 n1
              } else {
                mma_16816(o[w][j], a & 0x00ff00ffu, (a >> 8) & 0x00ff00ffu, c & 0x00ff00ffu, (c >> 8) & 0x00ff00ffu, pb[j][0], pb[j][1]);
              }
            }
          }
        }
      }
      __syncwarp();
      if (i + NST < cnt) issue(i + NST);
    }
    // ---- this warp's sums, [RT][HD], over its ring, whose tiles it is done with
    float* so = reinterpret_cast<float*>(ring);
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
        for (int k = 0; k < C::MT; k += 2) {  // four dims in a row: of two tiles of 16, this thread's two rows each
          const int at = 2 * k, g = at / (GS / 8);
          const float add = fmaf(z[g][j][c], -C::MID, bias[j][g][c]);
          float4 v;
          if constexpr (PER == 8)
            v = make_float4(fmaf(o[k][j][c], 0x1p24f, add), fmaf(o[k + 1][j][c] - o[k][j][c], 0x1p20f, add), fmaf(o[k][j][2 + c], 0x1p24f, add),
                            fmaf(o[k + 1][j][2 + c] - o[k][j][2 + c], 0x1p20f, add));
          else
            v = make_float4(fmaf(o[k][j][c], 0x1p24f, add), fmaf(o[k][j][2 + c], 0x1p24f, add), fmaf(o[k + 1][j][c], 0x1p24f, add),
                            fmaf(o[k + 1][j][2 + c], 0x1p24f, add));
          *reinterpret_cast<float4*>(so + r * HD + g * GS + r8 * (GS / 8) + at % (GS / 8)) = v;
        }
      }
    return true;
  };
  // The warps' results joined, four values a thread at a time: sink(row, dim, sum, reference, sum of weights).
  auto join_warps = [&](int nr, auto sink) {
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
      sink(r, d, acc, M, L);
    }
  };
  auto out_row = [&](int row_lo, int r, int h) { return (size_t)(row_lo + r / p.G) * p.Hq + h * p.G + r % p.G; };

  if constexpr (CLUSTER) {
    const int split = blockIdx.x % splits, group = blockIdx.x / splits, h = blockIdx.y, b = blockIdx.z;
    const int t0 = split * FR_WARPS + warp, step = splits * FR_WARPS;
    const int blocks0 = blocks_of(b, h, t0, step, 0);  // asked for before the lengths are there
    int row_lo, row_hi, n;
    request_rows(p, b, row_lo, row_hi, n);
    const int rows_b = (row_hi - row_lo) * p.G, len = request_len(p, b);
    for (int r0 = group * RT; r0 < rows_b; r0 += row_groups * RT) {
      const int nr = min(RT, rows_b - r0);
      const int own = max(0, min(len, len - n + (r0 + nr - 1) / p.G + 1));
      const int nt = np + (own + KT - 1) / KT;
      const bool ok = attend(b, h, row_lo, n, len, r0, nr, own, t0, step, max(0, (nt - t0 + step - 1) / step), blocks0);
      if (__syncthreads_or(!ok)) {  // (also: every ring is free)
        for (int r = r0; r < rows_b; r += row_groups * RT) {  // the others' barriers: two for this tile and for each that follows
          cluster_sync();
          cluster_sync();
        }
        break;
      }
      join_warps(nr, [&](int r, int d, const float4& acc, float M, float L) {
        *reinterpret_cast<float4*>(base + ((size_t)(RT + r) * HD + d) * 4) = acc;  // behind warp 0's result
        if (d == 0) s_ml[r] = make_float2(M, L);
      });
      __syncthreads();
      cluster_sync();
      join_cluster<__half, HD>(p, smem_u32(s_ml), smem_u32(base) + RT * HD * 4, split, splits, nr, row_lo, r0, h);
      __syncthreads();
      cluster_sync();  // before a result is written over, or its CTA exits
      // the rings hold the joined results: written by threads, next by copies
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncthreads();
    }
  } else {
    // ---- where the requests lie on the line: each thread a run of them, then a scan
    const int per = (p.B + FR_WARPS * 32 - 1) / (FR_WARPS * 32), b0 = min(p.B, (int)threadIdx.x * per), b1 = min(p.B, b0 + per);
    long long sum = 0;
    for (int b = b0; b < b1; ++b) sum += stream_request<RT, KT>(p, b, np).units;
    long long upto = sum;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const long long u = __shfl_up_sync(0xffffffffu, upto, d);
      if (lane >= d) upto += u;
    }
    if (lane == 31) s_sum[warp] = upto;
    __syncthreads();
    long long all = 0, at = upto - sum;
    for (int w = 0; w < FR_WARPS; ++w) {
      if (w < warp) at += s_sum[w];
      all += s_sum[w];
    }
    const long long quantum = max((all + gridDim.x - 1) / gridDim.x, (long long)(FQ_LEAST / KT));
    const long long lo = blockIdx.x * quantum, hi = min(all, lo + quantum);
    if (blockIdx.x == 0) {
      long long x = at;
      for (int b = b0; b < b1; ++b) {
        stream.offsets[b] = x;
        x += stream_request<RT, KT>(p, b, np).units;
      }
      if (threadIdx.x == 0) stream.offsets[p.B] = quantum;
    }
    if (lo >= at && lo < at + sum) {
      int b = b0;
      for (; b < b1; ++b) {
        const long long u = stream_request<RT, KT>(p, b, np).units;
        if (lo < at + u) break;
        at += u;
      }
      s_b = b;
      s_at = at;
    }
    __syncthreads();
    // ---- the CTA's piece of the line, unit by unit
    long long pos = lo, off = lo < hi ? s_at : 0;
    int b = lo < hi ? s_b : 0;
    StreamRequest q = stream_request<RT, KT>(p, b, np);
    int unit = 0;
    bool fresh = true;
    while (pos < hi) {
      if (pos >= off + q.units) {
        off += q.units;
        if (++b >= p.B) break;  // (offsets in q_start that cannot be, and their sums, lead nowhere)
        q = stream_request<RT, KT>(p, b, np);
        unit = 0;
        continue;
      }
      const int u = q.nt + FQ_UNIT / KT;
      if (fresh) {  // the first unit
        unit = (int)((pos - off) / u);
        fresh = false;
      }
      const int ta = (int)(pos - off - (long long)unit * u), tb = (int)min((long long)u, ta + (hi - pos));
      pos += tb - ta;
      const int at = unit;
      if (tb == u) ++unit;
      if (ta > 0 && ta >= q.nt) continue;  // nothing left of it
      if (at < 0 || at >= q.tiles * p.Hkv) break;
      const int h = at / q.tiles, r0 = (at - h * q.tiles) * RT, nr = min(RT, q.rows - r0);
      const int own = max(0, min(q.len, q.len - q.n + (r0 + nr - 1) / p.G + 1));
      const int end = min(tb, np + (own + KT - 1) / KT), t0 = ta + warp;
      const int cnt = max(0, (end - t0 + FR_WARPS - 1) / FR_WARPS);
      const bool ok = attend(b, h, q.row_lo, q.n, q.len, r0, nr, own, t0, FR_WARPS, cnt, blocks_of(b, h, t0, FR_WARPS, 0));
      if (__syncthreads_or(!ok)) break;
      const bool whole = ta == 0 && tb >= q.nt;
      const size_t place = (size_t)(2 * blockIdx.x + (ta == 0 ? 1 : 0)) * RT;
      join_warps(nr, [&](int r, int d, const float4& acc, float M, float L) {
        const size_t row = out_row(q.row_lo, r0 + r, h);
        if (!whole) {
          *reinterpret_cast<float4*>(stream.o + (place + r) * HD + d) = acc;
          if (d == 0) stream.ml[place + r] = make_float2(M, L);
        } else if (slot0 < 0) {
          store_out<__half>(reinterpret_cast<__half*>(p.out) + row * HD + d, acc, L);
        } else {
          const size_t to = (size_t)slot0 * p.T * p.Hq + row;
          *reinterpret_cast<float4*>(p.part_o + to * HD + d) = acc;
          if (d == 0) p.part_ml[to] = make_float2(M, L);
        }
      });
      // the rings hold the results: written by threads, next by copies
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncthreads();
    }
  }
  // copies in flight land before the CTA may exit (after a wait that ran out)
  if (lane == 0)
    for (; in_flight; --in_flight) {
      int ignore = 0;
      mbar_wait_bounded(&full[warp][s_out], phase, &ignore, PA_WAIT_NS);
      if (++s_out == NST) {
        s_out = 0;
        phase ^= 1u;
      }
    }
  if (threadIdx.x == 0 && s_abort) atomicExch(&g_prefix_attn_error, 1);
  if (with_prefix != PREFIX_ALL && blockIdx.x == gridDim.x - 1 && blockIdx.y == gridDim.y - 1 && blockIdx.z == gridDim.z - 1) pdl_wait();
}

// ---------------------------------------------------------------- join

// A row's partial results: the many-rows kernel's (slots 0 .. tc - 1, a value for every row), and of the CTAs that share the row's
// unit on the line.  WPR warps to a (row, head), which read every WPR-th of them (few rows have many), eight of them in flight,
// each with its (m, l); a block's rows are of one request.  Bound by latency: what does not hang on the results is asked for
// while the kernel before still runs.
template <int HD, int RT, int KT, int WPR>
__global__ void __launch_bounds__(256) join_stream_kernel(const PrefixAttnParams p, const StreamArgs stream, int with_prefix, int tc) {
  constexpr int V = HD / 32, ROWS = 8 / WPR, N = 8;
  __shared__ float s_o[WPR > 1 ? 8 : 1][HD];
  __shared__ float2 s_ml[WPR > 1 ? 8 : 1];
  const int b = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, part = warp % WPR, P = few_rows_prefix(p, with_prefix);
  const StreamRequest q = stream_request<RT, KT>(p, b, (int)(((long long)P + KT - 1) / KT));
  pdl_wait();
  pdl_trigger();
  const long long off = stream.offsets[b], quantum = stream.offsets[p.B];
  const size_t stride = (size_t)p.T * p.Hq;
  for (int i0 = blockIdx.y * ROWS; i0 < q.rows * p.Hkv; i0 += gridDim.y * ROWS) {
    const int i = i0 + warp / WPR;
    const bool live = i < q.rows * p.Hkv;
    const int h = live ? i / q.rows : 0, r = live ? i - h * q.rows : 0;
    const size_t row = (size_t)(q.row_lo + r / p.G) * p.Hq + h * p.G + r % p.G;
    const long long start = off + ((long long)h * q.tiles + r / RT) * (q.nt + FQ_UNIT / KT);
    const int c0 = (int)(start / quantum), last = q.nt ? (int)((start + q.nt - 1) / quantum) : c0, shares = last - c0 + 1;
    if (c0 < 0 || last < c0 || last >= stream.ctas) break;  // as there
    // a unit that one CTA had lies in slot tc, or was written already
    const int all = live ? tc + (shares > 1 ? shares : tc > 0 ? 1 : 0) : 0;
    float acc[V], L = 0.f, M = -INFINITY;
#pragma unroll
    for (int k = 0; k < V; ++k) acc[k] = 0.f;
    for (int s0 = part; s0 < all; s0 += N * WPR) {
      float2 ml[N];
      float v[N][V];
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const int s = s0 + k * WPR, c = s - tc;
        ml[k] = make_float2(-INFINITY, 0.f);
#pragma unroll
        for (int e = 0; e < V; ++e) v[k][e] = 0.f;
        if (s < all) {
          const bool line = c >= 0 && shares > 1;
          const size_t at = line ? (size_t)(2 * (c0 + c) + (c == 0 ? 1 : 0)) * RT + r % RT : s * stride + row;
          ml[k] = line ? stream.ml[at] : p.part_ml[at];
          const float* from = (line ? stream.o : p.part_o) + at * HD + lane * V;
          if constexpr (V == 4)
            *reinterpret_cast<float4*>(v[k]) = *reinterpret_cast<const float4*>(from);
          else
            *reinterpret_cast<float2*>(v[k]) = *reinterpret_cast<const float2*>(from);
        }
      }
      float top = M;
#pragma unroll
      for (int k = 0; k < N; ++k) top = fmaxf(top, ml[k].x);
      const float back = M == -INFINITY ? 0.f : ex2(M - top);
      M = top;
      L *= back;
#pragma unroll
      for (int e = 0; e < V; ++e) acc[e] *= back;
#pragma unroll
      for (int k = 0; k < N; ++k) {
        if (ml[k].x == -INFINITY && ml[k].y == 0.f) continue;  // no key: there may be no values either
        const float f = ex2(ml[k].x - M);
        L += f * ml[k].y;
#pragma unroll
        for (int e = 0; e < V; ++e) acc[e] += f * v[k][e];
      }
    }
    if constexpr (WPR > 1) {
#pragma unroll
      for (int e = 0; e < V; ++e) s_o[warp][lane * V + e] = acc[e];
      if (lane == 0) s_ml[warp] = make_float2(M, L);
      __syncthreads();
      if (part == 0) {
        for (int w = warp + 1; w < warp + WPR; ++w) M = fmaxf(M, s_ml[w].x);
        L = 0.f;
#pragma unroll
        for (int e = 0; e < V; ++e) acc[e] = 0.f;
        for (int w = warp; w < warp + WPR; ++w) {
          if (s_ml[w].x == -INFINITY && s_ml[w].y == 0.f) continue;
          const float f = ex2(s_ml[w].x - M);
          L += f * s_ml[w].y;
#pragma unroll
          for (int e = 0; e < V; ++e) acc[e] += f * s_o[w][lane * V + e];
        }
      }
      __syncthreads();
    }
    if (all == 0 || part != 0) continue;
    const float inv = L == 0.f ? 0.f : 1.f / L;
    __half* dst = reinterpret_cast<__half*>(p.out) + row * HD + lane * V;
#pragma unroll
    for (int k = 0; k < V; k += 2) *reinterpret_cast<__half2*>(dst + k) = __floats2half2_rn(acc[k] * inv, acc[k + 1] * inv);
  }
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

struct QuantPlan {
  AttnPlan::Kind kind;
  bool two;                // tiles of 16 rows in the few-rows kernel
  int splits, row_groups;  // its clusters; 0: its CTAs take pieces of the line
  int ctas;
  long long units;          // of the line, if every request has the mean number of rows
  int tc_splits, tc_items;  // many_rows_kernel
  int nslots;               // partial results that every row has
  size_t o_rows, ml_rows;   // rows of partial results in scratch: of values, with those of the line
  size_t bytes;
};

// How a call is cut, as plan_attn (sc_prefix_attn.cu) does, by what the tables hold.  `resident`: CTAs of the few-rows kernel that an
// SM takes, for tiles of 8 rows and of 16; `clusters`: of those that work in clusters.
static QuantPlan plan_quant_attn(int T, int B, int Hq, int Hkv, int hd, int bits, long long own_keys, long long prefix_keys, int sms,
                                 const int (&resident)[2], const int (&clusters)[2]) {
  QuantPlan a{};
  const int G = Hq / Hkv;
  const long long rows = (long long)T * G;
  const auto ceil_div = [](long long x, long long y) { return (x + y - 1) / y; };
  a.two = rows > 8ll * B;
  const long long groups = ceil_div(rows, (long long)B * (a.two ? 16 : 8)), slots = (long long)resident[a.two] * sms;
  a.units = (long long)B * Hkv * groups;
  // Few rows a request: the prefix is taken apart (SHARED) once the keys of it that a CTA slot of the few-rows kernel would stream
  // for its requests pass 1000 (us in a graph, 4 bits, few | shared: 8 kv heads of 128, 16 requests behind 2000 tokens 18 | 20, 8000 39 | 30,
  // 64 behind 700 19 | 19, 2000 38 | 23; 4 of 64, 16 behind 8000 18 | 20, 16000 30 | 26, 64 behind 2000 18 | 18).  64 rows and more:
  // the many-rows kernel over all keys, but for a few keys and tiles of rows, which clusters do with less of a start (cluster | chunks: one
  // request of 64 new tokens over 600 11 | 15, behind 6000 82 | 34; 3 of 32 over 600 16 | 17, behind 1000 23 | 20; 8 of 32 alone
  // 19 | 11), or where the prefix is most of what they see and a request has less than half a tile of rows (shared | chunks: 8 of 16 behind 6000
  // 52 | 93, of 32 78 | 80, of 64 138 | 97).
  const bool many = rows >= 64ll * B, shares = prefix_keys > 0 && B > 1;
  const double load = (double)(own_keys + prefix_keys) * std::max(slots / FR_CLUSTER, a.units) / slots;
  if (many ? a.units < 0.6 * slots && load <= 400 : !shares || (double)prefix_keys * a.units <= 1000.0 * slots)
    a.kind = AttnPlan::FEW;
  else if (!many || (shares && rows < 112ll * B && prefix_keys >= 4 * own_keys))
    a.kind = AttnPlan::SHARED;
  else
    a.kind = AttnPlan::CHUNKS;
  int line_sms = sms;
  if (a.kind == AttnPlan::CHUNKS) {
    // shares of the keys until there is a CTA for every SM, as in plan_attn; a request has a tile of rows of its own at least
    const long long tiles = ceil_div(prefix_keys + own_keys, TC_N), items = B * ceil_div(rows, (long long)B * 2 * TC_M);
    a.tc_items = (int)(ceil_div(rows, 2 * TC_M) + B);
    a.tc_splits = (int)std::max(1ll, std::min({(sms + items * Hkv / 2) / (items * Hkv), tiles, 32ll}));
    a.tc_splits = (int)ceil_div(tiles, ceil_div(tiles, a.tc_splits));
    if (tiles - ceil_div(tiles, a.tc_splits) < 3) a.tc_splits = 1;
    a.tc_splits = std::max(a.tc_splits, (int)std::min(32ll, ceil_div(tiles, 131072 / TC_N)));  // as in plan_attn
    a.nslots = a.tc_splits;
  } else if (a.kind == AttnPlan::SHARED) {
    // Shares of the prefix: the ones that end soonest with the own keys' kernel beside them, by a tile of 256 rows and 128 keys in 2.3 us
    // (heads of 64: 1.9) and 8 us for a CTA's start and end, own keys (half of what the tables hold) at 128 (230) a us and SM, and as much
    // again for those that are left when the last of the prefix's CTAs has ended (their SMs fill late).  64 requests behind 8197 tokens,
    // us with 4, 5, 6, 8, 10 shares: 57, 48, 45, 49, 52 (taken: 6); 256 behind 32768, 4, 6, 8, 10: 278, 256, 244, 243 (10).
    const long long tiles = ceil_div(prefix_keys, TC_N), items = ceil_div(rows, 2 * TC_M);
    const double tile = hd == 128 ? 2.3 : 1.9, few = (double)B * own_keys / 2 * Hkv * groups / (hd == 128 ? 128 : 230);
    double best = INFINITY;
    for (int s = 1; s <= 32 && s <= tiles; ++s) {
      if (ceil_div(tiles, ceil_div(tiles, s)) != s) continue;  // no more shares than their longest one needs
      const long long n = items * Hkv * s, waves = ceil_div(n, sms);
      const double one = tile * ceil_div(tiles, s) + 8, beside = (double)(waves * sms - n) * one;
      const double t = waves * one + 2 * std::max(0.0, few - beside) / sms;
      if (t < best) {
        best = t;
        a.tc_splits = s;
      }
    }
    a.tc_splits = std::max(a.tc_splits, (int)std::min(32ll, ceil_div(tiles, 131072 / TC_N)));
    a.tc_items = (int)items;
    a.nslots = a.tc_splits + 1;
    // as many CTAs as the SMs that the prefix's kernel leaves take at once
    const long long n = items * Hkv * a.tc_splits;
    if (n < sms) line_sms = std::max(sms / 4, sms - (int)n);
  } else {
    // Clusters of up to eight CTAs, which join their shares in place, while a share is short: up to 1800 keys (8 bits: 1600, heads of 64: 2200) of the longest
    // request there may be, or, with more requests than CTA slots, 4500 keys a slot (8 bits: 2700); past that pieces of the line and a join (us in a graph,
    // requests of any length up to the longest, cluster | line: 8 kv heads of 128, one of 5000 9 | 14, of 20000 22 | 17, 16 of 5000 22 | 23,
    // of 20000 71 | 54, 64 of 1200 22 | 25, of 5000 72 | 57, 128 of 5000 105 | 101; 4 of 64, 16 of 20000 23 | 24, of 60000 75 | 56).
    a.nslots = 1;
    const long long keys = own_keys + prefix_keys;
    // Sizes a power of two: 16 requests of up to 800 tokens, 8 kv heads of 128, 1 to 6 and 8 CTAs a cluster: 12.2, 9.9, 11.0, 9.8, 13.9,
    // 15.2, 16.2 us; as many as run at once, since a cluster of the next wave waits for one to end whole (8 kv heads of 128, 4 bits, 40 requests of up
    // to 100 tokens, 1 CTA a cluster | 2, a tenth too many: 7.3 | 13.4 us, to 300 10 | 14, 48 to 1000, a third too many, 18.6 | 20.3); up to a tenth more where
    // shares are long (40 of up to 2300: 27 | 25; 4 of 64, 8 bits, 80 of up to 2300: 23 | 19), and of tiles of 16 rows, some of whose CTAs have no rows, a
    // third (drafts of up to five tokens, 16 requests behind 1000, 4 kv heads of 64, three tiles of rows each, 1 to 4: 20.5, 14.1, 19.6, 19.6; 384 CTAs
    // in clusters of two on 296 places).
    // (CTAs for tiles of rows: those of requests with half as many rows again as the mean)
    a.row_groups = (int)(a.two ? ceil_div(3 * rows, 2ll * B * 16) : 1);
    const long long ctas = (long long)B * Hkv * a.row_groups, places = clusters[a.two] * sms;
    long long once = 1;
    while (once < FR_CLUSTER && 2 * once * ctas * 30 <= (a.two ? 40 : keys > 900 * once ? 33 : 30) * places && 2 * once <= ceil_div(keys, 64)) once *= 2;
    if (ctas >= places ? keys * ctas <= (bits == 4 ? 4500 : 2700) * places : keys <= (hd == 64 ? 2200 : bits == 4 ? 1800 : 1600) * once) a.splits = (int)once;
  }
  size_t rows_all = a.nslots > 1 ? (size_t)a.nslots * T * Hq : 0;
  a.o_rows = rows_all;
  if (a.kind != AttnPlan::CHUNKS && !a.splits) {
    a.ctas = resident[a.two] * line_sms;
    rows_all += 2 * (size_t)a.ctas * (a.two ? 16 : 8);
  }
  a.ml_rows = rows_all;
  a.bytes = rows_all * (hd + 2) * sizeof(float) + (a.ctas ? (size_t)(B + 1) * 8 : 0);
  return a;
}
static QuantPlan plan_quant_attn(int T, int B, int Hq, int Hkv, int hd, int bits, int group, int max_blocks, int max_prefix_blocks, int page_size) {
  QuantPlan a;
  with_quant_block(hd, bits, group, [&](auto block) {
    using QB = decltype(block);
    a = plan_quant_attn(T, B, Hq, Hkv, hd, bits, (long long)max_blocks * page_size, (long long)max_prefix_blocks * page_size, sm_count(),
                        {FewRowsQuant<QB, 1, false>::CTAS, FewRowsQuant<QB, 2, false>::CTAS}, {FewRowsQuant<QB, 1, true>::CTAS_CLUSTER, FewRowsQuant<QB, 2, true>::CTAS_CLUSTER});
    return 0;
  });
  return a;
}

template <typename QB, int NT, bool CLUSTER>
static int run_few_rows_quant(const PrefixAttnParams& p, const uint8_t* pages, const QuantPlan& a, const StreamArgs& line, cudaStream_t stream) {
  constexpr auto kern = few_rows_quant_kernel<QB, NT, CLUSTER>;
  constexpr int smem = FewRowsQuant<QB, NT, CLUSTER>::SMEM, KEYS = FewRowsQuant<QB, NT, CLUSTER>::KEYS;
  const cudaError_t e = opt_in<kern>(smem);
  if (e != cudaSuccess) return check_launch("prefix_attn_q", e);
  launch_clusters(CLUSTER ? a.splits : 1, kern, CLUSTER ? dim3(a.splits * a.row_groups, p.Hkv, p.B) : dim3(a.ctas), dim3(FR_WARPS * 32), smem,
                  stream, p, pages, a.kind == AttnPlan::FEW ? PREFIX_ALL : PREFIX_SHORT, a.splits, a.row_groups, a.kind == AttnPlan::SHARED ? a.tc_splits : -1, line);
  const int st = check_launch("prefix_attn_q");
  if (CLUSTER || st != SC_OK) return st;
  const long long rows = (long long)p.T * p.Hq;
  const bool wide = a.ctas >= 8 * a.units;  // each unit in eight pieces or more, if all are alike
  const long long y = std::min(std::max(16ll * sm_count() / p.B, 64ll), ((wide ? rows : rows / 8) * 2 + p.B - 1) / p.B);  // twice the mean: requests differ
  launch(wide ? join_stream_kernel<QB::HD, 8 * NT, KEYS, 8> : join_stream_kernel<QB::HD, 8 * NT, KEYS, 1>, dim3(p.B, (unsigned)std::max(1ll, y)), dim3(256), 0, stream, p, line,
         a.kind == AttnPlan::FEW ? PREFIX_ALL : PREFIX_SHORT, a.kind == AttnPlan::SHARED ? a.tc_splits : 0);
  return check_launch("prefix_attn_q_join");
}

template <typename QB, bool PACKED, bool TWO>
static int run_many_rows_quant(const PrefixAttnParams& p, const uint8_t* pages, const QuantPlan& a, cudaStream_t stream) {
  using C = ManyRows<QB::HD, QuantSource<QB>>;
  constexpr auto kern = many_rows_kernel<QB::HD, PACKED, QuantSource<QB>, TWO>;
  const cudaError_t e = opt_in<kern>(C::SMEM);
  if (e != cudaSuccess) return check_launch("prefix_attn_q", e);
  launch(kern, dim3((unsigned)(a.tc_splits * a.tc_items), p.Hkv), dim3(C::THREADS), C::SMEM, stream, p, QuantSource<QB>{pages}, a.tc_splits, 0);
  return check_launch("prefix_attn_q_many_rows");
}

template <typename QB>
static int run_quant_attn(const PrefixAttnParams& p, const uint8_t* pages, const QuantPlan& a, const StreamArgs& line, cudaStream_t stream) {
  if (a.kind == AttnPlan::CHUNKS) {
    const bool deep = ((long long)(p.max_prefix_blocks + p.max_blocks) << p.lg_page) >= TC_TWO_TERMS;
    int st = deep ? run_many_rows_quant<QB, false, false>(p, pages, a, stream) : SC_OK;
    PrefixAttnParams p2 = p;
    p2.beside = deep;
    if (st == SC_OK) st = run_many_rows_quant<QB, false, true>(p2, pages, a, stream);
    if (st != SC_OK || a.nslots == 1) return st;
    launch(join_slots_kernel<__half, QB::HD>, dim3((unsigned)(((size_t)p.T * p.Hq + 7) / 8)), dim3(256), 0, stream, p);
    return check_launch("prefix_attn_q_join");
  }
  if (a.kind == AttnPlan::SHARED) {
    const int st = run_many_rows_quant<QB, true, false>(p, pages, a, stream);
    if (st != SC_OK) return st;
  }
  if (a.splits)
    return a.two ? run_few_rows_quant<QB, 2, true>(p, pages, a, line, stream) : run_few_rows_quant<QB, 1, true>(p, pages, a, line, stream);
  return a.two ? run_few_rows_quant<QB, 2, false>(p, pages, a, line, stream) : run_few_rows_quant<QB, 1, false>(p, pages, a, line, stream);
}

}  // namespace sc

extern "C" {

size_t sc_prefix_attn_q_workspace_bytes(int T, int B, int Hq, int Hkv, int hd, int bits, int group, int max_blocks,
                                        int max_prefix_blocks, int page_size) {
  if (T < 1 || B < 1 || Hq < 1 || Hkv < 1 || max_blocks < 0 || max_prefix_blocks < 0 || page_size < 1) return 0;
  if (Hq % Hkv || !sc::quant_kind_ok(hd, bits, group)) return 0;
  return sc::plan_quant_attn(T, B, Hq, Hkv, hd, bits, group, max_blocks, max_prefix_blocks, page_size).bytes;
}

int sc_prefix_attn_q_plan(int T, int B, int Hq, int Hkv, int hd, int bits, int group, int max_blocks, int max_prefix_blocks, int page_size,
                          int32_t plan[4]) {
  using namespace sc;
  SC_REQUIRE(plan, SC_ERR_ARG, "prefix_attn_q_plan: null pointer");
  SC_REQUIRE(quant_kind_ok(hd, bits, group), SC_ERR_UNSUPPORTED,
             "prefix_attn_q_plan: head_dim %d in %d bits by groups of %d unsupported (64 or 128; 4 or 8; 32 or 64)", hd, bits, group);
  SC_REQUIRE(T >= 1 && B >= 1 && max_blocks >= 0 && max_prefix_blocks >= 0 && page_size >= 1 && Hkv >= 1 && Hq >= Hkv && Hq % Hkv == 0 &&
                 (long long)T * Hq <= (1 << 30),
             SC_ERR_SHAPE, "prefix_attn_q_plan: bad shape");
  const QuantPlan a = plan_quant_attn(T, B, Hq, Hkv, hd, bits, group, max_blocks, max_prefix_blocks, page_size);
  plan[0] = a.kind == AttnPlan::FEW ? 0 : a.kind == AttnPlan::SHARED ? 1 : 2;
  plan[1] = a.splits;
  plan[2] = a.ctas;
  plan[3] = a.tc_splits * a.tc_items * Hkv;
  return SC_OK;
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
  const QuantPlan a = plan_quant_attn(T, B, Hq, Hkv, hd, bits, group, max_blocks, max_prefix_blocks, page_size);
  const size_t need = a.bytes;
  SC_REQUIRE(workspace_bytes >= need && (need == 0 || workspace), SC_ERR_WORKSPACE,
             "prefix_attn_q: workspace of %zu bytes needed (got %zu)", need, workspace_bytes);
  SC_REQUIRE(((uintptr_t)workspace & 15) == 0, SC_ERR_ARG, "prefix_attn_q: the workspace must start on a 16-byte boundary");
  PrefixAttnParams p{};
  p.q = q;
  p.out = out;
  p.part_o = static_cast<float*>(workspace);
  // values of all rows, of the line; then (m, l) of both; then the line's offsets
  p.part_ml = reinterpret_cast<float2*>(p.part_o + a.ml_rows * hd);
  const StreamArgs line = {reinterpret_cast<long long*>(p.part_ml + a.ml_rows), p.part_o + a.o_rows * hd, p.part_ml + a.o_rows, a.ctas};
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
    return run_quant_attn<decltype(block)>(p, static_cast<const uint8_t*>(pages), a, line, stream);
  });
}

}  // extern "C"
