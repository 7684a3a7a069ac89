// Tokens into and out of a paged cache that is held in 8 or 4 bits.
//
// A group of GS values x of one token and head is held as codes c of BITS bits,
// a scale s and a bias b (fp16):
//   b = min x rounded down, s = the smallest fp16 value with MOST s >= max x - b,
//   c = rint((x - b) / s) in 0..MOST (0 where s is 0), and stands for s c + b
// so that b <= x <= b + MOST s, and x is at most s / 2 off.  Where b + MOST s would pass what fp16 holds, s is the
// fp16 value below: b + MOST s is then less than max x by no more than MOST 2^-10 s, and x still at most s / 2 off.  s and c are the ones that
// exact arithmetic gives: next to a border, fp32's roundings would decide.
#include <algorithm>

#include "sc_quant.cuh"

namespace sc {

struct AppendQuantParams {
  const void* qkv;
  const int32_t *rows_end, *slots, *positions;  // rows_end: one past the last row that is used
  const float *cos_tab, *sin_tab;
  __half* q_out;
  uint8_t* pages;
  int row0, items, Hq, Hkv, max_pos, n_pages;
  PageDiv page, per_row;  // items of a row
};

__device__ __forceinline__ void load4(const float* p, float (&v)[4]) {
  const float4 a = *reinterpret_cast<const float4*>(p);
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
}
__device__ __forceinline__ void load4(const __half* p, float (&v)[4]) {
  const uint2 a = *reinterpret_cast<const uint2*>(p);
  const float2 x = __half22float2(u32_as_h2(a.x)), y = __half22float2(u32_as_h2(a.y));
  v[0] = x.x; v[1] = x.y; v[2] = y.x; v[3] = y.y;
}

// NaN if either is.
__device__ __forceinline__ float min_nan(float a, float b) {
  float d;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// (scale, bias) of a group with these extremes.  Where either is not a finite value of fp16's range, the bias is NaN: the group stands for NaN, and no score of it is an infinity that would take the token out of the
// attention unseen.
template <int MOST>
__device__ __forceinline__ __half2 scale_bias(float lo, float hi) {
  const __half b = __float2half_rd(lo);
  const float fb = __half2float(b);
  // max x - b as a sum of two fp32 values t + e
  const float t = __fsub_rn(hi, fb), z = __fsub_rn(t, hi), e = __fsub_rn(__fsub_rn(hi, __fsub_rn(t, z)), __fadd_rn(fb, z));
  __half s = __float2half_ru(fmaxf(t, 0.f) * (1.f / MOST));
  // The estimate is within a few roundings of fp32, at most one fp16 value off.  MOST s needs no rounding, nor does its difference to t
  // where that is near.
  const unsigned short u = __half_as_ushort(s);
  if (__fsub_rn(__half2float(s) * MOST, t) < e)
    s = __ushort_as_half(u + 1);
  else if (u > 0 && u <= 0x7c00 && __fsub_rn(__half2float(__ushort_as_half(u - 1)) * MOST, t) >= e)
    s = __ushort_as_half(u - 1);
  const bool holds = fb >= -65504.f && hi <= 65504.f;
  // (fp32 may take a top next to 65504 for it: so does fp16)
  if (holds && fmaf(__half2float(s), (float)MOST, fb) > 65504.f) s = __ushort_as_half(__half_as_ushort(s) - 1);
  return __halves2half2(s, holds ? b : __ushort_as_half(0x7e00));
}

// rint((x - b) / s), `inv` about 1 / s.  The quotient in fp32 finds it or a neighbour; which, what is left over says exactly: x - b as
// a sum of two fp32 values t + e, and t - c s, which near the border of two codes needs no rounding, against half a step.
template <int MOST>
__device__ __forceinline__ uint32_t code_of(float x, float s, float b, float inv) {
  const float t = __fsub_rn(x, b), z = __fsub_rn(t, x), e = __fsub_rn(__fsub_rn(x, __fsub_rn(t, z)), __fadd_rn(b, z));
  const float c = rintf(__fmul_rn(t, inv)), r = __fmaf_rn(-c, s, t), h = 0.5f * s;
  const float over = __fsub_rn(r, h), under = __fadd_rn(r, h);  // beside -e: zero or more, zero or less
  const bool odd = (int)c & 1;
  const float up = over > -e || (over == -e && odd) ? 1.f : 0.f, down = under < -e || (under == -e && odd) ? 1.f : 0.f;
  return s > 0.f ? (uint32_t)fminf(fmaxf(c + up - down, 0.f), (float)MOST) : 0u;  // NaN: 0
}

// Four codes as the bytes that hold them.
template <int BITS>
__device__ __forceinline__ uint32_t pack4(const uint32_t (&c)[4]) {
  return c[0] | c[1] << BITS | c[2] << (2 * BITS) | c[3] << (3 * BITS);
}

// An item is eight values of a head of a row: four pairs (d, d + HD/2).  q and k
// are rotated, the products not fused (the bits of the append that does not
// quantise), and q is rounded once.  The HD/8 items of a k or v head lie in
// neighbouring lanes, which find their groups' extremes by shuffles and write
// the codes.  Moves its bytes once; bound by the loads' latency, three in a row (8150
// rows of 40 heads of 64, fp32, in 8 bits: 122 MB in 25.3 us, 4.8 TB/s, from fp16 23.1; 32 rows of 48 heads of 128: 2.6 us).  The 32 registers
// that eight CTAs an SM leave spill 16 to 24 bytes: with 40 it took 26.4 us for 24.6 then, with two items a thread 28.1, with four 35.5.
template <typename ST, typename QB>
__global__ void __launch_bounds__(256, 8) append_quant_kernel(const AppendQuantParams p) {
  constexpr int HD = QB::HD, HALF = HD / 2, LPH = HD / 8, NG = QB::NG, GS = QB::GS;
  pdl_trigger();
  pdl_wait();
  const int end = *p.rows_end;  // on its way together with the row
  const int it = blockIdx.x * 256 + threadIdx.x;
  bool live = it < p.items;
  const int r = live ? p.per_row.div(it) : 0, e = it - r * p.per_row.d, row = p.row0 + r, h = e / LPH, d = e % LPH * 4;
  const bool is_kv = h >= p.Hq, is_v = h >= p.Hq + p.Hkv;
  int pos = -1, slot = -1;
  float a[4] = {0.f, 0.f, 0.f, 0.f}, b[4] = {0.f, 0.f, 0.f, 0.f};
  if (live) {
    pos = p.positions[row];
    slot = p.slots[row];
    const ST* src = reinterpret_cast<const ST*>(p.qkv) + ((size_t)row * (p.Hq + 2 * p.Hkv) + h) * HD + d;
    load4(src, a);
    load4(src + HALF, b);
  }
  live = live && row < end;
  const bool there = pos >= 0 && pos < p.max_pos;
  if (live && !is_v && there) {
    float c[4], s[4];
    load4(p.cos_tab + (size_t)pos * HALF + d, c);
    load4(p.sin_tab + (size_t)pos * HALF + d, s);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float x = __fadd_rn(__fmul_rn(a[k], c[k]), __fmul_rn(-b[k], s[k]));
      b[k] = __fadd_rn(__fmul_rn(b[k], c[k]), __fmul_rn(a[k], s[k]));
      a[k] = x;
    }
  }
  if (live && !is_kv) {
    __half* dst = p.q_out + ((size_t)row * p.Hq + h) * HD + d;
    *reinterpret_cast<uint2*>(dst) = make_uint2(h2_as_u32(__floats2half2_rn(a[0], a[1])), h2_as_u32(__floats2half2_rn(a[2], a[3])));
    *reinterpret_cast<uint2*>(dst + HALF) = make_uint2(h2_as_u32(__floats2half2_rn(b[0], b[1])), h2_as_u32(__floats2half2_rn(b[2], b[3])));
  }
  if (!__any_sync(0xffffffffu, live && is_kv)) return;
  // ---- the groups of a's and of b's dims (one and the same where a head is a single group)
  float lo[2] = {min_nan(min_nan(a[0], a[1]), min_nan(a[2], a[3])), min_nan(min_nan(b[0], b[1]), min_nan(b[2], b[3]))};
  float hi[2] = {max_nan(max_nan(a[0], a[1]), max_nan(a[2], a[3])), max_nan(max_nan(b[0], b[1]), max_nan(b[2], b[3]))};
  if (NG == 1) {
    lo[0] = lo[1] = min_nan(lo[0], lo[1]);
    hi[0] = hi[1] = max_nan(hi[0], hi[1]);
  }
  constexpr int WIDTH = NG == 1 ? LPH : GS / 4;  // lanes that share a group
#pragma unroll
  for (int z = 1; z < WIDTH; z <<= 1)
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      lo[k] = min_nan(lo[k], __shfl_xor_sync(0xffffffffu, lo[k], z));
      hi[k] = max_nan(hi[k], __shfl_xor_sync(0xffffffffu, hi[k], z));
    }
  const int id = slot >= 0 ? p.page.div(slot) : p.n_pages;
  if (!live || !is_kv || !there || id >= p.n_pages) return;
  const int off = slot - id * p.page.d, tok = off & 15, head = h - p.Hq - (is_v ? p.Hkv : 0);
  uint8_t* block = p.pages + (((size_t)id * p.Hkv + head) * (p.page.d >> 4) + (off >> 4)) * QB::BYTES;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const __half2 sb = scale_bias<QB::MOST>(lo[k], hi[k]);
    const float scale = __low2float(sb), bias = __high2float(sb), inv = __frcp_rn(scale);
    const int dim = d + k * HALF;
    uint32_t code[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) code[j] = code_of<QB::MOST>(k ? b[j] : a[j], scale, bias, inv);
    const uint32_t w = pack4<QB::BITS>(code);
    if (is_v) {
      uint8_t* dst = block + QB::v_at(tok, dim);
      *reinterpret_cast<uint16_t*>(dst) = (uint16_t)w;
      if (QB::BITS == 8) *reinterpret_cast<uint16_t*>(dst + 4) = (uint16_t)(w >> 16);
    } else if (QB::BITS == 8) {
      *reinterpret_cast<uint32_t*>(block + QB::k_at(tok, dim)) = w;
    } else {
      *reinterpret_cast<uint16_t*>(block + QB::k_at(tok, dim)) = (uint16_t)w;
    }
    if (dim % GS == 0) *reinterpret_cast<__half2*>(block + (is_v ? QB::VM : QB::KM) + (tok * NG + dim / GS) * 4) = sb;
  }
}

struct ReadQuantParams {
  const uint8_t* pages;
  const int32_t *slots, *rows_end;  // rows_end: NULL: every row
  void *k_out, *v_out;
  int row0, items, Hkv, n_pages;
  PageDiv page, per_row;  // items of a row
};

// A code as fp32: 2^23 + c is its bit pattern.
__device__ __forceinline__ float code_f32(uint32_t c) { return __uint_as_float(0x4b000000u | c) - 8388608.f; }

// An item is sixteen values of a head of a row's K or V, four times four 32
// apart, so that the items of a head store whole sectors together: s c + b in fp32
// (one rounding, where a bias is far from its scale), then in the output's type.  With one group of four an item, finding its place was most of
// the instructions (40000 rows of 8 heads of 128 in 8 bits to fp32 114 us).
template <typename OT, typename QB>
__global__ void __launch_bounds__(256) read_quant_kernel(const ReadQuantParams p) {
  constexpr int HD = QB::HD, LPH = 8, Q = HD / 32, NG = QB::NG;
  pdl_trigger();
  pdl_wait();
  const int it = blockIdx.x * 256 + threadIdx.x;
  if (it >= p.items) return;
  const int r = p.per_row.div(it), e = it - r * p.per_row.d, row = p.row0 + r;
  const int slot = p.slots[row], end = p.rows_end ? *p.rows_end : INT32_MAX;
  if (row >= end) return;
  const int hh = e / LPH, side = hh >= p.Hkv, h = hh - (side ? p.Hkv : 0), d0 = e % LPH * 4;
  const int id = slot >= 0 ? p.page.div(slot) : p.n_pages;
  uint32_t w[Q], sb[NG];
#pragma unroll
  for (int k = 0; k < Q; ++k) w[k] = 0u;
#pragma unroll
  for (int g = 0; g < NG; ++g) sb[g] = 0u;
  if (id < p.n_pages) {
    const int off = slot - id * p.page.d, tok = off & 15;
    const uint8_t* block = p.pages + (((size_t)id * p.Hkv + h) * (p.page.d >> 4) + (off >> 4)) * QB::BYTES;
#pragma unroll
    for (int g = 0; g < NG; ++g) sb[g] = *reinterpret_cast<const uint32_t*>(block + (side ? QB::VM : QB::KM) + (tok * NG + g) * 4);
#pragma unroll
    for (int k = 0; k < Q; ++k) {
      const int d = d0 + 32 * k;
      if (side) {
        const uint8_t* src = block + QB::v_at(tok, d);
        w[k] = *reinterpret_cast<const uint16_t*>(src);
        if (QB::BITS == 8) w[k] |= (uint32_t)*reinterpret_cast<const uint16_t*>(src + 4) << 16;
      } else if (QB::BITS == 8) {
        w[k] = *reinterpret_cast<const uint32_t*>(block + QB::k_at(tok, d));
      } else {
        w[k] = *reinterpret_cast<const uint16_t*>(block + QB::k_at(tok, d));
      }
    }
  }
  OT* dst = reinterpret_cast<OT*>(side ? p.v_out : p.k_out) + ((size_t)row * p.Hkv + h) * HD + d0;
#pragma unroll
  for (int k = 0; k < Q; ++k) {
    const float2 f = __half22float2(u32_as_h2(sb[k * 32 / QB::GS]));
    float v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      v[j] = fmaf(code_f32(QB::BITS == 8 ? __byte_perm(w[k], 0u, 0x4440 + j) : (w[k] >> (4 * j)) & 15u), f.x, f.y);
    if constexpr (sizeof(OT) == 2)
      *reinterpret_cast<uint2*>(dst + 32 * k) = make_uint2(h2_as_u32(__floats2half2_rn(v[0], v[1])), h2_as_u32(__floats2half2_rn(v[2], v[3])));
    else
      *reinterpret_cast<float4*>(dst + 32 * k) = make_float4(v[0], v[1], v[2], v[3]);
  }
}

// Launches over rows [0, rows) of `per_row` items each, at most 2^30 items at a time, so that indexes fit in 32 bits.
template <typename P, typename F>
static int over_rows(P p, int rows, int per_row, F run) {
  const int most = (1 << 30) / per_row;
  for (int row0 = 0; row0 < rows; row0 += std::min(most, rows - row0)) {
    p.row0 = row0;
    p.items = std::min(most, rows - row0) * per_row;
    const int st = run(p);
    if (st != SC_OK) return st;
  }
  return SC_OK;
}

}  // namespace sc

extern "C" {

size_t sc_quant_page_bytes(int page_size, int hd, int bits, int group) {
  if (!sc::quant_kind_ok(hd, bits, group) || page_size < 16 || page_size % 16) return 0;
  return (size_t)(page_size / 16) * sc::quant_block_bytes(hd, bits, group);
}

int sc_paged_rope_append_q(const void* qkv, int qkv_dtype, int rows, const int32_t* rows_end, const int32_t* slots,
                           const int32_t* positions, const float* cos_tab, const float* sin_tab, int max_pos, int Hq,
                           int Hkv, int hd, void* q_out, void* pages, int bits, int group, int n_pages, int page_size,
                           cudaStream_t stream) {
  using namespace sc;
  SC_REQUIRE(qkv && rows_end && slots && positions && cos_tab && sin_tab && q_out && pages, SC_ERR_ARG, "paged_rope_append_q: null pointer");
  SC_REQUIRE(quant_kind_ok(hd, bits, group), SC_ERR_UNSUPPORTED,
             "paged_rope_append_q: head_dim %d in %d bits by groups of %d unsupported (64 or 128; 4 or 8; 32 or 64)", hd, bits, group);
  SC_REQUIRE(page_size >= 16 && page_size % 16 == 0, SC_ERR_UNSUPPORTED, "paged_rope_append_q: page size %d is not a multiple of 16", page_size);
  SC_REQUIRE(rows >= 1 && Hq >= 1 && Hkv >= 1 && n_pages >= 1 && max_pos >= 1, SC_ERR_SHAPE, "paged_rope_append_q: empty shape");
  SC_REQUIRE((long long)n_pages * page_size <= INT32_MAX, SC_ERR_SHAPE, "paged_rope_append_q: slots past 32 bits");
  SC_REQUIRE(qkv_dtype == SC_F16 || qkv_dtype == SC_F32, SC_ERR_ARG, "paged_rope_append_q: dtype");
  SC_REQUIRE((((uintptr_t)qkv | (uintptr_t)q_out | (uintptr_t)pages | (uintptr_t)cos_tab | (uintptr_t)sin_tab) & 15) == 0, SC_ERR_ARG,
             "paged_rope_append_q: tensors must start on 16-byte boundaries");
  SC_REQUIRE(((long long)Hq + 2ll * Hkv) * (hd / 8) <= (1 << 24), SC_ERR_SHAPE, "paged_rope_append_q: rows of %d + 2 * %d heads are too wide", Hq, Hkv);
  const AppendQuantParams p = {qkv, rows_end, slots, positions, cos_tab, sin_tab, static_cast<__half*>(q_out), static_cast<uint8_t*>(pages),
                               0, 0, Hq, Hkv, max_pos, n_pages, page_div(page_size), page_div((Hq + 2 * Hkv) * (hd / 8))};
  return with_quant_block(hd, bits, group, [&](auto block) {
    using QB = decltype(block);
    return over_rows(p, rows, (Hq + 2 * Hkv) * (hd / 8), [&](const AppendQuantParams& a) {
      auto kern = qkv_dtype == SC_F32 ? append_quant_kernel<float, QB> : append_quant_kernel<__half, QB>;
      launch(kern, dim3((unsigned)((a.items + 255) / 256)), dim3(256), 0, stream, a);
      return check_launch("paged_rope_append_q");
    });
  });
}

int sc_paged_read_q(const void* pages, int bits, int group, int n_pages, int page_size, int Hkv, int hd,
                    const int32_t* slots, int rows, const int32_t* rows_end, void* k_out, void* v_out, int out_dtype,
                    cudaStream_t stream) {
  using namespace sc;
  SC_REQUIRE(pages && slots && k_out && v_out, SC_ERR_ARG, "paged_read_q: null pointer");
  SC_REQUIRE(quant_kind_ok(hd, bits, group), SC_ERR_UNSUPPORTED,
             "paged_read_q: head_dim %d in %d bits by groups of %d unsupported (64 or 128; 4 or 8; 32 or 64)", hd, bits, group);
  SC_REQUIRE(page_size >= 16 && page_size % 16 == 0, SC_ERR_UNSUPPORTED, "paged_read_q: page size %d is not a multiple of 16", page_size);
  SC_REQUIRE(rows >= 1 && Hkv >= 1 && n_pages >= 1, SC_ERR_SHAPE, "paged_read_q: empty shape");
  SC_REQUIRE((long long)n_pages * page_size <= INT32_MAX, SC_ERR_SHAPE, "paged_read_q: slots past 32 bits");
  SC_REQUIRE(out_dtype == SC_F16 || out_dtype == SC_F32, SC_ERR_ARG, "paged_read_q: dtype");
  SC_REQUIRE((((uintptr_t)pages | (uintptr_t)k_out | (uintptr_t)v_out) & 15) == 0, SC_ERR_ARG,
             "paged_read_q: tensors must start on 16-byte boundaries");
  SC_REQUIRE(2ll * Hkv * 8 <= (1 << 24), SC_ERR_SHAPE, "paged_read_q: rows of 2 * %d heads are too wide", Hkv);
  const ReadQuantParams p = {static_cast<const uint8_t*>(pages), slots, rows_end, k_out, v_out, 0, 0, Hkv, n_pages,
                             page_div(page_size), page_div(2 * Hkv * 8)};
  return with_quant_block(hd, bits, group, [&](auto block) {
    using QB = decltype(block);
    return over_rows(p, rows, 2 * Hkv * 8, [&](const ReadQuantParams& a) {
      auto kern = out_dtype == SC_F32 ? read_quant_kernel<float, QB> : read_quant_kernel<__half, QB>;
      launch(kern, dim3((unsigned)((a.items + 255) / 256)), dim3(256), 0, stream, a);
      return check_launch("paged_read_q");
    });
  });
}

}  // extern "C"
