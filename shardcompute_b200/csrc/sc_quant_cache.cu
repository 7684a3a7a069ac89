// Tokens into and out of a paged cache that is held in 8 or 4 bits.
//
// A group of GS values x of one token and head is held as codes c of BITS bits,
// a scale s and a bias b (fp16):
//   b = min x rounded down, s = the smallest fp16 value with MOST s >= max x - b,
//   c = rint((x - b) / s) in 0..MOST (0 where s is 0), and stands for s c + b
// so that b <= x <= b + MOST s, and x is at most s / 2 off.
#include <algorithm>

#include "sc_quant.cuh"

namespace sc {

struct AppendQuantParams {
  const void* qkv;
  const int32_t *rows_end, *slots, *positions;  // rows_end: one past the last row that is used
  const float *cos_tab, *sin_tab;
  __half* q_out;
  uint8_t* pages;
  int row0, items, Hq, Hkv, max_pos, n_pages, page;
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

// (scale, bias) of a group with these extremes.  Where either is not finite the bias is NaN: the group stands for NaN, and
// no score of it is an infinity that would take the token out of the attention unseen.
template <int MOST>
__device__ __forceinline__ __half2 scale_bias(float lo, float hi) {
  const __half b = __float2half_rd(lo);
  const double need = fmax((double)hi - (double)__half2float(b), 0.0);
  __half s = __float2half_ru((float)need * (1.f / MOST));
  // the estimate is within a few roundings of fp32: at most one fp16 value off
  const unsigned short u = __half_as_ushort(s);
  if ((double)(__half2float(s) * MOST) < need)
    s = __ushort_as_half(u + 1);
  else if (u > 0 && u <= 0x7c00 && (double)(__half2float(__ushort_as_half(u - 1)) * MOST) >= need)
    s = __ushort_as_half(u - 1);
  const bool finite = (__half_as_ushort(s) & 0x7c00) != 0x7c00 && (__half_as_ushort(b) & 0x7c00) != 0x7c00;
  return __halves2half2(s, finite ? b : __ushort_as_half(0x7e00));
}

template <int MOST>
__device__ __forceinline__ uint32_t code_of(float x, float s, float b) {
  const float c = rintf(__fdiv_rn(x - b, s));
  return s > 0.f ? (uint32_t)fminf(fmaxf(c, 0.f), (float)MOST) : 0u;  // NaN: 0
}

// Four codes as the bytes that hold them.
template <int BITS>
__device__ __forceinline__ uint32_t pack4(const uint32_t (&c)[4]) {
  return c[0] | c[1] << BITS | c[2] << (2 * BITS) | c[3] << (3 * BITS);
}

constexpr int AQ_ITEMS = 2;  // of a thread

// An item is eight values of a head of a row: four pairs (d, d + HD/2).  q and k
// are rotated, the products not fused (the bits of the append that does not
// quantise), and q is rounded once.  The HD/8 items of a k or v head lie in
// neighbouring lanes, which find their groups' extremes by shuffles and write
// the codes; moves its bytes once.
template <typename ST, typename QB>
__global__ void __launch_bounds__(256) append_quant_kernel(const AppendQuantParams p) {
  constexpr int HD = QB::HD, HALF = HD / 2, LPH = HD / 8, NG = QB::NG, GS = QB::GS;
  pdl_trigger();
  pdl_wait();
  const int end = *p.rows_end, per_row = (p.Hq + 2 * p.Hkv) * LPH;
#pragma unroll
  for (int i = 0; i < AQ_ITEMS; ++i) {
    const int it = (blockIdx.x * AQ_ITEMS + i) * 256 + threadIdx.x;
    const int r = it / per_row, e = it - r * per_row, row = p.row0 + r, h = e / LPH, l = e % LPH, d = l * 4;
    const bool live = it < p.items && row < end, is_kv = h >= p.Hq, is_v = h >= p.Hq + p.Hkv;
    float a[4] = {0.f, 0.f, 0.f, 0.f}, b[4] = {0.f, 0.f, 0.f, 0.f};
    int pos = -1, slot = -1;
    if (live) {
      pos = p.positions[row];
      slot = p.slots[row];
      const ST* src = reinterpret_cast<const ST*>(p.qkv) + ((size_t)row * (p.Hq + 2 * p.Hkv) + h) * HD + d;
      load4(src, a);
      load4(src + HALF, b);
      if (!is_v && pos >= 0 && pos < p.max_pos) {
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
    }
    if (live && !is_kv) {
      __half* dst = p.q_out + ((size_t)row * p.Hq + h) * HD + d;
      *reinterpret_cast<uint2*>(dst) = make_uint2(h2_as_u32(__floats2half2_rn(a[0], a[1])), h2_as_u32(__floats2half2_rn(a[2], a[3])));
      *reinterpret_cast<uint2*>(dst + HALF) = make_uint2(h2_as_u32(__floats2half2_rn(b[0], b[1])), h2_as_u32(__floats2half2_rn(b[2], b[3])));
    }
    if (!__any_sync(0xffffffffu, live && is_kv)) continue;
    // ---- the groups of a's and of b's dims (one and the same where a head is a single group)
    float lo[2] = {min_nan(min_nan(a[0], a[1]), min_nan(a[2], a[3])), min_nan(min_nan(b[0], b[1]), min_nan(b[2], b[3]))};
    float hi[2] = {max_nan(max_nan(a[0], a[1]), max_nan(a[2], a[3])), max_nan(max_nan(b[0], b[1]), max_nan(b[2], b[3]))};
    if (NG == 1) {
      lo[0] = lo[1] = min_nan(lo[0], lo[1]);
      hi[0] = hi[1] = max_nan(hi[0], hi[1]);
    }
    constexpr int WIDTH = NG == 1 ? LPH : GS / 4;  // lanes that share a group
#pragma unroll
    for (int x = 1; x < WIDTH; x <<= 1)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        lo[k] = min_nan(lo[k], __shfl_xor_sync(0xffffffffu, lo[k], x));
        hi[k] = max_nan(hi[k], __shfl_xor_sync(0xffffffffu, hi[k], x));
      }
    const int id = slot >= 0 ? slot / p.page : p.n_pages;
    if (!live || !is_kv || pos < 0 || pos >= p.max_pos || id >= p.n_pages) continue;
    const int off = slot - id * p.page, tok = off & 15, head = h - p.Hq - (is_v ? p.Hkv : 0);
    uint8_t* block = p.pages + (((size_t)id * p.Hkv + head) * (p.page >> 4) + (off >> 4)) * QB::BYTES;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const __half2 sb = scale_bias<QB::MOST>(lo[k], hi[k]);
      const float s = __low2float(sb), bias = __high2float(sb);
      const float(&x)[4] = k ? b : a;
      const int dim = d + k * HALF;
      uint32_t c[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) c[j] = code_of<QB::MOST>(x[j], s, bias);
      const uint32_t w = pack4<QB::BITS>(c);
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
}

struct ReadQuantParams {
  const uint8_t* pages;
  const int32_t *slots, *rows_end;  // rows_end: NULL: every row
  void *k_out, *v_out;
  int row0, items, Hkv, n_pages, page;
};

// An item is eight consecutive values of a head of a row's K or V: s c + b in
// fp32, rounded once.  Bound by the writes.
template <typename OT, typename QB>
__global__ void __launch_bounds__(256) read_quant_kernel(const ReadQuantParams p) {
  constexpr int HD = QB::HD, LPH = HD / 8;
  pdl_trigger();
  pdl_wait();
  const int it = blockIdx.x * 256 + threadIdx.x, per_row = 2 * p.Hkv * LPH;
  if (it >= p.items) return;
  const int r = it / per_row, e = it - r * per_row, row = p.row0 + r, side = e / (p.Hkv * LPH), h = e / LPH - side * p.Hkv, d = e % LPH * 8;
  if (p.rows_end && row >= *p.rows_end) return;
  const int slot = p.slots[row], id = slot >= 0 ? slot / p.page : p.n_pages;
  float v[8];
  if (id < p.n_pages) {
    const int off = slot - id * p.page, tok = off & 15;
    const uint8_t* block = p.pages + (((size_t)id * p.Hkv + h) * (p.page >> 4) + (off >> 4)) * QB::BYTES;
    const __half2 sb = *reinterpret_cast<const __half2*>(block + (side ? QB::VM : QB::KM) + (tok * QB::NG + d / QB::GS) * 4);
    const float s = __low2float(sb), b = __high2float(sb);
    uint32_t w[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const uint8_t* src = block + (side ? QB::v_at(tok, d + 4 * k) : QB::k_at(tok, d + 4 * k));
      w[k] = *reinterpret_cast<const uint16_t*>(src);
      if (QB::BITS == 8) w[k] |= (uint32_t)*reinterpret_cast<const uint16_t*>(src + (side ? 4 : 2)) << 16;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = fmaf((float)((w[j >> 2] >> ((j & 3) * QB::BITS)) & QB::MOST), s, b);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = 0.f;
  }
  OT* dst = reinterpret_cast<OT*>(side ? p.v_out : p.k_out) + ((size_t)row * p.Hkv + h) * HD + d;
  if constexpr (sizeof(OT) == 2) {
    *reinterpret_cast<uint4*>(dst) = make_uint4(h2_as_u32(__floats2half2_rn(v[0], v[1])), h2_as_u32(__floats2half2_rn(v[2], v[3])),
                                                h2_as_u32(__floats2half2_rn(v[4], v[5])), h2_as_u32(__floats2half2_rn(v[6], v[7])));
  } else {
    *reinterpret_cast<float4*>(dst) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(dst + 4) = make_float4(v[4], v[5], v[6], v[7]);
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
                               0, 0, Hq, Hkv, max_pos, n_pages, page_size};
  return with_quant_block(hd, bits, group, [&](auto block) {
    using QB = decltype(block);
    return over_rows(p, rows, (Hq + 2 * Hkv) * (hd / 8), [&](const AppendQuantParams& a) {
      auto kern = qkv_dtype == SC_F32 ? append_quant_kernel<float, QB> : append_quant_kernel<__half, QB>;
      launch(kern, dim3((unsigned)((a.items + 256 * AQ_ITEMS - 1) / (256 * AQ_ITEMS))), dim3(256), 0, stream, a);
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
  SC_REQUIRE(2ll * Hkv * (hd / 8) <= (1 << 24), SC_ERR_SHAPE, "paged_read_q: rows of 2 * %d heads are too wide", Hkv);
  const ReadQuantParams p = {static_cast<const uint8_t*>(pages), slots, rows_end, k_out, v_out, 0, 0, Hkv, n_pages, page_size};
  return with_quant_block(hd, bits, group, [&](auto block) {
    using QB = decltype(block);
    return over_rows(p, rows, 2 * Hkv * (hd / 8), [&](const ReadQuantParams& a) {
      auto kern = out_dtype == SC_F32 ? read_quant_kernel<float, QB> : read_quant_kernel<__half, QB>;
      launch(kern, dim3((unsigned)((a.items + 255) / 256)), dim3(256), 0, stream, a);
      return check_launch("paged_read_q");
    });
  });
}

}  // extern "C"
