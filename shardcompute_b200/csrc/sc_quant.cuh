// How a paged cache in 8 or 4 bits lies in memory: what the append writes, the
// read and the attention take.
//
// A page of one kv head is a run of blocks of 16 tokens:
//   K codes [16 tokens][ROW] | V codes [8 pairs of tokens][2 ROW] |
//   K's (scale, bias) [16 tokens][NG] | V's, each pair two fp16
// so that 16 tokens of a head come with one bulk copy of BYTES, and every
// fragment of mma m16n8k16 with one conflict-free load per thread:
//   K  (A operand: tokens x dims).  Thread t of a row's four holds a quarter of
//      every group, its share of the row contiguous: share byte i of group g is
//      at t ROW/4 + g GS/4 + i (in dims).  A share of 32 bytes (8 bits, heads of
//      128) lies as two pieces of 16 in the row's halves, changed over for odd
//      tokens, so that 8 lanes' loads meet different banks.
//   V  (A operand: dims x tokens).  A register holds a dim of two neighbouring
//      tokens, so units of 2 bytes alternate between the two; a byte belongs to
//      one token all the same, and tokens are written apart.  Thread g of eight
//      holds an eighth of every group; the threads' pieces are exchanged by the
//      pair's number, against bank conflicts.
// Codes are taken as fp16 bit patterns: `w & 0x000f000f` is a pair of fp16
// subnormals code 2^-24 (0x00f000f0: code 2^-20), exact as operands of the tensor
// cores, so that no conversion stands between memory and the products.  A sum of
// products keeps the fewer bits, the lower a code lies (sc_quant_attn.cu, at q).
#pragma once

#include "sc_common.cuh"

namespace sc {

template <int HD_, int BITS_, int NG_>
struct QuantBlock {
  static constexpr int HD = HD_, BITS = BITS_, NG = NG_;
  static constexpr int GS = HD / NG;                  // dims of a group
  static constexpr int MOST = (1 << BITS) - 1;        // largest code
  static constexpr int ROW = HD * BITS / 8;           // code bytes of a token
  static constexpr int KSH = ROW / 4, VSH = ROW / 4;  // bytes of a thread's share: of a token's K, of a pair's V
  static constexpr int V = 16 * ROW, KM = 32 * ROW, VM = KM + 16 * 4 * NG, BYTES = KM + 32 * 4 * NG;

  // The byte of token `tok` that holds dim d (4 bits: dims d and d + 1, d even, the first in the low half).  Four dims
  // from a multiple of four on lie in the next bytes (K), or in the next 2 bytes and, 8 bits, 2 at + 4 (V).
  __device__ static int k_at(int tok, int d) {
    const int r = d % GS, share = (d / GS * (GS / 4) + r % (GS / 4)) * BITS / 8;
    return tok * ROW + piece_k(tok, r / (GS / 4), share);
  }
  __device__ static int v_at(int tok, int d) {
    const int r = d % GS, b = (d / GS * (GS / 8) + r % (GS / 8)) * BITS / 8;
    return V + (tok >> 1) * 2 * ROW + piece_v(tok >> 1, r / (GS / 8), b / 2 * 4 + (tok & 1) * 2 + b % 2);
  }
  // Byte `share` of thread t's share of a token's K, of thread g's of a pair's V, in the token's row, in the pair's.
  __device__ static int piece_k(int tok, int t, int share) {
    return KSH == 32 ? (((share >> 4) ^ (tok & 1)) << 6) + t * 16 + (share & 15) : t * KSH + share;
  }
  __device__ static int piece_v(int pair, int g, int share) {
    return VSH == 8 ? (g ^ ((pair & 2) << 1)) * 8 + share : (share >> 4) * 128 + ((g ^ ((pair & 3) << 1)) << 4) + (share & 15);
  }
};

inline bool quant_kind_ok(int hd, int bits, int group) {
  return (hd == 64 || hd == 128) && (bits == 4 || bits == 8) && (group == 32 || group == 64);
}
inline int quant_block_bytes(int hd, int bits, int group) { return 4 * hd * bits + 128 * (hd / group); }

// f(block) with the QuantBlock of the kind of pages that the arguments name.
template <typename F>
int with_quant_block(int hd, int bits, int group, F f) {
  if (hd == 128) {
    if (group == 64) return bits == 4 ? f(QuantBlock<128, 4, 2>{}) : f(QuantBlock<128, 8, 2>{});
    return bits == 4 ? f(QuantBlock<128, 4, 4>{}) : f(QuantBlock<128, 8, 4>{});
  }
  if (group == 64) return bits == 4 ? f(QuantBlock<64, 4, 1>{}) : f(QuantBlock<64, 8, 1>{});
  return bits == 4 ? f(QuantBlock<64, 4, 2>{}) : f(QuantBlock<64, 8, 2>{});
}

}  // namespace sc
