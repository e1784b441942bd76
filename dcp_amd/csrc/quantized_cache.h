// The layout of a paged K/V cache held in 4 bits.
//
// Every 32 neighbouring elements of a token's key or value are a block: x = c 2^e, c one of +-{0, 0.5, 1, 1.5, 2, 3, 4, 6} in 4 bits (a
// sign, two bits of exponent, one of mantissa), e one of [-127, 127] in a byte that holds e + 127 (255: the block is no number).  This is
// the 4-bit type that the device's conversions read, two elements and their scale an instruction, so what is held here costs half an
// instruction an element to multiply with.
//
// 16 tokens of a kv head lie together in 17 D bytes, in the order in which lane l = 16 g + n of a wave takes them as operands of
// 16x16x32 products:
//
//   [0, 8 D)       K's codes, token by token: lane (n, g) takes quarter g of token n's row
//   [8 D, 16 D)    V's codes, [4 g][16 n][4 tokens][D / 32 bytes]: lane (n, g) takes elements n D / 16 .. of tokens 4 g .. 4 g + 3
//   [16 D, +D/2)   K's exponents, [16 tokens][D / 32]
//   [.., +D/2)     V's exponents, [4 g][D / 32][4 tokens]
//
// so that a wave reads K or V of 16 tokens as 8 D contiguous bytes, straight into the lanes that need them: no LDS and no transposition.
// (V's rows whole, a lane would need four loads of 4 bytes.)  The low half of a byte is the earlier element.
#pragma once

#include "attn_common.h"

namespace dcp {

constexpr int kQuantTokens = 16, kQuantBlock = 32;
constexpr int kQuantFewRows = 32;  // rows of a kv head of a request that the attention's kernel of few rows takes

template <int D>
struct QuantTile {
  static constexpr int BYTES = 17 * D;
  static constexpr int BLOCKS = D / 32;              // of a row
  static constexpr int V = 8 * D, K_EXP = 16 * D, V_EXP = K_EXP + D / 2;
  static constexpr int V_PIECE = D / 32;             // bytes of a token's sixteenth
  // what lane (n, g) reads, and bytes that it takes of K or V
  static constexpr int LANE_BYTES = D / 8;
  typedef uint32_t Codes __attribute__((ext_vector_type(D / 32)));
  // where lane 16 g + n finds them
  static __device__ __forceinline__ int k_of(int lane) { return ((lane & 15) * 4 + (lane >> 4)) * LANE_BYTES; }
  static __device__ __forceinline__ int k_exp_of(int lane) { return K_EXP + ((lane & 15) * 4 + (lane >> 4)) * BLOCKS / 4; }
  static __device__ __forceinline__ int v_of(int lane) { return V + lane * LANE_BYTES; }
  static __device__ __forceinline__ int v_exp_of(int lane) { return V_EXP + lane * BLOCKS / 16 * 4; }  // (g BLOCKS + n BLOCKS / 16) 4
};

// Two elements of byte SEL of `codes`, times the power of two in scale's exponent bits (its other bits are ignored).
template <int DTYPE, int SEL>
__device__ __forceinline__ uint32_t two_of_codes(uint32_t codes, float scale) {
  if constexpr (DTYPE == DCP_DTYPE_BF16) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, SEL));
  else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, SEL));
}
// The eight of a word.
template <int DTYPE>
__device__ __forceinline__ u32x4 eight_of_codes(uint32_t codes, float scale) {
  return u32x4{two_of_codes<DTYPE, 0>(codes, scale), two_of_codes<DTYPE, 1>(codes, scale), two_of_codes<DTYPE, 2>(codes, scale),
               two_of_codes<DTYPE, 3>(codes, scale)};
}
// Byte `i` of exponents as a scale for them.
__device__ __forceinline__ float exponent_scale(uint32_t exponents, int i) {
  return __uint_as_float(i == 3 ? exponents >> 1 : exponents << (23 - 8 * i));
}

// What a lane reads of 16 tokens.
template <int D>
struct QuantGroup {
  typename QuantTile<D>::Codes k, v;
  uint32_t k_exp, v_exp;
  __device__ __forceinline__ void load_k(const char* at, int lane) {
    k = *reinterpret_cast<const typename QuantTile<D>::Codes*>(at + QuantTile<D>::k_of(lane));
    k_exp = *reinterpret_cast<const uint8_t*>(at + QuantTile<D>::k_exp_of(lane));
  }
  __device__ __forceinline__ void load_v(const char* at, int lane) {
    v = *reinterpret_cast<const typename QuantTile<D>::Codes*>(at + QuantTile<D>::v_of(lane));
    v_exp = *reinterpret_cast<const uint32_t*>(at + QuantTile<D>::v_exp_of(lane));
  }
  // what nobody sees of the lane's token j may hold anything: with this exponent it is finite
  __device__ __forceinline__ void clear_v(int j) { v_exp &= ~(0xffu << (8 * j)); }
};

}  // namespace dcp
