// The 4-bit key/value cache: its numbers and layout (kv4_cache.hip writes and
// reads it, kv4_attention.hip attends over it).
//
// A value is number * scale.  Numbers have a sign, two exponent bits and one of
// mantissa (0, 1/2, 1, 3/2, 2, 3, 4, 6); 32 dims of a token of a head share a
// scale, a positive number of five exponent bits and three of mantissa held in a
// byte: the upper bits of an fp16 number, up to 10240.  So a value has six significant
// bits: fp16 and bf16 hold it as it is, and what goes into a matrix product is what
// the cache holds.
//
// Layout (blocks of B tokens, Dp = head dim rounded up to 32):
//   K [blocks][heads][B][Dp/2]       two dims a byte, the even one in its lower half
//   V [blocks][heads][B/16][Dp][8]   16 tokens of one dim together, the even one in
//                                    the lower half: the operand of P.V's MFMAs
//   scales [blocks][heads][Dp/32][B] of K and of V
#pragma once

#include "hxmi_common.h"

namespace hxmi {
namespace kv4 {

constexpr float kMost = 61440.f;       // the largest value: 6 * 10240, the largest scale that fp16 holds six of
constexpr uint32_t kMostScale = 0xe2;  // that scale's byte

__device__ __forceinline__ float scale_value(uint32_t byte) {
  return (float)__builtin_bit_cast(_Float16, (unsigned short)(byte << 7));
}
// Two numbers of byte N of a word, the lower half first.
template <int N>
__device__ __forceinline__ half2v numbers(uint32_t w) {
  return __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.0f, N);
}
// A byte of scales as a pair of equal numbers: byte n by twice_byte(n).
__device__ __forceinline__ constexpr uint32_t twice_byte(uint32_t n) { return 0x0c000c00u | n << 16 | n; }  // (0x0c: zero)
__device__ __forceinline__ half2v scale_twice(uint32_t w, uint32_t byte) {
  return __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0u, w, byte) << 7);
}
template <int N>
__device__ __forceinline__ half2v scale_twice(uint32_t w) {
  return scale_twice(w, twice_byte(N));
}
// Bytes 2 N and 2 N + 1 of a word of scales as a pair.
template <int N>
__device__ __forceinline__ half2v scale_pair(uint32_t w) {
  constexpr uint32_t sel = 0x0c000c00u | (2 * N + 1) << 16 | 2 * N;
  return __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0u, w, sel) << 7);
}

}  // namespace kv4
}  // namespace hxmi
