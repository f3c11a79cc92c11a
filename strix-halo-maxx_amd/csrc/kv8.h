// The 8-bit KV cache: e4m3 codes with one power-of-two scale (E8M0 byte: exponent + 127) for each block of 64 tokens of
// one head, K and V apart. Value = code * 2^(byte - 127), exact in bf16. A block of K or V is 64 D bytes in the order in
// which the 32x32x64 MFMA takes its operands, 1 KB groups of 64 lanes x 16 bytes (lane = 32 h + l):
//  * K (rows = tokens): group t D / 32 + j, t < 2, j < D / 32: lane (h, l) holds token 32 t + l, columns
//    16 (2 j + h) .. + 15; groups 2 s, 2 s + 1 of a t are the operand of columns 64 s .. 64 s + 63.
//  * V (rows = columns of V, so that the product with the weights needs no transposition): group 2 t + j, t < D / 32,
//    j < 2: lane (h, l) holds column 32 t + l, byte r token 32 j + 8 (r / 4) + 4 h + r % 4. That is the token order in
//    which the MFMA leaves the scores of keys 32 j .. 32 j + 31 in the registers of lane (h, query), so the weights
//    go back into the next MFMA as they are.
// Both are read by 16-byte loads of 1 KB in a row, from memory or, after a linear copy, from LDS without bank conflicts.
// Caches: codes [slot][head][block][64 D], scales [slot][head][block].
#pragma once
#include "common.h"

constexpr int KV8_BLK = 64;

typedef int i32x8 __attribute__((ext_vector_type(8)));

__host__ __device__ __forceinline__ int kv8_blocks(int ctx) { return (ctx + KV8_BLK - 1) / KV8_BLK; }

// byte of token t (of 64), column d in a block
template <int D>
__device__ __forceinline__ int kv8_koff(int t, int d) {
  return (((t >> 5) * (D / 32) + (d >> 5)) * 64 + ((d >> 4) & 1) * 32 + (t & 31)) * 16 + (d & 15);
}
__device__ __forceinline__ int kv8_voff(int t, int d) {
  return (((d >> 5) * 2 + (t >> 5)) * 64 + ((t >> 2) & 1) * 32 + (d & 31)) * 16 + ((t >> 3) & 3) * 4 + (t & 3);
}

__device__ __forceinline__ float kv8_pow2(int byte) {  // 2^(byte - 127), byte 0 .. 254
  return __uint_as_float(byte ? (uint32_t)byte << 23 : 0x00400000u);
}
// The scale byte of a block whose largest finite |bf16| has these bits: the smallest e with amax <= 448 2^e, at least
// -127. amax = f 2^x with f in [1, 2) and 448 = 1.75 2^8: e = x - 8, one more where f > 1.75 (mantissa above 0x60).
__device__ __forceinline__ int kv8_scale_byte(uint32_t amax_bits) {
  const int b = (int)(amax_bits >> 7) - 8 + ((amax_bits & 0x7fu) > 0x60u ? 1 : 0);
  return b > 0 ? b : 0;
}
