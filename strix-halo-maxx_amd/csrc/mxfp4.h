// MXFP4 operands of this library: 4-bit e2m1 codes with one power-of-two scale (E8M0 byte: exponent + 127, 255 = NaN)
// for each block of 32 along a row, stored in the order the 32x32x64 scaled MFMA reads them.
//  * codes: tiles of 32 rows x 64 columns, 1 KB each, tile (rt, kt) at (rt * nkt + kt) * 1024, nkt even. Within a tile the
//    16 bytes of lane l are row (l & 31), columns 32 (l >> 5) .. + 31, the even column in the low nibble: one tile is one
//    operand, read by one 16-byte load per lane from 1 KB in a row, also after a linear copy to LDS (no bank conflicts, no
//    swizzle).
//  * scales: one dword per lane for two tiles along the row (128 columns) of two row tiles (64 rows), tile (rt, kt) in
//    byte 2 (rt & 1) + (kt & 1), at ((rt / 2 * (nkt / 2) + kt / 2) * 64 + l) * 4.
// Columns past K of a row have code 0 and scale byte 0; rows past the last one are not written (they meet no result that
// is stored).
#pragma once
#include "common.h"

typedef int i32x8 __attribute__((ext_vector_type(8)));

__host__ __device__ __forceinline__ int mx4_nk(int K) { return (K + 127) / 128; }       // steps of 128 columns
__host__ __device__ __forceinline__ int mx4_nkt(int K) { return 2 * mx4_nk(K); }        // tiles along a row
__host__ __device__ __forceinline__ long mx4_groups(long M) { return (M + 63) / 64; }   // groups of 64 rows

__device__ __forceinline__ i32x8 mx4_operand(u32x4 v) {
  return i32x8{(int)v.x, (int)v.y, (int)v.z, (int)v.w, 0, 0, 0, 0};
}
// D += A B^T on 4-bit operands, byte SA / SB of the scale registers.
// 32x32x64: one tile each. Lane l: D column (l & 31) (the row of b), D rows 8 (r / 4) + 4 (l >> 5) + r % 4 (rows of a).
template <int SA, int SB>
__device__ __forceinline__ f32x16 mfma_mx4(u32x4 a, u32x4 b, f32x16 c, int sa, int sb) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(mx4_operand(a), mx4_operand(b), c, 4, 4, SA, sa, SB, sb);
}
// 16x16x128: lane l gives row (l & 15), columns 32 (l >> 4) .. + 31 and their scale. D column (l & 15), rows
// 4 (l >> 4) + r.
__device__ __forceinline__ f32x4 mfma_mx4(u32x4 a, u32x4 b, f32x4 c, int sa, int sb) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(mx4_operand(a), mx4_operand(b), c, 4, 4, 0, sa, 0, sb);
}

// The scale byte of a block whose largest |bf16| has these bits (sign cleared): floor(log2 amax) - 2, at least 2^-127
// (amax with exponent field E is 2^(E - 127) times [1, 2), so the byte is E - 2; below, the clamp covers the subnormals);
// inf or NaN in the block: NaN.
__device__ __forceinline__ uint32_t mx4_scale_byte(uint32_t amax_bits) {
  const uint32_t E = amax_bits >> 7;
  return E == 255u ? 255u : (E > 2u ? E - 2u : 0u);
}
__device__ __forceinline__ float e8m0_float(uint32_t byte) {  // 2^(byte - 127); byte 0 is the subnormal 2^-127
  return __uint_as_float(byte ? byte << 23 : 0x00400000u);
}
// Eight bf16 values to eight codes. v_cvt_scalef32_pk_fp4_bf16 divides by the scale exactly, rounds to nearest even and
// saturates at 6 (checked on every bf16 at scales 2^-127 .. 2^125).
__device__ __forceinline__ uint32_t mx4_pack8(u32x4 v, float scale) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};  // (a bit cast of a vector's element itself takes element 0 here)
  uint32_t o = 0;
  o = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(o, __builtin_bit_cast(bf16x2, w[0]), scale, 0);
  o = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(o, __builtin_bit_cast(bf16x2, w[1]), scale, 1);
  o = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(o, __builtin_bit_cast(bf16x2, w[2]), scale, 2);
  o = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(o, __builtin_bit_cast(bf16x2, w[3]), scale, 3);
  return o;
}
// largest |bf16| (bits) of eight
__device__ __forceinline__ uint32_t amax8(u32x4 v) {
  uint32_t m = 0;
#pragma unroll
  for (int e = 0; e < 4; e++) {
    const uint32_t w = v[e] & 0x7fff7fffu;
    m = max(m, max(w & 0xffffu, w >> 16));
  }
  return m;
}
// max over the four lanes of a quad
__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xb1, 0xf, 0xf, false));  // quad_perm [1, 0, 3, 2]
  return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4e, 0xf, 0xf, false));  // quad_perm [2, 3, 0, 1]
}
// Columns k .. k + 7 of a row, zeros past K. Rows may start at any column: global memory takes 16-byte accesses at any
// address, which the compiler uses for a type that is aligned to 2 bytes.
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
__device__ __forceinline__ u32x4 load8(const uint16_t* __restrict__ row, int k, int K) {
  if (k + 8 <= K) return *reinterpret_cast<const u32x4_any*>(row + k);
  u32x4 v = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int e = 0; e < 8; e++)
    if (k + e < K) v[e >> 1] |= (uint32_t)row[k + e] << (16 * (e & 1));
  return v;
}
