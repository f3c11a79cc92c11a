// MXFP4 operands of this library: 4-bit e2m1 codes with one power-of-two scale (E8M0 byte: exponent + 127, 255 = NaN)
// for each block of 32 along a row, stored in the order the 16x16x128 scaled MFMA reads them.
//  * codes: tiles of 16 rows x 128 columns, 1 KB each, tile (rt, kt) at (rt * nkt + kt) * 1024. Within a tile the 16 bytes
//    of lane l are row (l & 15), columns 32 (l >> 4) .. + 31, the even column in the low nibble: one tile is one operand,
//    read by one 16-byte load per lane from 1 KB in a row, also after a linear copy to LDS (no bank conflicts, no swizzle).
//  * scales: one dword per lane and four tiles along the row, tile kt in byte kt & 3, at ((rt * nks + kt / 4) * 64 + l) * 4:
//    one register serves four MFMAs, which pick their byte.
// Rows past the last one and columns past K have code 0 and scale byte 0.
#pragma once
#include "common.h"

typedef int i32x8 __attribute__((ext_vector_type(8)));

__host__ __device__ __forceinline__ int mx4_nkt(int K) { return (K + 127) / 128; }
__host__ __device__ __forceinline__ int mx4_nks(int K) { return (mx4_nkt(K) + 3) / 4; }
__host__ __device__ __forceinline__ long mx4_rt(long M) { return (M + 15) / 16; }

// D += A B^T over 128 columns of one 16-row tile each; byte B of the scale registers. Lane l: D column (l & 15) (the row
// of b), D rows 4 (l >> 4) + r (the rows of a).
template <int BYTE>
__device__ __forceinline__ f32x4 mfma_mx4(u32x4 a, u32x4 b, f32x4 c, int sa, int sb) {
  const i32x8 A = {(int)a.x, (int)a.y, (int)a.z, (int)a.w, 0, 0, 0, 0};
  const i32x8 B = {(int)b.x, (int)b.y, (int)b.z, (int)b.w, 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(A, B, c, 4, 4, BYTE, sa, BYTE, sb);
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
// Columns k .. k + 7 of a row, zeros past K; vec: the row is 16-byte aligned and so is every multiple of 8 columns.
__device__ __forceinline__ u32x4 load8(const uint16_t* __restrict__ row, int k, int K, bool vec) {
  if (vec && k + 8 <= K) return *reinterpret_cast<const u32x4*>(row + k);
  u32x4 v = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int e = 0; e < 8; e++)
    if (k + e < K) v[e >> 1] |= (uint32_t)row[k + e] << (16 * (e & 1));
  return v;
}
