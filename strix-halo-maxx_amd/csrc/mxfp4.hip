// MXFP4 quantisation (bf16 rows to 4-bit codes with a power-of-two scale per 32 columns, OCP MX v1.0's conversion) and
// its inverse. Storage: mxfp4.h.
//   e = max(floor(log2(max |x|)) - 2, -127) over the block, code = e2m1(x 2^-e) to nearest even, saturating at 6.
// Every step is exact but the rounding of the code, so the codes follow from the formula bit for bit.
#include "mxfp4.h"

namespace {

// A workgroup of 4 waves covers 64 rows x 128 columns, wave w the rows 16 w ... Four lanes share a block of 32: each loads
// 16 bytes, the block's maximum goes over the quad by DPP, each lane stores a dword of codes; a wave's load takes 256
// bytes from each of 4 rows. The bound is HBM: 2 bytes read and 0.53 written per value. 186624 x 1152 96 us (5.7 TB/s, a copy
// of 1 GiB 5.2), 9477 x 2048 11.6, 794 x 2048 3.2, 40000 x 588 17.4 (37.4 with 2-byte loads at its odd row starts).
__global__ __launch_bounds__(256) void quant_mxfp4_kernel(const uint16_t* __restrict__ x, long ldx,
                                                          uint8_t* __restrict__ codes, uint32_t* __restrict__ scales,
                                                          int M, int K) {
  __shared__ uint8_t sc[64][4];
  const int nk = mx4_nk(K);
  const int ks = blockIdx.x % nk;
  const long rg = blockIdx.x / nk;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int part = lane & 3, g = (lane >> 2) & 3;
  const int k = ks * 128 + g * 32 + part * 8;
  u32x4 v[4];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const long row = rg * 64 + wave * 16 + 4 * i + (lane >> 4);
    v[i] = u32x4{0u, 0u, 0u, 0u};
    if (row < M && k < K) v[i] = load8(x + row * ldx, k, K);
  }
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int r = wave * 16 + 4 * i + (lane >> 4);
    const uint32_t byte = mx4_scale_byte(quad_max(amax8(v[i])));
    const uint32_t c = byte == 255u ? 0u : mx4_pack8(v[i], e8m0_float(byte));
    const int l = 32 * (g & 1) + (r & 31);
    if (rg * 64 + r < M)
      reinterpret_cast<uint32_t*>(codes)[((2 * rg + (r >> 5)) * 2 * nk + 2 * ks + (g >> 1)) * 256 + l * 4 + part] = c;
    if (part == 0) sc[l][2 * (r >> 5) + (g >> 1)] = (uint8_t)byte;
  }
  __syncthreads();
  if (wave == 0) scales[(rg * nk + ks) * 64 + lane] = *reinterpret_cast<const uint32_t*>(sc[lane]);
}

// The same cells: a wave writes 256 bytes of each of 4 rows at a time, a lane 8 columns from one dword of codes. The loads
// have no branches (rows past the end repeat the last one), so they go out together. HBM bound: 186624 x 1152 112 us (4.9
// TB/s, 131 with branches), 794 x 2048 4.0.
__global__ __launch_bounds__(256) void mxfp4_values_kernel(const uint8_t* __restrict__ codes,
                                                           const uint32_t* __restrict__ scales,
                                                           uint16_t* __restrict__ y, long ldy, int M, int K) {
  const int nk = mx4_nk(K);
  const int ks = blockIdx.x % nk;
  const long rg = blockIdx.x / nk;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int part = lane & 3, g = (lane >> 2) & 3;
  const int k = ks * 128 + g * 32 + part * 8;
  const uint32_t* tile = reinterpret_cast<const uint32_t*>(codes) + (2 * rg * 2 * nk + 2 * ks + (g >> 1)) * 256;
  uint32_t c[4], sc[4];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int r = (int)min((long)(wave * 16 + 4 * i + (lane >> 4)), M - 1 - rg * 64), l = 32 * (g & 1) + (r & 31);
    c[i] = tile[(r >> 5) * 2 * nk * 256 + l * 4 + part];
    sc[i] = (scales[(rg * nk + ks) * 64 + l] >> (16 * (r >> 5) + 8 * (g >> 1))) & 255u;
  }
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const long row = rg * 64 + wave * 16 + 4 * i + (lane >> 4);
    if (row >= M || k >= K) continue;
    const float s = e8m0_float(sc[i]);
    u32x4 v;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      float f[2];
#pragma unroll
      for (int h = 0; h < 2; h++) {
        // e2m1 code m (3 bits): 0, 0.5, then 2^(m / 2 - 1) (1 + (m & 1) / 2)
        const uint32_t q = c[i] >> (8 * e + 4 * h), m = q & 7u;
        const float a = m < 2u ? 0.5f * (float)m : __uint_as_float(((126u + (m >> 1)) << 23) | ((m & 1u) << 22));
        f[h] = ((q & 8u) ? -a : a) * s;
      }
      v[e] = sc[i] == 255u ? 0x7fc07fc0u : pack2(f[0], f[1]);
    }
    uint16_t* out = y + row * ldy + k;
    if (k + 8 <= K) {  // not kept in the caches: 112 us for 117 at 186624 x 1152, 12.1 for 14.9 at 9477 x 2048
      __builtin_nontemporal_store(v, reinterpret_cast<u32x4_any*>(out));
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++)
        if (k + e < K) out[e] = (uint16_t)(v[e >> 1] >> (16 * (e & 1)));
    }
  }
}

}  // namespace

extern "C" long mx_mxfp4_code_bytes(int M, int K) { return M < 1 || K < 1 ? 0 : mx4_groups(M) * mx4_nk(K) * 4096; }
extern "C" long mx_mxfp4_scale_bytes(int M, int K) { return M < 1 || K < 1 ? 0 : mx4_groups(M) * mx4_nk(K) * 256; }

extern "C" int mx_quant_mxfp4(hipStream_t st, const uint16_t* x, long ldx, uint8_t* codes, uint8_t* scales, int M, int K) {
  if (!x || !codes || !scales) return MX_ENULL;
  if (M < 1 || K < 1 || ldx < 0) return MX_ESHAPE;
  if (((uintptr_t)x & 1) || ((uintptr_t)codes & 15) || ((uintptr_t)scales & 3)) return MX_ELAYOUT;
  const long wgs = mx4_groups(M) * mx4_nk(K);
  if (wgs > 0xffffffL) return MX_ESHAPE;  // 2^32 threads in a grid
  hipLaunchKernelGGL(quant_mxfp4_kernel, dim3((unsigned)wgs), dim3(256), 0, st, x, ldx, codes, (uint32_t*)scales, M, K);
  return hipGetLastError() == hipSuccess ? MX_OK : MX_ELAUNCH;
}

extern "C" int mx_mxfp4_values(hipStream_t st, const uint8_t* codes, const uint8_t* scales, uint16_t* y, long ldy, int M,
                               int K) {
  if (!codes || !scales || !y) return MX_ENULL;
  if (M < 1 || K < 1 || ldy < (M > 1 ? K : 0)) return MX_ESHAPE;
  if (((uintptr_t)y & 1) || ((uintptr_t)codes & 15) || ((uintptr_t)scales & 3)) return MX_ELAYOUT;
  const long wgs = mx4_groups(M) * mx4_nk(K);
  if (wgs > 0xffffffL) return MX_ESHAPE;  // 2^32 threads in a grid
  hipLaunchKernelGGL(mxfp4_values_kernel, dim3((unsigned)wgs), dim3(256), 0, st, codes, (const uint32_t*)scales, y, ldy, M,
                     K);
  return hipGetLastError() == hipSuccess ? MX_OK : MX_ELAUNCH;
}
