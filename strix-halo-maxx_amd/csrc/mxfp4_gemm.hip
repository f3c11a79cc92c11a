// MXFP4 Linear: C[m, n] = act(sum_k Xq[m, k] Wq[n, k] + b[n]) + R[m, n], both operands in MXFP4 (mxfp4.h), on the
// 16x16x128 scaled MFMA, which multiplies every block's product by both scales itself. The sum, the bias, the activation
// and the residual stay in fp32; the one rounding is the store to bf16.
#include "mxfp4.h"

#include <type_traits>

namespace {

struct Mx4Epi {
  const float* bias;
  const uint16_t* R;
  long ldr;
  int r_rows;
  uint16_t* C;
  long ldc;
  int M, N, act_from, vec;
};

// Columns n .. n + 3 of row m (both may lie outside). vec: N % 4 == 0 and rows of C and R allow 8-byte accesses.
template <int ACT>
__device__ __forceinline__ void mx4_store(const Mx4Epi& p, int m, int n, f32x4 v) {
  if (m >= p.M || n >= p.N) return;
  const long rrow = p.R ? (long)(p.r_rows > 0 ? m % p.r_rows : m) * p.ldr : 0;
  const int cnt = min(4, p.N - n);
  float r[4] = {0.f, 0.f, 0.f, 0.f};
  if (p.R) {
    if (p.vec) {
      const u32x2 w = *reinterpret_cast<const u32x2*>(p.R + rrow + n);
      r[0] = lo_bf(w.x), r[1] = hi_bf(w.x), r[2] = lo_bf(w.y), r[3] = hi_bf(w.y);
    } else {
#pragma unroll
      for (int e = 0; e < 4; e++)
        if (e < cnt) r[e] = bf2f(p.R[rrow + n + e]);
    }
  }
#pragma unroll
  for (int e = 0; e < 4; e++) {
    float y = v[e];
    if (p.bias && e < cnt) y += p.bias[n + e];
    if (ACT && n + e >= p.act_from) y = ACT == 1 ? gelu_tanh(y) : gelu_erf(y);
    v[e] = p.R ? y + r[e] : y;
  }
  uint16_t* out = p.C + (long)m * p.ldc + n;
  if (p.vec) {
    *reinterpret_cast<u32x2*>(out) = u32x2{pack2(v[0], v[1]), pack2(v[2], v[3])};
  } else {
#pragma unroll
    for (int e = 0; e < 4; e++)
      if (e < cnt) out[e] = f2bf(v[e]);
  }
}

// ---------------------------------------------------------------------------------------------- few rows
// At most 16 MT rows. A workgroup owns 16 columns of C (16 rows of W); its waves take the groups of 512 columns of K in
// turn (4 KB of W each, read in one piece) and their sums meet in LDS. PRE = false: x arrives in bf16 and each wave
// quantises the 512 columns it multiplies (its own slice: no wave waits for another before the end).
template <int NW, int MT, bool PRE, int ACT>
__global__ __launch_bounds__(64 * NW) void mx4_rows_kernel(const uint16_t* __restrict__ x, long ldx, int vecx,
                                                           const uint8_t* __restrict__ xc,
                                                           const uint32_t* __restrict__ xs,
                                                           const uint8_t* __restrict__ wc,
                                                           const uint32_t* __restrict__ ws, int K, Mx4Epi p) {
  static_assert(PRE || MT == 1, "bf16 rows come in one tile");
  __shared__ __attribute__((aligned(16))) uint32_t xq[PRE ? 1 : NW][16][64];  // a row's codes of the wave's 512 columns
  __shared__ __attribute__((aligned(16))) uint8_t xsc[PRE ? 1 : NW][16][16];  // its scale bytes, [32-block % 4][tile]
  __shared__ f32x4 red[NW][MT][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int nkt = mx4_nkt(K), nks = mx4_nks(K);
  const long nt = blockIdx.x;
  const int r16 = lane & 15, g = lane >> 4;
  f32x4 acc[MT];
#pragma unroll
  for (int i = 0; i < MT; i++) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int ks = wave; ks < nks; ks += NW) {
    u32x4 w[4], b[MT][4];
    const int left = nkt - 4 * ks;
    const uint8_t* wt = wc + (nt * nkt + 4 * ks) * 1024 + lane * 16;
#pragma unroll
    for (int t = 0; t < 4; t++) {
      w[t] = u32x4{0u, 0u, 0u, 0u};
      if (t < left) w[t] = *reinterpret_cast<const u32x4*>(wt + t * 1024);
    }
    const int sw = (int)ws[(nt * nks + ks) * 64 + lane];
    int sx[MT];
    if constexpr (PRE) {
#pragma unroll
      for (int i = 0; i < MT; i++) {
        const uint8_t* xt = xc + ((long)i * nkt + 4 * ks) * 1024 + lane * 16;
        const bool on = 16 * i < p.M;
#pragma unroll
        for (int t = 0; t < 4; t++) {
          b[i][t] = u32x4{0u, 0u, 0u, 0u};
          if (on && t < left) b[i][t] = *reinterpret_cast<const u32x4*>(xt + t * 1024);
        }
        sx[i] = on ? (int)xs[((long)i * nks + ks) * 64 + lane] : 0;
      }
    } else {
      const int blk = lane >> 2, k = ks * 512 + lane * 8;
      for (int m = 0; m < p.M; m++) {
        u32x4 v = {0u, 0u, 0u, 0u};
        if (k < K) v = load8(x + m * ldx, k, K, vecx);
        const uint32_t byte = mx4_scale_byte(quad_max(amax8(v)));
        xq[wave][m][lane] = byte == 255u ? 0u : mx4_pack8(v, e8m0_float(byte));
        if ((lane & 3) == 0) xsc[wave][m][(blk & 3) * 4 + (blk >> 2)] = (uint8_t)byte;
      }
      // the wave reads only what it wrote: in order, once its LDS writes are done
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_wave_barrier();
      const bool on = r16 < p.M;
#pragma unroll
      for (int t = 0; t < 4; t++) {
        b[0][t] = u32x4{0u, 0u, 0u, 0u};
        if (on) b[0][t] = *reinterpret_cast<const u32x4*>(&xq[wave][r16][(4 * t + g) * 4]);
      }
      sx[0] = on ? *reinterpret_cast<const int*>(&xsc[wave][r16][g * 4]) : 0;
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_wave_barrier();
    }
#pragma unroll
    for (int i = 0; i < MT; i++) {
      acc[i] = mfma_mx4<0>(w[0], b[i][0], acc[i], sw, sx[i]);
      acc[i] = mfma_mx4<1>(w[1], b[i][1], acc[i], sw, sx[i]);
      acc[i] = mfma_mx4<2>(w[2], b[i][2], acc[i], sw, sx[i]);
      acc[i] = mfma_mx4<3>(w[3], b[i][3], acc[i], sw, sx[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < MT; i++) red[wave][i][lane] = acc[i];
  __syncthreads();
  for (int i = wave; i < MT; i += NW) {
    f32x4 s = red[0][i][lane];
#pragma unroll
    for (int u = 1; u < NW; u++) s += red[u][i][lane];
    mx4_store<ACT>(p, 16 * i + r16, (int)nt * 16 + 4 * g, s);
  }
}

// ---------------------------------------------------------------------------------------------- tiles
// 128 x 128 tiles, 4 waves of 64 x 64, operands straight from memory.
template <int ACT>
__global__ __launch_bounds__(256) void mx4_tile_kernel(const uint8_t* __restrict__ xc, const uint32_t* __restrict__ xs,
                                                       const uint8_t* __restrict__ wc, const uint32_t* __restrict__ ws,
                                                       int K, Mx4Epi p, int tiles_n) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int nkt = mx4_nkt(K), nks = mx4_nks(K);
  const int m0 = (blockIdx.x / tiles_n) * 128 + (wave & 1) * 64, n0 = (blockIdx.x % tiles_n) * 128 + (wave >> 1) * 64;
  const int mrt = (p.M + 15) / 16 - 1, nrt = (p.N + 15) / 16 - 1;  // last row tiles
  long xr[4], wr[4];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    xr[i] = min(m0 / 16 + i, mrt);
    wr[i] = min(n0 / 16 + i, nrt);
  }
  f32x4 acc[4][4];
#pragma unroll
  for (int i = 0; i < 4; i++)
#pragma unroll
    for (int j = 0; j < 4; j++) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int ks = 0; ks < nks; ks++) {
    int sx[4], sw[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      sx[i] = (int)xs[(xr[i] * nks + ks) * 64 + lane];
      sw[i] = (int)ws[(wr[i] * nks + ks) * 64 + lane];
    }
    auto step = [&](auto tc) {
      constexpr int t = decltype(tc)::value;
      if (4 * ks + t >= nkt) return;
      u32x4 a[4], b[4];
#pragma unroll
      for (int i = 0; i < 4; i++) {
        b[i] = *reinterpret_cast<const u32x4*>(xc + (xr[i] * nkt + 4 * ks + t) * 1024 + lane * 16);
        a[i] = *reinterpret_cast<const u32x4*>(wc + (wr[i] * nkt + 4 * ks + t) * 1024 + lane * 16);
      }
#pragma unroll
      for (int j = 0; j < 4; j++)
#pragma unroll
        for (int i = 0; i < 4; i++) acc[i][j] = mfma_mx4<t>(a[j], b[i], acc[i][j], sw[j], sx[i]);
    };
    step(std::integral_constant<int, 0>{});
    step(std::integral_constant<int, 1>{});
    step(std::integral_constant<int, 2>{});
    step(std::integral_constant<int, 3>{});
  }
  const int r16 = lane & 15, g = lane >> 4;
#pragma unroll
  for (int i = 0; i < 4; i++)
#pragma unroll
    for (int j = 0; j < 4; j++) mx4_store<ACT>(p, m0 + 16 * i + r16, n0 + 16 * j + 4 * g, acc[i][j]);
}

int check(const void* wc, const void* ws, const float* bias, const uint16_t* R, long ldr, int r_rows, const uint16_t* C,
          long ldc, int M, int N, int K, int act, int act_from) {
  if (!wc || !ws || !C) return MX_ENULL;
  if (act < 0 || act > 2) return MX_EBADCFG;
  if (M < 1 || N < 1 || K < 1 || act_from < 0 || r_rows < 0 || (M > 1 && ldc < N)) return MX_ESHAPE;
  if (R && ldr < 0) return MX_ESHAPE;
  if ((((uintptr_t)wc) & 15) || ((uintptr_t)ws & 3) || ((uintptr_t)bias & 3) || ((uintptr_t)R & 1) || ((uintptr_t)C & 1))
    return MX_ELAYOUT;
  return MX_OK;
}

Mx4Epi epi(const float* bias, const uint16_t* R, long ldr, int r_rows, uint16_t* C, long ldc, int M, int N, int act_from) {
  const bool vec = N % 4 == 0 && !((uintptr_t)C & 7) && ldc % 4 == 0 && (!R || (!((uintptr_t)R & 7) && ldr % 4 == 0));
  return Mx4Epi{bias, R, ldr, r_rows, C, ldc, M, N, act_from, vec};
}

template <int MT, bool PRE>
hipError_t launch_rows(hipStream_t st, const uint16_t* x, long ldx, int vecx, const uint8_t* xc, const uint8_t* xs,
                       const uint8_t* wc, const uint8_t* ws, int K, int act, const Mx4Epi& p) {
  const dim3 grid((unsigned)((p.N + 15) / 16));
  auto go = [&](auto kern, int nw) {
    hipLaunchKernelGGL(kern, grid, dim3(64 * nw), 0, st, x, ldx, vecx, xc, (const uint32_t*)xs, wc, (const uint32_t*)ws, K,
                       p);
    return hipGetLastError();
  };
  if (mx4_nks(K) <= 4) {
    if (act == 0) return go(mx4_rows_kernel<4, MT, PRE, 0>, 4);
    if (act == 1) return go(mx4_rows_kernel<4, MT, PRE, 1>, 4);
    return go(mx4_rows_kernel<4, MT, PRE, 2>, 4);
  }
  if (act == 0) return go(mx4_rows_kernel<8, MT, PRE, 0>, 8);
  if (act == 1) return go(mx4_rows_kernel<8, MT, PRE, 1>, 8);
  return go(mx4_rows_kernel<8, MT, PRE, 2>, 8);
}

}  // namespace

// Rows that mx_gemv_mxfp4 takes.
extern "C" int mx_gemv_mxfp4_rows(void) { return 16; }

extern "C" int mx_gemv_mxfp4(hipStream_t st, const uint16_t* x, long ldx, const uint8_t* wc, const uint8_t* ws,
                             const float* bias, const uint16_t* R, long ldr, int r_rows, uint16_t* C, long ldc, int M,
                             int N, int K, int act, int act_from) {
  if (!x) return MX_ENULL;
  const int rc = check(wc, ws, bias, R, ldr, r_rows, C, ldc, M, N, K, act, act_from);
  if (rc) return rc;
  if (M > 16 || ldx < 0) return MX_ESHAPE;
  if ((uintptr_t)x & 1) return MX_ELAYOUT;
  const int vecx = !((uintptr_t)x & 15) && ldx % 8 == 0;
  const hipError_t e = launch_rows<1, false>(st, x, ldx, vecx, nullptr, nullptr, wc, ws, K, act,
                                             epi(bias, R, ldr, r_rows, C, ldc, M, N, act_from));
  return e == hipSuccess ? MX_OK : MX_ELAUNCH;
}

extern "C" int mx_gemm_mxfp4(hipStream_t st, const uint8_t* xc, const uint8_t* xs, const uint8_t* wc, const uint8_t* ws,
                             const float* bias, const uint16_t* R, long ldr, int r_rows, uint16_t* C, long ldc, int M,
                             int N, int K, int act, int act_from) {
  if (!xc || !xs) return MX_ENULL;
  const int rc = check(wc, ws, bias, R, ldr, r_rows, C, ldc, M, N, K, act, act_from);
  if (rc) return rc;
  if (((uintptr_t)xc & 15) || ((uintptr_t)xs & 3)) return MX_ELAYOUT;
  const Mx4Epi p = epi(bias, R, ldr, r_rows, C, ldc, M, N, act_from);
  hipError_t e;
  if (M <= 16) {
    e = launch_rows<1, true>(st, nullptr, 0, 0, xc, xs, wc, ws, K, act, p);
  } else if (M <= 32) {
    e = launch_rows<2, true>(st, nullptr, 0, 0, xc, xs, wc, ws, K, act, p);
  } else if (M <= 64) {
    e = launch_rows<4, true>(st, nullptr, 0, 0, xc, xs, wc, ws, K, act, p);
  } else {
    const long tm = (M + 127) / 128, tn = (N + 127) / 128;
    if (tm * tn > 0xffffffL) return MX_ESHAPE;  // 2^32 threads in a grid
    auto go = [&](auto kern) {
      hipLaunchKernelGGL(kern, dim3((unsigned)(tm * tn)), dim3(256), 0, st, xc, (const uint32_t*)xs, wc,
                         (const uint32_t*)ws, K, p, (int)tn);
      return hipGetLastError();
    };
    e = act == 0 ? go(mx4_tile_kernel<0>) : act == 1 ? go(mx4_tile_kernel<1>) : go(mx4_tile_kernel<2>);
  }
  return e == hipSuccess ? MX_OK : MX_ELAUNCH;
}
