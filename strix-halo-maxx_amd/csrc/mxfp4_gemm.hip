// MXFP4 Linear: C[m, n] = act(sum_k Xq[m, k] Wq[n, k] + b[n]) + R[m, n], both operands in MXFP4 (mxfp4.h), on the
// scaled MFMA, which multiplies every block's product by both scales itself. The sum, the bias, the activation
// and the residual stay in fp32; the one rounding is the store to bf16.
#include "mxfp4.h"

#include <algorithm>
#include <type_traits>
#include <utility>

namespace {

constexpr int GEMV_ROWS = 8;  // rows that the bf16 form takes

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

// LayerNorm of the one row of x before its quantisation.
struct Mx4Ln {
  const uint16_t *gamma, *beta;
  float eps;
};
// The sum over a wave in the order of wave_sum (xor 32, 16, 8, 4, 2, 1), without its round trips through LDS.
__device__ __forceinline__ float wave_sum_reg(float v) {
  v = halves_sum(v);
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  v += dpp_mov<0x128>(0.f, v);                     // row_ror 8: lane ^ 8
  v += dpp_mov<0x1b>(0.f, dpp_mov<0x141>(0.f, v));  // quad_perm [3, 2, 1, 0] of row_half_mirror: lane ^ 3 ^ 7
  v += dpp_mov<0x4e>(0.f, v);                      // lane ^ 2
  return v + dpp_mov<0xb1>(0.f, v);                // lane ^ 1
}

// ---------------------------------------------------------------------------------------------- few rows
// 16 MT rows per workgroup (grid y). It owns 16 columns of C (16 rows of W); its waves take the groups of 512 columns of K in
// turn (4 KB of W each, read in one piece) and their sums meet in LDS. PRE = false: x arrives in bf16, XR rows at most (XV: K
// is a multiple of 8, whole 16-byte loads), and each wave quantises the 512 columns it multiplies (its own slice: no wave waits
// for another before the end). The bound is the fetch of W from HBM behind one latency: us for 1 / 8 / 16 / 64 rows, weights
// not in any cache, 2048 x 10240 5.7 / 9.4 / 6.6 / 10.0 (11 MB; 9.9 / 13.3 / 9.9 / 14.7 with branches around the loads, which
// then wait for each other), 8192 x 2048 4.8 / 6.3 / 4.9 / 6.5, 768 x 768 2.8 / 4.1 / 2.9 / 3.8 (a launch alone takes about
// 2). With 8 rows the quantisation, which every workgroup repeats, takes the time.
// LN (one row of at most 512 NW columns): the row is normalised first, in layernorm_kernel's arithmetic and order. Every wave
// takes the row's sums, whose lanes hold the columns that they hold there, and normalises the 512 that it multiplies, while
// its part of W is on the way: us in one launch / two, weights from HBM, 14336 x 2048 8.6 / 9.2, 8192 x 2048 6.3 / 7.8, 4304
// x 1152 4.7 / 6.1 (every workgroup repeats the norm, so a wider W gains less).
template <int NW, int MT, bool PRE, int XR, bool XV, bool LN, int ACT>
__global__ __launch_bounds__(64 * NW) void mx4_rows_kernel(const uint16_t* __restrict__ x, long ldx,
                                                           const uint8_t* __restrict__ xc,
                                                           const uint32_t* __restrict__ xs,
                                                           const uint8_t* __restrict__ wc,
                                                           const uint32_t* __restrict__ ws, int K, Mx4Epi p, Mx4Ln ln) {
  static_assert(PRE || MT == 1, "bf16 rows come in one tile");
  static_assert(!LN || (!PRE && XR == 1 && XV), "one row is normalised");
  __shared__ __attribute__((aligned(16))) uint32_t xq[PRE ? 1 : NW][XR][64];  // a row's codes of the wave's columns
  __shared__ __attribute__((aligned(16))) uint8_t xsc[PRE ? 1 : NW][XR][16];  // its scale bytes, [block % 4][step]
  __shared__ f32x4 red[NW][MT][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int nk = mx4_nk(K), nks = (nk + 3) / 4;
  const long nt = blockIdx.x;
  const int mt = blockIdx.y * MT;  // first row tile
  const int r16 = lane & 15, g = lane >> 4;
  // The 16 rows of tile u in the operand order of the 16x16x128 MFMA: half u & 1 of row tile u / 2, lane (r16, g) the 16
  // bytes of block g & 1 of column tile g / 2; its scale byte 2 ((u / 2) & 1) + g / 2 of dword lane 32 (g & 1) + row.
  auto codes = [&](const uint8_t* c, long u) {
    return c + ((u >> 1) * 2 * nk + (g >> 1)) * 1024 + (32 * (g & 1) + 16 * (u & 1) + r16) * 16;
  };
  auto scale = [&](const uint32_t* s, long u, int k) {
    return (int)(s[((u >> 2) * nk + k) * 64 + 32 * (g & 1) + 16 * (u & 1) + r16] >> (16 * ((u >> 1) & 1) + 8 * (g >> 1)));
  };
  f32x4 acc[MT];
#pragma unroll
  for (int i = 0; i < MT; i++) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  // What a step reads. The loads have no branches (past the end they repeat the last place and x counts as zero), so the
  // compiler can count them: the next step's are in flight while this one's are multiplied.
  struct Step {
    u32x4 w[4], x[PRE ? MT : 1][PRE ? 4 : XR];  // W; x: its codes, or its rows in bf16
    int sw[4], sx[PRE ? MT : 1][4];
    u32x4 row[LN ? NW : 1], gamma, beta;
  };
  auto fetch = [&](Step& q, int ks) {
    const int left = nk - 4 * ks;
    if constexpr (LN) {
#pragma unroll
      for (int i = 0; i < NW; i++)
        q.row[i] = *reinterpret_cast<const u32x4_any*>(x + min(i * 512 + lane * 8, K - 8));
      const int k = min(ks * 512 + lane * 8, K - 8);
      q.gamma = *reinterpret_cast<const u32x4_any*>(ln.gamma + k);
      q.beta = *reinterpret_cast<const u32x4_any*>(ln.beta + k);
    }
    const uint8_t* wt = codes(wc, nt) + (long)ks * 8192;
#pragma unroll
    for (int t = 0; t < 4; t++) {
      const int u = min(t, left - 1);
      q.w[t] = *reinterpret_cast<const u32x4*>(wt + u * 2048);
      q.sw[t] = scale(ws, nt, 4 * ks + u);
    }
    if constexpr (PRE) {
#pragma unroll
      for (int i = 0; i < MT; i++) {
        const int ut = min(mt + i, (p.M - 1) / 16);
        const uint8_t* xt = codes(xc, ut) + (long)ks * 8192;
#pragma unroll
        for (int t = 0; t < 4; t++) {
          const int u = min(t, left - 1);
          q.x[i][t] = *reinterpret_cast<const u32x4*>(xt + u * 2048);
          q.sx[i][t] = scale(xs, ut, 4 * ks + u);
        }
      }
    } else if constexpr (!LN) {
      const int k = ks * 512 + lane * 8;
#pragma unroll
      for (int m = 0; m < XR; m++) {
        const uint16_t* row = x + min(m, p.M - 1) * ldx;
        if constexpr (XV)
          q.x[0][m] = *reinterpret_cast<const u32x4_any*>(row + min(k, K - 8));
        else
          q.x[0][m] = load8(row, k, K);
      }
    }
  };
  auto normalise = [&](Step& q, int ks) {
    float s = 0.f, ss = 0.f;
#pragma unroll
    for (int i = 0; i < NW; i++) {
      const bool on = i * 512 + lane * 8 < K;
#pragma unroll
      for (int e = 0; e < 4; e++) {
        s += on ? lo_bf(q.row[i][e]) : 0.f;
        s += on ? hi_bf(q.row[i][e]) : 0.f;
      }
    }
    const float mean = wave_sum_reg(s) / (float)K;
#pragma unroll
    for (int i = 0; i < NW; i++) {
      const bool on = i * 512 + lane * 8 < K;
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const float a = lo_bf(q.row[i][e]) - mean, b = hi_bf(q.row[i][e]) - mean;
        ss += on ? a * a : 0.f;
        ss += on ? b * b : 0.f;
      }
    }
    const float rstd = 1.0f / sqrtf(wave_sum_reg(ss) / (float)K + ln.eps);
    u32x4 own = q.row[0];
#pragma unroll
    for (int i = 1; i < NW; i++) own = ks == i ? q.row[i] : own;
#pragma unroll
    for (int e = 0; e < 4; e++)
      q.x[0][0][e] = pack2((lo_bf(own[e]) - mean) * rstd * lo_bf(q.gamma[e]) + lo_bf(q.beta[e]),
                           (hi_bf(own[e]) - mean) * rstd * hi_bf(q.gamma[e]) + hi_bf(q.beta[e]));
  };
  auto multiply = [&](Step& q, int ks) {
    if constexpr (LN) normalise(q, ks);
    const int left = nk - 4 * ks;
    const u32x4 none = {0u, 0u, 0u, 0u};
    if constexpr (PRE) {
#pragma unroll
      for (int t = 0; t < 4; t++)
#pragma unroll
        for (int i = 0; i < MT; i++)
          acc[i] = mfma_mx4(q.w[t], t < left ? q.x[i][t] : none, acc[i], q.sw[t], t < left ? q.sx[i][t] : 0);
    } else {
      const int blk = lane >> 2, k = ks * 512 + lane * 8;
#pragma unroll
      for (int m = 0; m < XR; m++) {
        const u32x4 v = k < K ? q.x[0][m] : none;
        const uint32_t byte = mx4_scale_byte(quad_max(amax8(v)));
        xq[wave][m][lane] = byte == 255u ? 0u : mx4_pack8(v, e8m0_float(byte));
        if ((lane & 3) == 0) xsc[wave][m][(blk & 3) * 4 + (blk >> 2)] = (uint8_t)byte;
      }
      // the wave reads only what it wrote: in order, once its LDS writes are done
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_wave_barrier();
      const int r = min(r16, XR - 1);  // rows of the operand past XR meet no result that is stored
      const uint32_t s4 = *reinterpret_cast<const uint32_t*>(&xsc[wave][r][g * 4]);
      u32x4 b[4];
#pragma unroll
      for (int t = 0; t < 4; t++) b[t] = *reinterpret_cast<const u32x4*>(&xq[wave][r][(4 * t + g) * 4]);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int t = 0; t < 4; t++) acc[0] = mfma_mx4(q.w[t], b[t], acc[0], q.sw[t], (int)(s4 >> (8 * t)));
    }
  };
  if (wave < nks) {
    Step cur;
    fetch(cur, wave);
    int ks = wave;
    for (; ks + NW < nks; ks += NW) {
      if constexpr (MT == 1) {
        Step nxt;
        fetch(nxt, ks + NW);
        multiply(cur, ks);
        cur = nxt;
      } else {  // (the registers of two steps would not fit)
        multiply(cur, ks);
        fetch(cur, ks + NW);
      }
    }
    multiply(cur, ks);
  }
#pragma unroll
  for (int i = 0; i < MT; i++) red[wave][i][lane] = acc[i];
  __syncthreads();
  for (int i = wave; i < MT; i += NW) {
    f32x4 s = red[0][i][lane];
#pragma unroll
    for (int u = 1; u < NW; u++) s += red[u][i][lane];
    mx4_store<ACT>(p, 16 * (mt + i) + r16, (int)nt * 16 + 4 * g, s);
  }
}

// ---------------------------------------------------------------------------------------------- tiles
// 64 lanes x 16 bytes through a buffer resource (byte offset per lane; lanes outside the resource read zeros) into LDS at
// lds + LO + 16 * lane.
template <int LO>
__device__ __forceinline__ void dma16r(u32x4 rsrc, uint32_t voff, uint32_t lds) {
  asm volatile("s_add_u32 m0, %2, %3\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(voff), "s"(rsrc), "s"(lds),
               "n"(LO)
               : "memory", "m0", "scc");
}
__device__ __forceinline__ u32x4 resource(const void* base, long bytes) {
  const uint64_t u = (uint64_t)(uintptr_t)base;
  return u32x4{(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)u),
               (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(u >> 32) & 0xffffu),
               (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(bytes < 0x7ffffff0L ? bytes : 0x7ffffff0L)), 0x00020000u};
}

// 64 FB rows of x against 64 FA rows of W per tile, 4 waves (2 x 2), each 32 FB x 32 FA of it in registers; persistent
// workgroups. A step is 128 columns: two column tiles of every row tile and one dword of scales per 64 rows. The LDS ring
// holds S steps, copied by the asynchronous LDS-DMA load, across the end of a tile into the next one. Two sets of operand
// registers take turns, one multiplied while the other is read. Between the two halves of a step lies its only barrier:
// the next step has landed, and this one's slot, all read, is refilled. The loop has no branch around its products (the
// compiler would move them over it, to the end): the loads' tile changes by selection.
template <int FA, int FB, int S, int GM, int ACT, bool VEC>
__global__ __launch_bounds__(256, FA * FB > 8 ? 1 : 2) void mx4_ring_kernel(const uint8_t* __restrict__ xc,
                                                                          const uint8_t* __restrict__ xs,
                                                                          const uint8_t* __restrict__ wc,
                                                                          const uint8_t* __restrict__ ws, int K, Mx4Epi p,
                                                                          int tiles_m, int tiles_n) {
  constexpr int XB = FB * 4096, WB = FA * 4096;  // a step's codes
  constexpr int SI = (FA + FB + 3) / 4;          // load instructions of scales: 4 groups each, one by each of SI waves
  constexpr int STG = XB + WB + SI * 1024;
  constexpr int LPS = FA + FB;                   // load instructions of codes per wave and step
  constexpr int NST = VEC ? 2 * FA * FB : 0;
  constexpr int GA = (FA + 1) / 2, GB = (FB + 1) / 2;  // scale registers
  static_assert((S - 2) * (LPS + 1) + NST <= 63 && S * STG + 2048 <= 160 * 1024 && FA <= 4, "schedule");
  __shared__ __attribute__((aligned(1024))) uint8_t smem[S * STG + 2048];  // the ring, two bias rows
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave & 1, wn = wave >> 1;
  const uint32_t sbase = lds_off(smem);
  const int nk = mx4_nk(K);  // > S (the caller)
  const int mrt = (p.M + 31) / 32, nrt = (p.N + 31) / 32;

  // this workgroup's tiles: XCD x (= block % 8) owns a contiguous run of the tile sequence, its workgroups take the
  // run's tiles in turn
  const int nt = tiles_m * tiles_n, nx = min(8, (int)gridDim.x);
  const int xcd = blockIdx.x % nx, stride = ((int)gridDim.x - xcd + nx - 1) / nx;
  const int per = nt / nx, rem = nt % nx;
  const int run0 = xcd * per + min(xcd, rem), run1 = run0 + per + (xcd < rem ? 1 : 0);
  const int t0 = run0 + (int)blockIdx.x / nx;
  if (t0 >= run1) return;
  auto origin = [&](int t, int& mt, int& ntl) {  // row groups of GM tiles, column-major inside a group
    const int grp = t / (GM * tiles_n), first = grp * GM, gs = min(tiles_m - first, GM);
    const int r = t - grp * GM * tiles_n;
    mt = first + r % gs;
    ntl = r / gs;
  };

  // ---- what is loaded next: step pk of the tile that rx, rw, psc describe; n*: the tile after it (past the last tile it
  // repeats that tile: the loads keep the counts of the waits true)
  struct Src {
    u32x4 x, w;
    const uint8_t* sc;  // this lane's 16 bytes of scales of the tile's first step
  };
  const int piece = min(min(wave, SI - 1) * 4 + (lane >> 4), FA + FB - 1);
  auto aim = [&](int t) {
    int mt, ntl;
    origin(t, mt, ntl);
    Src s;
    s.x = resource(xc + (long)mt * (2 * FB) * nk * 2048, (long)(mrt - mt * 2 * FB) * nk * 2048);
    s.w = resource(wc + (long)ntl * (2 * FA) * nk * 2048, (long)(nrt - ntl * 2 * FA) * nk * 2048);
    const bool isx = piece < FB;
    const long grp = isx ? min((long)mt * FB + piece, (mrt - 1L) / 2) : min((long)ntl * FA + piece - FB, (nrt - 1L) / 2);
    s.sc = (isx ? xs : ws) + grp * nk * 256 + (lane & 15) * 16;
    return s;
  };
  Src src = aim(t0), nxt = aim(min(t0 + stride, run1 - 1));
  int pk = 0;
  uint32_t pdst = sbase;
  const uint32_t rs = (uint32_t)nk * 2048;  // a row tile's codes
  // instruction q = wave F + e of an operand: 1 KB, column tile q & 1 of row tile q / 2
  const uint32_t vx = lane * 16 + (wave * FB / 2) * rs + (wave * FB % 2) * 1024;
  const uint32_t vw = lane * 16 + (wave * FA / 2) * rs + (wave * FA % 2) * 1024;
  auto load = [&](auto ec) {
    constexpr int e = decltype(ec)::value, f = e < FB ? FB : FA, i = e < FB ? e : e - FB;
    // the wave's first instruction may be the second half of a row tile (odd f)
    const uint32_t step = f % 2 == 0 ? (i / 2) * rs + (i % 2) * 1024
                                     : (uint32_t)((wave * f + i) / 2 - wave * f / 2) * rs + (uint32_t)((wave * f + i) % 2 - wave * f % 2) * 1024;
    dma16r<e < FB ? 0 : XB>(e < FB ? src.x : src.w, (e < FB ? vx : vw) + (uint32_t)pk * 2048 + step, pdst + (wave * f + i) * 1024);
  };
  auto load_scales = [&]() {  // every wave (one count for the waits): those past SI repeat the last
    dma16(src.sc + (long)pk * 256, pdst + XB + WB + min(wave, SI - 1) * 1024);
  };
  auto next = [&]() {
    pdst = pdst == sbase + (S - 1) * STG ? sbase : pdst + STG;
    const bool wrap = ++pk == nk;
    pk = wrap ? 0 : pk;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      src.x[e] = wrap ? nxt.x[e] : src.x[e];
      src.w[e] = wrap ? nxt.w[e] : src.w[e];
    }
    src.sc = wrap ? nxt.sc : src.sc;
  };

  f32x16 acc[FA][FB];
  u32x4 a[2][FA], b[2][FB];
  int sa[GA], sb[GB], na[GA], nb[GB];
  const uint8_t* xb = smem + wm * FB * 2048 + lane * 16;
  const uint8_t* wb = smem + XB + wn * FA * 2048 + lane * 16;
  const uint8_t* scb = smem + XB + WB + lane * 4;
  auto ld = [](const uint8_t* q) { return *reinterpret_cast<const u32x4*>(q); };
  // scale dwords in the slot at so; a wave with one row tile takes the half of its group that is its own
  auto scale_a = [&](uint32_t so, int i) {
    const int v = *reinterpret_cast<const int*>(scb + so + (FB + (FA == 1 ? 0 : wn * GA + i)) * 256);
    return FA == 1 ? v >> (16 * wn) : v;
  };
  auto scale_b = [&](uint32_t so, int j) {
    const int v = *reinterpret_cast<const int*>(scb + so + (FB == 1 ? 0 : wm * GB + j) * 256);
    return FB == 1 ? v >> (16 * wm) : v;
  };
  static_assert(FA == 1 || FA % 2 == 0, "a wave's rows of W start with a scale group");
  static_assert(FB == 1 || FB % 2 == 0, "a wave's rows of x start with a scale group");

  int after = 0;     // waits left whose counts include the write-out's stores
  uint32_t cur = 0;  // slot of the step being multiplied
  auto step = [&](auto firstc) {  // FIRST: the sums start at 0
    constexpr bool FIRST = decltype(firstc)::value;
    constexpr int NM = FA * FB;
    // ---- first half: set 0, while set 1 is read
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < FA; i++)
#pragma unroll
      for (int j = 0; j < FB; j++) {
        f32x16 z = acc[i][j];
        if (FIRST)
#pragma unroll
          for (int e = 0; e < 16; e++) z[e] = 0.f;
        acc[i][j] = (i & 1) ? ((j & 1) ? mfma_mx4<2, 2>(a[0][i], b[0][j], z, sa[i / 2], sb[j / 2])
                                       : mfma_mx4<2, 0>(a[0][i], b[0][j], z, sa[i / 2], sb[j / 2]))
                            : ((j & 1) ? mfma_mx4<0, 2>(a[0][i], b[0][j], z, sa[i / 2], sb[j / 2])
                                       : mfma_mx4<0, 0>(a[0][i], b[0][j], z, sa[i / 2], sb[j / 2]));
        __builtin_amdgcn_sched_barrier(0);
        if (j == 0) a[1][i] = ld(wb + cur + (2 * i + 1) * 1024);
        if (i == 0) b[1][j] = ld(xb + cur + (2 * j + 1) * 1024);
        __builtin_amdgcn_sched_barrier(0);
      }
    // ---- second half: set 1, while set 0 of the next step is read and the slot refilled
    if (after > 0) {
      after--;
      wait_vm<(S - 2) * (LPS + 1) + NST>();
    } else {
      wait_vm<(S - 2) * (LPS + 1)>();
    }
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    cur = cur == (S - 1) * STG ? 0 : cur + STG;
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < FA; i++)
#pragma unroll
      for (int j = 0; j < FB; j++) {
        acc[i][j] = (i & 1) ? ((j & 1) ? mfma_mx4<3, 3>(a[1][i], b[1][j], acc[i][j], sa[i / 2], sb[j / 2])
                                       : mfma_mx4<3, 1>(a[1][i], b[1][j], acc[i][j], sa[i / 2], sb[j / 2]))
                            : ((j & 1) ? mfma_mx4<1, 3>(a[1][i], b[1][j], acc[i][j], sa[i / 2], sb[j / 2])
                                       : mfma_mx4<1, 1>(a[1][i], b[1][j], acc[i][j], sa[i / 2], sb[j / 2]));
        __builtin_amdgcn_sched_barrier(0);
        if (j == 0) {
          a[0][i] = ld(wb + cur + 2 * i * 1024);
          if (i % 2 == 0) na[i / 2] = scale_a(cur, i / 2);
        }
        if (i == 0) {
          b[0][j] = ld(xb + cur + 2 * j * 1024);
          if (j % 2 == 0) nb[j / 2] = scale_b(cur, j / 2);
        }
        if (i + j == 0) load_scales();
        [&]<int... e>(std::integer_sequence<int, e...>) {
          ((e * NM / LPS == i * FB + j ? load(std::integral_constant<int, e>{}) : void()), ...);
        }(std::make_integer_sequence<int, LPS>{});
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
    for (int i = 0; i < GA; i++) sa[i] = na[i];
#pragma unroll
    for (int j = 0; j < GB; j++) sb[j] = nb[j];
    next();
  };

  // ---- prologue
#pragma unroll
  for (int i = 0; i < S; i++) {
    load_scales();
    [&]<int... e>(std::integer_sequence<int, e...>) { (load(std::integral_constant<int, e>{}), ...); }
    (std::make_integer_sequence<int, LPS>{});
    next();
  }
  wait_vm<(S - 1) * (LPS + 1)>();
  __syncthreads();
#pragma unroll
  for (int i = 0; i < FA; i++) a[0][i] = ld(wb + 2 * i * 1024);
#pragma unroll
  for (int j = 0; j < FB; j++) b[0][j] = ld(xb + 2 * j * 1024);
#pragma unroll
  for (int i = 0; i < GA; i++) sa[i] = scale_a(0, i);
#pragma unroll
  for (int j = 0; j < GB; j++) sb[j] = scale_b(0, j);

  int brow = 0;
  for (int t = t0; t < run1; t += stride) {
    int mt0, nt0;
    origin(t, mt0, nt0);
    const int m0 = mt0 * 64 * FB, n0 = nt0 * 64 * FA, mw = wm * FB * 32, nw = wn * FA * 32;
    if (VEC && p.bias && wave == 0)  // read after nk > S steps, whose waits and barriers cover it
      dma16s(p.bias, (uint32_t)min(n0 + 4 * lane, p.N - 4) * 4, sbase + S * STG + brow * 1024);
    step(std::true_type{});
    for (int k = 1; k < nk; k++) step(std::false_type{});
    // the loads have gone on to the next tile (nk > S steps ago they were at most S ahead): the one after it
    nxt = aim(min(t + 2 * stride, run1 - 1));

    int ln = lane;
    asm volatile("" : "+v"(ln));  // the lane's addresses are computed here, per tile: hoisted they would take registers
    const int lr = ln & 31, hk = ln >> 5;
    if constexpr (VEC) {
      // A lane holds 4 columns in a row at 8 u + 4 hk, the lane 32 further the other 4 of the 8: a swap of halves between u
      // and u + 1 leaves 8 in a row in every lane. Stores go through a buffer resource, always the same number of them.
      const long cb = ((long)(p.M - m0 - 1) * p.ldc + p.N - n0) * 2, rb = p.R ? ((long)(p.M - m0 - 1) * p.ldr + p.N - n0) * 2 : 0;
      const __amdgpu_buffer_rsrc_t rc = __builtin_amdgcn_make_buffer_rsrc(p.C + (long)m0 * p.ldc + n0, (short)0,
                                                                          (int)(cb < 0x7ffffff0L ? cb : 0x7ffffff0L), 0x00020000);
      const __amdgpu_buffer_rsrc_t rr = __builtin_amdgcn_make_buffer_rsrc(
          const_cast<uint16_t*>(p.R ? p.R + (long)m0 * p.ldr + n0 : nullptr), (short)0,
          (int)(rb < 0x7ffffff0L ? rb : 0x7ffffff0L), 0x00020000);
      // Unit q: row tile q / 2, columns 16 (q & 1) .. + 15. The residuals are loaded units ahead: memory operations finish in
      // order, so a load behind a unit's stores would wait for them.
      constexpr int NU = 2 * FA, RD = NU < 4 ? NU : 4;
      u32x4 res[RD][FB];
      auto column = [&](int q) { return nw + 32 * (q >> 1) + 16 * (q & 1) + 8 * hk; };  // of the lane's stores
      auto row = [&](int j) { return mw + 32 * j + lr; };
      auto fetch = [&](int q) {
#pragma unroll
        for (int j = 0; j < FB; j++)
          res[q % RD][j] = __builtin_bit_cast(
              u32x4, __builtin_amdgcn_raw_buffer_load_b128(
                         rr, n0 + column(q) < p.N ? (uint32_t)(row(j) * (int)p.ldr + column(q)) * 2 : 0x80000000u, 0, 0));
      };
      const uint8_t* brp = smem + S * STG + brow * 1024 + (nw + 4 * hk) * 4;
      brow ^= 1;
      if (p.R)
#pragma unroll
        for (int q = 0; q < RD - 1; q++) fetch(q);
#pragma unroll
      for (int q = 0; q < NU; q++) {
        if (p.R && q + RD - 1 < NU) fetch(q + RD - 1);
        f32x4 bias[2];
#pragma unroll
        for (int v = 0; v < 2; v++)
          bias[v] = p.bias ? *reinterpret_cast<const f32x4*>(brp + (32 * (q >> 1) + 16 * (q & 1) + 8 * v) * 4)
                           : f32x4{0.f, 0.f, 0.f, 0.f};
        const int i = q >> 1, u = 2 * (q & 1);
        const bool on = n0 + column(q) < p.N;
#pragma unroll
        for (int j = 0; j < FB; j++) {
          u32x4 r = {0u, 0u, 0u, 0u};
          if (p.R) {
            r = res[q % RD][j];
#pragma unroll
            for (int e = 0; e < 2; e++) {
              const auto w = __builtin_amdgcn_permlane32_swap(r[e], r[2 + e], false, false);
              r[e] = w[0], r[2 + e] = w[1];
            }
          }
          uint32_t o[2][2];
#pragma unroll
          for (int v = 0; v < 2; v++) {
            float y[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
              y[e] = acc[i][j][4 * (u + v) + e] + bias[v][e];
              if (ACT && n0 + nw + 32 * i + 8 * (u + v) + 4 * hk + e >= p.act_from)
                y[e] = ACT == 1 ? gelu_tanh(y[e]) : gelu_erf(y[e]);
              if (p.R) y[e] += (e & 1) ? hi_bf(r[2 * v + (e >> 1)]) : lo_bf(r[2 * v + (e >> 1)]);
            }
            o[v][0] = pack2(y[0], y[1]), o[v][1] = pack2(y[2], y[3]);
          }
          const auto x = __builtin_amdgcn_permlane32_swap(o[0][0], o[1][0], false, false);
          const auto z = __builtin_amdgcn_permlane32_swap(o[0][1], o[1][1], false, false);
          __builtin_amdgcn_raw_buffer_store_b128(u32x4{x[0], z[0], x[1], z[1]}, rc,
                                                 on ? (uint32_t)(row(j) * (int)p.ldc + column(q)) * 2 : 0x80000000u, 0, 0);
        }
      }
      after = S - 1;
    } else {
#pragma unroll
      for (int i = 0; i < FA; i++)
#pragma unroll
        for (int j = 0; j < FB; j++)
#pragma unroll
          for (int u = 0; u < 4; u++)
            mx4_store<ACT>(p, m0 + mw + 32 * j + lr, n0 + nw + 32 * i + 8 * u + 4 * hk,
                           f32x4{acc[i][j][4 * u], acc[i][j][4 * u + 1], acc[i][j][4 * u + 2], acc[i][j][4 * u + 3]});
    }
  }
  wait_vm<0>();  // the loads past the last tile land before the workgroup's LDS is given away
}

template <int FA, int FB, int S, int GM>
hipError_t launch_ring(hipStream_t st, const uint8_t* xc, const uint8_t* xs, const uint8_t* wc, const uint8_t* ws, int K,
                       int act, const Mx4Epi& p) {
  const long tm = ((long)p.M + 64 * FB - 1) / (64 * FB), tn = ((long)p.N + 64 * FA - 1) / (64 * FA), nt = tm * tn;
  int dev = 0, cus = 0;
  hipError_t e = hipGetDevice(&dev);
  if (e == hipSuccess) e = hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev);
  if (e != hipSuccess) return e;
  constexpr int lds = S * ((FA + FB) * 4096 + (FA + FB + 3) / 4 * 1024) + 2048;
  const long most = (long)cus * std::min(FA * FB > 8 ? 1 : FA * FB > 4 ? 2 : 3, 160 * 1024 / lds);
  if (nt > 0x3fffffffL) return hipErrorInvalidValue;
  const dim3 grid((unsigned)(nt < most ? nt : most));
  auto go = [&](auto kern) {
    hipLaunchKernelGGL(kern, grid, dim3(256), 0, st, xc, xs, wc, ws, K, p, (int)tm, (int)tn);
    return hipGetLastError();
  };
  // 16-byte accesses to whole chunks of 8 columns at 32-bit offsets
  const bool vec = p.N % 8 == 0 && p.ldc % 8 == 0 && !((uintptr_t)p.C & 15) && p.ldc < (1L << 21) && p.r_rows == 0 &&
                   (!p.R || (p.ldr % 8 == 0 && !((uintptr_t)p.R & 15) && p.ldr < (1L << 21))) && !((uintptr_t)p.bias & 15);
  if (vec)
    return act == 0   ? go(mx4_ring_kernel<FA, FB, S, GM, 0, true>)
           : act == 1 ? go(mx4_ring_kernel<FA, FB, S, GM, 1, true>)
                      : go(mx4_ring_kernel<FA, FB, S, GM, 2, true>);
  return act == 0   ? go(mx4_ring_kernel<FA, FB, S, GM, 0, false>)
         : act == 1 ? go(mx4_ring_kernel<FA, FB, S, GM, 1, false>)
                    : go(mx4_ring_kernel<FA, FB, S, GM, 2, false>);
}

int check(const void* wc, const void* ws, const float* bias, const uint16_t* R, long ldr, int r_rows, const uint16_t* C,
          long ldc, int M, int N, int K, int act, int act_from) {
  if (!wc || !ws || !C) return MX_ENULL;
  if (act < 0 || act > 2) return MX_EBADCFG;
  if (M < 1 || N < 1 || K < 1 || act_from < 0 || r_rows < 0 || (M > 1 && ldc < N)) return MX_ESHAPE;
  if (N > 1 << 27) return MX_ESHAPE;  // few rows: 16 columns a workgroup of up to 512 threads, 2^32 threads in a grid
  if (R && ldr < 0) return MX_ESHAPE;
  if ((((uintptr_t)wc) & 15) || ((uintptr_t)ws & 3) || ((uintptr_t)bias & 3) || ((uintptr_t)R & 1) || ((uintptr_t)C & 1))
    return MX_ELAYOUT;
  return MX_OK;
}

Mx4Epi epi(const float* bias, const uint16_t* R, long ldr, int r_rows, uint16_t* C, long ldc, int M, int N, int act_from) {
  const bool vec = N % 4 == 0 && !((uintptr_t)C & 7) && ldc % 4 == 0 && (!R || (!((uintptr_t)R & 7) && ldr % 4 == 0));
  return Mx4Epi{bias, R, ldr, r_rows, C, ldc, M, N, act_from, vec};
}

template <int MT, bool PRE, int XR, bool XV>
hipError_t launch_rows(hipStream_t st, const uint16_t* x, long ldx, const uint8_t* xc, const uint8_t* xs, const uint8_t* wc,
                       const uint8_t* ws, int K, int act, const Mx4Epi& p) {
  const dim3 grid((unsigned)((p.N + 15L) / 16), (unsigned)((p.M + 16L * MT - 1) / (16 * MT)));
  auto go = [&](auto kern, int nw) {
    hipLaunchKernelGGL(kern, grid, dim3(64 * nw), 0, st, x, ldx, xc, (const uint32_t*)xs, wc, (const uint32_t*)ws, K, p,
                       Mx4Ln{});
    return hipGetLastError();
  };
  if (mx4_nk(K) <= 16) {
    if (act == 0) return go(mx4_rows_kernel<4, MT, PRE, XR, XV, false, 0>, 4);
    if (act == 1) return go(mx4_rows_kernel<4, MT, PRE, XR, XV, false, 1>, 4);
    return go(mx4_rows_kernel<4, MT, PRE, XR, XV, false, 2>, 4);
  }
  if (act == 0) return go(mx4_rows_kernel<8, MT, PRE, XR, XV, false, 0>, 8);
  if (act == 1) return go(mx4_rows_kernel<8, MT, PRE, XR, XV, false, 1>, 8);
  return go(mx4_rows_kernel<8, MT, PRE, XR, XV, false, 2>, 8);
}

// Which kernel, by the grid it makes (us on one MI355X; N x K after the rows):
//  * the few-row kernel up to 32 rows, and beyond while its grid (16 columns x 64 rows each) is at most two workgroups per
//    CU: loads alone, on all CUs, reach 50 bytes a clock and CU from the XCD's own L2 and 11 from beyond it, so the product of
//    few rows goes as fast as its weights are spread. Against tiles, weights from HBM: 2048 x 8192, 64 rows 8.8 / 17.4, 256
//    rows 14.3 / 17.2, 384 rows 19.8 / 17.5; 2048 x 2048, 256 rows 5.3 / 6.7, 384 rows 7.6 / 6.9; 64 rows, 8192 x 2048 6.5
//    / 7.6, 14336 x 2048 10.6 / 8.2;
//  * the smallest tile whose grid is at most one workgroup per CU, for the same reason (64 x 64, 64 x 128, 128 x 128,
//    128 x 256): 512 rows, 2048 x 2048 7.9 / 9.4 / 10.4 / 14.6; 256 rows, 8192 x 2048 10.5 / 10.0 / 10.8 / 14.7;
//  * 128 x 128 below two full rounds of 128 x 256: 4096 rows, 4304 x 1152 30.2 / 26.6 / 22.6 / 25.7;
//  * 128 x 256 beyond, for its fewer LDS reads per product: 9477 rows, 8192 x 2048 182 / 142 / 110 / 105; 8192^3 492 /
//    380 / 306 / 272 (289 in the median: the clock falls with the power);
//  * K up to 256: the few-row kernel (the tiles' loads run at most one tile ahead, so they need more steps than the ring has),
//    up to 512 a ring of two steps.
enum Mx4Kernel { ROWS16, ROWS32, ROWS64, SHORT128X128, RING64X64, RING64X128, RING128X128, RING128X256 };
Mx4Kernel mx4_kernel(int M, int N, int K) {
  const auto tiles = [&](int bm, int bn) { return ((long)M + bm - 1) / bm * (((long)N + bn - 1) / bn); };
  const int nk = mx4_nk(K);
  if (M <= 16) return ROWS16;
  if (M <= 32) return ROWS32;
  if (tiles(64, 16) <= 512 || nk <= 2) return ROWS64;
  if (nk <= 4) return SHORT128X128;
  if (tiles(64, 64) <= 256) return RING64X64;
  if (tiles(64, 128) <= 256) return RING64X128;
  return tiles(128, 256) < 1024 ? RING128X128 : RING128X256;
}

}  // namespace

// Rows that mx_gemv_mxfp4 takes.
extern "C" int mx_gemv_mxfp4_rows(void) { return GEMV_ROWS; }

extern "C" int mx_gemv_mxfp4(hipStream_t st, const uint16_t* x, long ldx, const uint8_t* wc, const uint8_t* ws,
                             const float* bias, const uint16_t* R, long ldr, int r_rows, uint16_t* C, long ldc, int M,
                             int N, int K, int act, int act_from) {
  if (!x) return MX_ENULL;
  const int rc = check(wc, ws, bias, R, ldr, r_rows, C, ldc, M, N, K, act, act_from);
  if (rc) return rc;
  if (M > GEMV_ROWS || ldx < 0) return MX_ESHAPE;
  if ((uintptr_t)x & 1) return MX_ELAYOUT;
  const bool vec = K % 8 == 0;
  const Mx4Epi p = epi(bias, R, ldr, r_rows, C, ldc, M, N, act_from);
  auto go = [&](auto launch) { return launch(st, x, ldx, nullptr, nullptr, wc, ws, K, act, p); };
  const hipError_t e = !vec     ? go(launch_rows<1, false, GEMV_ROWS, false>)
                       : M == 1 ? go(launch_rows<1, false, 1, true>)
                       : M <= 4 ? go(launch_rows<1, false, 4, true>)
                                : go(launch_rows<1, false, GEMV_ROWS, true>);
  return e == hipSuccess ? MX_OK : MX_ELAUNCH;
}

// Widest row that mx_ln_gemv_mxfp4 takes: four waves' 512 columns.
extern "C" int mx_ln_gemv_mxfp4_cols(void) { return 2048; }

extern "C" int mx_ln_gemv_mxfp4(hipStream_t st, const uint16_t* x, const uint16_t* gamma, const uint16_t* beta, float eps,
                                const uint8_t* wc, const uint8_t* ws, const float* bias, uint16_t* C, int N, int K, int act,
                                int act_from) {
  if (!x || !gamma || !beta) return MX_ENULL;
  const int rc = check(wc, ws, bias, nullptr, 0, 0, C, N, 1, N, K, act, act_from);
  if (rc) return rc;
  if (K % 8 || K > 2048) return MX_ESHAPE;
  if (((uintptr_t)x | (uintptr_t)gamma | (uintptr_t)beta) & 1) return MX_ELAYOUT;
  const dim3 grid((unsigned)((N + 15L) / 16));
  const Mx4Epi p = epi(bias, nullptr, 0, 0, C, N, 1, N, act_from);
  auto go = [&](auto kern) {
    hipLaunchKernelGGL(kern, grid, dim3(256), 0, st, x, 0L, nullptr, nullptr, wc, (const uint32_t*)ws, K, p,
                       Mx4Ln{gamma, beta, eps});
    return hipGetLastError();
  };
  const hipError_t e = act == 0   ? go(mx4_rows_kernel<4, 1, false, 1, true, true, 0>)
                       : act == 1 ? go(mx4_rows_kernel<4, 1, false, 1, true, true, 1>)
                                  : go(mx4_rows_kernel<4, 1, false, 1, true, true, 2>);
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
  if (((long)M + 63) / 64 * (((long)N + 63) / 64) > 0x3fffffffL || mx4_nk(K) > (1 << 15)) return MX_ESHAPE;
  switch (mx4_kernel(M, N, K)) {
    case ROWS16: e = launch_rows<1, true, 1, true>(st, nullptr, 0, xc, xs, wc, ws, K, act, p); break;
    case ROWS32: e = launch_rows<2, true, 1, true>(st, nullptr, 0, xc, xs, wc, ws, K, act, p); break;
    case ROWS64:
      if (M > 64 * 65535) return MX_ESHAPE;
      e = launch_rows<4, true, 1, true>(st, nullptr, 0, xc, xs, wc, ws, K, act, p);
      break;
    case SHORT128X128: e = launch_ring<2, 2, 2, 8>(st, xc, xs, wc, ws, K, act, p); break;
    case RING64X64: e = launch_ring<1, 1, 4, 8>(st, xc, xs, wc, ws, K, act, p); break;
    case RING64X128: e = launch_ring<2, 1, 4, 8>(st, xc, xs, wc, ws, K, act, p); break;
    case RING128X128: e = launch_ring<2, 2, 4, 8>(st, xc, xs, wc, ws, K, act, p); break;
    default: e = launch_ring<4, 2, 3, 8>(st, xc, xs, wc, ws, K, act, p);
  }
  return e == hipSuccess ? MX_OK : MX_ELAUNCH;
}

// The kernel that mx_gemm_mxfp4 takes: t = rows and columns of C per workgroup, steps in the LDS ring (0: the few-row kernel),
// waves per workgroup.
extern "C" void mx_gemm_mxfp4_tiling(int M, int N, int K, int* t) {
  static constexpr int shape[8][3] = {{16, 16, 0}, {32, 16, 0}, {64, 16, 0}, {128, 128, 2}, {64, 64, 4}, {64, 128, 4},
                                      {128, 128, 4}, {128, 256, 3}};
  std::fill(t, t + 4, 0);
  if (M < 1 || N < 1 || K < 1) return;
  const int k = mx4_kernel(M, N, K);
  std::copy(shape[k], shape[k] + 3, t);
  t[3] = k <= ROWS64 && mx4_nk(K) > 16 ? 8 : 4;
}
