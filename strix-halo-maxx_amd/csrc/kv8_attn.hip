// Attention over the 8-bit KV cache (kv8.h) for head dims 64 and 128, G query heads per key head:
//   O[b, i, h] = sum_j softmax_j(scale <Q[b, h, i], K[b, h / G, j]>) V[b, h / G, j]   over the visible keys j
//   key j is visible to query i of sequence b iff j < len_b and (j < causal_from or j <= qpos_b + i); a query that sees
//   no key gets zeros.
//
// The codes go from the cache into the 32x32x64 MFMA as they are; nothing is converted to bf16.
//  * S^T = K Q^T: Q is two e4m3 terms, q = 2^e (hi + lo / 16) with one exponent per row, which hold a bf16's 8 bits (what
//    falls below 2^-23 of the row's largest value is lost), so both products together are the bf16 product. The scales
//    of the K block and of Q are the MFMA's own scale operands.
//  * O^T += V^T P^T: the weights of 64 keys are two e4m3 terms too, with a power of two of their own for every query and
//    block: p = 2^(el - 8 - m) (hi + lo / 16), el the next integer above the block's largest score (base 2), m the
//    running one. Relative to the block's largest weight that keeps 2^-9 of each weight and everything above 2^-22. The
//    running maximum is an integer, so rescaling is exact. Sums of weights are taken in fp32 before that rounding.
//  * The token order inside a V block is the order in which S^T leaves its keys in a lane's registers (kv8.h).
// The fp8 MFMA adds its 64 products to the fp32 accumulator with an error of about 2^-16 of the result's size (measured:
// 1.3e-5 of the root mean square on normal data, without bias), a hundredth of the bf16 rounding of the output.
// A query wave owns 32 rows, the (query, head of the group) pairs of one key head; a lane holds one row's scores of 32 of
// the 64 keys of a block, the other 32 sit in lane ^ 32.
//
// A masked key must not reach any result: its weight is zero, but the MFMA would multiply a NaN code by it. Blocks that
// need a mask are therefore searched for NaN codes, and where there is one (never in ordinary data) the codes are cleared
// and a second product, of NaN indicators with the visibility, finds the outputs that become NaN.
#include "kv8.h"

namespace {

constexpr int M_NONE = -(1 << 30);

struct Attn8Args {
  const uint16_t* q;
  long sq_b, sq_h, sq_t;
  const uint8_t *kc, *vc, *ks, *vs;
  uint16_t* o;
  long so_b, so_t;
  float* part;
  const int* len;
  long len_s;
  int base, qpos, qend, causal_from;  // qend: queries are the last Tq positions of the sequence (qpos is not read)
  int B, H, G, Tq, ctx, nrt, splits, chunk;
  float sl2;
};

__device__ __forceinline__ f32x16 mfma8(i32x8 a, i32x8 b, f32x16 c, int sa, int sb) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, c, 0, 0, 0, sa, 0, sb);
}
__device__ __forceinline__ i32x8 join(u32x4 a, u32x4 b) {
  return i32x8{(int)a.x, (int)a.y, (int)a.z, (int)a.w, (int)b.x, (int)b.y, (int)b.z, (int)b.w};
}
// a, b, c, d (|.| <= 448) as hi + lo / 16
__device__ __forceinline__ void split4(float a, float b, float c, float d, uint32_t& hi, uint32_t& lo) {
  uint32_t h = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  h = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, h, true);
  const auto x = __builtin_amdgcn_cvt_pk_f32_fp8(h, false), y = __builtin_amdgcn_cvt_pk_f32_fp8(h, true);
  uint32_t l = __builtin_amdgcn_cvt_pk_fp8_f32((a - x[0]) * 16.f, (b - x[1]) * 16.f, 0, false);
  l = __builtin_amdgcn_cvt_pk_fp8_f32((c - y[0]) * 16.f, (d - y[1]) * 16.f, l, true);
  hi = h, lo = l;
}

// What a sequence's length and position give.
struct Seq {
  int len, qpos;
};
__device__ __forceinline__ Seq sequence(const Attn8Args& p, int b) {
  const long l = (long)p.base + (p.len ? p.len[b * p.len_s] : 0);
  Seq s;
  s.len = (int)min(max(l, 0L), (long)p.ctx);
  s.qpos = p.qend ? s.len - p.Tq : p.qpos;
  return s;
}
// keys visible to query i: 0 .. limit - 1
__device__ __forceinline__ int limit(const Attn8Args& p, const Seq& s, int i) {
  return min(s.len, max(p.causal_from, (int)min((long)s.qpos + i + 1, 0x7fffffffL)));
}

template <int D>
struct Rows {  // one query wave's 32 rows
  i32x8 qh[D / 64], ql[D / 64];
  int sqh, sql;
  f32x16 o[D / 32];
  int m;
  float l;

  __device__ __forceinline__ void load(const uint16_t* qrow, int hk) {
    u32x4 x[D / 32][2];
    uint32_t mx = 0;
#pragma unroll
    for (int j = 0; j < D / 32; j++)
#pragma unroll
      for (int u = 0; u < 2; u++) {
        x[j][u] = *reinterpret_cast<const u32x4*>(qrow + 32 * j + 16 * hk + 8 * u);
#pragma unroll
        for (int e = 0; e < 4; e++) mx = max(mx, max(x[j][u][e] & 0x7fffu, (x[j][u][e] >> 16) & 0x7fffu));
      }
    mx = (uint32_t)halves_max((float)mx);
    // scaled maximum in [128, 256); an infinity or NaN stays one and makes its row NaN, as the formula does
    const int code = max((int)(mx >> 7) - 7, 8);
    const float f = __uint_as_float((uint32_t)(254 - code) << 23);
    sqh = code, sql = code - 4;
#pragma unroll
    for (int s = 0; s < D / 64; s++)
#pragma unroll
      for (int w = 0; w < 8; w++) {  // dword w: columns 4 w .. 4 w + 3 of the lane's 32
        const u32x4 v = x[2 * s + (w >> 2)][(w >> 1) & 1];
        const uint32_t a = v[2 * (w & 1)], b = v[2 * (w & 1) + 1];
        uint32_t hi, lo;
        split4(lo_bf(a) * f, hi_bf(a) * f, lo_bf(b) * f, hi_bf(b) * f, hi, lo);
        if (mx >= 0x7f80u) hi = 0x7f7f7f7fu;
        qh[s][w] = (int)hi, ql[s][w] = (int)lo;
      }
  }
  __device__ __forceinline__ void clear() {
    m = M_NONE, l = 0.f;
#pragma unroll
    for (int t = 0; t < D / 32; t++)
#pragma unroll
      for (int e = 0; e < 16; e++) o[t][e] = 0.f;
  }
  // S^T of 64 keys, k[t][j] = group t D / 32 + j
  __device__ __forceinline__ void scores(const u32x4 (&k)[2][D / 32], int sk, f32x16 (&st)[2]) const {
#pragma unroll
    for (int t = 0; t < 2; t++) {
#pragma unroll
      for (int e = 0; e < 16; e++) st[t][e] = 0.f;
#pragma unroll
      for (int s = 0; s < D / 64; s++) st[t] = mfma8(join(k[t][2 * s], k[t][2 * s + 1]), qh[s], st[t], sk, sqh);
#pragma unroll
      for (int s = 0; s < D / 64; s++) st[t] = mfma8(join(k[t][2 * s], k[t][2 * s + 1]), ql[s], st[t], sk, sql);
    }
  }
  // Scores to weights: rescales o and l, returns the two terms of the weights and their scale. Keys >= lim (within the
  // block) are masked where MASK.
  template <bool MASK>
  __device__ __forceinline__ void weights(f32x16 (&st)[2], float sl2, int lim, int hk, i32x8& ph, i32x8& pl, int& sp) {
    float mx = -INFINITY;
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
      for (int r = 0; r < 16; r++) {
        if (MASK) {
          const int key = 32 * t + 8 * (r >> 2) + 4 * hk + (r & 3);
          st[t][r] = key < lim ? st[t][r] : -INFINITY;
        }
        mx = fmaxf(mx, st[t][r]);
      }
    mx = halves_max(mx) * sl2;
    const int el = (int)fminf(fmaxf(ceilf(mx), (float)M_NONE), (float)-M_NONE);
    const int mn = max(m, el);
    if (__any(mn != m)) {
      const float al = __builtin_amdgcn_ldexpf(1.f, m - mn);
      l *= al;
#pragma unroll
      for (int t = 0; t < D / 32; t++)
#pragma unroll
        for (int e = 0; e < 16; e++) o[t][e] *= al;
      m = mn;
    }
    const float sh = (float)(8 - el);
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < 8; w++) {
      float x[4];
#pragma unroll
      for (int e = 0; e < 4; e++) {
        x[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(st[w >> 2][4 * (w & 3) + e], sl2, sh));
        sum += x[e];
      }
      uint32_t hi, lo;
      split4(x[0], x[1], x[2], x[3], hi, lo);
      ph[w] = (int)hi, pl[w] = (int)lo;
    }
    l += __builtin_amdgcn_ldexpf(halves_sum(sum), el - 8 - mn);
    sp = max(127 + max(el - mn, -240) - 8, 4);
  }
  __device__ __forceinline__ void add(int t, u32x4 v0, u32x4 v1, int sv, i32x8 ph, i32x8 pl, int sp) {
    const i32x8 v = join(v0, v1);
    o[t] = mfma8(v, ph, o[t], sv, sp);
    o[t] = mfma8(v, pl, o[t], sv, sp - 4);
  }
};

__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }
// Clears the NaN codes of V groups (columns 32 t ..) and makes the outputs of the queries that see one NaN.
__device__ __forceinline__ void clear_nan(u32x4& v0, u32x4& v1, f32x16& o, int lim, int hk) {
  i32x8 ind, vis;
#pragma unroll
  for (int w = 0; w < 8; w++) {
    const uint32_t c = w < 4 ? v0[w & 3] : v1[w & 3], nb = nan_bytes(c) >> 7, clean = c & ~(nb * 0xffu);
    if (w < 4) v0[w & 3] = clean;
    else v1[w & 3] = clean;
    ind[w] = (int)(nb * 0x38u);  // 1.0
    uint32_t z = 0;
#pragma unroll
    for (int e = 0; e < 4; e++)
      if (32 * (w >> 2) + 8 * (w & 3) + 4 * hk + e < lim) z |= 0x38u << (8 * e);
    vis[w] = (int)z;
  }
  f32x16 c;
#pragma unroll
  for (int e = 0; e < 16; e++) c[e] = 0.f;
  c = mfma8(ind, vis, c, 127, 127);
#pragma unroll
  for (int e = 0; e < 16; e++)
    if (c[e] > 0.f) o[e] = __uint_as_float(0x7fc00000u);
}

// Sums the shares of NK waves (each 32 rows, the same ones) in LDS, in wave order. Wave kw leaves with the total's m and
// l, and with the total in the groups of four registers u of o with u % NK = kw. sm: NK * (128 + 32 D) floats.
template <int D, int NK>
__device__ __forceinline__ void merge(float* sm, int kw, int lane, Rows<D>& r) {
  float* cm = sm + kw * 128;
  float* co = sm + NK * 128;
  cm[lane] = __int_as_float(r.m);
  cm[64 + lane] = r.l;
#pragma unroll
  for (int t = 0; t < D / 32; t++)
#pragma unroll
    for (int e = 0; e < 16; e++) co[((kw * (D / 32) + t) * 16 + e) * 64 + lane] = r.o[t][e];
  __syncthreads();
  int M = M_NONE;
#pragma unroll
  for (int k = 0; k < NK; k++) M = max(M, __float_as_int(sm[k * 128 + lane]));
  float L = 0.f, f[NK];
#pragma unroll
  for (int k = 0; k < NK; k++) {
    f[k] = __builtin_amdgcn_ldexpf(1.f, __float_as_int(sm[k * 128 + lane]) - M);
    L += sm[k * 128 + 64 + lane] * f[k];
  }
  r.m = M, r.l = L;
#pragma unroll
  for (int t = 0; t < D / 32; t++)
#pragma unroll
    for (int e = 0; e < 16; e++) {
      if ((t * 4 + e / 4) % NK != kw) continue;
      float a = 0.f;
#pragma unroll
      for (int k = 0; k < NK; k++) a += co[((k * (D / 32) + t) * 16 + e) * 64 + lane] * f[k];
      r.o[t][e] = a;
    }
}

// ---------------------------------------------------------------------------------------------- few rows
// One workgroup per (sequence, key head, 32 rows, run of `chunk` blocks); its NK waves take the blocks in turn, straight
// from memory into the MFMA's registers, the next block's K in flight through this block's softmax and its V through
// the next block's scores. splits > 1: unnormalised shares to p.part, put together by kv8_join_kernel.
template <int D, int NK>
__global__ __launch_bounds__(64 * NK) void kv8_rows_kernel(Attn8Args p) {
  __shared__ __attribute__((aligned(16))) float sm[NK * (128 + 32 * D)];
  const int lane = threadIdx.x & 63, kw = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), hk = lane >> 5;
  const int s = blockIdx.x % p.splits;
  const long cell = blockIdx.x / p.splits;
  const int rt = (int)(cell % p.nrt), bh = (int)(cell / p.nrt), b = bh / p.H, h = bh % p.H;
  const Seq sq = sequence(p, b);
  const int R = p.Tq * p.G, row = rt * 32 + (lane & 31), rc = min(row, R - 1);
  const int lim = limit(p, sq, rc / p.G);
  const int kend = limit(p, sq, min(rt * 32 + 31, R - 1) / p.G);                  // keys that any row sees
  const int kall = limit(p, sq, rt * 32 / p.G);                                    // keys that every row sees
  const int b0 = s * p.chunk, b1 = min(b0 + p.chunk, (kend + 63) / 64);
  Rows<D> r;
  r.clear();
  if (b0 < b1) {
    r.load(p.q + b * p.sq_b + (long)(h * p.G + rc % p.G) * p.sq_h + (long)(rc / p.G) * p.sq_t, hk);
    const long c0 = (long)bh * kv8_blocks(p.ctx);
    const uint8_t* kp = p.kc + c0 * (64 * D) + lane * 16;
    const uint8_t* vp = p.vc + c0 * (64 * D) + lane * 16;
    u32x4 k[2][D / 32], v[D / 32][2];
    int sk = 0, sv = 0, nsk = 0, nsv = 0;
    auto get_k = [&](int blk) {
#pragma unroll
      for (int t = 0; t < 2; t++)
#pragma unroll
        for (int j = 0; j < D / 32; j++)
          k[t][j] = *reinterpret_cast<const u32x4*>(kp + (long)blk * (64 * D) + (t * (D / 32) + j) * 1024);
      nsk = p.ks[c0 + blk];
      nsv = p.vs[c0 + blk];
    };
    auto get_v = [&](int blk) {
#pragma unroll
      for (int t = 0; t < D / 32; t++)
#pragma unroll
        for (int j = 0; j < 2; j++)
          v[t][j] = *reinterpret_cast<const u32x4*>(vp + (long)blk * (64 * D) + (t * 2 + j) * 1024);
    };
    int blk = b0 + kw;
    if (blk < b1) {
      get_k(blk);
      get_v(blk);
    }
    for (; blk < b1; blk += NK) {
      f32x16 st[2];
      sk = nsk, sv = nsv;
      r.scores(k, sk, st);
      const bool more = blk + NK < b1;
      if (more) get_k(blk + NK);
      i32x8 ph, pl;
      int sp;
      if ((blk + 1) * 64 > kall) {
        r.template weights<true>(st, p.sl2, lim - blk * 64, hk, ph, pl, sp);
        uint32_t nb = 0;
#pragma unroll
        for (int t = 0; t < D / 32; t++)
#pragma unroll
          for (int j = 0; j < 2; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) nb |= nan_bytes(v[t][j][e]);
        if (__any(nb != 0)) {
#pragma unroll
          for (int t = 0; t < D / 32; t++) clear_nan(v[t][0], v[t][1], r.o[t], lim - blk * 64, hk);
        }
      } else {
        r.template weights<false>(st, p.sl2, 64, hk, ph, pl, sp);
      }
#pragma unroll
      for (int t = 0; t < D / 32; t++) r.add(t, v[t][0], v[t][1], sv, ph, pl, sp);
      if (more) get_v(blk + NK);
    }
  }
  merge<D, NK>(sm, kw, lane, r);
  if (row >= R) return;
  const bool whole = p.splits == 1;
  const float inv = r.l == 0.f ? 0.f : 1.f / r.l;
  uint16_t* out = p.o + b * p.so_b + (long)(row / p.G) * p.so_t + (long)(h * p.G + row % p.G) * D;
  // shares: [cell][split][row of 32][D], then [cell][split][2][32] behind all of them
  const long rec = (long)blockIdx.x;
  float* po = p.part + (rec * 32 + (lane & 31)) * D;
  float* pm = p.part + (long)gridDim.x * 32 * D + rec * 64;
  if (!whole && kw == 0 && hk == 0) {
    pm[lane & 31] = __int_as_float(r.m);
    pm[32 + (lane & 31)] = r.l;
  }
#pragma unroll
  for (int t = 0; t < D / 32; t++)
#pragma unroll
    for (int u = 0; u < 4; u++) {
      if ((t * 4 + u) % NK != kw) continue;
      const int d = 32 * t + 8 * u + 4 * hk;
      if (whole)
        *reinterpret_cast<u32x2*>(out + d) = u32x2{pack2(r.o[t][4 * u] * inv, r.o[t][4 * u + 1] * inv),
                                                   pack2(r.o[t][4 * u + 2] * inv, r.o[t][4 * u + 3] * inv)};
      else
        *reinterpret_cast<f32x4*>(po + d) = f32x4{r.o[t][4 * u], r.o[t][4 * u + 1], r.o[t][4 * u + 2], r.o[t][4 * u + 3]};
    }
}

// One workgroup per row: 256 / D groups of threads add the shares in turn, in a fixed order.
template <int D>
__global__ __launch_bounds__(256) void kv8_join_kernel(Attn8Args p, long ncell) {
  constexpr int NG = 256 / D;
  __shared__ float so[NG][D];
  __shared__ float sl[NG];
  const int R = p.Tq * p.G, d = threadIdx.x % D, g = threadIdx.x / D;
  const long bh = blockIdx.x / R;
  const int row = (int)(blockIdx.x % R), b = (int)(bh / p.H), h = (int)(bh % p.H);
  const long rec0 = (bh * p.nrt + row / 32) * p.splits;
  const float* po = p.part + (rec0 * 32 + row % 32) * D + d;
  const float* pm = p.part + ncell * p.splits * 32 * D + rec0 * 64 + row % 32;
  int M = M_NONE;
  for (int s = 0; s < p.splits; s++) M = max(M, __float_as_int(pm[s * 64]));
  float a = 0.f, L = 0.f;
  for (int s = g; s < p.splits; s += NG) {
    const float f = __builtin_amdgcn_ldexpf(1.f, __float_as_int(pm[s * 64]) - M);
    L += pm[s * 64 + 32] * f;
    a += po[(long)s * 32 * D] * f;
  }
  so[g][d] = a;
  if (d == 0) sl[g] = L;
  __syncthreads();
  if (g) return;
  a = 0.f, L = 0.f;
#pragma unroll
  for (int u = 0; u < NG; u++) {
    a += so[u][d];
    L += sl[u];
  }
  p.o[b * p.so_b + (long)(row / p.G) * p.so_t + (long)(h * p.G + row % p.G) * D + d] = f2bf(L == 0.f ? 0.f : a / L);
}

}  // namespace

// Blocks of 64 keys per workgroup and runs per sequence of mx_kv8_sdpa; part needs mx_kv8_sdpa_ws floats.
static void plan(int B, int H, int G, int Tq, int ctx, int D, int* nrt, int* splits, int* chunk) {
  const int nb = kv8_blocks(ctx);
  *nrt = (int)(((long)Tq * G + 31) / 32);
  const long cells = (long)B * H * *nrt;
  long sp = (1024 + cells - 1) / cells;
  const long most = (nb + 15) / 16;
  if (sp > most) sp = most;
  if (sp < 1) sp = 1;
  *chunk = (int)((nb + sp - 1) / sp);
  *splits = (nb + *chunk - 1) / *chunk;
}

extern "C" long mx_kv8_sdpa_ws(int B, int H, int G, int Tq, int ctx, int D) {
  if (B < 1 || H < 1 || G < 1 || Tq < 1 || ctx < 1 || (D != 64 && D != 128)) return 0;
  int nrt, sp, ch;
  plan(B, H, G, Tq, ctx, D, &nrt, &sp, &ch);
  return sp == 1 ? 0 : (long)B * H * nrt * sp * 32 * (D + 2);
}

extern "C" int mx_kv8_sdpa(hipStream_t st, const uint16_t* q, long sq_b, long sq_h, long sq_t, const uint8_t* kc,
                           const uint8_t* vc, const uint8_t* ks, const uint8_t* vs, uint16_t* o, long so_b, long so_t,
                           int B, int H, int G, int Tq, int D, int ctx, const int* len, long len_s, int base, int qpos,
                           int qend, int causal_from, float scale, float* part, long part_elems) {
  if (!q || !kc || !vc || !ks || !vs || !o) return MX_ENULL;
  if (D != 64 && D != 128) return MX_EBADCFG;
  if (B < 1 || H < 1 || G < 1 || Tq < 1 || ctx < 1 || ctx > 0x7fffff00 || (long)Tq * G > 0x7fffff00L) return MX_ESHAPE;
  if (!(scale > 0.f) || !(scale < INFINITY) || causal_from < 0) return MX_ESHAPE;
  if ((sq_b | sq_h | sq_t) % 8 || (so_b | so_t) % 4) return MX_ESHAPE;
  if (((uintptr_t)q | (uintptr_t)kc | (uintptr_t)vc) & 15 || ((uintptr_t)o & 7) || ((uintptr_t)len & 3)) return MX_ELAYOUT;
  Attn8Args a{q, sq_b, sq_h, sq_t, kc, vc, ks, vs, o, so_b, so_t, part, len, len_s, base, qpos, qend, causal_from,
              B, H, G, Tq, ctx, 0, 0, 0, scale * 1.4426950408889634f};
  plan(B, H, G, Tq, ctx, D, &a.nrt, &a.splits, &a.chunk);
  if (a.splits > 1 && (!part || part_elems < mx_kv8_sdpa_ws(B, H, G, Tq, ctx, D) || ((uintptr_t)part & 15))) return MX_ESPLIT;
  const long ncell = (long)B * H * a.nrt, rows = (long)B * H * Tq * G;
  if (ncell * a.splits > 0x7fffffL || (a.splits > 1 && rows > 0xffffffL)) return MX_ESHAPE;
  const dim3 grid((unsigned)(ncell * a.splits));
  if (D == 64)
    hipLaunchKernelGGL((kv8_rows_kernel<64, 8>), grid, dim3(512), 0, st, a);
  else
    hipLaunchKernelGGL((kv8_rows_kernel<128, 8>), grid, dim3(512), 0, st, a);
  if (a.splits > 1) {
    if (D == 64)
      hipLaunchKernelGGL(kv8_join_kernel<64>, dim3((unsigned)rows), dim3(256), 0, st, a, ncell);
    else
      hipLaunchKernelGGL(kv8_join_kernel<128>, dim3((unsigned)rows), dim3(256), 0, st, a, ncell);
  }
  return hipGetLastError() == hipSuccess ? MX_OK : MX_ELAUNCH;
}
