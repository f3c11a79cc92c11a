// Attention over the 8-bit KV cache (kv8.h) for head dims 64 and 128, G query heads per key head:
//   O[b, i, h] = sum_j softmax_j(scale <Q[b, h, i], K[b, h / G, j]>) V[b, h / G, j]   over the visible keys j
//   key j is visible to query i of sequence b iff j < len_b and (j < causal_from or j <= qpos_b + i); a query that sees
//   no key gets zeros.
//
// The codes go from the cache into the 32x32x64 MFMA as they are; nothing is converted to bf16.
//  * S^T = K Q^T: Q is two e4m3 terms, q = 2^e (hi + lo / 16) with one exponent per row, which hold a bf16's 8 bits, so both
//    products together are the bf16 product. The row's largest value lies in [128, 256) and lo's last step is 2^-13, so
//    values below 2^-14, which is 2^-22 to 2^-21 of the largest, become 0. The scales of the K block and of Q are the
//    MFMA's own scale operands.
//  * O^T += V^T P^T: the weights of 64 keys are two e4m3 terms too, with a power of two of their own for every query and
//    block: p = 2^(el - 8 - m) (hi + lo / 16), el the next integer above the block's largest score (base 2), m the
//    running one. That keeps each weight to 2^-9 of itself, and every weight above 2^-21 of the block's largest. The
//    running maximum is an integer, so rescaling is exact. Sums of weights are taken in fp32 before that rounding.
//    Scores up to 2^29 in size (2^30 in base 2, where the integers end) give what the formula gives; beyond, 0 or NaN.
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
  int B, H, G, Tq, ctx;
  int rw, nrt, splits, chunk;  // rows per workgroup, row groups, runs of `chunk` blocks per sequence
  float sl2;
};

__device__ __forceinline__ f32x16 mfma8(i32x8 a, i32x8 b, f32x16 c, int sa, int sb) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, c, 0, 0, 0, sa, 0, sb);
}
__device__ __forceinline__ f32x4 mfma8(i32x8 a, i32x8 b, f32x4 c, int sa, int sb) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, sa, 0, sb);
}
__device__ __forceinline__ i32x8 join(u32x4 a, u32x4 b) {
  return i32x8{(int)a.x, (int)a.y, (int)a.z, (int)a.w, (int)b.x, (int)b.y, (int)b.z, (int)b.w};
}
typedef short s16x2 __attribute__((ext_vector_type(2)));
// a, b, c, d (|.| <= 448) as hi + lo / 16; with a power of two `unit` a / unit .. are
__device__ __forceinline__ void split4(float a, float b, float c, float d, uint32_t& hi, uint32_t& lo) {
  uint32_t h = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  h = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, h, true);
  const auto x = __builtin_amdgcn_cvt_pk_f32_fp8(h, false), y = __builtin_amdgcn_cvt_pk_f32_fp8(h, true);
  s16x2 l = {0, 0};
  l = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(l, a - x[0], b - x[1], 0.0625f, false);
  l = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(l, c - y[0], d - y[1], 0.0625f, true);
  hi = h, lo = __builtin_bit_cast(uint32_t, l);
}

__device__ __forceinline__ void split4(float a, float b, float c, float d, float unit, uint32_t& hi, uint32_t& lo) {
  s16x2 h = {0, 0}, l = {0, 0};
  h = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(h, a, b, unit, false);
  h = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(h, c, d, unit, true);
  hi = __builtin_bit_cast(uint32_t, h);
  const auto x = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(hi, unit, false);
  const auto y = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(hi, unit, true);
  const float part = unit * 0.0625f;
  l = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(l, a - x[0], b - x[1], part, false);
  l = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(l, c - y[0], d - y[1], part, true);
  lo = __builtin_bit_cast(uint32_t, l);
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

// The larger of the four values that lanes l, l ^ 16, l ^ 32, l ^ 48 hold / their sum.
__device__ __forceinline__ float quarters_max(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return halves_max(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
__device__ __forceinline__ float quarters_sum(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return halves_sum(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

// One row's query: NC chunks of 16 columns (two 16-byte loads each) as hi and lo dwords, 4 per chunk; its scale byte for
// hi (lo: 4 less). The scaled maximum lies in [128, 256); an infinity or NaN makes its row NaN, as the formula does.
template <int NC>
__device__ __forceinline__ int split_row(const u32x4 (&x)[NC][2], uint32_t mx, uint32_t (&hi)[4 * NC], uint32_t (&lo)[4 * NC]) {
  const int code = max((int)(mx >> 7) - 7, 8);
  const float f = __uint_as_float((uint32_t)(254 - code) << 23);
#pragma unroll
  for (int w = 0; w < 4 * NC; w++) {
    const u32x4 v = x[w >> 2][(w >> 1) & 1];
    const uint32_t a = v[2 * (w & 1)], b = v[2 * (w & 1) + 1];
    split4(lo_bf(a) * f, hi_bf(a) * f, lo_bf(b) * f, hi_bf(b) * f, hi[w], lo[w]);
    if (mx >= 0x7f80u) hi[w] = 0x7f7f7f7fu;
  }
  return code;
}
__device__ __forceinline__ uint32_t bits_max(u32x4 v) {
  uint32_t m = 0;
#pragma unroll
  for (int e = 0; e < 4; e++) m = max(m, max(v[e] & 0x7fffu, (v[e] >> 16) & 0x7fffu));
  return m;
}
// What a block whose largest score is mx makes of its scores s: weights exp2(fma(s, sl2, neg)), at most 256 unit, whose codes
// count 2^(el - 8), for a power of two unit near 2^-8. neg is a float exactly and the fma rounds once, next to 0, so this also
// holds where mx sl2 is rounded to far more than 1 (from 2^24 on): what that rounding is off by goes into unit.
struct Block8 {
  float neg, unit;
  int el, e0;  // e0 = -neg
};
__device__ __forceinline__ Block8 block_scale(float mx, float sl2) {
  Block8 s;
  const float top = fminf(fmaxf(ceilf(mx * sl2), (float)M_NONE), -(float)M_NONE - 128.f);
  const int over = (int)fminf(fmaxf(ceilf(__builtin_fmaf(mx, sl2, -top)), -64.f), 64.f);  // 0, but for that rounding
  s.neg = -top, s.e0 = (int)top;
  s.el = max(s.e0 + over, M_NONE);
  s.unit = __uint_as_float((uint32_t)(127 - 8 + over) << 23);
  return s;
}
// scale byte of a block's weights (hi; lo: 4 less)
__device__ __forceinline__ int weight_byte(int el, int m) { return max(127 - 8 + max(el - m, -240), 4); }

__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }
__device__ __forceinline__ uint32_t nan_bytes(u32x4 v) {
  return nan_bytes(v.x) | nan_bytes(v.y) | nan_bytes(v.z) | nan_bytes(v.w);
}
// NaN codes of 16: cleared, and 1.0 in their places
__device__ __forceinline__ u32x4 take_nan(u32x4& v) {
  u32x4 ind;
#pragma unroll
  for (int e = 0; e < 4; e++) {
    const uint32_t nb = nan_bytes(v[e]) >> 7;
    v[e] &= ~(nb * 0xffu);
    ind[e] = nb * 0x38u;
  }
  return ind;
}
// 1.0 for the four keys from `key` on that lie below lim
__device__ __forceinline__ uint32_t seen4(int key, int lim) {
  const int n = lim - key;
  return n <= 0 ? 0u : n >= 4 ? 0x38383838u : 0x38383838u & ((1u << (8 * n)) - 1u);
}
template <class V>
__device__ __forceinline__ void mark_nan(const V& hits, V& o, int n) {
#pragma unroll
  for (int e = 0; e < n; e++)
    if (hits[e] > 0.f) o[e] = __uint_as_float(0x7fc00000u);
}

// Where a row's result goes: bf16 output, or (splits > 1) the share of record rec, row r of rw: [record][row][D] and
// behind all of them [record][2][rw] (m and l).
struct Out {
  uint16_t* out;
  float *po, *pm;
  float inv;
  bool whole;
};
template <int D>
__device__ __forceinline__ Out target(const Attn8Args& p, int b, int h, int row, long rec, long nrec, float l) {
  Out t;
  const int r = row % p.rw;
  t.whole = p.splits == 1;
  t.out = p.o + b * p.so_b + (long)(row / p.G) * p.so_t + (long)(h * p.G + row % p.G) * D;
  t.po = p.part + (rec * p.rw + r) * D;
  t.pm = p.part + nrec * p.rw * D + rec * 2 * p.rw + r;
  t.inv = l == 0.f ? 0.f : 1.f / l;
  return t;
}
__device__ __forceinline__ void put4(const Out& t, int d, float a, float b, float c, float e) {
  if (t.whole)
    *reinterpret_cast<u32x2*>(t.out + d) = u32x2{pack2(a * t.inv, b * t.inv), pack2(c * t.inv, e * t.inv)};
  else
    *reinterpret_cast<f32x4*>(t.po + d) = f32x4{a, b, c, e};
}

// ---------------------------------------------------------------------------------------------- few rows
// At most 16 rows per workgroup, on the 16x16x128 MFMA: (sequence, key head, 16 rows, run of `chunk` blocks); its NK waves
// take the blocks in turn, straight from memory into the MFMA's registers, the next block's K in flight through this
// block's softmax and its V through the next block's scores. A score tile tt holds keys 32 (g >> 1) + 4 (g & 1) + 8 tt + r
// (g = lane / 16, r = register): with that choice of rows the four tiles of a block leave, in a lane, the 16 keys whose V
// codes are one 16-byte group of the cache, in its order. The MFMA's 128 columns take hi and lo at once where the sum is
// 64 long (V's 64 keys; K at head dim 64): the same codes twice against (hi, lo), whose scales differ by lane (the scale
// of columns 32 u .. comes from lanes 16 u .., columns 64 .. are the second 16 bytes).
// The bound is the cache's bytes from HBM for long or many sequences (1 x 8 x 4 heads x 128, 262144 keys: 99 us, 5.4 TB/s
// with the join; 32 x 8 x 4, 6000 keys 80 us, 4.9 TB/s), for short ones a launch and one block's chain load -> scores ->
// maximum -> weights -> product (1 x 32 x 64: 128 keys 4.7 us, 794 keys 6.8).
template <int D, int NK>
__global__ __launch_bounds__(64 * NK) void kv8_rows_kernel(Attn8Args p) {
  constexpr int NQ = D / 64, NT = D / 16;
  __shared__ __attribute__((aligned(16))) float sm[NK * (32 + 16 * D)];
  const int lane = threadIdx.x & 63, kw = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int s = blockIdx.x % p.splits;
  const long cell = blockIdx.x / p.splits;
  const int rt = (int)(cell % p.nrt), bh = (int)(cell / p.nrt), b = bh / p.H, h = bh % p.H;
  const int R = p.Tq * p.G, row = rt * 16 + c, rc = min(row, R - 1);
  const Seq sq = sequence(p, b);
  const int lim = limit(p, sq, rc / p.G);
  const int kend = limit(p, sq, min(rt * 16 + 15, R - 1) / p.G);  // keys that any row sees
  const int kall = limit(p, sq, rt * 16 / p.G);                    // keys that every row sees
  const int b0 = s * p.chunk, b1 = min(b0 + p.chunk, (kend + 63) / 64);
  f32x4 o[NT];
#pragma unroll
  for (int t = 0; t < NT; t++) o[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  int m = M_NONE;
  float l = 0.f;
  int blk = b0 + kw;
  if (blk < b1) {
    const long c0 = (long)bh * kv8_blocks(p.ctx);
    // K: token 32 (c >> 3) + (c & 7) + 8 tt, columns 16 g .. (and 64 + 16 g ..); V: column c + 16 t, token group g
    const uint8_t* kp = p.kc + c0 * (64 * D) + (((c >> 3) * (D / 32) + (g >> 1)) * 64 + (g & 1) * 32 + (c & 7)) * 16;
    const uint8_t* vp = p.vc + c0 * (64 * D) + ((g >> 1) * 64 + (g & 1) * 32 + c) * 16;
    u32x4 k[4][NQ], v[NT];
    int nsk = 0, nsv = 0;
    auto get_k = [&](int i) {
#pragma unroll
      for (int tt = 0; tt < 4; tt++)
#pragma unroll
        for (int u = 0; u < NQ; u++)
          k[tt][u] = *reinterpret_cast<const u32x4*>(kp + (long)i * (64 * D) + tt * 128 + u * 2048);
      nsk = p.ks[c0 + i];
      nsv = p.vs[c0 + i];
    };
    auto get_v = [&](int i) {
#pragma unroll
      for (int t = 0; t < NT; t++)
        v[t] = *reinterpret_cast<const u32x4*>(vp + (long)i * (64 * D) + (t >> 1) * 2048 + (t & 1) * 256);
    };
    u32x4 x[NQ][2];
    const uint16_t* qrow = p.q + b * p.sq_b + (long)(h * p.G + rc % p.G) * p.sq_h + (long)(rc / p.G) * p.sq_t + 16 * g;
#pragma unroll
    for (int u = 0; u < NQ; u++)
#pragma unroll
      for (int e = 0; e < 2; e++) x[u][e] = *reinterpret_cast<const u32x4*>(qrow + 64 * u + 8 * e);
    get_k(blk);
    get_v(blk);
    uint32_t mx0 = 0, qhi[4 * NQ], qlo[4 * NQ];
#pragma unroll
    for (int u = 0; u < NQ; u++) mx0 = max(mx0, max(bits_max(x[u][0]), bits_max(x[u][1])));
    mx0 = (uint32_t)quarters_max((float)mx0);
    const int sqh = split_row<NQ>(x, mx0, qhi, qlo);
    const int half = g < 2 ? 0 : 4;  // lanes whose scale is that of the second 64 columns
    i32x8 qa, qb;
    if constexpr (D == 64) {
#pragma unroll
      for (int w = 0; w < 4; w++) qa[w] = (int)qhi[w], qa[4 + w] = (int)qlo[w];
    } else {
#pragma unroll
      for (int w = 0; w < 8; w++) qa[w] = (int)qhi[w], qb[w] = (int)qlo[w];
    }
    for (; blk < b1; blk += NK) {
      const int sk = nsk, sv = nsv;
      f32x4 st[4];
#pragma unroll
      for (int tt = 0; tt < 4; tt++) {
        st[tt] = f32x4{0.f, 0.f, 0.f, 0.f};
        if constexpr (D == 64) {
          st[tt] = mfma8(join(k[tt][0], k[tt][0]), qa, st[tt], sk, sqh - half);
        } else {
          st[tt] = mfma8(join(k[tt][0], k[tt][NQ - 1]), qa, st[tt], sk, sqh);
          st[tt] = mfma8(join(k[tt][0], k[tt][NQ - 1]), qb, st[tt], sk, sqh - 4);
        }
      }
      const bool more = blk + NK < b1;
      if (more) get_k(blk + NK);
      const bool masked = (blk + 1) * 64 > kall;
      const int key0 = blk * 64 + 32 * (g >> 1) + 4 * (g & 1);
      float mx = -INFINITY;
      if (masked) {
        asm volatile("");  // keeps the branch: as selects the mask would be computed for every block
#pragma unroll
        for (int tt = 0; tt < 4; tt++)
#pragma unroll
          for (int r = 0; r < 4; r++) st[tt][r] = key0 + 8 * tt + r < lim ? st[tt][r] : -INFINITY;
      }
#pragma unroll
      for (int tt = 0; tt < 4; tt++)
#pragma unroll
        for (int r = 0; r < 4; r++) mx = fmaxf(mx, st[tt][r]);
      const Block8 bs = block_scale(quarters_max(mx), p.sl2);
      const int el = bs.el, mn = max(m, el);
      if (__any(mn != m)) {
        const float al = __builtin_amdgcn_ldexpf(1.f, m - mn);
        l *= al;
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
          for (int r = 0; r < 4; r++) o[t][r] *= al;
        m = mn;
      }
      float sum = 0.f;
      u32x4 hi, lo;
#pragma unroll
      for (int tt = 0; tt < 4; tt++) {
        float y[4];
#pragma unroll
        for (int r = 0; r < 4; r++) {
          y[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(st[tt][r], p.sl2, bs.neg));
          sum += y[r];
        }
        uint32_t a, d;
        split4(y[0], y[1], y[2], y[3], bs.unit, a, d);
        hi[tt] = a, lo[tt] = d;
      }
      l += __builtin_amdgcn_ldexpf(quarters_sum(sum), bs.e0 - mn);
      if (masked) {
        uint32_t nb = 0;
#pragma unroll
        for (int t = 0; t < NT; t++) nb |= nan_bytes(v[t]);
        if (__any(nb != 0)) {
          const u32x4 none = {0u, 0u, 0u, 0u};
          u32x4 vis;
#pragma unroll
          for (int tt = 0; tt < 4; tt++) vis[tt] = seen4(key0 + 8 * tt, lim);
#pragma unroll
          for (int t = 0; t < NT; t++) {
            const u32x4 ind = take_nan(v[t]);
            mark_nan(mfma8(join(ind, none), join(vis, none), f32x4{0.f, 0.f, 0.f, 0.f}, 127, 127), o[t], 4);
          }
        }
      }
      const int sp = weight_byte(el, mn) - half;
      const i32x8 w = join(hi, lo);
#pragma unroll
      for (int t = 0; t < NT; t++) o[t] = mfma8(join(v[t], v[t]), w, o[t], sv, sp);
      if (more) get_v(blk + NK);
    }
  }
  // ---- the waves' shares meet in LDS, added in wave order; wave kw finishes the tiles t with t % NK = kw
  float* cm = sm + kw * 32;
  f32x4* co = reinterpret_cast<f32x4*>(sm + NK * 32);
  if (g == 0) {
    cm[c] = __int_as_float(m);
    cm[16 + c] = l;
  }
#pragma unroll
  for (int t = 0; t < NT; t++) co[(kw * NT + t) * 64 + lane] = o[t];
  __syncthreads();
  if (row >= R) return;
  int M = M_NONE;
#pragma unroll
  for (int w = 0; w < NK; w++) M = max(M, __float_as_int(sm[w * 32 + c]));
  float L = 0.f, f[NK];
#pragma unroll
  for (int w = 0; w < NK; w++) {
    f[w] = __builtin_amdgcn_ldexpf(1.f, __float_as_int(sm[w * 32 + c]) - M);
    L += sm[w * 32 + 16 + c] * f[w];
  }
  const Out t = target<D>(p, b, h, row, blockIdx.x, gridDim.x, L);
  if (!t.whole && kw == 0 && g == 0) {
    t.pm[0] = __int_as_float(M);
    t.pm[p.rw] = L;
  }
  for (int u = kw; u < NT; u += NK) {
    f32x4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < NK; w++) {
      const f32x4 y = co[(w * NT + u) * 64 + lane];
#pragma unroll
      for (int e = 0; e < 4; e++) a[e] += y[e] * f[w];
    }
    put4(t, 16 * u + 4 * g, a[0], a[1], a[2], a[3]);
  }
}

// ---------------------------------------------------------------------------------------------- many rows
// 32 NQW rows per workgroup, on the 32x32x64 MFMA: NQW query waves x NKW key waves. A stage of the LDS ring holds NKW
// blocks of K and V as they lie in the cache, copied by the asynchronous LDS-DMA load a stage or more ahead; key wave u
// takes block u of every stage, and the shares of the key waves are added at the end. The bound is the vector ALU beside
// the MFMA: per key and row, four products of 8-bit terms, and an exponential and two roundings to e4m3. 2048 rows of a
// 16001-key sequence, 32 heads x 128 over 8: 535 us, 0.93 PFLOP/s of the bf16 product (MFMA pipes busy in 41 % of the cycles,
// ALU in 46 %; 600 us in a trace, at a lower clock).
template <int D, int NQW, int NKW, int S>
struct Tile8 {
  static constexpr int NW = NQW * NKW;
  static constexpr int BLK_B = 128 * D;               // K and V of a block
  static constexpr int STAGE_B = NKW * BLK_B;
  static constexpr int LPS = STAGE_B / 1024 / NW;      // load instructions per wave and stage
  static constexpr int RING_B = S * STAGE_B;
  static constexpr int COMB_B = NKW > 1 ? NW * 64 * (2 + D / 2) * 4 : 0;
  static constexpr int BYTES = RING_B > COMB_B ? RING_B : COMB_B;
  static_assert(64 % NKW == 0 && STAGE_B % (1024 * NW) == 0 && BYTES <= 160 * 1024, "ring");
};

template <int D, int NQW, int NKW, int S>
__global__ __launch_bounds__(64 * NQW * NKW, 2) void kv8_tile_kernel(Attn8Args p) {
  using C = Tile8<D, NQW, NKW, S>;
  constexpr int NT = D / 32, NS = D / 64;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[C::BYTES];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int qg = wave % NQW, kw = wave / NQW, c = lane & 31, hk = lane >> 5;
  const int s = blockIdx.x % p.splits;
  const long cell = blockIdx.x / p.splits;
  // the row groups of a causal prompt's end see the most keys: they start first
  const int rt = p.nrt - 1 - (int)(cell % p.nrt), bh = (int)(cell / p.nrt), b = bh / p.H, h = bh % p.H;
  const long rec = ((long)bh * p.nrt + rt) * p.splits + s;  // the share's record (rows in order, not as they start)
  const int R = p.Tq * p.G, r0 = rt * 32 * NQW, row = r0 + 32 * qg + c, rc = min(row, R - 1);
  const Seq sq = sequence(p, b);
  const int lim = limit(p, sq, rc / p.G);
  const int kend = limit(p, sq, min(r0 + 32 * NQW - 1, R - 1) / p.G);               // keys that any row sees
  const int wend = limit(p, sq, min(r0 + 32 * qg + 31, R - 1) / p.G);               // ... any row of this wave
  const int kall = limit(p, sq, min(r0 + 32 * qg, R - 1) / p.G);                    // ... every row of this wave
  const int b0 = s * p.chunk, b1 = min(b0 + p.chunk, (kend + 63) / 64);
  const int ns = b1 > b0 ? (b1 - b0 + NKW - 1) / NKW : 0;
  const long c0 = (long)bh * kv8_blocks(p.ctx);
  const uint32_t sbase = lds_off(smem);
  // stage i: K then V of each block; instruction q brings 1 KB; blocks past the last repeat it (never used)
  auto issue = [&](int i) {
    const uint32_t dst = sbase + (uint32_t)(i % S) * C::STAGE_B;
#pragma unroll
    for (int e = 0; e < C::LPS; e++) {
      const int q = wave * C::LPS + e, u = q / (C::BLK_B / 1024), r = q % (C::BLK_B / 1024);
      const long blk = c0 + min(b0 + i * NKW + u, b1 - 1);
      const uint8_t* src = r < D / 16 ? p.kc + blk * (64 * D) + r * 1024 : p.vc + blk * (64 * D) + (r - D / 16) * 1024;
      dma16s(src, (uint32_t)lane * 16, dst + q * 1024);
    }
  };
  f32x16 o[NT];
#pragma unroll
  for (int t = 0; t < NT; t++)
#pragma unroll
    for (int e = 0; e < 16; e++) o[t][e] = 0.f;
  int m = M_NONE;
  float l = 0.f;
  i32x8 qh[NS], ql[NS];
  int sqh;
  // the scale bytes of the next 64 blocks, one per lane (a load per block would wait for the copies in flight behind it)
  int skl = 0, svl = 0;
  auto get_scales = [&](int first) {
    const long i = c0 + min(first + lane, b1 - 1);
    skl = p.ks[i], svl = p.vs[i];
  };
  if (ns > 0) {
    get_scales(b0);
    issue(0);
  }
  {
    u32x4 x[NT][2];
    uint32_t mx = 0, hi[4 * NT], lo[4 * NT];
    const uint16_t* qrow = p.q + b * p.sq_b + (long)(h * p.G + rc % p.G) * p.sq_h + (long)(rc / p.G) * p.sq_t + 16 * hk;
#pragma unroll
    for (int j = 0; j < NT; j++)
#pragma unroll
      for (int e = 0; e < 2; e++) {
        x[j][e] = *reinterpret_cast<const u32x4*>(qrow + 32 * j + 8 * e);
        mx = max(mx, bits_max(x[j][e]));
      }
    mx = (uint32_t)halves_max((float)mx);
    sqh = split_row<NT>(x, mx, hi, lo);
#pragma unroll
    for (int u = 0; u < NS; u++)
#pragma unroll
      for (int w = 0; w < 8; w++) qh[u][w] = (int)hi[8 * u + w], ql[u][w] = (int)lo[8 * u + w];
  }
  __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): the compiler does not count the LDS-DMA loads, so nothing of its own may
                                       // be in flight beside them (gfx9 encoding; expcnt, lgkmcnt not waited)
#pragma unroll
  for (int i = 1; i < S - 1; i++)
    if (i < ns) issue(i);

  for (int i = 0; i < ns; i++) {
    wait_stages<C::LPS, S - 2>(ns - 1 - i);
    __syncthreads();
    if (i + S - 1 < ns) issue(i + S - 1);
    const int rel = i * NKW + kw, blk = b0 + rel;
    if (i > 0 && i * NKW % 64 == 0) get_scales(b0 + i * NKW);
    if (blk >= b1 || blk * 64 >= wend) continue;
    const uint8_t* kst = smem + (i % S) * C::STAGE_B + kw * C::BLK_B + lane * 16;
    const uint8_t* vst = kst + 64 * D;
    auto ld = [](const uint8_t* q) { return *reinterpret_cast<const u32x4*>(q); };
    const int sk = __builtin_amdgcn_readlane(skl, rel % 64), sv = __builtin_amdgcn_readlane(svl, rel % 64);
    f32x16 st[2];
    // a wave in its products goes first: the two waves of a SIMD fall out of step, and one's softmax runs under the other's
    // products (3 % of the time, 2048 rows x 16001 keys, 32 heads x 128)
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int t = 0; t < 2; t++) {
      i32x8 kk[NS];
#pragma unroll
      for (int u = 0; u < NS; u++)
        kk[u] = join(ld(kst + (t * NT + 2 * u) * 1024), ld(kst + (t * NT + 2 * u + 1) * 1024));
#pragma unroll
      for (int e = 0; e < 16; e++) st[t][e] = 0.f;
#pragma unroll
      for (int u = 0; u < NS; u++) st[t] = mfma8(kk[u], qh[u], st[t], sk, sqh);
#pragma unroll
      for (int u = 0; u < NS; u++) st[t] = mfma8(kk[u], ql[u], st[t], sk, sqh - 4);
    }
    __builtin_amdgcn_s_setprio(0);
    const bool masked = (blk + 1) * 64 > kall;
    const int key0 = blk * 64 + 4 * hk;
    float mx = -INFINITY;
    if (masked) {
      asm volatile("");  // keeps the branch: as selects the mask would cost every block 100 instructions
#pragma unroll
      for (int t = 0; t < 2; t++)
#pragma unroll
        for (int r = 0; r < 16; r++)
          st[t][r] = key0 + 32 * t + 8 * (r >> 2) + (r & 3) < lim ? st[t][r] : -INFINITY;
    }
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
      for (int r = 0; r < 16; r++) mx = fmaxf(mx, st[t][r]);
    const Block8 bs = block_scale(halves_max(mx), p.sl2);
    const int el = bs.el, mn = max(m, el);
    if (__any(mn != m)) {
      const float al = __builtin_amdgcn_ldexpf(1.f, m - mn);
      l *= al;
#pragma unroll
      for (int e = 0; e < 16; e++) {
#pragma unroll
        for (int t = 0; t < NT; t++) o[t][e] *= al;
      }
      m = mn;
    }
    float sum = 0.f;
    i32x8 ph, pl;
#pragma unroll
    for (int w = 0; w < 8; w++) {
      float y[4];
#pragma unroll
      for (int e = 0; e < 4; e++) y[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(st[w >> 2][4 * (w & 3) + e], p.sl2, bs.neg));
      sum += (y[0] + y[1]) + (y[2] + y[3]);
      uint32_t a, d;
      split4(y[0], y[1], y[2], y[3], bs.unit, a, d);
      ph[w] = (int)a, pl[w] = (int)d;
    }
    const int sp = weight_byte(el, mn);
    l += __builtin_amdgcn_ldexpf(halves_sum(sum), bs.e0 - mn);
    __builtin_amdgcn_s_setprio(1);
    bool nan = false;
    if (masked) {
      uint32_t nb = 0;
#pragma unroll
      for (int t = 0; t < 2 * NT; t++) nb |= nan_bytes(ld(vst + t * 1024));
      nan = __any(nb != 0);
    }
#pragma unroll
    for (int t = 0; t < NT; t++) {
      u32x4 v0 = ld(vst + 2 * t * 1024), v1 = ld(vst + (2 * t + 1) * 1024);
      if (nan) {
        const u32x4 i0 = take_nan(v0), i1 = take_nan(v1);
        i32x8 vis;
#pragma unroll
        for (int w = 0; w < 8; w++) vis[w] = (int)seen4(key0 + 32 * (w >> 2) + 8 * (w & 3), lim);
        f32x16 z;
#pragma unroll
        for (int e = 0; e < 16; e++) z[e] = 0.f;
        mark_nan(mfma8(join(i0, i1), vis, z, 127, 127), o[t], 16);
      }
      o[t] = mfma8(join(v0, v1), ph, o[t], sv, sp);
      o[t] = mfma8(join(v0, v1), pl, o[t], sv, sp - 4);
    }
    __builtin_amdgcn_s_setprio(0);
  }

  float L = l;
  if constexpr (NKW > 1) {
    // ---- the key waves' shares, added in wave order; wave kw finishes the register groups u with u % NKW = kw
    float* cm = reinterpret_cast<float*>(smem);
    f32x4* co = reinterpret_cast<f32x4*>(cm + C::NW * 128);
    wait_vm<0>();
    __syncthreads();
    cm[wave * 128 + lane] = __int_as_float(m);
    cm[wave * 128 + 64 + lane] = L;
#pragma unroll
    for (int u = 0; u < 4 * NT; u++)
      co[(wave * 4 * NT + u) * 64 + lane] =
          f32x4{o[u / 4][4 * (u % 4)], o[u / 4][4 * (u % 4) + 1], o[u / 4][4 * (u % 4) + 2], o[u / 4][4 * (u % 4) + 3]};
    __syncthreads();
    m = M_NONE;
#pragma unroll
    for (int w = 0; w < NKW; w++) m = max(m, __float_as_int(cm[(w * NQW + qg) * 128 + lane]));
    float f[NKW];
    L = 0.f;
#pragma unroll
    for (int w = 0; w < NKW; w++) {
      f[w] = __builtin_amdgcn_ldexpf(1.f, __float_as_int(cm[(w * NQW + qg) * 128 + lane]) - m);
      L += cm[(w * NQW + qg) * 128 + 64 + lane] * f[w];
    }
    if (row >= R) return;
    const Out t = target<D>(p, b, h, row, rec, gridDim.x, L);
    if (!t.whole && kw == 0 && hk == 0) {
      t.pm[0] = __int_as_float(m);
      t.pm[p.rw] = L;
    }
    for (int u = kw; u < 4 * NT; u += NKW) {
      f32x4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < NKW; w++) {
        const f32x4 y = co[((w * NQW + qg) * 4 * NT + u) * 64 + lane];
#pragma unroll
        for (int e = 0; e < 4; e++) a[e] += y[e] * f[w];
      }
      put4(t, 8 * u + 4 * hk, a[0], a[1], a[2], a[3]);
    }
  } else {
    if (row >= R) return;
    const Out t = target<D>(p, b, h, row, rec, gridDim.x, L);
    if (!t.whole && hk == 0) {
      t.pm[0] = __int_as_float(m);
      t.pm[p.rw] = L;
    }
#pragma unroll
    for (int u = 0; u < 4 * NT; u++)
      put4(t, 8 * u + 4 * hk, o[u / 4][4 * (u % 4)], o[u / 4][4 * (u % 4) + 1], o[u / 4][4 * (u % 4) + 2],
           o[u / 4][4 * (u % 4) + 3]);
  }
}

// One workgroup per row: the shares' factors first, then 1024 / D groups of threads with 4 columns each add the shares in
// turn, in a fixed order.
template <int D>
__global__ __launch_bounds__(256) void kv8_join_kernel(Attn8Args p, long nrec) {
  constexpr int TD = D / 4, NG = 256 / TD;
  __shared__ float fs[1024];
  __shared__ f32x4 so[NG][TD];
  __shared__ float red[2][4];
  const int tid = threadIdx.x, wave = tid >> 6;
  const int R = p.Tq * p.G, d = tid % TD, g = tid / TD;
  const long bh = blockIdx.x / R;
  const int row = (int)(blockIdx.x % R), b = (int)(bh / p.H), h = (int)(bh % p.H);
  const long rec0 = (bh * p.nrt + row / p.rw) * p.splits;
  const float* pm = p.part + nrec * p.rw * D + rec0 * 2 * p.rw + row % p.rw;
  int m = M_NONE;
  for (int s = tid; s < p.splits; s += 256) m = max(m, __float_as_int(pm[(long)s * 2 * p.rw]));
  // integers of at most 2^30: the comparison goes by halves that a float holds
  const float top = wave_max((float)((m >> 15) + 32768));
  const int hi = (int)top - 32768;
  const float bot = wave_max((m >> 15) == hi ? (float)(m & 32767) : -1.f);
  if ((tid & 63) == 0) red[0][wave] = __int_as_float(hi * 32768 + (int)bot);
  __syncthreads();
  int M = M_NONE;
#pragma unroll
  for (int w = 0; w < 4; w++) M = max(M, __float_as_int(red[0][w]));
  float l = 0.f;
  for (int s = tid; s < p.splits; s += 256) {
    const float f = __builtin_amdgcn_ldexpf(1.f, __float_as_int(pm[(long)s * 2 * p.rw]) - M);
    fs[s] = f;
    l += pm[(long)s * 2 * p.rw + p.rw] * f;
  }
  l = wave_total(l);
  if ((tid & 63) == 0) red[1][wave] = l;
  __syncthreads();
  const float* po = p.part + (rec0 * p.rw + row % p.rw) * D + 4 * d;
  f32x4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = g; s < p.splits; s += NG) {
    const f32x4 y = *reinterpret_cast<const f32x4*>(po + (long)s * p.rw * D);
#pragma unroll
    for (int e = 0; e < 4; e++) a[e] += y[e] * fs[s];
  }
  so[g][d] = a;
  __syncthreads();
  if (g) return;
#pragma unroll
  for (int u = 1; u < NG; u++) a += so[u][d];
  const float L = red[1][0] + red[1][1] + red[1][2] + red[1][3], inv = L == 0.f ? 0.f : 1.f / L;
  *reinterpret_cast<u32x2*>(p.o + b * p.so_b + (long)(row / p.G) * p.so_t + (long)(h * p.G + row % p.G) * D + 4 * d) =
      u32x2{pack2(a[0] * inv, a[1] * inv), pack2(a[2] * inv, a[3] * inv)};
}

// How a problem is cut, by the cache's capacity (grid and workspace have to be known on the host, the lengths may be on the
// device; 1 x 8 x 4, 128, 1, 16000 keys take 11.2 with ctx 16000, 28.4 with 262144): rw rows per
// workgroup (16: the few-row kernel), nkw key waves, nrt row groups, `splits` runs of `chunk` blocks. us on one MI355X (query waves x key waves; sequences x key heads x group, head dim, queries, keys):
//  * up to 32 rows: the few-row kernel; runs of keys until there are 3 workgroups per CU (a CU holds 2 or 3), of 16 blocks
//    at least. Where those leave half of the CUs idle, runs of 8 (the join costs 3 us; caches that no other call has just
//    read: 1 x 8 x 4, 128, 1, 4000 11.0, runs of 16 13.0; 4 x 8 x 4, 128, 1, 2000 11.6 / 13.6), or one run up to 24 blocks (1
//    x 32 x 1, 64, 1, 1100 7.5, two runs 9.2; 4 x 8 x 4, 128, 1, 1536 12.3, runs of 8 11.2). 8 waves instead of 4 where
//    there is at most one workgroup per CU (8 x 32 x 1, 64, 1, 794 7.4 / 8.1; with 512 workgroups, 64 x 8 x 4, 128, 1, 1000,
//    24.8 / 23.8);
//  * 4 x 1 where 128-row groups give two workgroups per CU: 4 x 8 x 4, 128, 512, 512 30.2 (4 x 2 37.7, 2 x 2 37.4);
//  * 4 x 2 down to three quarters of one per CU: 1 x 8 x 4, 128, 1024, 8000 152 (4 x 1 209, 2 x 4 183, 1 x 4 314);
//  * 2 x 4, 64-row groups, down to the same: 1 x 8 x 4, 128, 512, 4000 54 (4 x 2 70, 1 x 4 92);
//  * 1 x 8 (head dim 128: 1 x 4, its LDS) below: 1 x 32 x 1, 64, 64, 794 9.9 (2 x 4 13.1, 4 x 2 17.6); 1 x 8 x 4, 128, 256,
//    2000 27 (2 x 4 35, 4 x 2 42);
//  * few rows over 16384 keys or more (bound by the keys' bytes): all rows of a head in a workgroup, if 64 or 128 hold
//    them, and runs of keys: 1 x 8 x 4, 128, 16, 100000 2 x 4 56, 1 x 4 80, 4 x 2 73.
struct Plan {
  int rw, nkw, nrt, splits, chunk;
};
Plan plan(int B, int H, int G, int Tq, int ctx, int D) {
  Plan q;
  const long R = (long)Tq * G;
  const int nb = kv8_blocks(ctx);
  const auto cells = [&](int rw) { return (long)B * H * ((R + rw - 1) / rw); };
  if (R <= 32) {
    q.rw = 16, q.nkw = 4;
  } else if (cells(128) >= 512) {
    q.rw = 128, q.nkw = 1;
  } else if (cells(128) >= 192) {
    q.rw = 128, q.nkw = 2;
  } else if (cells(64) >= 192) {
    q.rw = 64, q.nkw = 4;
  } else if (nb >= 256) {
    q.rw = R <= 64 ? 64 : 128, q.nkw = R <= 64 ? 4 : 2;
  } else {
    q.rw = 32, q.nkw = D == 64 ? 8 : 4;
  }
  const long n = cells(q.rw);
  q.nrt = (int)((R + q.rw - 1) / q.rw);
  long sp = q.rw == 16 ? (768 + n - 1) / n : n <= 128 ? 256 / n : 1;
  long most = (nb + 15) / 16;
  if (q.rw == 16 && n * most <= 128) most = nb <= 24 ? 1 : (nb + 7) / 8;
  if (sp > most) sp = most;
  if (sp > 1024) sp = 1024;
  if (sp < 1) sp = 1;
  q.chunk = (int)((nb + sp - 1) / sp);
  q.splits = (nb + q.chunk - 1) / q.chunk;
  if (q.rw == 16 && n * q.splits <= 256) q.nkw = 8;
  return q;
}

template <int D>
hipError_t launch(hipStream_t st, Attn8Args a, const Plan& q) {
  const long nrec = (long)a.B * a.H * q.nrt * q.splits;
  a.rw = q.rw, a.nrt = q.nrt, a.splits = q.splits, a.chunk = q.chunk;
  const dim3 grid((unsigned)nrec);
  auto go = [&](auto kern, int waves) { hipLaunchKernelGGL(kern, grid, dim3(64 * waves), 0, st, a); };
  if (q.rw == 16) {
    if (q.nkw == 8) go(kv8_rows_kernel<D, 8>, 8);
    else go(kv8_rows_kernel<D, 4>, 4);
  } else if (q.rw == 128) {
    if (q.nkw == 1) go(kv8_tile_kernel<D, 4, 1, 3>, 4);
    else go(kv8_tile_kernel<D, 4, 2, 2>, 8);
  } else if (q.rw == 64) {
    go(kv8_tile_kernel<D, 2, 4, 2>, 8);
  } else if constexpr (D == 64) {
    go(kv8_tile_kernel<D, 1, 8, 2>, 8);
  } else {
    go(kv8_tile_kernel<D, 1, 4, 2>, 4);
  }
  hipError_t e = hipGetLastError();
  if (e == hipSuccess && q.splits > 1) {
    hipLaunchKernelGGL(kv8_join_kernel<D>, dim3((unsigned)((long)a.B * a.H * a.Tq * a.G)), dim3(256), 0, st, a, nrec);
    e = hipGetLastError();
  }
  return e;
}

}  // namespace

// Sizes that plan() can take: heads that a grid holds, and counts that stay in their types.
static bool sizes_ok(int B, int H, int G, int Tq, int ctx) {
  return B >= 1 && H >= 1 && G >= 1 && Tq >= 1 && ctx >= 1 && ctx <= 0x7fffff00 && (long)Tq * G <= 0x7fffff00L &&
         (long)B * H <= 0x7fffffL;
}

extern "C" long mx_kv8_sdpa_ws(int B, int H, int G, int Tq, int ctx, int D) {
  if (!sizes_ok(B, H, G, Tq, ctx) || (D != 64 && D != 128)) return 0;
  const Plan q = plan(B, H, G, Tq, ctx, D);
  return q.splits == 1 ? 0 : (long)B * H * q.nrt * q.splits * q.rw * (D + 2);
}

// How mx_kv8_sdpa cuts a call: t = rows per workgroup (16: the few-row kernel), waves that share the keys, runs of keys, blocks
// of 64 keys per run.
extern "C" void mx_kv8_sdpa_tiling(int B, int H, int G, int Tq, int ctx, int D, int* t) {
  t[0] = t[1] = t[2] = t[3] = 0;
  if (!sizes_ok(B, H, G, Tq, ctx) || (D != 64 && D != 128)) return;
  const Plan q = plan(B, H, G, Tq, ctx, D);
  t[0] = q.rw, t[1] = q.nkw, t[2] = q.splits, t[3] = q.chunk;
}

extern "C" int mx_kv8_sdpa(hipStream_t st, const uint16_t* q, long sq_b, long sq_h, long sq_t, const uint8_t* kc,
                           const uint8_t* vc, const uint8_t* ks, const uint8_t* vs, uint16_t* o, long so_b, long so_t,
                           int B, int H, int G, int Tq, int D, int ctx, const int* len, long len_s, int base, int qpos,
                           int qend, int causal_from, float scale, float* part, long part_elems) {
  if (!q || !kc || !vc || !ks || !vs || !o) return MX_ENULL;
  if (D != 64 && D != 128) return MX_EBADCFG;
  if (!sizes_ok(B, H, G, Tq, ctx)) return MX_ESHAPE;
  if (!(scale > 0.f) || !(scale * 1.4426950408889634f < INFINITY) || causal_from < 0) return MX_ESHAPE;
  if ((sq_b | sq_h | sq_t) % 8 || (so_b | so_t) % 4) return MX_ESHAPE;
  if (((uintptr_t)q | (uintptr_t)kc | (uintptr_t)vc) & 15 || ((uintptr_t)o & 7) || ((uintptr_t)len & 3)) return MX_ELAYOUT;
  const Plan pl = plan(B, H, G, Tq, ctx, D);
  const long nrec = (long)B * H * pl.nrt * pl.splits, rows = (long)B * H * Tq * G;
  if (nrec > 0x7fffffL || (pl.splits > 1 && rows > 0xffffffL)) return MX_ESHAPE;  // 2^32 threads in a grid
  if (pl.splits > 1 && (!part || part_elems < mx_kv8_sdpa_ws(B, H, G, Tq, ctx, D) || ((uintptr_t)part & 15)))
    return MX_ESPLIT;
  const Attn8Args a{q, sq_b, sq_h, sq_t, kc, vc, ks, vs, o, so_b, so_t, part, len, len_s, base, qpos, qend, causal_from,
                    B, H, G, Tq, ctx, 0, 0, 0, 0, scale * 1.4426950408889634f};
  const hipError_t e = D == 64 ? launch<64>(st, a, pl) : launch<128>(st, a, pl);
  return e == hipSuccess ? MX_OK : MX_ELAUNCH;
}
