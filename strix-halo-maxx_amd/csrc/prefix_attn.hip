// Attention of sequences that share a prefix, head dims 64 and 128, G query heads per key head. Sequence b = n S + j of
// prefix n has the prefix's keys (one copy for its S sequences) and keys of its own:
//   O[b, i, h] = sum softmax(scale <Q[b, h, i], key>) value   over the prefix's first plen_n keys and its own keys that it sees
//   own key t is visible to query i iff t < len_b and (not causal or t <= len_b - Tq + i); a query without a key gets zeros.
// A row is a (sequence, query, head of the group) of one key head h: row = (j Tq + i) G + g of the S Tq G that share K and V.
//
// Three ways to cut it (plan()):
//  * rows: 16 or 32 rows per workgroup, from any sequences; its waves go through one list of blocks of keys: the prefix's,
//    then those of each sequence in the tile, which the rows of the others do not see. Few rows: a workgroup reads all keys
//    of its rows once.
//  * both: tiles of 64 or 128 rows over the prefix, which is so read once for each, and in the same launch 16-row
//    tiles over the sequences' own keys. Many sequences of few rows each.
//  * tiles: tiles of 32 - 256 rows of one sequence through the prefix and then its own keys. Prompts.
// Each may cut its list of blocks into runs ("splits"): a run's share (maximum, sum, unnormalised output in fp32) goes to
// memory and the join adds the shares of a row in a fixed order. The host knows capacities only (lengths may be on the
// device), so it fixes the number of runs and the device cuts each list evenly.
//
// Numerics: fp32 scores, sums and outputs; a weight is rounded to bf16 for its product (2^-9 of it on average), its sum takes it
// before that. A masked key reaches no result: blocks that need a mask are searched for infinities and NaN among the values, and
// where there is one (never in ordinary data) it is cleared and two products of indicators with the visibility find the outputs
// that it belongs to. An infinite value of a key that is seen, but whose weight underflows to 0 in fp32, leaves infinity or NaN in its
// column of that row, by which block, wave and run it lies in: 0 times it in a product or a joining factor is NaN, an indicator's
// output infinity.
#include "common.h"

namespace {

struct Seg {  // K or V of one segment: element strides
  const uint16_t* p;
  long s_b, s_h;
  int s_t;
};

struct Args {
  const uint16_t* q;
  long sq_b, sq_h, sq_t;
  Seg pk, pv, k, v;
  uint16_t* o;
  long so_b, so_t;
  const int *plen, *len;  // null: pbase, base alone
  long plen_s, len_s;
  int pbase, base, P, T;
  int N, S, H, G, Tq, causal;
  float sl2;
  // the shares of the tile kernel (a) and of the 16-row kernel (b): rows per tile, tiles per cell, runs, first float of
  // the outputs and of the (maximum, sum) pairs in part
  int rwa, nta, spa, rwb, ntb, spb;
  long na;  // workgroups of the tile kernel
  float *oa, *ma, *ob, *mb;
};

__device__ __forceinline__ int prefix_len(const Args& p, int n) {
  const long l = (long)p.pbase + (p.plen ? p.plen[n * p.plen_s] : 0);
  return (int)min(max(l, 0L), (long)p.P);
}
__device__ __forceinline__ int own_len(const Args& p, int b) {
  const long l = (long)p.base + (p.len ? p.len[b * p.len_s] : 0);
  return (int)min(max(l, 0L), (long)p.T);
}
// own keys that query i of a sequence of len sees
__device__ __forceinline__ int limit(const Args& p, int len, int i) {
  return p.causal ? min(max(len - p.Tq + 1 + i, 0), len) : len;
}

// The order of the 16-byte slots of a key's row in LDS: slot s of key lies at s ^ swz(key). 64 banks hold one row of 128 or
// two of 64 columns; with these bits both the operand reads of K (one slot of 16 keys) and the transposed reads of V (two
// slots of 8 keys, or four of 4) meet every bank once.
template <int D>
__device__ __forceinline__ int swz(int key) {
  const int lo = ((key >> 2) & 1) * 2 + ((key >> 3) & 1);
  return D == 128 ? ((key >> 1) & 1) * 8 + (key & 1) * 4 + lo : ((key >> 1) & 1) * 4 + lo;
}

__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(a), as_bf16x8(b), c, 0, 0, 0);
}
__device__ __forceinline__ float quarters_max(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return halves_max(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
__device__ __forceinline__ float quarters_sum(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return halves_sum(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

// bit 15 of each bf16 of a pair: infinity or NaN; with them, 1.0 where it is +infinity (neg: -infinity) or NaN; cleared
__device__ __forceinline__ uint32_t odd(uint32_t w) {
  return ~(((w & 0x7f807f80u) ^ 0x7f807f80u) + 0x7fff7fffu) & 0x80008000u;
}
__device__ __forceinline__ uint32_t odd(u32x4 v) { return odd(v.x) | odd(v.y) | odd(v.z) | odd(v.w); }
__device__ __forceinline__ uint32_t mark(uint32_t w, uint32_t neg) {  // neg: 0 or ~0
  const uint32_t nan = (w & 0x007f007fu) + 0x7fff7fffu;
  return ((odd(w) & (nan | (w ^ ~neg))) >> 15) * 0x3f80u;
}
__device__ __forceinline__ u32x4 mark(u32x4 v, uint32_t neg) {
  return u32x4{mark(v.x, neg), mark(v.y, neg), mark(v.z, neg), mark(v.w, neg)};
}
__device__ __forceinline__ uint32_t finite(uint32_t w) { return w & ~((odd(w) >> 15) * 0xffffu); }
__device__ __forceinline__ u32x4 finite(u32x4 v) { return u32x4{finite(v.x), finite(v.y), finite(v.z), finite(v.w)}; }
// Column d of the values of keys key .. key + 3 and key + far .. + 3 (0 from `end` on), as an MFMA operand. Slow: for the blocks
// that hold an infinity or NaN.
__device__ __forceinline__ u32x4 column(const uint16_t* v, int st, int d, int key, int far, int end) {
  u32x4 a;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int k = key + (i >> 1) * far + 2 * (i & 1);
    const uint32_t lo = k < end ? v[(long)k * st + d] : 0, hi = k + 1 < end ? v[(long)(k + 1) * st + d] : 0;
    a[i] = lo | hi << 16;
  }
  return a;
}
// 1.0 for the two keys from `key` on that lie below lim
__device__ __forceinline__ uint32_t seen2(int key, int lim) { return (key < lim ? 0x3f80u : 0u) | (key + 1 < lim ? 0x3f800000u : 0u); }

// 2^x of the distance to a maximum that may still be -infinity.
__device__ __forceinline__ float base_of(float m) { return m == -INFINITY ? 0.f : m; }

// A row's sequence, query and head of the group (unsigned 32-bit divisions: signed or 64-bit ones cost a microsecond here).
struct Row {
  int j, i, g;
};
__device__ __forceinline__ Row row_of(const Args& p, int row, int M) {
  Row w;
  w.j = (int)((uint32_t)row / (uint32_t)M);
  const uint32_t r = row - w.j * M;
  w.i = (int)(r / (uint32_t)p.G);
  w.g = (int)r - w.i * p.G;
  return w;
}
// Blocks of run s of `runs` over a list of `total`.
__device__ __forceinline__ int2 run_of(int total, int s, int runs) {
  const uint32_t q = (uint32_t)total / (uint32_t)runs, rest = total - q * runs;
  const int x0 = (int)(s * q + min((uint32_t)s, rest));
  return int2{x0, x0 + (int)q + ((uint32_t)s < rest ? 1 : 0)};
}

// Where the result of a row goes: bf16, or (runs > 1) the share of its record.
struct Out {
  uint16_t* o;
  float *po, *pm;
  float inv;
};
__device__ __forceinline__ uint16_t* out_row(const Args& p, int n, int h, int row, int D) {
  const Row w = row_of(p, row, p.G * p.Tq);
  return p.o + (long)(n * p.S + w.j) * p.so_b + (long)w.i * p.so_t + (long)(h * p.G + w.g) * D;
}
__device__ __forceinline__ void put4(const Out& t, int d, float a, float b, float c, float e) {
  if (t.po)
    *reinterpret_cast<f32x4*>(t.po + d) = f32x4{a, b, c, e};
  else
    *reinterpret_cast<u32x2*>(t.o + d) = u32x2{pack2(a * t.inv, b * t.inv), pack2(c * t.inv, e * t.inv)};
}

// ---------------------------------------------------------------------------------------------- few rows
template <int D, int NW, int RT>
constexpr int rows_lds() {
  return NW * RT * (32 + 16 * D) * 4 > NW * 8192 ? NW * RT * (32 + 16 * D) * 4 : NW * 8192;
}

// Item = (prefix and key head, run, 16 RT rows). The NW waves take the blocks of the run in turn, 8 KB of K and 8 of V each (64
// keys of 64 columns, 32 of 128): K from memory into the 16x16x32 MFMA's registers, V through a piece of LDS of the wave's own
// for the transposed read; the next block is in flight through this one's softmax and product. S^T leaves keys
// 16 t + 4 (lane / 16) + r of row lane % 16 in a lane, and the product with V takes its keys in that order.
// Bound by bytes: where the keys of a head are one workgroup's, by what one CU gets from beyond its L2, about 30 bytes per ns (1 x
// 4 x 32 x 1, 64, 1, 794 + 64 as in plan(): 268 KB a workgroup in 10.4 us); where runs fill the chip, by memory (6 x 8 x 8 x 4,
// 128, 1, 16000 + 200: 432 MB, some of them still in the 256 MB cache, in 60 us); where lengths on the device differ widely, by the
// longest lists, whose runs on_xcd keeps on one or two XCDs (the same with prefixes of 1 - 16000 keys: 52 us). 8 or 16 waves per
// workgroup brought nothing, nor did dealing the runs out by the lengths on the device (3 - 8 us more for lists that are alike, 4 less
// for the most unlike).
template <int D, int NW, int RT, bool PREFIX>
__device__ __forceinline__ void rows_body(const Args& p, uint32_t item, uint8_t* smem) {
  constexpr int KB = 4096 / D, KT = KB / 16, NS = D / 32, NT = D / 16, NV = 8, CPR = D / 8, RW = 16 * RT;
  const int lane = threadIdx.x & 63, kw = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  const uint32_t run = item / (uint32_t)p.ntb, cell = run / (uint32_t)p.spb;
  const int rt = (int)(item - run * p.ntb), s = (int)(run - cell * p.spb), n = (int)(cell / (uint32_t)p.H), h = (int)cell - n * p.H;
  const int M = p.G * p.Tq, R = p.S * M, r0 = rt * RW, rl = min(r0 + RW - 1, R - 1);
  const int j0 = (uint32_t)r0 / (uint32_t)M, jl = (uint32_t)rl / (uint32_t)M;  // the tile's sequences
  u32x4 qf[RT][NS];  // loaded first: everything else waits for the lengths
  int j[RT], iq[RT], lim_own[RT];
#pragma unroll
  for (int y = 0; y < RT; y++) {
    const Row w = row_of(p, min(r0 + 16 * y + c, R - 1), M);
    j[y] = w.j, iq[y] = w.i;
    const uint16_t* qrow = p.q + (long)(n * p.S + w.j) * p.sq_b + (long)(h * p.G + w.g) * p.sq_h + (long)w.i * p.sq_t + 8 * g;
#pragma unroll
    for (int e = 0; e < NS; e++) qf[y][e] = *reinterpret_cast<const u32x4*>(qrow + 32 * e);
  }
  // lane u of 32: sequence j0 + u, the keys that any / every row of it in this tile sees, blocks up to and with it
  const int us = lane & 31, ju = min(j0 + us, jl), lenu = own_len(p, n * p.S + ju);
  const int kendu = limit(p, lenu, (uint32_t)min(rl - ju * M, M - 1) / (uint32_t)p.G);
  const int kallu = limit(p, lenu, (uint32_t)max(r0 - ju * M, 0) / (uint32_t)p.G);
  const int plen = PREFIX ? prefix_len(p, n) : 0, npb = (plen + KB - 1) / KB;
  int cum = j0 + us <= jl ? (kendu + KB - 1) / KB : 0;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const int o = __shfl_up(cum, d, 32);
    cum += us >= d ? o : 0;
  }
  cum += npb;
  const int2 share = run_of(__builtin_amdgcn_readlane(cum, 31), s, p.spb);
  const int x0 = share.x, x1 = share.y;
#pragma unroll
  for (int y = 0; y < RT; y++) lim_own[y] = limit(p, own_len(p, n * p.S + j[y]), iq[y]);

  struct Blk {
    const uint16_t *k, *v;
    int sk, sv, key0, kend, seq;  // seq: the sequence whose own keys these are, or -1
    bool masked;
  } b;
  int u = 0;
  auto locate = [&](int x) {
    if (PREFIX && x < npb) {
      b.key0 = KB * x, b.kend = plen, b.seq = -1, b.masked = b.key0 + KB > plen;
      b.sk = p.pk.s_t, b.sv = p.pv.s_t;
      b.k = p.pk.p + n * p.pk.s_b + h * p.pk.s_h + (long)b.key0 * b.sk;
      b.v = p.pv.p + n * p.pv.s_b + h * p.pv.s_h + (long)b.key0 * b.sv;
      return;
    }
    while (x >= __builtin_amdgcn_readlane(cum, u)) u++;
    const int first = u ? __builtin_amdgcn_readlane(cum, u - 1) : npb;
    const long seq = n * p.S + j0 + u;
    b.key0 = KB * (x - first), b.kend = __builtin_amdgcn_readlane(kendu, u), b.seq = j0 + u;
    b.masked = jl > j0 || b.key0 + KB > __builtin_amdgcn_readlane(kallu, u);
    b.sk = p.k.s_t, b.sv = p.v.s_t;
    b.k = p.k.p + seq * p.k.s_b + h * p.k.s_h + (long)b.key0 * b.sk;
    b.v = p.v.p + seq * p.v.s_b + h * p.v.s_h + (long)b.key0 * b.sv;
  };
  u32x4 k[KT][NS], v[NV];
  auto get = [&]() {  // keys past the last are the last one again (masked); 32-bit offsets from the block's first key
    const int last = b.kend - 1 - b.key0;
    const uint8_t *kb = reinterpret_cast<const uint8_t*>(b.k), *vb = reinterpret_cast<const uint8_t*>(b.v);
#pragma unroll
    for (int t = 0; t < KT; t++) {
      const uint32_t off = (uint32_t)min(16 * t + c, last) * (uint32_t)(2 * b.sk) + 16 * g;
#pragma unroll
      for (int e = 0; e < NS; e++) k[t][e] = *reinterpret_cast<const u32x4*>(kb + off + 64 * e);
    }
#pragma unroll
    for (int e = 0; e < NV; e++) {
      const uint32_t off = (uint32_t)min(lane / CPR + 64 / CPR * e, last) * (uint32_t)(2 * b.sv) + lane % CPR * 16;
      v[e] = *reinterpret_cast<const u32x4*>(vb + off);
    }
  };
  f32x4 o[RT][NT];
  float m[RT], l[RT];
#pragma unroll
  for (int y = 0; y < RT; y++) {
    m[y] = -INFINITY, l[y] = 0.f;
#pragma unroll
    for (int t = 0; t < NT; t++) o[y][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  // Addresses in the wave's V block: the slots of a lane differ by constants in the bits of the swizzle. They are made in the
  // loop (the empty asm keeps them there): kept across it they would take 24 registers.
  const int ra = lane / CPR, q0 = 4 * g + (c >> 2);
  const uint32_t wr0 = kw * 8192 + ra * 2 * D + (((lane % CPR) ^ swz<D>(ra)) * 16);
  const uint32_t rd0 = kw * 8192 + q0 * 2 * D + (((c & 3) >> 1) ^ swz<D>(q0)) * 16 + (c & 1) * 8;
  uint32_t wr = wr0, rd = rd0;
  auto stage = [&](const u32x4(&x)[NV]) {
#pragma unroll
    for (int e = 0; e < NV; e++)
      *reinterpret_cast<u32x4*>(smem + ((wr ^ (swz<D>(64 / CPR * e) * 16)) + 64 / CPR * e * 2 * D)) = x[e];
  };
  auto operand = [&](int t, int e) {
    const u32x2 lo = lds_read_tr16(reinterpret_cast<const uint16_t*>(smem + (rd ^ (32 * t)) + 64 * D * e));
    const u32x2 hi = lds_read_tr16(reinterpret_cast<const uint16_t*>(smem + (rd ^ (32 * t)) + 64 * D * e + 32 * D));
    return u32x4{lo.x, lo.y, hi.x, hi.y};
  };
  int x = x0 + kw;
  bool late = false;  // a block with a mask holds an infinity or NaN
  if (x < x1) {
    locate(x);
    get();
    for (;;) {
      asm volatile("" : "+v"(wr), "+v"(rd));
      f32x4 st[RT][KT];
#pragma unroll
      for (int y = 0; y < RT; y++)
#pragma unroll
        for (int t = 0; t < KT; t++) {
          st[y][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int e = 0; e < NS; e++) st[y][t] = mfma16(k[t][e], qf[y][e], st[y][t]);
        }
      if (b.masked) {
        const int key = b.key0 + 4 * g;
        int lim[RT];
#pragma unroll
        for (int y = 0; y < RT; y++) lim[y] = b.seq < 0 ? b.kend : b.seq == j[y] ? lim_own[y] : 0;
        asm volatile("");  // keeps the branch: as selects all this would be computed for every block
        uint32_t bad = 0;
#pragma unroll
        for (int e = 0; e < NV; e++) bad |= odd(v[e]);
        if (__any(bad != 0)) {
          late = true;
#pragma unroll
          for (int e = 0; e < NV; e++) v[e] = finite(v[e]);
        }
#pragma unroll
        for (int y = 0; y < RT; y++)
#pragma unroll
          for (int t = 0; t < KT; t++)
#pragma unroll
            for (int r = 0; r < 4; r++) st[y][t][r] = key + 16 * t + r < lim[y] ? st[y][t][r] : -INFINITY;
      }
      stage(v);
      x += NW;
      const bool more = x < x1;
      if (more) {
        locate(x);
        get();
      }
      u32x4 w[RT][KT / 2];
#pragma unroll
      for (int y = 0; y < RT; y++) {
        float mx = -INFINITY;
#pragma unroll
        for (int t = 0; t < KT; t++)
#pragma unroll
          for (int r = 0; r < 4; r++) mx = fmaxf(mx, st[y][t][r]);
        mx = quarters_max(mx) * p.sl2;
        const bool grow = mx > m[y];
        if (__any(grow)) {
          const float al = grow ? __builtin_amdgcn_exp2f(m[y] - mx) : 1.f;
          l[y] *= al;
#pragma unroll
          for (int t = 0; t < NT; t++)
#pragma unroll
            for (int r = 0; r < 4; r++) o[y][t][r] *= al;
          m[y] = grow ? mx : m[y];
        }
        const float mb = base_of(m[y]);
#pragma unroll
        for (int t = 0; t < KT; t++)
#pragma unroll
          for (int r = 0; r < 4; r += 2) {
            const float a = __builtin_amdgcn_exp2f(__builtin_fmaf(st[y][t][r], p.sl2, -mb));
            const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(st[y][t][r + 1], p.sl2, -mb));
            l[y] += a + e;
            w[y][t / 2][2 * (t % 2) + r / 2] = pack2(a, e);
          }
      }
#pragma unroll
      for (int e = 0; e < KT / 2; e++)
#pragma unroll
        for (int t = 0; t < NT; t++) {
          const u32x4 a = operand(t, e);
#pragma unroll
          for (int y = 0; y < RT; y++) o[y][t] = mfma16(a, w[y][e], o[y][t]);
        }
      if (!more) break;
    }
  }
  if (late) {
    u = 0;
    for (x = x0 + kw; x < x1; x += NW) {
      locate(x);
      if (!b.masked) continue;
      for (int key = 4 * g; key < 4 * g + KB; key += 32) {
#pragma unroll
        for (int t = 0; t < NT; t++) {
          const u32x4 a = column(b.v, b.sv, 16 * t + c, key, 16, b.kend - b.key0);
#pragma unroll
          for (int y = 0; y < RT; y++) {
            const int lim = (b.seq < 0 ? b.kend : b.seq == j[y] ? lim_own[y] : 0) - b.key0;
            const u32x4 vis = {seen2(key, lim), seen2(key + 2, lim), seen2(key + 16, lim), seen2(key + 18, lim)};
            const f32x4 none = {0.f, 0.f, 0.f, 0.f};
            const f32x4 up = mfma16(mark(a, 0u), vis, none), dn = mfma16(mark(a, ~0u), vis, none);
#pragma unroll
            for (int r = 0; r < 4; r++) {
              o[y][t][r] += up[r] > 0.f ? INFINITY : 0.f;
              o[y][t][r] -= dn[r] > 0.f ? INFINITY : 0.f;
            }
          }
        }
      }
    }
  }
  // ---- the waves' shares meet in LDS, added in wave order; wave kw finishes the tiles e with e % NW = kw
  __syncthreads();
  float* cm = reinterpret_cast<float*>(smem);
  f32x4* co = reinterpret_cast<f32x4*>(cm + NW * 2 * RW);
#pragma unroll
  for (int y = 0; y < RT; y++) {
    const float ly = quarters_sum(l[y]);
    if (g == 0) {
      cm[kw * 2 * RW + 16 * y + c] = m[y];
      cm[kw * 2 * RW + RW + 16 * y + c] = ly;
    }
#pragma unroll
    for (int t = 0; t < NT; t++) co[((kw * RT + y) * NT + t) * 64 + lane] = o[y][t];
  }
  __syncthreads();
#pragma unroll
  for (int y = 0; y < RT; y++) {
    const int rr = 16 * y + c, row = r0 + rr;
    if (row >= R) continue;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < NW; w++) top = fmaxf(top, cm[w * 2 * RW + rr]);
    const float tb = base_of(top);
    float L = 0.f, f[NW];
#pragma unroll
    for (int w = 0; w < NW; w++) {
      f[w] = __builtin_amdgcn_exp2f(cm[w * 2 * RW + rr] - tb);
      L += cm[w * 2 * RW + RW + rr] * f[w];
    }
    Out t;
    t.o = out_row(p, n, h, row, D);
    t.po = p.ob ? p.ob + ((long)item * RW + rr) * D : nullptr;
    t.inv = L == 0.f ? 0.f : 1.f / L;
    if (t.po && kw == 0 && g == 0) {
      p.mb[(long)item * 2 * RW + rr] = top;
      p.mb[(long)item * 2 * RW + RW + rr] = L;
    }
    for (int e = kw; e < NT; e += NW) {
      f32x4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < NW; w++) {
        const f32x4 z = co[((w * RT + y) * NT + e) * 64 + lane];
#pragma unroll
        for (int r = 0; r < 4; r++) a[r] += z[r] * f[w];
      }
      put4(t, 16 * e + 4 * g, a[0], a[1], a[2], a[3]);
    }
  }
}

// The dispatcher sends workgroup i to XCD i % 8; neighbouring items (the row tiles over the same keys) go to one XCD, whose
// L2 then holds those keys once.
__device__ __forceinline__ uint32_t on_xcd(uint32_t i, uint32_t n) {
  const uint32_t per = n / 8, rem = n % 8, x = i % 8, idx = i / 8;
  return x < rem ? x * (per + 1) + idx : rem * (per + 1) + (x - rem) * per + idx;
}

template <int D, int NW, int RT>
__global__ __launch_bounds__(64 * NW, 2) void prefix_rows_kernel(Args p) {
  __shared__ __attribute__((aligned(1024))) uint8_t smem[rows_lds<D, NW, RT>()];
  rows_body<D, NW, RT, true>(p, on_xcd(blockIdx.x, gridDim.x), smem);
}

// ---------------------------------------------------------------------------------------------- many rows
template <int D, int NQW, int NKW, int KB, int S>
struct Tile {
  static constexpr int CPR = D / 8, KBW = KB / NKW, NST = KBW / 32, NW = NQW * NKW, DT = D / 32;
  static constexpr int STAGE_B = 4 * KB * D;             // K and V of a block
  static constexpr int NIW = STAGE_B / 1024 / NW;        // load instructions per wave and block
  static constexpr int RING_B = S * STAGE_B;
  static constexpr int COMB_B = NKW > 1 ? NW * 64 * (2 + D / 2) * 4 : 0;
  static constexpr int BYTES = RING_B > COMB_B ? RING_B : COMB_B;
  static_assert(KBW % 32 == 0 && STAGE_B % (1024 * NW) == 0 && BYTES <= 160 * 1024, "ring");
};

// Item = (cell, run, 32 NQW rows) on the 32x32x16 MFMA; a cell is a prefix and a key head, and (SEQ) one of its sequences.
// NQW query waves x NKW key waves; blocks of KB keys go through an LDS ring of S stages by the asynchronous load, the
// block's keys shared among the key waves, whose shares are added at the end. S^T = K Q^T leaves a lane the scores of one
// row, in the key order that the product with V (transposed reads) takes.
// Prompts are bound by a SIMD's two waves issuing softmax and products by turns: 2 x 2 x 8 x 4, 128, 1024, 8001 + 1500 takes 560 us
// = 0.87 PFLOP/s (a large library product 1.13), the matrix unit busy 39 % of the time, the vector ALU 36 %, no bank conflicts.
// Tried and slower: the next block's scores before this one's softmax in one wave (588 - 620 us: registers), waves in two groups
// that swap softmax and products at barriers (1217 us and more), rings of 3 and 4 stages (the same). Over a long prefix with few
// rows it is bound by memory: 1 x 16 x 8 x 4, 128, 1, 131071 + 512 reads 557 MB in 104 us, 5.4 TB/s.
template <int D, int NQW, int NKW, int KB, int S, bool SEQ>
__device__ __forceinline__ void tile_body(const Args& p, uint32_t item, uint8_t* smem) {
  using C = Tile<D, NQW, NKW, KB, S>;
  constexpr int CPR = C::CPR, KBW = C::KBW, NST = C::NST, DT = C::DT, RB = 2 * D;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int qg = wave % NQW, kw = wave / NQW, c = lane & 31, hk = lane >> 5;
  const int M = p.G * p.Tq, R = SEQ ? M : p.S * M;
  const uint32_t run = item / (uint32_t)p.nta, cell = run / (uint32_t)p.spa, nh = SEQ ? cell / (uint32_t)p.S : cell;
  const int rt = (int)(item - run * p.nta), s = (int)(run - cell * p.spa), j0 = SEQ ? (int)(cell - nh * p.S) : 0;
  const int n = (int)(nh / (uint32_t)p.H), h = (int)nh - n * p.H;
  const int r0 = rt * 32 * NQW, row = r0 + 32 * qg + c, rc = min(row, R - 1);
  const int plen = prefix_len(p, n), npb = (plen + KB - 1) / KB;
  int lim_own = 0, kend = 0, kmin = 0, wend = 0, kall = 0;  // own keys that the row, any / every row, any / every row of this wave sees
  if (SEQ) {
    const int len = own_len(p, n * p.S + j0);
    const auto query = [&](int row) { return (int)((uint32_t)min(row, R - 1) / (uint32_t)p.G); };
    lim_own = limit(p, len, query(rc));
    kend = limit(p, len, query(r0 + 32 * NQW - 1));
    kmin = limit(p, len, query(r0));
    wend = limit(p, len, query(r0 + 32 * qg + 31));
    kall = limit(p, len, query(r0 + 32 * qg));
  }
  const int2 share = run_of(npb + (kend + KB - 1) / KB, s, p.spa);
  const int x0 = share.x, x1 = share.y;
  const uint32_t sbase = lds_off(smem);
  const uint16_t *pkb = p.pk.p + n * p.pk.s_b + h * p.pk.s_h, *pvb = p.pv.p + n * p.pv.s_b + h * p.pv.s_h;
  const uint16_t *kb = p.k.p + (long)(n * p.S + j0) * p.k.s_b + h * p.k.s_h, *vb = p.v.p + (long)(n * p.S + j0) * p.v.s_b + h * p.v.s_h;
  const int spk = p.pk.s_t, spv = p.pv.s_t, sok = p.k.s_t, sov = p.v.s_t;
  // instruction q of a block brings 1 KB of the K part, then of the V part, in LDS order; keys past the last are it again
  auto issue = [&](int x) {
    const bool pre = !SEQ || x < npb;
    const int first = (pre ? x : x - npb) * KB, last = (pre ? plen : kend) - 1 - first;
    const uint32_t dst = sbase + (uint32_t)((uint32_t)(x - x0) % S) * C::STAGE_B;
    int stk = spk, stv = spv;
    const uint16_t *kf = pkb, *vf = pvb;
    if (!pre) stk = sok, stv = sov, kf = kb, vf = vb;
    kf += (long)first * stk, vf += (long)first * stv;
#pragma unroll
    for (int e = 0; e < C::NIW; e++) {
      const int q = wave * C::NIW + e;
      const bool isv = q >= KB * CPR / 64;
      const int ch = (q * 64 + lane) % (KB * CPR), key = ch / CPR, slot = (ch % CPR) ^ swz<D>(key);
      dma16s(isv ? vf : kf, (uint32_t)min(key, last) * (uint32_t)(2 * (isv ? stv : stk)) + slot * 16, dst + q * 1024);
    }
  };
  f32x16 o[DT];
#pragma unroll
  for (int t = 0; t < DT; t++)
#pragma unroll
    for (int e = 0; e < 16; e++) o[t][e] = 0.f;
  float m = -INFINITY, l = 0.f;
  bool late = false;  // a block with a mask holds an infinity or NaN
  bf16x8 qf[D / 16];
  if (x0 < x1) issue(x0);
  {
    const Row w = row_of(p, rc, M);
    const uint16_t* qrow = p.q + (long)(n * p.S + j0 + w.j) * p.sq_b + (long)(h * p.G + w.g) * p.sq_h + (long)w.i * p.sq_t + 8 * hk;
#pragma unroll
    for (int e = 0; e < D / 16; e++) qf[e] = as_bf16x8(*reinterpret_cast<const u32x4*>(qrow + 16 * e));
  }
  __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): the compiler does not count the LDS-DMA loads, so nothing of its own may
                                       // be in flight beside them (gfx9 encoding; expcnt, lgkmcnt not waited)
#pragma unroll
  for (int e = 1; e < S - 1; e++)
    if (x0 + e < x1) issue(x0 + e);

  for (int x = x0; x < x1; x++) {
    wait_stages<C::NIW, S - 2>(x1 - 1 - x);
    __syncthreads();
    if (x + S - 1 < x1) issue(x + S - 1);
    const bool pre = !SEQ || x < npb;
    const int kx = (pre ? x : x - npb) * KB, k0 = kx + kw * KBW;  // the block's first key, and that of this wave's share
    if (kx + KB > (pre ? plen : kmin)) {
      // some row does not see all of these keys: their values must be finite
      uint8_t* vb0 = smem + ((uint32_t)(x - x0) % S) * C::STAGE_B + KB * RB;
      int bad = 0;
#pragma unroll 1
      for (int i = threadIdx.x; i < KB * CPR; i += 64 * C::NW) {
        const u32x4 y = *reinterpret_cast<const u32x4*>(vb0 + 16 * i);
        if (odd(y)) *reinterpret_cast<u32x4*>(vb0 + 16 * i) = finite(y), bad = 1;
      }
      late |= __syncthreads_or(bad) != 0;
    }
    if (k0 >= (pre ? plen : wend)) continue;
    const uint8_t* kst = smem + ((uint32_t)(x - x0) % S) * C::STAGE_B + kw * KBW * RB;
    const uint8_t* vst = kst + KB * RB;
    f32x16 st[NST];
#pragma unroll
    for (int t = 0; t < NST; t++)
#pragma unroll
      for (int e = 0; e < 16; e++) st[t][e] = 0.f;
#pragma unroll
    for (int e = 0; e < D / 16; e++)
#pragma unroll
      for (int t = 0; t < NST; t++) {
        const int key = 32 * t + c;  // the swizzle depends on key % 16 only
        const u32x4 a = *reinterpret_cast<const u32x4*>(kst + key * RB + ((2 * e + hk) ^ swz<D>(key)) * 16);
        st[t] = mfma32(as_bf16x8(a), qf[e], st[t]);
      }
    const bool masked = k0 + KBW > (pre ? plen : kall);
    const int lim = pre ? plen : lim_own, key0 = k0 + 4 * hk;
    float mx = -INFINITY;
    if (masked) {
      asm volatile("");  // keeps the branch: as selects the mask would be computed for every block
#pragma unroll
      for (int t = 0; t < NST; t++)
#pragma unroll
        for (int r = 0; r < 16; r++)
          st[t][r] = key0 + 32 * t + 8 * (r >> 2) + (r & 3) < lim ? st[t][r] : -INFINITY;
    }
#pragma unroll
    for (int t = 0; t < NST; t++)
#pragma unroll
      for (int r = 0; r < 16; r++) mx = fmaxf(mx, st[t][r]);
    // the running maximum is raised when a row's block maximum passes it by more than 8: weights stay below 2^8, and what
    // they are relative to cancels in the end
    mx = halves_max(mx) * p.sl2;
    const bool grow = mx > m + 8.f;
    if (__any(grow)) {
      const float al = grow ? __builtin_amdgcn_exp2f(m - mx) : 1.f;
      l *= al;
#pragma unroll
      for (int t = 0; t < DT; t++)
#pragma unroll
        for (int e = 0; e < 16; e++) o[t][e] *= al;
      m = grow ? mx : m;
    }
    const float mb = base_of(m);
    uint32_t w[NST][8];
#pragma unroll
    for (int t = 0; t < NST; t++)
#pragma unroll
      for (int r = 0; r < 16; r += 2) {
        const float a = __builtin_amdgcn_exp2f(__builtin_fmaf(st[t][r], p.sl2, -mb));
        const float b = __builtin_amdgcn_exp2f(__builtin_fmaf(st[t][r + 1], p.sl2, -mb));
        l += a + b;
        w[t][r >> 1] = pack2(a, b);
      }
    // ---- O^T += V^T P^T: step (t, e) takes keys 32 t + 16 e + {4 hk .. 4 hk + 3, 8 + 4 hk ..}
    const int jr = (lane & 15) >> 2, jc = 4 * (lane & 3) + 16 * ((lane >> 4) & 1);
    auto operand = [&](int t, int e, int dt) {
      const int r1 = 32 * t + 16 * e + 4 * hk + jr, slot = (32 * dt + jc) >> 3, sub = (jc & 7) * 2;
      const u32x2 lo = lds_read_tr16(reinterpret_cast<const uint16_t*>(vst + r1 * RB + (slot ^ swz<D>(r1)) * 16 + sub));
      const u32x2 hi = lds_read_tr16(reinterpret_cast<const uint16_t*>(vst + (r1 + 8) * RB + (slot ^ swz<D>(r1 + 8)) * 16 + sub));
      return u32x4{lo.x, lo.y, hi.x, hi.y};
    };
#pragma unroll
    for (int t = 0; t < NST; t++)
#pragma unroll
      for (int e = 0; e < 2; e++) {
        const u32x4 pb = {w[t][4 * e], w[t][4 * e + 1], w[t][4 * e + 2], w[t][4 * e + 3]};
#pragma unroll
        for (int dt = 0; dt < DT; dt++) o[dt] = mfma32(as_bf16x8(operand(t, e, dt)), as_bf16x8(pb), o[dt]);
      }
  }
  if (late) {
    for (int x = x0; x < x1; x++) {
      const bool pre = !SEQ || x < npb;
      const int kx = (pre ? x : x - npb) * KB, k0 = kx + kw * KBW, end = pre ? plen : kend;
      if (kx + KB <= (pre ? plen : kmin) || k0 >= (pre ? plen : wend)) continue;
      const int lim = pre ? plen : lim_own;
#pragma unroll 1
      for (int k1 = k0 + 4 * hk; k1 < k0 + 4 * hk + KBW; k1 += 16) {
        const u32x4 vis = {seen2(k1, lim), seen2(k1 + 2, lim), seen2(k1 + 8, lim), seen2(k1 + 10, lim)};
#pragma unroll
        for (int dt = 0; dt < DT; dt++) {
          __builtin_amdgcn_sched_barrier(0);  // one at a time: few registers for what never happens
          const u32x4 a = column(pre ? pvb : vb, pre ? p.pv.s_t : p.v.s_t, 32 * dt + c, k1, 8, end);
#pragma unroll
          for (int neg = 0; neg < 2; neg++) {
            __builtin_amdgcn_sched_barrier(0);
            f32x16 hit;
#pragma unroll
            for (int r = 0; r < 16; r++) hit[r] = 0.f;
            hit = mfma32(as_bf16x8(mark(a, neg ? ~0u : 0u)), as_bf16x8(vis), hit);
#pragma unroll
            for (int r = 0; r < 16; r++) o[dt][r] += hit[r] > 0.f ? (neg ? -INFINITY : INFINITY) : 0.f;
          }
        }
      }
    }
  }

  float L = halves_sum(l);
  Out t;
  auto aim = [&]() {
    t.o = out_row(p, n, h, SEQ ? j0 * M + row : row, D);
    t.po = p.oa ? p.oa + ((long)item * p.rwa + 32 * qg + c) * D : nullptr;
    t.inv = L == 0.f ? 0.f : 1.f / L;
    if (t.po && kw == 0 && hk == 0) {
      p.ma[(long)item * 2 * p.rwa + 32 * qg + c] = m;
      p.ma[(long)item * 2 * p.rwa + p.rwa + 32 * qg + c] = L;
    }
  };
  if constexpr (NKW > 1) {
    // ---- the key waves' shares, added in wave order; wave kw finishes the register groups u with u % NKW = kw
    float* cm = reinterpret_cast<float*>(smem);
    f32x4* co = reinterpret_cast<f32x4*>(cm + C::NW * 128);
    wait_vm<0>();
    __syncthreads();
    cm[wave * 128 + lane] = m;
    cm[wave * 128 + 64 + lane] = L;
#pragma unroll
    for (int u = 0; u < 4 * DT; u++)
      co[(wave * 4 * DT + u) * 64 + lane] =
          f32x4{o[u / 4][4 * (u % 4)], o[u / 4][4 * (u % 4) + 1], o[u / 4][4 * (u % 4) + 2], o[u / 4][4 * (u % 4) + 3]};
    __syncthreads();
    m = -INFINITY;
#pragma unroll
    for (int w = 0; w < NKW; w++) m = fmaxf(m, cm[(w * NQW + qg) * 128 + lane]);
    const float mb = base_of(m);
    float f[NKW];
    L = 0.f;
#pragma unroll
    for (int w = 0; w < NKW; w++) {
      f[w] = __builtin_amdgcn_exp2f(cm[(w * NQW + qg) * 128 + lane] - mb);
      L += cm[(w * NQW + qg) * 128 + 64 + lane] * f[w];
    }
    if (row >= R) return;
    aim();
    for (int u = kw; u < 4 * DT; u += NKW) {
      f32x4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < NKW; w++) {
        const f32x4 y = co[((w * NQW + qg) * 4 * DT + u) * 64 + lane];
#pragma unroll
        for (int r = 0; r < 4; r++) a[r] += y[r] * f[w];
      }
      put4(t, 8 * u + 4 * hk, a[0], a[1], a[2], a[3]);
    }
  } else {
    if (row >= R) return;
    aim();
#pragma unroll
    for (int u = 0; u < 4 * DT; u++)
      put4(t, 8 * u + 4 * hk, o[u / 4][4 * (u % 4)], o[u / 4][4 * (u % 4) + 1], o[u / 4][4 * (u % 4) + 2],
           o[u / 4][4 * (u % 4) + 3]);
  }
}

template <int D, int NQW, int NKW, int KB, int S>
__global__ __launch_bounds__(64 * NQW * NKW, 2) void prefix_tile_kernel(Args p) {
  __shared__ __attribute__((aligned(1024))) uint8_t smem[Tile<D, NQW, NKW, KB, S>::BYTES];
  tile_body<D, NQW, NKW, KB, S, true>(p, on_xcd(blockIdx.x, p.na), smem);
}
template <int D, int NQW, int NKW, int KB, int S>
__global__ __launch_bounds__(64 * NQW * NKW, 2) void prefix_both_kernel(Args p) {
  constexpr int A = Tile<D, NQW, NKW, KB, S>::BYTES, B = rows_lds<D, NQW * NKW, 1>();
  __shared__ __attribute__((aligned(1024))) uint8_t smem[A > B ? A : B];
  if (blockIdx.x < p.na) tile_body<D, NQW, NKW, KB, S, false>(p, on_xcd(blockIdx.x, p.na), smem);
  else rows_body<D, NQW * NKW, 1, false>(p, blockIdx.x - p.na, smem);
}

// The shares of one row: 256 / WPR threads... one workgroup has 4 / WPR rows of WPR waves; D / 4 threads with 4 columns each
// form a group, and the groups take the shares in turn, in a fixed order. Bound by the latency of two trips to memory (pairs, then
// outputs, of which the first four are asked for at once): four waves a row 4.9 us for 512 rows of 36 runs, one wave 5.9 for 2048
// of 17.
template <int D, int WPR>
__global__ __launch_bounds__(256) void prefix_join_kernel(Args p, uint32_t rows) {
  constexpr int TD = D / 4, NT = 64 * WPR, NG = NT / TD, RPB = 256 / NT;
  __shared__ f32x4 so[RPB][NG][TD];
  __shared__ float red[RPB][2][WPR];
  const int tid = threadIdx.x % NT, rb = threadIdx.x / NT, wave = tid >> 6, d = tid % TD, grp = tid / TD;
  const uint32_t at = blockIdx.x * RPB + rb;  // (prefix and key head, row); rows beyond the last do the last again
  const int M = p.G * p.Tq, R = p.S * M;
  const uint32_t ic = min(at, rows - 1), cell = ic / (uint32_t)R;
  const int row = (int)(ic - cell * R), n = (int)(cell / (uint32_t)p.H), h = (int)cell - n * p.H;
  // the row's shares: spa of the tile kernel (if any), then spb of the 16-row kernel
  const bool seq = p.oa && !p.ob;  // tiles of one sequence
  const int js = seq ? (int)((uint32_t)row / (uint32_t)M) : 0, ra = row - js * M, ta = p.oa ? (int)((uint32_t)ra / (uint32_t)p.rwa) : 0;
  const int qa = ra - ta * p.rwa, tb = row / p.rwb, qb = row % p.rwb;
  const long ca = seq ? (long)cell * p.S + js : cell;
  const int na = p.oa ? p.spa : 0, nr = na + (p.ob ? p.spb : 0);
  auto rec_a = [&](int s) { return (ca * p.spa + s) * p.nta + ta; };
  auto rec_b = [&](int s) { return ((long)cell * p.spb + s - na) * p.ntb + tb; };
  auto stat = [&](int s, int which) {
    return s < na ? p.ma[rec_a(s) * 2 * p.rwa + which * p.rwa + qa] : p.mb[rec_b(s) * 2 * p.rwb + which * p.rwb + qb];
  };
  const auto source = [&](int s) {
    return reinterpret_cast<const f32x4*>((s < na ? p.oa + (rec_a(s) * p.rwa + qa) * D : p.ob + (rec_b(s) * p.rwb + qb) * D) + 4 * d);
  };
  // the first four shares of a group are on their way while the factors are found
  f32x4 y0[4];
  float m0[4];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int s = min(grp + NG * i, nr - 1);
    y0[i] = *source(s);
    m0[i] = stat(s, 0);
  }
  float m = -INFINITY, l = 0.f;
  if (tid < nr) m = stat(tid, 0), l = stat(tid, 1);
  for (int s = tid + NT; s < nr; s += NT) m = fmaxf(m, stat(s, 0));
  const float first = m;
  m = wave_max(m);
  if (WPR > 1) {
    if ((tid & 63) == 0) red[rb][0][wave] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WPR; w++) m = fmaxf(m, red[rb][0][w]);
  }
  const float mb = base_of(m);
  if (nr <= NT) {
    l *= __builtin_amdgcn_exp2f(first - mb);
  } else {
    l = 0.f;
    for (int s = tid; s < nr; s += NT) l += stat(s, 1) * __builtin_amdgcn_exp2f(stat(s, 0) - mb);
  }
  l = wave_total(l);
  if (WPR > 1) {
    if ((tid & 63) == 0) red[rb][1][wave] = l;
    __syncthreads();
    l = 0.f;
#pragma unroll
    for (int w = 0; w < WPR; w++) l += red[rb][1][w];
  }
  f32x4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const float f = __builtin_amdgcn_exp2f(m0[i] - mb);
    if (grp + NG * i < nr) {
#pragma unroll
      for (int e = 0; e < 4; e++) a[e] += y0[i][e] * f;
    }
  }
#pragma unroll 4
  for (int s = grp + 4 * NG; s < nr; s += NG) {
    const float f = __builtin_amdgcn_exp2f(stat(s, 0) - mb);
    const f32x4 y = *source(s);
#pragma unroll
    for (int e = 0; e < 4; e++) a[e] += y[e] * f;
  }
  so[rb][grp][d] = a;
  __syncthreads();
  if (grp || at >= rows) return;
#pragma unroll
  for (int u = 1; u < NG; u++) a += so[rb][u][d];
  const float inv = l == 0.f ? 0.f : 1.f / l;
  *reinterpret_cast<u32x2*>(out_row(p, n, h, row, D) + 4 * d) = u32x2{pack2(a[0] * inv, a[1] * inv), pack2(a[2] * inv, a[3] * inv)};
}

// How a problem is cut, by its capacities. M rows of a sequence, R of the sequences of a prefix; us on one MI355X (HIP-graph
// replays; prefixes x sequences x key heads x group, head dim, queries, prefix + own keys):
//  * M < 32 and R <= 32 or R P < 2^20: rows. Up to 24 blocks of keys (1536 keys of 64 values, 768 of 128) in one run: one launch
//    and no workspace (1 x 4 x 32 x 1, 64, 1, 794 + 64 10.8 in a graph and, bound by the host, 11.5 called eagerly; 8 runs and the
//    join 9.2 and 15.5: a captured step, as the text decoder's, pays 1.6 a layer for it). More of them in 256 workgroups where
//    runs of 128 keys give that many (1 x 8 x 8 x 4, 128, 1, 2000 + 200 12.3, in 128 workgroups 13.4). 32 rows per workgroup instead of 16 where the keys would be read again too often, from R P =
//    400000 on (6 x 8 x 8 x 4, 128, 1, 16000 + 200 60, 16 rows 88; 1 x 8 x 8 x 4, 128, 1, 2000 + 200 14.0, 16 rows 12.6);
//  * more rows of M < 32: both. Up to 64 rows 2 x 4 waves (1 x 16 x 8 x 4, 128, 1, 131071 + 512 109, 4 x 1 112), else 4 x 1 (1 x
//    64 x 8 x 4, 128, 1, 65536 + 200 99, 2 x 2 111; rows of 32 175). Below, rows (5 x 48 x 4 x 7, 128, 1, 2000 + 500 53, both 60;
//    1 x 16 x 8 x 4, 128, 1, 2000 + 1000 19.1, both 21.6);
//  * M >= 32: tiles of no more than twice M's rows, 8 x 1 waves where 256-row tiles give two workgroups per CU (2 x 2 x 8 x 4,
//    128, 1024, 8001 + 1500 565, 4 x 1 595), 4 x 1 where 128-row ones do, 4 x 2 down to three quarters of one per CU (1 x 4 x 8 x
//    4, 128, 200, 3000 + 300 63, 4 x 1 73, 2 x 4 79), 2 x 4 with 64-row tiles down to the same, 1 x 4 below (1 x 4 x 8 x 4, 128,
//    64, 2000 + 100 26, 2 x 4 29, 4 x 1 in runs 37; 1 x 8 x 32 x 1, 64, 32, 730 + 32 12.2). Over 8192 keys or more instead of
//    those two as many rows as M has, and runs (1 x 1 x 8 x 4, 128, 256, 16000 + 256 8 x 1 in 8 runs 82, 4 x 2 in 4 90, 1 x 4 in
//    one 141).
struct Plan {
  int kind, nqw, nkw, nta, spa, rtb, ntb, spb;  // kind 0: rows, 1: both, 2: tiles
  long na, nb;                                  // workgroups of the tile kernel and of the 16-row kernel
};
long cdiv(long a, long b) { return (a + b - 1) / b; }
long clamped(long v, long lo, long hi) { return v < lo || hi < lo ? lo : v > hi ? hi : v; }
Plan plan(int N, int S, int H, int G, int Tq, int P, int T, int D) {
  Plan q = {};
  const long M = (long)G * Tq, R = S * M, cells = (long)N * H;
  q.spa = q.spb = 1;
  if (M >= 32) {
    q.kind = 2;
    const auto wgs = [&](int rw) { return cells * S * cdiv(M, rw); };
    const long nb = cdiv(P, 64) + cdiv(T, 64);
    if (M > 128 && wgs(256) >= 512) q.nqw = 8, q.nkw = 1;
    else if (M > 64 && wgs(128) >= 512) q.nqw = 4, q.nkw = 1;
    else if (M > 64 && wgs(128) >= 192) q.nqw = 4, q.nkw = 2;
    else if (M > 32 && nb >= 128) q.nqw = M <= 64 ? 2 : M <= 128 ? 4 : 8, q.nkw = M <= 64 ? 4 : M <= 128 ? 2 : 1;
    else if (M > 32 && wgs(64) >= 192) q.nqw = 2, q.nkw = 4;
    else q.nqw = 1, q.nkw = 4;
    q.nta = (int)cdiv(M, 32 * q.nqw);
    const long w = cells * S * q.nta;
    q.spa = (int)clamped(w <= 128 ? 256 / w : 1, 1, clamped(nb / 16, 1, 1024));
    q.na = w * q.spa;
    return q;
  }
  const double work = (double)R * P;
  q.kind = R <= 32 || work < 1048576. ? 0 : 1;
  q.rtb = q.kind == 0 && R > 16 && work >= 400000. ? 2 : 1;
  q.ntb = (int)cdiv(R, 16 * q.rtb);
  const long wb = cells * q.ntb, seqs = clamped(cdiv(16 * q.rtb, M), 1, S);  // sequences in a tile, nearly
  const long kb = 4096 / D, nb = (q.kind == 0 ? cdiv(P, kb) : 0) + seqs * cdiv(T, kb);
  q.spb = (int)clamped(256 / wb, 1, clamped(nb * kb / (q.kind == 0 ? 128 : 512), 1, 1024));
  if (q.kind == 0 && nb <= 24) q.spb = 1;
  q.nb = wb * q.spb;
  if (q.kind == 0) return q;
  q.nqw = R <= 64 ? 2 : 4, q.nkw = R <= 64 ? 4 : 1;
  q.nta = (int)cdiv(R, 32 * q.nqw);
  const long wa = cells * q.nta;
  q.spa = (int)clamped((R <= 64 ? 256 : 512) / wa, 1, clamped(cdiv(P, 64) / 8, 1, 1024));
  q.na = wa * q.spa;
  return q;
}
bool shares(const Plan& q) { return q.kind == 1 || q.spa > 1 || q.spb > 1; }
long ws_floats(const Plan& q, int D) {
  return shares(q) ? q.na * 32 * q.nqw * (D + 2) + q.nb * 16 * q.rtb * (D + 2) : 0;
}

template <int D>
hipError_t launch(hipStream_t st, const Args& a, const Plan& q) {
  const auto go = [&](auto kern, int waves) {
    hipLaunchKernelGGL(kern, dim3((unsigned)(q.na + q.nb)), dim3(64 * waves), 0, st, a);
  };
  if (q.kind == 0) {
    if (q.rtb == 2) go(prefix_rows_kernel<D, 4, 2>, 4);
    else go(prefix_rows_kernel<D, 4, 1>, 4);
  } else if (q.kind == 1) {
    if (q.nqw == 4) go(prefix_both_kernel<D, 4, 1, 64, 2>, 4);
    else go(prefix_both_kernel<D, 2, 4, 128, 2>, 8);
  } else if (q.nqw == 8) {
    go(prefix_tile_kernel<D, 8, 1, 64, 2>, 8);
  } else if (q.nqw == 4) {
    if (q.nkw == 1) go(prefix_tile_kernel<D, 4, 1, 64, 2>, 4);
    else go(prefix_tile_kernel<D, 4, 2, 64, 2>, 8);
  } else if (q.nqw == 2) {
    go(prefix_tile_kernel<D, 2, 4, 128, 2>, 8);
  } else {
    go(prefix_tile_kernel<D, 1, 4, 128, 2>, 4);
  }
  hipError_t e = hipGetLastError();
  if (e == hipSuccess && shares(q)) {
    const long rows = (long)a.N * a.S * a.H * a.G * a.Tq;
    // four waves a row for many shares, fewer of them where few rows leave CUs idle (24 rows of 21 shares, the whole call: 9.1 us, by
    // single waves 10.0; 2048 rows of 17: 60.6, single 58.6)
    if (q.spa + q.spb > (rows < 1024 ? 16 : 32))
      hipLaunchKernelGGL((prefix_join_kernel<D, 4>), dim3((unsigned)rows), dim3(256), 0, st, a, (uint32_t)rows);
    else
      hipLaunchKernelGGL((prefix_join_kernel<D, 1>), dim3((unsigned)cdiv(rows, 4)), dim3(256), 0, st, a, (uint32_t)rows);
    e = hipGetLastError();
  }
  return e;
}

bool sizes_ok(int N, int S, int H, int G, int Tq, int P, int T) {
  return N >= 1 && S >= 1 && H >= 1 && G >= 1 && Tq >= 1 && P >= 0 && T >= 0 && P <= 0x7fffff00 && T <= 0x7fffff00 &&
         (long)N * S <= 0x7fffff && (long)N * S * H <= 0x7fffff && (long)G * Tq <= 0x7fffff00L &&
         (long)S * G * Tq <= 0x7fffff00L && (double)N * S * H * G * Tq <= 16777215.0;
}

}  // namespace

extern "C" long mx_sdpa_prefix_ws(int N, int S, int H, int G, int Tq, int P, int T, int D) {
  if (!sizes_ok(N, S, H, G, Tq, P, T) || (D != 64 && D != 128)) return 0;
  return ws_floats(plan(N, S, H, G, Tq, P, T, D), D);
}

// t: 0 rows, 1 both, 2 tiles; query and key waves of the tile kernel, its runs; rows per workgroup and runs of the few-row kernel.
extern "C" void mx_sdpa_prefix_tiling(int N, int S, int H, int G, int Tq, int P, int T, int D, int* t) {
  for (int i = 0; i < 6; i++) t[i] = 0;
  if (!sizes_ok(N, S, H, G, Tq, P, T) || (D != 64 && D != 128)) return;
  const Plan q = plan(N, S, H, G, Tq, P, T, D);
  t[0] = q.kind, t[1] = q.nqw, t[2] = q.nkw, t[3] = q.kind ? q.spa : 0, t[4] = 16 * q.rtb, t[5] = q.kind < 2 ? q.spb : 0;
}

extern "C" int mx_sdpa_prefix(hipStream_t st, const uint16_t* q, const uint16_t* pk, const uint16_t* pv, const uint16_t* k,
                              const uint16_t* v, uint16_t* o, const long* strides, long so_b, long so_t, int N, int S, int H, int G,
                              int Tq, int D, int P, int T, const int* plen, long plen_s, int pbase, const int* len, long len_s,
                              int base, int causal, float scale, float* part, long part_elems) {
  if (!q || !o || !strides || (P > 0 && (!pk || !pv)) || (T > 0 && (!k || !v))) return MX_ENULL;
  if (D != 64 && D != 128) return MX_EBADCFG;
  if (!sizes_ok(N, S, H, G, Tq, P, T)) return MX_ESHAPE;
  if (!(scale > 0.f) || !(scale * 1.4426950408889634f < INFINITY)) return MX_ESHAPE;
  long any = 0;
  for (int i = 0; i < 15; i++) any |= strides[i];
  if (any % 8 || (so_b | so_t) % 4) return MX_ESHAPE;
  for (int i = 5; i < 15; i += 3)  // a block's rows are addressed by 32-bit byte offsets from its first
    if (strides[i] < 0 || strides[i] > 0x7fffffL) return MX_ESHAPE;
  if (((uintptr_t)q | (uintptr_t)pk | (uintptr_t)pv | (uintptr_t)k | (uintptr_t)v) & 15 || ((uintptr_t)o & 7) ||
      ((uintptr_t)plen & 3) || ((uintptr_t)len & 3))
    return MX_ELAYOUT;
  const auto seg = [&](const uint16_t* x, int i) { return Seg{x, strides[i], strides[i + 1], (int)strides[i + 2]}; };
  const Plan pl = plan(N, S, H, G, Tq, P, T, D);
  if (pl.na + pl.nb > 0x7fffffL) return MX_ESHAPE;  // 2^32 threads in a grid
  const long need = ws_floats(pl, D);
  if (need && (!part || part_elems < need || ((uintptr_t)part & 15))) return MX_ESPLIT;
  Args a{q, strides[0], strides[1], strides[2], seg(pk, 3), seg(pv, 6), seg(k, 9), seg(v, 12),
         o, so_b, so_t, plen, len, plen_s, len_s, pbase, base, P, T, N, S, H, G, Tq, causal, scale * 1.4426950408889634f,
         32 * pl.nqw, pl.nta, pl.spa, 16 * pl.rtb, pl.ntb, pl.spb, pl.na, nullptr, nullptr, nullptr, nullptr};
  if (need) {
    const long fa = pl.na * a.rwa, fb = pl.nb * a.rwb;
    if (pl.na) a.oa = part, a.ma = part + fa * D + fb * D;
    if (pl.nb) a.ob = part + fa * D, a.mb = part + fa * D + fb * D + 2 * fa;
  }
  const hipError_t e = D == 64 ? launch<64>(st, a, pl) : launch<128>(st, a, pl);
  return e == hipSuccess ? MX_OK : MX_ELAUNCH;
}
