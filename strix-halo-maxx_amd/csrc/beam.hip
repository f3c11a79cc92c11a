// Beam search: the selection over beams and vocabulary, and the reordering of the slots of a cache.
//
// Selection. Beam w of search b with score s_w offers each token v at the value
//   s_w + x[w, v] - log sum_u exp(x[w, u]);
// a finished beam offers eos alone, at s_w. The k largest of the W V values, in falling order, ties by the lower w V + v.
// Two launches:
//  * parts: a workgroup reads 4 x 64 E logits of a row once: their maximum, the sum of their exponentials, and their k largest
//    as (logit, token) keys. Within a row the order of the values is that of the logits, so no sum is needed yet.
//  * merge: one workgroup per search adds the parts' sums, and takes the k largest of all parts' keys by their values.
// The sums are fp32 within a part and fp64 from there on, values are fp64 and rounded to fp32 once; where two of one beam are
// equal in fp64, their logits decide, as they do exactly.
#include <float.h>

#include "common.h"

namespace {

typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));  // rows start at any element
constexpr float LOG2E = 1.4426950408889634f;
constexpr int MAXW = 64, MAXK = 64, MT = 1024, MAXL = 8192;  // MT, MAXL: threads and lists of the merge

// Order-preserving bits of a float; -0 counts as 0. NONE: -infinity and below, no candidate.
__device__ __forceinline__ uint32_t bits_of(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float float_of(uint32_t b) { return __uint_as_float(b ^ ((b >> 31) ? 0x80000000u : 0xffffffffu)); }
constexpr uint32_t NONE = 0x007fffffu;  // bits_of(-infinity)

struct SelArgs {
  const void* x;
  long sx_b, sx_w;  // elements
  const float* score;
  const uint8_t* done;  // may be null
  int B, W, V, k, eos, segs;
  uint64_t* keys;  // [row][seg][k]: bits << 32 | ~token, falling; 0: none
  float* stat;     // [row][seg][2]: maximum, sum of exp(x - maximum)
  float* o_score;
  int *o_parent, *o_token;
  uint8_t* o_done;  // may be null
};

// 8 logits from v0 on; -infinity past the row's end
template <class T>
__device__ __forceinline__ void load8(const T* row, int v0, int V, float (&f)[8]) {
  if (v0 + 8 <= V) {
    if constexpr (sizeof(T) == 2) {
      const u32x4 w = *reinterpret_cast<const u32x4_any*>(row + v0);
#pragma unroll
      for (int e = 0; e < 4; e++) f[2 * e] = lo_bf(w[e]), f[2 * e + 1] = hi_bf(w[e]);
    } else {
      const u32x4 a = *reinterpret_cast<const u32x4_any*>(row + v0), b = *reinterpret_cast<const u32x4_any*>(row + v0 + 4);
#pragma unroll
      for (int e = 0; e < 4; e++) f[e] = __uint_as_float(a[e]), f[4 + e] = __uint_as_float(b[e]);
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; e++) {
    f[e] = -INFINITY;
    if (v0 + e < V) {
      if constexpr (sizeof(T) == 2) f[e] = bf2f(row[v0 + e]);
      else f[e] = row[v0 + e];
    }
  }
}

// A lane holds E / 8 chunks of 8 neighbouring logits, chunk i of a wave's lanes 512 in a row. The wave's threshold is the
// k-th largest of its lanes' maxima (found bit by bit from ballots: 32 steps whatever k is): k lanes have a logit that large,
// so no smaller one is among the k largest, and the larger ones lie in fewer than k lanes. What passes the largest of the four
// waves' thresholds, and the first k of a wave that equal it, go to LDS, where every one counts the larger ones: its rank.
// Bound by the vector ALU's work per logit (maximum, subtraction, scaling, exponential, sum, comparison) and, in fp32, nearly by
// memory: 16 x 16 rows of 131071 fp32 logits 27.6 us = 4.9 TB/s; 32 x 8 of 51200 bf16 11.
template <class T, int E>
__global__ __launch_bounds__(256) void beam_parts_kernel(SelArgs p) {
  extern __shared__ uint64_t cand[];  // 4 ((k - 1) E + k)
  __shared__ int count;
  __shared__ float ms[4][2];
  __shared__ uint32_t bound[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int seg = blockIdx.x % p.segs;
  const long row = blockIdx.x / p.segs;
  const float score = p.score[row];
  if ((p.done && p.done[row]) || !(fabsf(score) < INFINITY)) return;  // the merge does not look at it
  const T* x = reinterpret_cast<const T*>(p.x) + row / p.W * p.sx_b + row % p.W * p.sx_w;
  if (tid == 0) count = 0;
  const int v0 = seg * 256 * E + wave * 64 * E + lane * 8;
  float f[E];
#pragma unroll
  for (int i = 0; i < E / 8; i++) load8(x, v0 + 512 * i, p.V, *reinterpret_cast<float(*)[8]>(f + 8 * i));
  float m = f[0];
#pragma unroll
  for (int e = 1; e < E; e++) m = fmaxf(m, f[e]);
  const float mw = wave_max(m), mb = mw == -INFINITY ? 0.f : mw;
  float s = 0.f;
#pragma unroll
  for (int e = 0; e < E; e++) s += __builtin_amdgcn_exp2f((f[e] - mb) * LOG2E);
  s = wave_total(s);
  if (lane == 0) ms[wave][0] = mw, ms[wave][1] = s;
  // ---- the wave's threshold, from the lanes' maxima (bf16 logits: their upper half is all there is)
  constexpr int LOW = sizeof(T) == 2 ? 16 : 0;
  const uint32_t top = m > -INFINITY ? bits_of(m) >> LOW : 0u;  // (NaN is no maximum)
  uint32_t t = 0;
#pragma unroll 4
  for (int b = 31 - LOW; b >= 0; b--) {
    const uint32_t c = t | (1u << b);
    if (__popcll(__ballot(top >= c)) >= p.k) t = c;
  }
  if constexpr (E == 16) {  // more than 32 to select: many lanes' smallest maximum is a poor bound: the k-th largest logit itself
    uint32_t u[E];
#pragma unroll
    for (int e = 0; e < E; e++) u[e] = f[e] > -INFINITY ? bits_of(f[e]) >> LOW : 0u;
    uint32_t c0 = 0;
#pragma unroll 1
    for (int b = 31 - LOW; b >= 0; b--) {
      const uint32_t c = c0 | (1u << b);
      int n = 0;
#pragma unroll
      for (int e = 0; e < E; e++) n += __popcll(__ballot(u[e] >= c));
      if (n >= p.k) c0 = c;
    }
    t = c0;
  }
  if (lane == 0) bound[wave] = t;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 4; w++) t = max(t, bound[w]);  // the largest of the waves' thresholds serves them all
  // fewer than k lanes in each, or -infinity: every finite logit
  const bool all = t <= NONE >> LOW;
  const float tf = all ? -INFINITY : float_of(t << LOW | (LOW && !(t >> 15) ? 0xffffu : 0u)), least = all ? -FLT_MAX : tf;
  uint32_t ge = 0, eq = 0;  // of the lane's logits, a bit for each
#pragma unroll
  for (int e = 0; e < E; e++) ge |= f[e] >= least ? 1u << e : 0u;
  for (; ge; ge &= ge - 1) {  // a few logits in a few lanes: read again, which costs less than work on each of the E registers
    const int e = __ffs(ge) - 1, v = v0 + 512 * (e / 8) + e % 8;
    float g;
    if constexpr (sizeof(T) == 2) g = bf2f(x[v]);
    else g = x[v];
    if (g > tf) cand[atomicAdd(&count, 1)] = (uint64_t)bits_of(g) << 32 | ~(uint32_t)v;
    else eq |= 1u << e;
  }
  if (!all) {
    int left = p.k;  // places for logits that equal the threshold, in the order of their tokens
#pragma unroll
    for (int i = 0; i < E / 8; i++) {
      const uint32_t mine = eq >> (8 * i) & 0xffu;
      uint64_t who = __ballot(mine != 0);
      while (who && left > 0) {  // wave-uniform
        const int l = __ffsll((unsigned long long)who) - 1;
        who &= who - 1;
        uint32_t bits = __builtin_amdgcn_readlane(mine, l);
        const int nl = __popc(bits);
        if (lane == l)
          for (int j = left; bits && j > 0; j--, bits &= bits - 1)
            cand[atomicAdd(&count, 1)] = (uint64_t)bits_of(tf) << 32 | ~(uint32_t)(v0 + 512 * i + __ffs(bits) - 1);
        left -= nl;
      }
    }
  }
  __syncthreads();
  const int n = count;
  uint64_t* out = p.keys + (row * p.segs + seg) * p.k;
  for (int i = tid; i < n; i += 256) {
    const uint64_t mine = cand[i];
    int rank = 0;
#pragma unroll 4
    for (int j = 0; j < n; j++) rank += cand[j] > mine;
    if (rank < p.k) out[rank] = mine;
  }
  if (tid >= n && tid < p.k) out[tid] = 0;
  if (tid == 0) {
    float M = -INFINITY, S = 0.f;
#pragma unroll
    for (int w = 0; w < 4; w++) M = fmaxf(M, ms[w][0]);
    const float Mb = M == -INFINITY ? 0.f : M;
#pragma unroll
    for (int w = 0; w < 4; w++) S += ms[w][1] * __builtin_amdgcn_exp2f((ms[w][0] == -INFINITY ? -INFINITY : ms[w][0] - Mb) * LOG2E);
    float* st = p.stat + (row * p.segs + seg) * 2;
    st[0] = M, st[1] = S;
  }
}

// Order-preserving bits of a double (not NaN); 0 stands for no candidate.
__device__ __forceinline__ uint64_t bits_of(double x) {
  const uint64_t u = (uint64_t)__double_as_longlong(x + 0.);
  return u ^ ((uint64_t)((int64_t)u >> 63) | 0x8000000000000000ull);
}
__device__ __forceinline__ double double_of(uint64_t b) {
  return __longlong_as_double((int64_t)(b ^ ((b >> 63) ? 0x8000000000000000ull : ~0ull)));
}
typedef uint64_t u64x2 __attribute__((ext_vector_type(2)));

// A list is a part's keys; a finished beam's is its one continuation. The k-th largest head of the lists bounds what can be
// selected, and a key at place i of a list whose head has rank r has i + r larger ones: few keys are left to be ranked. What
// takes the time is three rounds to memory, one after the other: the sums, the heads, the keys behind them (32 searches of 8 beams
// of 7 parts 6.2 us, 16 of 16 of 16 9.7).
__global__ __launch_bounds__(MT) void beam_merge_kernel(SelArgs p) {
  extern __shared__ u64x2 sh[];  // (value, key), key = ~logit's bits << 32 | token: the lists' heads [nl], then candidates
  __shared__ double base[MAXW];  // score - log of the sum
  __shared__ float big[MAXW];    // largest logit
  __shared__ int state[MAXW];    // 0: offers nothing, 1: its logits, 2: eos
  __shared__ int best[MAXK], count;
  __shared__ int above[2][31];
  const int tid = threadIdx.x, nl = p.W * p.segs;
  const long b = blockIdx.x;
  u64x2 *head = sh, *cand = head + nl;
  int* rank = reinterpret_cast<int*>(cand + p.k * (p.k + 1) / 2);  // heads and their ranks, then the candidates' beams and ranks
  int *cw = rank, *cr = rank + p.k * (p.k + 1) / 2;
  if (tid == 0) count = 0;
  if (tid < p.k) best[tid] = -1;
  if (tid < 62) above[tid / 31][tid % 31] = 0;
  const uint64_t* keys = p.keys + b * nl * p.k;
  const uint64_t first = tid < nl ? keys[(long)tid * p.k] : 0;
  int per = 1;  // threads of a row: no more than it has parts, a wave with few rows spends long on their fp64 functions
  while (per < p.segs && per < 64 && 2 * per * p.W <= MT) per *= 2;
  const int w0 = tid / per, in = tid % per;
  if (w0 < p.W) {
    const long row = b * p.W + w0;
    const float score = p.score[row];
    int st = fabsf(score) < INFINITY ? (p.done && p.done[row] ? 2 : 1) : 0;
    double c = score;
    float M = -INFINITY;
    if (st == 1) {  // the same for all threads of the row
      const float* s = p.stat + row * p.segs * 2;
      double sum = 0.;  // NaN stays: the comparisons leave the maximum alone
      for (int i = in; i < p.segs; i += per) {
        const float m = s[2 * i], x = s[2 * i + 1];
        if (m > M) sum *= M == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((M - m) * LOG2E), M = m;
        sum += m == -INFINITY ? x : x * __builtin_amdgcn_exp2f((m - M) * LOG2E);
      }
      for (int d = per / 2; d; d >>= 1) {
        const float m = __shfl_xor(M, d, 64);
        const double x = __shfl_xor(sum, d, 64);
        const float top = fmaxf(M, m), tb = top == -INFINITY ? 0.f : top;
        sum = (M == -INFINITY ? sum : sum * __builtin_amdgcn_exp2f((M - tb) * LOG2E)) +
              (m == -INFINITY ? x : x * __builtin_amdgcn_exp2f((m - tb) * LOG2E));
        M = top;
      }
      c = (double)score - log(sum);
      if (!(fabs(c) < INFINITY && fabsf(M) < INFINITY)) st = 0;  // NaN or +infinity among the logits, or nothing above -infinity
    }
    if (in == 0) base[w0] = c, big[w0] = M, state[w0] = st;
  }
  __syncthreads();
  const auto value = [&](int w, uint64_t key) {
    return u64x2{bits_of(((double)float_of((uint32_t)(key >> 32)) - (double)big[w]) + base[w]), ~key};
  };
  for (int l = tid; l < nl; l += MT) {
    const int w = (int)((uint32_t)l / (uint32_t)p.segs);
    u64x2 c = {0, 0};
    const uint64_t key = l < MT ? first : keys[(long)l * p.k];
    if (state[w] == 2 && l == w * p.segs) c = u64x2{bits_of(base[w]), (uint64_t)p.eos};
    if (state[w] == 1 && key) c = value(w, key);
    head[l] = c;
  }
  __syncthreads();
  // The ranks of those of n values that can be among the k largest: place[i] = which << 16 | rank. Returns how many they are
  const auto ranks = [&](int n, const u64x2* v, int* place, int (&above)[31], auto beam) {
    int nc = n;
    if (n > 128) {  // those whose upper 20 bits are no less than the k-th largest's (0 without so many), two bits at a time. Two
                    // searches of 400 and of 224 lists: 20 and 23 us, all ranked 40 and 31; 256 by 16 waves: 38.1 and 37.7
      uint32_t top[MAXL / MT], t = 0;
#pragma unroll
      for (int j = 0; j < MAXL / MT; j++) top[j] = tid + j * MT < n ? (uint32_t)(v[tid + j * MT].x >> 32) : 0u;
      for (int bit = 0; bit < 20; bit += 2) {
        const uint32_t d = 0x40000000u >> bit;
        int* cnt = above + 1 + 3 * bit / 2;
        int some[3] = {0, 0, 0};
#pragma unroll
        for (int j = 0; j < MAXL / MT; j++) {
#pragma unroll
          for (int i = 0; i < 3; i++) some[i] += __popcll(__ballot(top[j] >= t + (i + 1) * d));
          if (n <= (j + 1) * MT) break;
        }
        if ((tid & 63) < 3) atomicAdd(cnt + (tid & 63), (tid & 63) == 0 ? some[0] : (tid & 63) == 1 ? some[1] : some[2]);
        __syncthreads();
        t += cnt[2] >= p.k ? 3 * d : cnt[1] >= p.k ? 2 * d : cnt[0] >= p.k ? d : 0u;
      }
      for (int i = tid; i < n; i += MT)
        if (v[i].x && (uint32_t)(v[i].x >> 32) >= t) place[atomicAdd(above, 1)] = i << 16;
      __syncthreads();
      nc = above[0];
    } else {
      for (int i = tid; i < n; i += MT) place[i] = i << 16;
      __syncthreads();
    }
    // every thread compares one with a share of all
    const int ways = nc && nc < MT ? MT / nc : 1, share = (n + ways - 1) / ways;
    for (int e = tid; e < nc * ways; e += MT) {
      const int at = (int)((uint32_t)e % (uint32_t)nc), i0 = (int)((uint32_t)e / (uint32_t)nc) * share, i1 = min(i0 + share, n);
      const int a = place[at] >> 16;
      const u64x2 c = v[a];
      if (!c.x) continue;
      int r = 0, same = a >= i0 && a < i1 ? -1 : 0;
#pragma unroll 8
      for (int i = i0; i < i1; i++) {
        const uint64_t y = v[i].x;
        r += y > c.x;
        same += y == c.x;
      }
      if (same) {  // rare, so that the loop above is two comparisons a value
        const int w = beam(a);
        for (int i = i0; i < i1; i++)
          if (v[i].x == c.x) r += beam(i) < w || (beam(i) == w && v[i].y < c.y);
      }
      atomicAdd(place + at, r);
    }
    __syncthreads();
    return nc;
  };
  const int nh = ranks(nl, head, rank, above[0], [&](int l) { return l / p.segs; });
  for (int a = tid; a < nh; a += MT) {
    const int r = rank[a] & 0xffff, l = rank[a] >> 16;
    if (r < p.k && head[l].x) best[r] = l;
  }
  __syncthreads();
  const uint64_t least = best[p.k - 1] < 0 ? 0 : head[best[p.k - 1]].x;
#pragma unroll 2
  for (int q = tid; q < p.k * p.k; q += MT) {
    const int r = q / p.k, i = q % p.k, l = best[r];
    if (l < 0 || i + r >= p.k) continue;
    const int w = l / p.segs;
    u64x2 c = head[l];
    if (i) {
      const uint64_t key = state[w] == 1 ? keys[(long)l * p.k + i] : 0;
      if (!key) continue;
      c = value(w, key);
    }
    if (c.x < least) continue;
    const int at = atomicAdd(&count, 1);
    cand[at] = c, cw[at] = w;
  }
  __syncthreads();
  const int n = count, nc = ranks(n, cand, cr, above[1], [&](int i) { return cw[i]; });
  const long o = b * p.k;
  for (int i = tid; i < nc; i += MT) {
    const int r = cr[i] & 0xffff, a = cr[i] >> 16, token = (int)(uint32_t)cand[a].y;
    if (r >= p.k) continue;
    p.o_score[o + r] = (float)double_of(cand[a].x);
    p.o_parent[o + r] = cw[a];
    p.o_token[o + r] = token;
    if (p.o_done) p.o_done[o + r] = token == p.eos;
  }
  if (tid >= n && tid < p.k) {  // fewer candidates than places
    p.o_score[o + tid] = -INFINITY;
    p.o_parent[o + tid] = 0;
    p.o_token[o + tid] = max(p.eos, 0);
    if (p.o_done) p.o_done[o + tid] = 1;
  }
}

// Logits per lane. Fewer fill the CUs earlier, but leave the merge longer lists, which costs more (us for the whole selection with
// 32, 16, 8 per lane: 1 x 4 x 51200 11.8, 11.5, 12.6; 8 x 8 x 51200 13.7, 15.3, 17.5; 32 x 8 x 51200 18.0, 21.9, 32.3; 16 x 16 x
// 131071 fp32 38, 53, 66). More than 32 to select: 16, for the LDS of what is handed over (1 x 64 x 51200: 44, 8 per lane 52).
int per_lane(int k) { return k <= 32 ? 32 : 16; }
int segments(int V, int k) { return (V + 256 * per_lane(k) - 1) / (256 * per_lane(k)); }

// ---------------------------------------------------------------------------------------------- slots
struct MoveArgs {
  uint8_t* x;
  long s_n, s_s, s_h, s_t;  // bytes
  const int* parent;
  long sp_g, sp_w;
  const int* len;  // may be null: base
  long len_s;
  int base, unit, first, T, G, W, H, cpr;  // cpr: pieces per row
  unsigned nblk;
};

// x[n, g W + w, h, t] = x[n, g W + parent[g, w], h, t] for first <= t < rows of the parent. A thread owns one piece (16, 4 or 1
// bytes) of a row in every slot of a group, loads what moves and then stores it, so the copy is in place in any order and no
// two threads meet. Bound by the bytes: slots that do not change are not touched. What a beam step of
// the text decoder moves (48 K and V of 4 slots x 32 heads x 40 rows x 128 bytes) takes 8.4 us among others, 10.7 waited for; 16 of 64
// slots x 8 heads x 1 - 500 rows x 256 bytes 143. The 8-bit cache's four buffers of each layer are a call each, bound by the
// launches: 96 of them for 24 layers of 4 slots take 264 us in a graph, for some 50 MB.
template <class U, int WM>
__global__ __launch_bounds__(256) void move_kernel(MoveArgs p) {
  __shared__ long from[WM];  // byte offset of slot w's parent; the rows that it takes from it
  __shared__ int rows[WM];
  const unsigned blk = blockIdx.x % p.nblk;
  long c = blockIdx.x / p.nblk;
  const int h = (int)(c % p.H), g = (int)(c / p.H % p.G);
  const long n = c / p.H / p.G;
  if (threadIdx.x < WM) {
    const int w = threadIdx.x, src = w < p.W ? p.parent[g * p.sp_g + w * p.sp_w] : w;
    int r = 0;
    if (src != w && src >= 0 && src < p.W) {
      const long len = (long)p.base + (p.len ? p.len[(g * p.W + src) * p.len_s] : 0);
      r = (int)min((max(len, 0L) + p.unit - 1) / p.unit, (long)p.T);
    }
    rows[w] = r;
    from[w] = (long)src * p.s_s;
  }
  __syncthreads();
  int most = 0;
  long spare = 0;
#pragma unroll
  for (int w = 0; w < WM; w++)
    if (rows[w] > most) most = rows[w], spare = from[w];
  const long q = (long)blk * 256 + threadIdx.x;
  const long t = p.first + q / p.cpr;
  if (t >= most) return;
  uint8_t* at = p.x + n * p.s_n + (long)g * p.W * p.s_s + h * p.s_h + t * p.s_t + q % p.cpr * sizeof(U);
  U v[WM];
#pragma unroll
  for (int w = 0; w < WM; w++)  // what does not move loads what the slot that moves most does: one run of loads, no branches
    v[w] = *reinterpret_cast<const U*>(at + (t < rows[w] ? from[w] : spare));
#pragma unroll
  for (int w = 0; w < WM; w++)
    if (t < rows[w]) *reinterpret_cast<U*>(at + w * p.s_s) = v[w];
}

template <class U>
void move(hipStream_t st, const MoveArgs& a, unsigned grid) {
  const auto go = [&](auto kern) { hipLaunchKernelGGL(kern, dim3(grid), dim3(256), 0, st, a); };
  if (a.W <= 4) go(move_kernel<U, 4>);
  else if (a.W <= 8) go(move_kernel<U, 8>);
  else if (a.W <= 16) go(move_kernel<U, 16>);
  else if (a.W <= 32) go(move_kernel<U, 32>);
  else go(move_kernel<U, 64>);
}

// the merge's LDS: values and keys of heads and candidates; ranks of heads, and in the same place beams and ranks of candidates
long merge_lds(int W, int segs, int k) {
  const long nl = (long)W * segs, nc = k * (k + 1) / 2;
  return 16 * (nl + nc) + 4 * (nl > 2 * nc ? nl : 2 * nc);
}
bool select_ok(int B, int W, int V, int k) {
  if (B < 1 || W < 1 || W > MAXW || V < 1 || V > 0x7fff0000 || k < 1 || k > MAXK || (long)B * W > 0x7fffffL) return false;
  const long rows = (long)B * W, segs = segments(V, k);
  // (2^32 threads in a grid: B workgroups of MT in the merge, one of 256 for each part. 2048 bytes: what the merge has beside its
  // lists)
  return (long)B * MT <= 0xffffffffL && rows * segs <= 0x7fffffL && W * segs <= MAXL && merge_lds(W, (int)segs, k) <= 160 * 1024 - 2048;
}

}  // namespace

// Bytes of workspace of mx_beam_select; 0 for what it refuses.
extern "C" long mx_beam_select_ws(int B, int W, int V, int k) {
  if (!select_ok(B, W, V, k)) return 0;
  return (long)B * W * segments(V, k) * (8L * k + 8);
}

extern "C" int mx_beam_select(hipStream_t st, const void* x, int fp32, long sx_b, long sx_w, const float* score,
                              const uint8_t* done, int eos, int B, int W, int V, int k, float* o_score, int* o_parent,
                              int* o_token, uint8_t* o_done, void* ws, long ws_bytes) {
  if (!x || !score || !o_score || !o_parent || !o_token) return MX_ENULL;
  if (!select_ok(B, W, V, k)) return MX_ESHAPE;
  if (eos >= V || (eos < 0 && done)) return MX_ESHAPE;
  if (((uintptr_t)x & (fp32 ? 3 : 1)) || (((uintptr_t)score | (uintptr_t)o_score | (uintptr_t)o_parent | (uintptr_t)o_token) & 3))
    return MX_ELAYOUT;
  const long rows = (long)B * W;
  const int segs = segments(V, k), E = per_lane(k);
  const long lds = merge_lds(W, segs, k);
  if (!ws || ws_bytes < mx_beam_select_ws(B, W, V, k) || ((uintptr_t)ws & 7)) return MX_ESPLIT;
  uint64_t* keys = reinterpret_cast<uint64_t*>(ws);
  const SelArgs a{x, sx_b, sx_w, score, done, B, W, V, k, eos, segs, keys, reinterpret_cast<float*>(keys + rows * segs * k),
                  o_score, o_parent, o_token, o_done};
  const dim3 grid((unsigned)(rows * segs));
  const auto go = [&](auto kern) {
    const size_t sh = 4 * ((k - 1) * (size_t)E + k) * 8;  // what four waves can hand over
    hipLaunchKernelGGL(kern, grid, dim3(256), sh, st, a);
  };
  const auto parts = [&](auto t) {
    typedef decltype(t) T;
    E == 32 ? go(beam_parts_kernel<T, 32>) : go(beam_parts_kernel<T, 16>);
  };
  fp32 ? parts(0.f) : parts(uint16_t{});
  if (hipGetLastError() != hipSuccess) return MX_ELAUNCH;
  hipLaunchKernelGGL(beam_merge_kernel, dim3((unsigned)B), dim3(MT), (size_t)lds, st, a);
  return hipGetLastError() == hipSuccess ? MX_OK : MX_ELAUNCH;
}

extern "C" int mx_reorder_slots(hipStream_t st, void* x, long s_n, long s_s, long s_h, long s_t, int N, int G, int W, int H, int T,
                                int row_bytes, const int* parent, long sp_g, long sp_w, const int* len, long len_s, int base,
                                int unit, int first) {
  if (!x || !parent) return MX_ENULL;
  if (N < 1 || G < 1 || W < 1 || W > 64 || H < 1 || T < 1 || row_bytes < 1 || unit < 1 || first < 0) return MX_ESHAPE;
  if (((uintptr_t)parent & 3) || ((uintptr_t)len & 3)) return MX_ELAYOUT;
  if (W == 1 || first >= T) return MX_OK;
  const uintptr_t bits = (uintptr_t)x | (uintptr_t)s_n | (uintptr_t)s_s | (uintptr_t)s_h | (uintptr_t)s_t | (uintptr_t)row_bytes;
  const int size = bits & 3 ? 1 : bits & 15 ? 4 : 16;
  const int cpr = row_bytes / size;
  const double blocks = ((double)(T - first) * cpr + 255) / 256 * N * G * H;
  if (blocks > 0x7fffff) return MX_ESHAPE;  // 2^31 threads; a grid has less than 2^32
  const unsigned nblk = (unsigned)(((long)(T - first) * cpr + 255) / 256);
  const MoveArgs a{(uint8_t*)x, s_n, s_s, s_h, s_t, parent, sp_g, sp_w, len, len_s, base, unit, first, T, G, W, H, cpr, nblk};
  const unsigned grid = nblk * (unsigned)(N * G * H);
  if (size == 16) move<u32x4>(st, a, grid);
  else if (size == 4) move<uint32_t>(st, a, grid);
  else move<uint8_t>(st, a, grid);
  return hipGetLastError() == hipSuccess ? MX_OK : MX_ELAUNCH;
}
