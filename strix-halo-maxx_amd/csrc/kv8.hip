// The 8-bit KV cache (kv8.h): rows into the cache, and the cache back as bf16.
//
// Append. Rows t = 0 .. n_b - 1 of sequence b go to positions pos_b + t. For each block of 64 positions that a row falls
// into, K and V apart:
//   need = smallest e with max |finite row value| <= 448 2^e,   e' = max(e, need) where the block holds earlier rows
//   (positions of the block before pos_b), else need;
//   the earlier rows' codes become e4m3(code 2^(e - e')) if e' > e, the new rows' codes e4m3(x 2^-e'), both to nearest
//   even; infinities and NaN become the NaN code, e4m3 has no infinity.
// Scaling by powers of two is exact, so the codes follow from this bit for bit. The sequence ends behind the new rows: the
// codes of the block after them stay, their exponent does not.
#include "kv8.h"

namespace {

struct AppendArgs {
  const uint16_t *k, *v, *q;
  long sk_b, sk_h, sk_t, sv_b, sv_h, sv_t, sq_b, sq_h, sq_t;
  uint8_t *kc, *vc, *ks, *vs;
  uint16_t* q_out;
  const int *pos, *count;
  const float* cs;
  long pos_s, count_s;
  int H, Hq, n, ctx, base, ncs, bcast, nslots;
};

// Four codes times 2^-d (d > 0), rounded again.
__device__ __forceinline__ uint32_t requant4(uint32_t c, float f) {
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(c, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(c, true);
  uint32_t o = __builtin_amdgcn_cvt_pk_fp8_f32(lo[0] * f, lo[1] * f, 0, false);
  return __builtin_amdgcn_cvt_pk_fp8_f32(hi[0] * f, hi[1] * f, o, true);
}
// Four bf16 (two words) times f to codes. f = 2^-e: the products are exact (or underflow far below half a code step).
// v_cvt_pk_fp8_f32 saturates what is too large, which leaves infinity: it becomes NaN first.
__device__ __forceinline__ float fin(float x) { return fabsf(x) < INFINITY ? x : __uint_as_float(0x7fc00000u); }
__device__ __forceinline__ uint32_t code4(uint32_t w0, uint32_t w1, float f) {
  uint32_t o = __builtin_amdgcn_cvt_pk_fp8_f32(fin(lo_bf(w0)) * f, fin(hi_bf(w0)) * f, 0, false);
  return __builtin_amdgcn_cvt_pk_fp8_f32(fin(lo_bf(w1)) * f, fin(hi_bf(w1)) * f, o, true);
}
__device__ __forceinline__ uint32_t amax_fin(uint32_t w) {
  const uint32_t a = w & 0x7fffu, b = (w >> 16) & 0x7fffu;
  return max(a < 0x7f80u ? a : 0u, b < 0x7f80u ? b : 0u);
}
// 1 / 2^(byte - 127); byte 0: 2^127, byte 254 does not occur (bf16 needs at most 247)
__device__ __forceinline__ float inv_pow2(int byte) { return __uint_as_float((uint32_t)(254 - byte) << 23); }

// Rows may start at any column: global memory takes wide accesses at any address, which the compiler uses for types that
// are aligned to 2 bytes.
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(2)));
__device__ __forceinline__ u32x4 ld8(const uint16_t* p) { return *reinterpret_cast<const u32x4_any*>(p); }
// Columns 8 c .. 8 c + 7 of a 64-wide row after the rotary embedding of rope.hip (rotary width 32: out[2j] =
// a_j cos - b_j sin, out[2j + 1] = a_j sin + b_j cos with a = x[0:16], b = x[16:32]), in its arithmetic and rounding.
__device__ __forceinline__ u32x4 roped8(const uint16_t* row, int c, const float* cp) {
  if (c >= 4) return ld8(row + 8 * c);
  u32x4 o;
#pragma unroll
  for (int e = 0; e < 4; e++) {
    const int j = 4 * c + e;
    const float a = bf2f(row[j]), b = bf2f(row[16 + j]), cc = cp[2 * j], sn = cp[2 * j + 1];
    o[e] = pack2(__fsub_rn(__fmul_rn(a, cc), __fmul_rn(b, sn)), __fadd_rn(__fmul_rn(a, sn), __fmul_rn(b, cc)));
  }
  return o;
}

// One workgroup per (block, head, slot); with a rotary table, heads H .. H + Hq - 1 of the grid rotate the queries.
// K: thread = (token, 8 columns). V: thread = 4 tokens x D / 16 columns, whose codes are transposed in registers to a dword
// per column. The block is put together in LDS and leaves in 16-byte stores; a block that keeps earlier rows is read
// first, together with the new rows (every load is issued before the first is used). The bound is HBM for long prompts (4
// sequences x 8001 rows x 8 heads x 128: 36 us, 4.5 TB/s), and for single rows the chain position -> rows -> maximum ->
// stores behind a launch (1 x 32 heads x 64 3.8 us, 32 x 8 x 128 10).
template <int D, bool ROPE>
__global__ __launch_bounds__(256) void kv8_append_kernel(AppendArgs p) {
  constexpr int CPR = D / 8, NC = 64 * CPR / 256;   // K: chunks of 8 columns per row, per thread
  constexpr int VC = D / 16, NO = 64 * D / 16 / 256;  // V: columns per thread; 16-byte pieces of the block per thread
  __shared__ __attribute__((aligned(16))) uint8_t kb[64 * D], vb[64 * D];
  __shared__ uint32_t red[2][4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int slot = blockIdx.z, b = p.bcast ? 0 : slot;
  const long pos = (long)p.base + (p.pos ? p.pos[b * p.pos_s] : 0);
  int n = p.n;
  if (p.count) n = min(n, max(0, p.count[b * p.count_s]));
  if (ROPE && (int)blockIdx.y >= p.H) {  // queries: rows 64 x .. 64 x + 63, every row (count bounds the cache only)
    const int hq = blockIdx.y - p.H, t0 = blockIdx.x * 64;
    if (p.bcast && slot) return;
    for (int c = tid; c < 64 * CPR; c += 256) {
      const int t = t0 + c / CPR;
      if (t >= p.n) break;
      const long cp = min(max(pos + t, 0L), (long)p.ncs - 1) * 32;
      *reinterpret_cast<u32x4*>(p.q_out + (((long)b * p.Hq + hq) * p.n + t) * D + 8 * (c % CPR)) =
          roped8(p.q + b * p.sq_b + hq * p.sq_h + t * p.sq_t, c % CPR, p.cs + cp);
    }
    return;
  }
  const int h = blockIdx.y;
  const long first = max(pos, 0L), last = min(pos + n, (long)p.ctx);  // positions written
  const long blk = first / 64 + blockIdx.x;
  const long lo = max(first, blk * 64), hi = min(last, blk * 64 + 64);
  if (lo >= hi) return;
  const int t_lo = (int)(lo - blk * 64), t_hi = (int)(hi - blk * 64);
  const int nblk = kv8_blocks(p.ctx);
  const long cell = ((long)slot * p.H + h) * nblk + blk;
  const uint16_t* kr = p.k + b * p.sk_b + h * p.sk_h + (blk * 64 - pos) * p.sk_t;  // token 0 of the block
  const uint16_t* vr = p.v + b * p.sv_b + h * p.sv_h + (blk * 64 - pos) * p.sv_t;

  uint8_t* kg = p.kc + cell * (64 * D);
  uint8_t* vg = p.vc + cell * (64 * D);
  const bool part = t_lo > 0 || t_hi < 64;  // the block keeps some of its bytes
  u32x4 xk[NC], ok[NO], ov[NO];
  uint32_t xv[4][VC / 2];
  uint32_t mk = 0, mv = 0;
  const int vq = 4 * (tid / 16), vcol = VC * (tid % 16);
  const int bk0 = p.ks[cell], bv0 = p.vs[cell];
  if (part)
#pragma unroll
    for (int i = 0; i < NO; i++) {
      ok[i] = *reinterpret_cast<const u32x4*>(kg + 16 * (tid + 256 * i));
      ov[i] = *reinterpret_cast<const u32x4*>(vg + 16 * (tid + 256 * i));
    }
#pragma unroll
  for (int i = 0; i < NC; i++) {
    const int c = tid + 256 * i, t = c / CPR, cc = c % CPR;
    xk[i] = u32x4{0u, 0u, 0u, 0u};
    if (t >= t_lo && t < t_hi) {
      if constexpr (ROPE)
        xk[i] = roped8(kr + (long)t * p.sk_t, cc, p.cs + min(blk * 64 + t, (long)p.ncs - 1) * 32);
      else
        xk[i] = ld8(kr + (long)t * p.sk_t + 8 * cc);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int t = vq + i;
    const uint16_t* row = vr + (long)t * p.sv_t + vcol;
#pragma unroll
    for (int e = 0; e < VC / 2; e++) xv[i][e] = 0;
    if (t >= t_lo && t < t_hi) {
      if constexpr (VC == 8) {
        const u32x4 v = ld8(row);
#pragma unroll
        for (int e = 0; e < 4; e++) xv[i][e] = v[e];
      } else {
        const u32x2 v = *reinterpret_cast<const u32x2_any*>(row);
        xv[i][0] = v.x, xv[i][1] = v.y;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < NC; i++)
#pragma unroll
    for (int e = 0; e < 4; e++) mk = max(mk, amax_fin(xk[i][e]));
#pragma unroll
  for (int i = 0; i < 4; i++)
#pragma unroll
    for (int e = 0; e < VC / 2; e++) mv = max(mv, amax_fin(xv[i][e]));
  mk = (uint32_t)wave_max((float)mk);  // exact: below 2^15
  mv = (uint32_t)wave_max((float)mv);
  if (lane == 0) {
    red[0][wave] = mk;
    red[1][wave] = mv;
  }
  __syncthreads();
  int bk = kv8_scale_byte(max(max(red[0][0], red[0][1]), max(red[0][2], red[0][3])));
  int bv = kv8_scale_byte(max(max(red[1][0], red[1][1]), max(red[1][2], red[1][3])));
  if (t_lo > 0) {
    bk = max(bk, bk0);
    bv = max(bv, bv0);
  }
  if (part) {  // keep what is there, rounded to the block's new exponent before the new rows
    const float fk = bk > bk0 ? inv_pow2(min(127 + bk - bk0, 254)) : 1.f, fv = bv > bv0 ? inv_pow2(min(127 + bv - bv0, 254)) : 1.f;
#pragma unroll
    for (int i = 0; i < NO; i++) {
      const int c = tid + 256 * i, l = c & 31, hh = (c >> 5) & 1, grp = c >> 6;
      u32x4 a = ok[i], w = ov[i];
      if (bk > bk0 && (grp / (D / 32)) * 32 + l < t_lo)
#pragma unroll
        for (int e = 0; e < 4; e++) a[e] = requant4(a[e], fk);
      if (bv > bv0)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const int t = (grp & 1) * 32 + 8 * e + 4 * hh, keep = t_lo - t;  // tokens t .. t + 3, the first keep are earlier
          if (keep <= 0) continue;
          const uint32_t msk = keep >= 4 ? 0xffffffffu : (1u << (8 * keep)) - 1u;
          w[e] = (requant4(w[e], fv) & msk) | (w[e] & ~msk);
        }
      *reinterpret_cast<u32x4*>(kb + 16 * c) = a;
      *reinterpret_cast<u32x4*>(vb + 16 * c) = w;
    }
    __syncthreads();
  }
  const float fk = inv_pow2(bk), fv = inv_pow2(bv);
#pragma unroll
  for (int i = 0; i < NC; i++) {
    const int c = tid + 256 * i, t = c / CPR, cc = c % CPR;
    if (t >= t_lo && t < t_hi)
      *reinterpret_cast<u32x2*>(kb + kv8_koff<D>(t, 8 * cc)) =
          u32x2{code4(xk[i][0], xk[i][1], fk), code4(xk[i][2], xk[i][3], fk)};
  }
#pragma unroll
  for (int e = 0; e < VC; e += 4) {  // 4 tokens x 4 columns
    uint32_t c[4];
#pragma unroll
    for (int i = 0; i < 4; i++) c[i] = code4(xv[i][e / 2], xv[i][e / 2 + 1], fv);
    const uint32_t a0 = __builtin_amdgcn_perm(c[1], c[0], 0x05010400u), a1 = __builtin_amdgcn_perm(c[3], c[2], 0x05010400u);
    const uint32_t b0 = __builtin_amdgcn_perm(c[1], c[0], 0x07030602u), b1 = __builtin_amdgcn_perm(c[3], c[2], 0x07030602u);
    const uint32_t t[4] = {__builtin_amdgcn_perm(a1, a0, 0x05040100u), __builtin_amdgcn_perm(a1, a0, 0x07060302u),
                           __builtin_amdgcn_perm(b1, b0, 0x05040100u), __builtin_amdgcn_perm(b1, b0, 0x07060302u)};
#pragma unroll
    for (int j = 0; j < 4; j++) {
      uint8_t* o = vb + kv8_voff(vq, vcol + e + j);
      if (vq >= t_lo && vq + 4 <= t_hi) {
        *reinterpret_cast<uint32_t*>(o) = t[j];
      } else {
#pragma unroll
        for (int i = 0; i < 4; i++)
          if (vq + i >= t_lo && vq + i < t_hi) o[i] = (uint8_t)(t[j] >> (8 * i));
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < NO; i++) {
    const int c = 16 * (tid + 256 * i);
    *reinterpret_cast<u32x4*>(kg + c) = *reinterpret_cast<const u32x4*>(kb + c);
    *reinterpret_cast<u32x4*>(vg + c) = *reinterpret_cast<const u32x4*>(vb + c);
  }
  if (tid == 0) {
    p.ks[cell] = (uint8_t)bk;
    p.vs[cell] = (uint8_t)bv;
  }
}

// Rows 0 .. n - 1 of every slot and head back as bf16: one workgroup per (block, head x slot), the block by way of LDS. HBM
// bound: 4 slots x 8 heads x 16002 x 128 74 us (5.3 TB/s); the stores are not kept in the caches (79 us if they are).
template <int D>
__global__ __launch_bounds__(256) void kv8_read_kernel(const uint8_t* __restrict__ kc, const uint8_t* __restrict__ vc,
                                                       const uint8_t* __restrict__ ks, const uint8_t* __restrict__ vs,
                                                       uint16_t* __restrict__ k, uint16_t* __restrict__ v, int n, int ctx) {
  constexpr int CPR = D / 8;
  __shared__ __attribute__((aligned(16))) uint8_t kb[64 * D], vb[64 * D];
  const int tid = threadIdx.x, nb = kv8_blocks(n);
  const long blk = blockIdx.x % nb, sh = blockIdx.x / nb;
  const long cell = sh * kv8_blocks(ctx) + blk;
#pragma unroll
  for (int i = 0; i < 64 * D / 16 / 256; i++) {
    const int c = 16 * (tid + 256 * i);
    *reinterpret_cast<u32x4*>(kb + c) = *reinterpret_cast<const u32x4*>(kc + cell * (64 * D) + c);
    *reinterpret_cast<u32x4*>(vb + c) = *reinterpret_cast<const u32x4*>(vc + cell * (64 * D) + c);
  }
  const float fk = kv8_pow2(ks[cell]), fv = kv8_pow2(vs[cell]);
  __syncthreads();
  for (int c = tid; c < 64 * CPR; c += 256) {
    const int t = c / CPR, d = 8 * (c % CPR);
    if (blk * 64 + t >= n) break;
    const long o = (sh * n + blk * 64 + t) * D + d;
    const u32x2 kk = *reinterpret_cast<const u32x2*>(kb + kv8_koff<D>(t, d));
    u32x4 yk, yv;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const auto a = (e & 1) ? __builtin_amdgcn_cvt_pk_f32_fp8(kk[e >> 1], true) : __builtin_amdgcn_cvt_pk_f32_fp8(kk[e >> 1], false);
      yk[e] = pack2(a[0] * fk, a[1] * fk);
      const uint32_t w = (uint32_t)vb[kv8_voff(t, d + 2 * e)] | (uint32_t)vb[kv8_voff(t, d + 2 * e + 1)] << 8;
      const auto z = __builtin_amdgcn_cvt_pk_f32_fp8(w, false);
      yv[e] = pack2(z[0] * fv, z[1] * fv);
    }
    __builtin_nontemporal_store(yk, reinterpret_cast<u32x4*>(k + o));
    __builtin_nontemporal_store(yv, reinterpret_cast<u32x4*>(v + o));
  }
}

}  // namespace

extern "C" int mx_kv8_append(hipStream_t st, const uint16_t* k, long sk_b, long sk_h, long sk_t, const uint16_t* v,
                             long sv_b, long sv_h, long sv_t, uint8_t* kc, uint8_t* vc, uint8_t* ks, uint8_t* vs, int B,
                             int H, int n, int D, int ctx, int nslots, int bcast, const int* pos, long pos_s, int base,
                             const int* count, long count_s, const float* cs, int ncs, const uint16_t* q, long sq_b,
                             long sq_h, long sq_t, int Hq, uint16_t* q_out) {
  if (!k || !v || !kc || !vc || !ks || !vs) return MX_ENULL;
  if (D != 64 && D != 128) return MX_EBADCFG;
  if (B < 1 || H < 1 || n < 1 || ctx < 1 || nslots < B || (bcast && B != 1) || ctx > 0x7fffff00) return MX_ESHAPE;
  const int nz = bcast ? nslots : B, ny = H + (cs && q ? Hq : 0);
  if (nz > 65535 || ny > 65535 || n > 0x7fffff00) return MX_ESHAPE;
  if (!pos && (base < 0 || (long)base + n > ctx)) return MX_ESHAPE;
  if (cs && (D != 64 || ncs < 1)) return MX_EBADCFG;
  if (q && (!cs || !q_out || Hq < 1)) return MX_ENULL;
  if (((uintptr_t)k | (uintptr_t)v | (uintptr_t)q) & 1) return MX_ELAYOUT;
  if (((uintptr_t)kc | (uintptr_t)vc | (uintptr_t)q_out) & 15) return MX_ELAYOUT;
  if (((uintptr_t)pos | (uintptr_t)count | (uintptr_t)cs) & 3) return MX_ELAYOUT;
  const AppendArgs a{k, v, q, sk_b, sk_h, sk_t, sv_b, sv_h, sv_t, sq_b, sq_h, sq_t, kc, vc, ks, vs, q_out, pos, count, cs, pos_s,
               count_s, H, Hq, n, ctx, base, ncs, bcast, nslots};
  // blocks that n rows can touch wherever they start; the queries need ceil(n / 64), which is no more
  const int nx = pos ? (int)(((long)n + 62) / 64 + 1) : (base + n - 1) / 64 - base / 64 + 1;
  const int gx = cs && q ? (nx > (n + 63) / 64 ? nx : (n + 63) / 64) : nx;
  if (gx > 0xffffff) return MX_ESHAPE;
  const dim3 grid((unsigned)gx, (unsigned)ny, (unsigned)nz);
  if (cs)
    hipLaunchKernelGGL((kv8_append_kernel<64, true>), grid, dim3(256), 0, st, a);
  else if (D == 64)
    hipLaunchKernelGGL((kv8_append_kernel<64, false>), grid, dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((kv8_append_kernel<128, false>), grid, dim3(256), 0, st, a);
  return hipGetLastError() == hipSuccess ? MX_OK : MX_ELAUNCH;
}

extern "C" int mx_kv8_read(hipStream_t st, const uint8_t* kc, const uint8_t* vc, const uint8_t* ks, const uint8_t* vs,
                           uint16_t* k, uint16_t* v, int nslots, int H, int n, int D, int ctx) {
  if (!kc || !vc || !ks || !vs || !k || !v) return MX_ENULL;
  if (D != 64 && D != 128) return MX_EBADCFG;
  if (nslots < 1 || H < 1 || n < 1 || n > ctx || ctx > 0x7fffff00) return MX_ESHAPE;
  if (((uintptr_t)kc | (uintptr_t)vc | (uintptr_t)k | (uintptr_t)v) & 15) return MX_ELAYOUT;
  const long heads = (long)nslots * H, wgs = kv8_blocks(n) * heads;
  if (heads > 0xffffffL || wgs > 0xffffffL) return MX_ESHAPE;
  if (D == 64)
    hipLaunchKernelGGL(kv8_read_kernel<64>, dim3((unsigned)wgs), dim3(256), 0, st, kc, vc, ks, vs, k, v, n, ctx);
  else
    hipLaunchKernelGGL(kv8_read_kernel<128>, dim3((unsigned)wgs), dim3(256), 0, st, kc, vc, ks, vs, k, v, n, ctx);
  return hipGetLastError() == hipSuccess ? MX_OK : MX_ELAUNCH;
}
