"""The reduced-bit operators in 64 bits on the CPU: MXFP4 (OCP MX v1.0: e2m1 codes, a power of two per 32 columns), its
Linear, the 8-bit KV cache (e4m3 codes, a power of two per 64 tokens of a head) and attention over it. Quantised values are
returned as the doubles they stand for. No reference counterpart: the reference's narrowest formats are W8A8 and a bf16
cache."""
import math

import torch

F64 = torch.float64
E2M1 = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=F64)
E4M3 = torch.tensor([m * 2.0 ** -9 for m in range(8)] +
                    [(1 + m / 8) * 2.0 ** e for e in range(-6, 9) for m in range(8)][:-1], dtype=F64)  # last: NaN


def nearest(v, levels):
    """Nearest level, halfway to the level of even index (the even code); magnitudes beyond the last saturate."""
    a = v.abs().contiguous()
    mid = (levels[1:] + levels[:-1]) / 2
    lo, hi = torch.bucketize(a, mid, right=False), torch.bucketize(a, mid, right=True)
    return torch.copysign(levels[torch.where(lo % 2 == 0, lo, hi)], v)


def floor_log2(x):
    """Exact for every positive double that a bf16 can be; -inf for 0."""
    m, e = torch.frexp(x)
    return torch.where(x > 0, (e - 1).to(F64), torch.full_like(x, -math.inf))


def mxfp4(x):
    """(M, K) to MXFP4 values."""
    M, K = x.shape
    y = torch.zeros(M, -(-K // 32) * 32, dtype=F64)
    y[:, :K] = x.to(F64)
    y = y.view(M, -1, 32)
    bad = ~torch.isfinite(y).all(2, keepdim=True)
    unit = torch.exp2((floor_log2(torch.where(bad, 1.0, y.abs().amax(2, keepdim=True))) - 2).clamp(min=-127))
    v = torch.where(bad, math.nan, nearest(torch.where(bad, 0.0, y) / unit, E2M1) * unit)
    return v.reshape(M, -1)[:, :K]


def gelu(y, act):
    if act == "tanh":
        return 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))
    return 0.5 * y * (1 + torch.erf(y / math.sqrt(2))) if act == "erf" else y


def mxfp4_linear(x, w, b=None, act=None, res=None, act_from=0):
    """(y, magnitude): the Linear, and sum |x w| + |b|, which rounding errors of the sum go by."""
    xq, wq = mxfp4(x), mxfp4(w)
    y, mag = xq @ wq.t(), xq.abs() @ wq.t().abs()
    if b is not None:
        y, mag = y + b.to(F64), mag + b.to(F64).abs()
    y = torch.cat([y[:, :act_from], gelu(y[:, act_from:], act)], 1)
    return (y if res is None else y + res.to(F64)), mag


class KV8:
    """One tensor (K or V) of the cache: values (slots, H, ctx, D), exponents per block (slots, H, blocks)."""

    def __init__(self, slots, H, ctx, D):
        self.val = torch.zeros(slots, H, ctx, D, dtype=F64)
        self.exp = torch.full((slots, H, -(-ctx // 64)), -127.0, dtype=F64)
        self.ctx = ctx

    def append(self, slot, rows, pos):
        """rows (H, n, D) at pos ..; rows outside the cache are dropped."""
        for t0 in range(max(pos, 0) // 64 * 64, min(pos + rows.shape[1], self.ctx), 64):
            lo, hi = max(pos, t0), min(pos + rows.shape[1], t0 + 64, self.ctx)
            if lo >= hi:
                continue
            x = rows[:, lo - pos:hi - pos].to(F64)
            x = torch.where(torch.isfinite(x), x, math.nan)
            big = torch.nan_to_num(x.abs(), nan=0.0).amax((1, 2))
            fl = floor_log2(big)
            need = (fl - 8 + (big > 1.75 * torch.exp2(fl)).to(F64)).clamp(min=-127)
            e = torch.maximum(self.exp[slot, :, t0 // 64], need) if lo > t0 else need
            unit = torch.exp2(e)[:, None, None]
            if lo > t0:
                old = self.val[slot, :, t0:lo] / unit
                self.val[slot, :, t0:lo] = torch.where(old.isnan(), math.nan, nearest(torch.nan_to_num(old), E4M3)) * unit
            x = x / unit
            self.val[slot, :, lo:hi] = torch.where(x.isnan(), math.nan, nearest(torch.nan_to_num(x), E4M3)) * unit
            self.exp[slot, :, t0 // 64] = e


def sdpa(q, k, v, length, scale=None, qpos0=None, causal_from=None):
    """One sequence: q (Hq, Tq, D), k, v (H, ctx, D). Returns (out (Tq, Hq, D), average |v| under the weights (same
    shape), largest sum |q k| scale of a row (Tq, Hq, 1))."""
    Hq, Tq, D = q.shape
    G = Hq // k.shape[0]
    q = q.to(F64)
    scale = D ** -0.5 if scale is None else scale
    qpos0 = length - Tq if qpos0 is None else qpos0
    j, i = torch.arange(length)[None], torch.arange(Tq)[:, None]
    seen = torch.ones(Tq, length, dtype=torch.bool) if causal_from is None else (j < causal_from) | (j <= qpos0 + i)
    out, avg, size = (torch.zeros(Tq, Hq, n, dtype=F64) for n in (D, D, 1))
    for h in range(Hq):
        kk, vv = k[h // G, :length], v[h // G, :length]
        for t in range(Tq):
            ks, vs = kk[seen[t]], vv[seen[t]]
            if not len(ks):
                continue
            p = torch.softmax(ks @ q[h, t] * scale, 0)
            out[t, h] = p @ vs
            avg[t, h] = p @ vs.abs()
            size[t, h] = (ks.abs() @ q[h, t].abs()).max() * scale
    return out, avg, size
