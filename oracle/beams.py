"""Attention over shared prefixes, beam selection and slot reordering in 64 bits on the CPU, straight from their definitions.
No reference counterpart: the reference copies its image prefix into every question's cache slot and never decodes."""
import math
from fractions import Fraction

import torch

F64 = torch.float64


def sdpa_prefix(q, pk, pv, k, v, kv_len=None, prefix_len=None, scale=None, causal=True):
    """(o, mag, size): (B, Tq, Hq D) outputs, sum p |v| at the same places, and the largest sum |q k| scale of a row that has keys.
    Keys that a row does not see are left out of its sums, whatever they hold."""
    B, Hq, Tq, D = q.shape
    N, H, P = pk.shape[:3]
    T, G = k.shape[2], Hq // H
    scale = D ** -0.5 if scale is None else scale
    lens = [T] * B if kv_len is None else [min(max(int(x), 0), T) for x in kv_len]
    plens = [P] * N if prefix_len is None else [min(max(int(x), 0), P) for x in prefix_len]
    o, mag, size = torch.zeros(B, Tq, Hq, D, dtype=F64), torch.zeros(B, Tq, Hq, D, dtype=F64), 0.0
    for b in range(B):
        n, t = b // (B // N), lens[b]
        p = plens[n]
        for h in range(H):
            kk = torch.cat([pk[n, h, :p], k[b, h, :t]]).to(F64)
            vv = torch.cat([pv[n, h, :p], v[b, h, :t]]).to(F64)
            qq = q[b, h * G:(h + 1) * G].to(F64)
            if not causal or Tq == 1:
                groups = [(slice(None), p + t)]
            else:
                groups = [(slice(i, i + 1), p + min(max(t - Tq + 1 + i, 0), t)) for i in range(Tq)]
            for rows, m in groups:
                if not m:
                    continue
                x = qq[:, rows]
                s = torch.matmul(x, kk[:m].t()) * scale
                w = torch.softmax(s, -1)
                w = torch.where(s == -math.inf, 0.0, w)
                o[b, rows, h * G:(h + 1) * G] = _product(w, vv[:m]).transpose(0, 1)
                mag[b, rows, h * G:(h + 1) * G] = _product(w, vv[:m].abs()).transpose(0, 1)
                fin = torch.nan_to_num(x, 0, 0, 0).abs(), torch.nan_to_num(kk[:m], 0, 0, 0).abs()
                size = max(size, float(torch.matmul(fin[0], fin[1].t()).max()) * scale)
    return o.flatten(2), mag.flatten(2), size


def _product(w, v):
    """w v, with 0 v = 0 only where the weight is 0 by definition (never: a softmax weight is positive however small)."""
    if torch.isfinite(v).all():
        return torch.matmul(w, v)
    tiny = torch.where(w == 0, torch.full_like(w, 1e-300), w)
    return (tiny[..., None] * v).sum(-2)


def beam_select(logits, scores, k, done=None, eos=None):
    """(values (B, k) fp64, parent, token, done)."""
    B, W, V = logits.shape
    val, par, tok, fin = [], [], [], []
    for b in range(B):
        cand = []
        for w in range(W):
            s = float(scores[b, w])
            if not math.isfinite(s):
                continue
            if done is not None and bool(done[b, w]):
                cand.append((-Fraction(s), w * V + eos))
                continue
            x = logits[b, w].to(F64)
            lse = float(torch.logsumexp(x, 0))
            if not math.isfinite(lse):
                continue
            # the order within a beam is exact: logits that lie closer than the sum's spacing are still apart
            for v in x.sort(descending=True, stable=True)[1][:k].tolist():
                if x[v] > -math.inf:
                    cand.append((-(Fraction(s) + Fraction(float(x[v])) - Fraction(lse)), w * V + v))
        cand.sort()
        cand = [(float(c), i) for c, i in cand[:k]]
        e = 0 if eos is None else eos
        val.append([-c for c, _ in cand] + [-math.inf] * (k - len(cand)))
        par.append([i // V for _, i in cand] + [0] * (k - len(cand)))
        tok.append([i % V for _, i in cand] + [e] * (k - len(cand)))
        fin.append([i % V == eos for _, i in cand] + [True] * (k - len(cand)))
    i32 = torch.int32
    return torch.tensor(val, dtype=F64), torch.tensor(par, dtype=i32), torch.tensor(tok, dtype=i32), torch.tensor(fin)


def reorder_slots(x, parent, n=None, first=0, unit=1):
    """A reordered copy of x (L, slots, H, T, ...)."""
    parent = parent if parent.dim() == 2 else parent[None]
    G, W = parent.shape
    T = x.shape[3]
    n = [T * unit] * (G * W) if n is None else ([n] * (G * W) if isinstance(n, int) else [int(v) for v in n])
    y = x.clone()
    for g in range(G):
        for w in range(W):
            p = int(parent[g, w])
            if 0 <= p < W:
                hi = min(max(-(-n[g * W + p] // unit), 0), T)
                lo = first // unit
                if lo < hi:
                    y[:, g * W + w, :, lo:hi] = x[:, g * W + p, :, lo:hi]
    return y
