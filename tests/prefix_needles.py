"""Checks of the shared-prefix attention that see a single key lost, counted twice or taken for another, in keys of any number:
`attend(q, pk, pv, k, v, kv_len, prefix_len)` is ops.sdpa_prefix or a plain form. Two sets of inputs:

  counts   q = 0, so that all of a row's n keys weigh 1 / n, and values 0 but for four keys of each column, of values 1, 2, 4, 8:
           an output is the sum of the marks that the row sees over n. A mark lost or doubled is at least 1 / 15 of it.
  needles  every row looks for one key, whose score is 512 or more above the others': their weights are 2^-738 = 0 in fp32, and the
           output is that key's value, bit for bit.
"""
import torch

BF, F64 = torch.bfloat16, torch.float64


def geometry(case, lens, plens, dev):
    """(kv_len, prefix_len) tensors or None, own keys (B, Tq) and prefix keys (N,) that are seen."""
    N, S, H, G, D, Tq, P, T = case
    B = N * S
    kv = None if lens is None else torch.tensor((list(lens) * B)[:B], dtype=torch.int32, device=dev)
    pl = None if plens is None else torch.tensor((list(plens) * N)[:N], dtype=torch.int32, device=dev)
    own = torch.full((B,), T, device=dev) if kv is None else kv.long()
    own = torch.minimum((own[:, None] - Tq + 1 + torch.arange(Tq, device=dev)).clamp(min=0), own[:, None])
    return kv, pl, own, torch.full((N,), P, device=dev) if pl is None else pl.long()


def marks(keys, D, first, dev):
    m = torch.zeros(keys, D, device=dev)
    at = torch.arange(first, min(first + 4 * D, keys), device=dev)
    m[at, at % D] = 2.0 ** ((at - first) // D).float()
    return m


def counts(attend, case, lens=None, plens=None, dev="cpu"):
    N, S, H, G, D, Tq, P, T = case
    B = N * S
    kv, pl, own, pre = geometry(case, lens, plens, dev)
    gen = torch.Generator().manual_seed(P + T)
    rnd = lambda *s: torch.randn(*s, generator=gen).to(BF).to(dev)
    q = torch.zeros(B, H * G, Tq, D, device=dev, dtype=BF)
    pk, k = rnd(N, H, P, D), rnd(B, H, T, D)
    n = (pre.repeat_interleave(S)[:, None] + own).double()
    for where, keys in (("prefix", P), ("own", T)):
        for first in range(0, keys, 4 * D):
            m = marks(keys, D, first, dev)
            held = lambda x, here: (m.to(BF) if here else torch.zeros_like(m[:1]).to(BF).expand(x.shape[2], D)).expand(x.shape).contiguous()
            out = attend(q, pk, held(pk, where == "prefix"), k, held(k, where == "own"), kv, pl).view(B, Tq, H * G, D).to(F64)
            total = torch.cat([torch.zeros(1, D, device=dev, dtype=F64), m.to(F64).cumsum(0)])
            seen = total[pre].repeat_interleave(S, 0)[:, None].expand(B, Tq, D) if where == "prefix" else total[own]
            want = torch.where(n[..., None] > 0, seen / n[..., None], 0.0)[:, :, None]
            # weights, their sum and the sums of marks are whole numbers, exact; the reciprocal, the product with it and the output's
            # rounding to bf16 (2^-8 of it) are not
            over = (out - want).abs() - (2.0 ** -8 + 2.0 ** -20) * want
            assert float(over.max()) <= 0, (where, first, float(over.max()))


def _look(attend, case, kv, pl, x, rows, target, value, dev):
    """Rows (B, H, Tq, G: true where it looks) have to find their value (B, H, Tq, G, D)."""
    N, S, H, G, D, Tq, P, T = case
    out = attend(*x, kv, pl).view(N * S, Tq, H, G, D).permute(0, 2, 1, 3, 4)
    wrong = ((out != value).any(4) & rows).nonzero()
    assert not wrong.numel(), (target, wrong[:4].tolist())


def needles(attend, case, lens=None, plens=None, dev="cpu", calls=24):
    N, S, H, G, D, Tq, P, T = case
    B = N * S
    kv, pl, own, pre = geometry(case, lens, plens, dev)
    gen = torch.Generator().manual_seed(P + T + 1)
    rnd = lambda *s: torch.randn(*s, generator=gen).to(BF).to(dev)
    pv, v = rnd(N, H, P, D), rnd(B, H, T, D)
    big = (512.0 * D ** 0.5) ** 0.5  # squared and scaled: 512
    big = 2.0 ** torch.tensor(big).log2().ceil().item()
    # row r = (j Tq + i) G + g of a prefix and head looks along axis r % D, all rows of an axis for one key
    r = torch.arange(S * Tq * G, device=dev)
    axis = (r % D).view(S, Tq, G)
    q = torch.zeros(N, S, H, Tq, G, D, device=dev)
    q.scatter_(5, axis[None, :, None, :, :, None].expand(N, S, H, Tq, G, 1), big)
    q = q.permute(0, 1, 2, 4, 3, 5).reshape(B, H * G, Tq, D).to(BF)
    # ---- keys of the prefix: both sides of every 32nd, the first and the last, a few at random
    used = min(D, S * Tq * G)
    for n in range(N):
        p = int(pre[n])
        if not p:
            continue
        edge = [i for i in range(p) if i % 32 in (0, 31)] + [p - 1]
        edge += torch.randint(0, p, (len(edge) // 4 + 1,), generator=gen).tolist()
        edge = [edge[i] for i in torch.randperm(len(edge), generator=gen).tolist()]
        edge = [0, p - 1] + edge
        for at in range(0, min(len(edge), calls * used), used):
            part = list(dict.fromkeys(edge[at:at + used]))  # one key has one axis
            t = torch.tensor(part, device=dev)
            pk = torch.zeros(N, H, P, D, device=dev, dtype=BF)
            pk[n, :, t, torch.arange(len(part), device=dev)] = big
            ax = axis[None].expand(N, S, Tq, G).reshape(B, Tq, G)
            look = (ax < len(part)) & (torch.arange(B, device=dev) // S == n)[:, None, None]
            value = pv[n][:, t[ax.clamp(max=len(part) - 1)]].permute(1, 0, 2, 3, 4)  # (H, B, Tq, G, D) before
            _look(attend, case, kv, pl, (q, pk, pv, torch.zeros_like(v), v), look[:, None].expand(B, H, Tq, G), ("prefix", n, part), value, dev)
            if N > 4:
                break  # many prefixes of few keys: the edges of each
    if not T:
        return
    # ---- the last own keys that a query sees, D queries at a time (more would share an axis)
    pk = torch.zeros(N, H, P, D, device=dev, dtype=BF)
    for i0 in range(0, Tq, D):
        i = torch.arange(i0, min(i0 + D, Tq), device=dev)
        for back in (0, 1, 31, 64):
            k = torch.zeros(B, H, T, D, device=dev, dtype=BF)
            at = own[:, i] - 1 - back  # (B, queries)
            for b in range(B):
                ok = at[b] >= 0
                k[b, :, at[b][ok], (i - i0)[ok]] = big
            qs = torch.zeros(B, H * G, Tq, D, device=dev, dtype=BF)
            qs[:, :, i, i - i0] = big
            look = torch.zeros(B, Tq, dtype=torch.bool, device=dev)
            look[:, i] = at >= 0
            place = (own - 1 - back).clamp(min=0)
            value = v[torch.arange(B, device=dev)[:, None], :, place].transpose(1, 2)  # (B, H, Tq, D)
            _look(attend, case, kv, pl, (qs, pk, pv, k, v), look[:, None, :, None].expand(B, H, Tq, G), ("own", i0, back),
                  value[:, :, :, None].expand(B, H, Tq, G, D), dev)
