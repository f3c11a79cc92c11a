"""Attention over shared prefixes on the MI355X against the 64-bit oracle, within a bound derived from its roundings."""
import math

import pytest
import torch

import oracle.beams as ob
import strix_halo_maxx_amd.ops as ops
from beam_cases import ATTENTION, MASKED

pytestmark = pytest.mark.gpu
BF, F64 = torch.bfloat16, torch.float64


def gen(seed):
    return torch.Generator().manual_seed(seed)


def rnd(g, *shape):
    return torch.randn(*shape, generator=g).to(BF)


def i32(dev, v):
    return torch.tensor(v, device=dev, dtype=torch.int32)


def inputs(g, N, S, H, G, D, Tq, P, T):
    B = N * S
    return dict(q=rnd(g, B, H * G, Tq, D), pk=rnd(g, N, H, P, D), pv=rnd(g, N, H, P, D), k=rnd(g, B, H, T, D), v=rnd(g, B, H, T, D))


def within(got, want, mag, size, keys, D):
    """The bf16 weights are off by 2^-8 of themselves at most, in the sum and under the fraction alike, which moves the mean of v
    by at most 2^-8 (sum p |v| + |o|); the output's rounding is 2^-8 of it. fp32: a dot product of D terms is off by D 2^-24 of
    sum |q k| (as an exponent: of the weight), its scale and exponent by 2^-22 of the score and 2^-20; sums over the keys by
    keys 2^-24 of sum p |v|."""
    got = got.cpu().to(F64)
    u = 2.0 ** -8
    fine = torch.isfinite(want) & torch.isfinite(mag)
    bad = ~fine & (torch.isnan(want) | torch.isinf(want))
    same = (got[bad] == want[bad]) | (got[bad].isnan() & want[bad].isnan())
    assert bool(same.all()), "infinities and NaN"
    slack = 2 * (size * (D + 8) * 2.0 ** -24 + size * 2.0 ** -22 + 2.0 ** -20) + keys * 2.0 ** -24
    tol = u * (1 + u) * (mag + want.abs()) + u * (1 + u) * want.abs() + slack * (mag + want.abs()) + 2.0 ** -133
    over = ((got - want).abs() / tol)[fine]
    assert not over.numel() or float(over.max()) <= 1.0, float(over.max())


def check(dev, x, kv_len=None, prefix_len=None, **kw):
    d = {n: t.to(dev) for n, t in x.items()}
    li = None if kv_len is None else (kv_len if isinstance(kv_len, int) else i32(dev, kv_len))
    pi = None if prefix_len is None else (prefix_len if isinstance(prefix_len, int) else i32(dev, prefix_len))
    got = ops.sdpa_prefix(d["q"], d["pk"], d["pv"], d["k"], d["v"], li, pi, **kw)
    B, N = x["q"].shape[0], x["pk"].shape[0]
    want = ob.sdpa_prefix(*x.values(), kv_len=[kv_len] * B if isinstance(kv_len, int) else kv_len,
                          prefix_len=[prefix_len] * N if isinstance(prefix_len, int) else prefix_len, **kw)
    within(got, *want, x["pk"].shape[2] + x["k"].shape[2], x["q"].shape[3])
    return got


@pytest.mark.parametrize("case", ATTENTION, ids=str)
def test_every_kernel(dev, case):
    (N, S, H, G, D, Tq, P, T), lens, plens = case
    print(case, ops.sdpa_prefix_tiling(N, S, H, G, Tq, P, T, D), flush=True)
    x = inputs(gen(P + T), N, S, H, G, D, Tq, P, T)
    kv = (list(lens) * (N * S))[:N * S] if lens else None
    pl = (list(plens) * N)[:N] if plens else None
    got = check(dev, x, kv, pl)
    again = ops.sdpa_prefix(*(t.to(dev) for t in x.values()), None if kv is None else i32(dev, kv), None if pl is None else i32(dev, pl))
    assert torch.equal(got, again)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("P,T", [(0, 0), (0, 1), (1, 0), (1, 1), (31, 33), (32, 32), (33, 31), (64, 0), (0, 64), (65, 129)])
@pytest.mark.parametrize("S,Tq", [(1, 1), (3, 1), (2, 5), (40, 1), (2, 40)])
def test_short_lengths(dev, D, P, T, S, Tq):
    x = inputs(gen(P * 7 + T), 1, S, 2, 2, D, Tq, P, T)
    check(dev, x)
    check(dev, x, causal=False)


@pytest.mark.parametrize("D", [64, 128])
def test_lengths_on_the_device(dev, D):
    """Ragged, zero, negative and too large lengths; rows without a key are zero."""
    x = inputs(gen(3), 3, 4, 2, 3, D, 1, 100, 70)
    kv = [0, 1, 70, 33, 0, 64, -5, 1000, 2 ** 31 - 1, -2 ** 31, 0, 5]
    got = check(dev, x, kv, [0, 100, 2 ** 31 - 1])
    assert not bool(got[0].any())
    check(dev, x, kv, [-7, 33, 64])
    check(dev, x, 12, 40)
    xq = inputs(gen(4), 2, 2, 2, 2, D, 9, 50, 40)
    got = check(dev, xq, [0, 3, 9, 40], [0, 50])  # the first queries of a sequence shorter than Tq see the prefix alone
    assert not bool(got[:1].any()) and not bool(got[1, :6].any())


@pytest.mark.parametrize("case", MASKED, ids=str)
def test_what_is_masked_reaches_nothing(dev, case):
    """Behind the lengths, in other sequences, and after a query: NaN and infinities change no other row."""
    N, S, H, G, D, Tq, P, T = case
    B = N * S
    lens = [(T - 5 * b) % (T + 1) for b in range(B)]
    plens = [max(P - 13 * n, 0) for n in range(N)]
    x = inputs(gen(9), N, S, H, G, D, Tq, P, T)
    clean = {n: t.clone() for n, t in x.items()}
    for b in range(B):
        for y in (x["k"], x["v"]):
            y[b, :, lens[b]:] = torch.tensor([math.nan, math.inf, -math.inf, 3e38])[torch.arange(D) % 4].to(BF)
    for n in range(N):
        for y in (x["pk"], x["pv"]):
            y[n, :, plens[n]:] = math.nan
    a = check(dev, x, lens, plens)
    assert torch.equal(a, check(dev, clean, lens, plens))
    # values of single keys that some rows see: those become what the formula says, the others stay
    b = max(range(B), key=lambda i: lens[i])
    if lens[b] > 3:
        t = lens[b]
        x["v"][b, 0, t - 1, 3], x["v"][b, 0, t - 2, 4], x["v"][b, 1, t // 2, 5] = math.nan, math.inf, -math.inf
        x["v"][b, 1, t - 1, 6], x["v"][b, 1, t - 2, 6] = math.inf, -math.inf
        got = check(dev, x, lens, plens)
        others = [i for i in range(B) if i != b]
        assert torch.equal(got[others], a[others])
        x["k"][b, 0, t - 1, 0] = math.nan
        got = check(dev, x, lens, plens)
        assert torch.equal(got[others], a[others])


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("S,Tq", [(3, 1), (40, 1), (2, 50)])
def test_large_scores(dev, D, S, Tq):
    """Scores up to 2^28: one key takes all the weight, or keys share it where their scores are equal."""
    x = inputs(gen(D), 1, S, 2, 1, D, Tq, 200, 60)
    e = torch.zeros(D)
    e[0] = 1.0
    x["q"] = (e * 2.0 ** 16 * (1 + torch.arange(Tq)[None, None, :, None] % 3)).expand(S, 2, Tq, D).to(BF)
    for n in ("pk", "k"):
        x[n][..., 0] = (torch.randint(-8, 9, x[n].shape[:3], generator=gen(1)) * 256.0).to(BF)
    check(dev, x, scale=2.0)
    x["q"] = x["q"] * 0
    check(dev, x)


def test_strides_and_alignment(dev):
    """Views of fused projections, odd addresses and strides, one prefix for all heads and sequences, out in q's memory."""
    g = gen(11)
    N, S, H, G, D, Tq, P, T = 2, 3, 2, 2, 64, 4, 90, 50
    x = inputs(g, N, S, H, G, D, Tq, P, T)
    want = ops.sdpa_prefix(*(t.to(dev) for t in x.values()))
    shift = lambda t: torch.cat([t.new_zeros(1), t.flatten()]).to(dev)[1:].view(t.shape)              # 2 bytes off 16
    wide = lambda t: torch.cat([t, t.new_zeros(*t.shape[:3], 3)], 3).to(dev)[..., :t.shape[3]]         # odd row stride
    swap = lambda t: t.transpose(1, 2).contiguous().to(dev).transpose(1, 2)                            # heads innermost
    cols = lambda t: t.transpose(2, 3).contiguous().to(dev).transpose(2, 3)                            # column stride
    for f in (shift, wide, swap, cols):
        assert torch.equal(ops.sdpa_prefix(*(f(t) for t in x.values())), want), f
    one = lambda t: t[:1, :1].to(dev).expand(N, H, *t.shape[2:])
    a = ops.sdpa_prefix(x["q"].to(dev), one(x["pk"]), one(x["pv"]), x["k"].to(dev), x["v"].to(dev))
    b = ops.sdpa_prefix(x["q"].to(dev), one(x["pk"]).contiguous(), one(x["pv"]).contiguous(), x["k"].to(dev), x["v"].to(dev))
    assert torch.equal(a, b)
    # a batch of one: the stride of its dimension is never walked
    q1 = x["q"][:1].to(dev).as_strided((1, H * G, Tq, D), (3, Tq * D, D, 1))
    y1 = {n: x[n][:1].to(dev) for n in ("pk", "pv", "k", "v")}
    assert torch.equal(ops.sdpa_prefix(q1, *y1.values()), ops.sdpa_prefix(x["q"][:1].to(dev), *y1.values()))
    # out over q, and as columns of a wider buffer
    buf = x["q"].transpose(1, 2).contiguous().to(dev)
    q = buf.transpose(1, 2)
    ops.sdpa_prefix(q, *(x[n].to(dev) for n in ("pk", "pv", "k", "v")), out=buf.view(N * S, Tq, -1))
    assert torch.equal(buf.view(N * S, Tq, -1), want)
    big = torch.full((N * S, Tq, H * G * D + 8), 7.0, device=dev, dtype=BF)
    ops.sdpa_prefix(*(t.to(dev) for t in x.values()), out=big[..., 4:-4])
    assert torch.equal(big[..., 4:-4], want) and bool((big[..., :4] == 7).all()) and bool((big[..., -4:] == 7).all())


def test_far_offsets(dev):
    """Own caches whose slots lie more than 2^32 bytes apart, and keys beyond 2^31 elements in a prefix."""
    D, H, T = 128, 1, 70
    slot = 2 ** 31 // 2 + 2 ** 28  # elements
    buf = torch.zeros(3 * slot + T * D, device=dev, dtype=BF)
    g = gen(5)
    x = inputs(g, 1, 4, H, 2, D, 1, 40, T)
    k = buf.as_strided((4, H, T, D), (slot, T * D, D, 1))
    k.copy_(x["k"])
    want = ops.sdpa_prefix(*(t.to(dev) for t in x.values()))
    assert torch.equal(ops.sdpa_prefix(x["q"].to(dev), x["pk"].to(dev), x["pv"].to(dev), k, x["v"].to(dev)), want)
    st = 2 ** 23 - 8  # rows 2^24 bytes apart: the last lies 2^32 bytes and more behind the first
    pk = buf.as_strided((1, H, buf.numel() // st, D), (0, 0, st, 1))
    assert (pk.shape[2] - 1) * st * 2 > 2 ** 32
    y = rnd(g, *pk.shape)
    pk.copy_(y)
    for Tq in (1, 40):
        q = rnd(g, 4, 2, Tq, D).to(dev)
        got = ops.sdpa_prefix(q, pk, y.to(dev), x["k"].to(dev), x["v"].to(dev))
        assert torch.equal(got, ops.sdpa_prefix(q, y.to(dev), y.to(dev), x["k"].to(dev), x["v"].to(dev)))


def test_streams_and_graphs(dev):
    """Two captured graphs replayed in turn with eager calls between, on streams of their own; lengths change between replays."""
    shapes = [(1, 6, 4, 2, 64, 1, 3000, 200), (2, 20, 2, 1, 128, 1, 900, 50), (1, 3, 2, 2, 128, 30, 2500, 100)]
    runs = []
    for i, s in enumerate(shapes):
        x = {n: t.to(dev) for n, t in inputs(gen(i), *s).items()}
        kv, pl = i32(dev, [s[7]] * (s[0] * s[1])), i32(dev, [s[6]] * s[0])
        call = lambda x=x, kv=kv, pl=pl: ops.sdpa_prefix(*x.values(), kv, pl)
        call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        runs.append((graph, out, call, kv, pl, s))
    g = gen(77)
    side = [torch.cuda.Stream() for _ in runs]
    for _ in range(4):
        for graph, out, call, kv, pl, s in runs:
            kv.copy_(torch.randint(0, s[7] + 1, kv.shape, generator=g))
            pl.copy_(torch.randint(0, s[6] + 1, pl.shape, generator=g))
        want = [r[2]().clone() for r in runs]
        torch.cuda.synchronize()
        for st, (graph, *_) in zip(side, runs):
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        for w, r in zip(want, runs):
            assert torch.equal(w, r[1])


def test_a_run_of_one_prefix_is_the_plain_attention(dev):
    """With the prefix's keys copied before each sequence's own, sdpa gives the same within the bound."""
    N, S, H, G, D, Tq, P, T = 1, 4, 3, 1, 64, 20, 130, 45
    x = inputs(gen(2), N, S, H, G, D, Tq, P, T)
    got = check(dev, x)
    full = lambda a, b: torch.cat([a.expand(S, -1, -1, -1), b], 2).contiguous().to(dev)
    ref = ops.sdpa(x["q"].to(dev), full(x["pk"], x["k"]), full(x["pv"], x["v"]), qpos0=P + T - Tq, causal_from=P)
    o, mag, _ = ob.sdpa_prefix(*x.values())
    assert bool(((got.cpu().to(F64) - ref.cpu().to(F64)).abs() <= 2 * 3.1 * 2.0 ** -8 * (mag + o.abs())).all())
