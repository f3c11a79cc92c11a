"""Beam selection, slot reordering and the rotary embedding at rows on the device, on the MI355X against the 64-bit oracle:
choices exactly, scores within a bound derived from their roundings."""
import math

import pytest
import torch

import oracle.beams as ob
import strix_halo_maxx_amd.ops as ops
from beam_cases import SELECT
from strix_halo_maxx_amd import _lib
from strix_halo_maxx_amd.synth import freqs_cis

pytestmark = pytest.mark.gpu
BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64
INF, NAN = math.inf, math.nan


def gen(seed):
    return torch.Generator().manual_seed(seed)


def model_logits(g, B, W, V, dtype=BF):
    """A broad bulk, a few dozen likely tokens."""
    x = torch.randn(B, W, V, generator=g) * 2 + 9 * torch.rand(B, W, V, generator=g) * (torch.rand(B, W, V, generator=g) < 32 / V)
    return x.to(dtype)


def check(dev, logits, scores, k=None, done=None, eos=None, view=lambda t: t):
    k = logits.shape[1] if k is None else k
    want = ob.beam_select(logits, scores, k, done, eos)
    to = lambda t: None if t is None else t.to(dev)
    got = ops.beam_select(view(to(logits)), to(scores), k, done=to(done), eos=eos)
    s, p, t, d = (None if x is None else x.cpu() for x in got)
    assert s.dtype == F32 and p.dtype == t.dtype == torch.int32 and torch.equal(p, want[1]) and torch.equal(t, want[2])
    assert (d is None) == (eos is None) and (d is None or torch.equal(d, want[3]))
    # the log-sum: exponentials off by 2^-22 of themselves (their argument, up to 2^5 in base 2 where it counts, and the
    # instruction), sums of at most 32 terms a lane and 8 steps between lanes by 2^-18; the value's rounding by 2^-24 of it
    fine = want[0] > -INF
    assert torch.equal(fine, s > -INF)
    err = (s.to(F64) - want[0]).abs()[fine]
    assert bool((err <= 2.0 ** -17 + 2.0 ** -24 * want[0].abs()[fine]).all()), float(err.max())
    return got


def falling(g, B, W):
    return -(torch.rand(B, W, generator=g) * 20).sort(1)[0]


@pytest.mark.parametrize("case", SELECT, ids=str)
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
def test_select(dev, case, dtype):
    B, W, V, k = case
    g = gen(V + W)
    x, s = model_logits(g, B, W, V, dtype), falling(g, B, W)
    a = check(dev, x, s, k)
    b = ops.beam_select(x.to(dev), s.to(dev), k)
    assert all(torch.equal(u, v) for u, v in zip(a[:3], b[:3]))
    done = torch.rand(B, W, generator=g) < 0.4
    check(dev, x, s, k, done, eos=V - 1)
    check(dev, x, s, k, None, eos=0)


def test_select_ties(dev):
    """Equal logits, equal beams, -0 and 0: the lowest beam, then the lowest token."""
    g = gen(1)
    for V in (1, 7, 300, 5000, 20001):
        for k in (1, 5, 64):
            check(dev, torch.zeros(2, 3, V, dtype=BF), torch.zeros(2, 3), k)
            x = torch.randint(-2, 3, (2, 3, V), generator=g).to(BF)
            check(dev, x, torch.zeros(2, 3), k)                    # whole steps between values: ties and no near ones
            check(dev, x[:, :1].expand(2, 3, V).contiguous(), torch.tensor([[0.0, -1, 0], [0, 0, 0]]), k)
            z = torch.where(torch.rand(2, 3, V, generator=g) < 0.5, 0.0, -0.0).to(BF)
            check(dev, z, torch.zeros(2, 3), k)
            check(dev, torch.arange(V).expand(1, 2, V).float().contiguous(), torch.tensor([[0.0, -0.5]]), k)  # rising
            check(dev, -torch.arange(V).expand(1, 2, V).float().contiguous(), torch.tensor([[0.0, -0.5]]), k)


def test_select_large_ties(dev):
    """The same where a lane holds 32 logits."""
    check(dev, torch.zeros(40, 16, 9000, dtype=BF), torch.zeros(40, 16), 16)
    x = torch.randint(-1, 2, (40, 16, 9000), generator=gen(2)).to(BF)
    check(dev, x, torch.zeros(40, 16), 32)
    check(dev, torch.arange(9000).expand(40, 16, 9000).float().contiguous(), torch.zeros(40, 16), 20)


def test_select_many_lists(dev):
    """More parts of rows than can all be ranked: ties among them, beams of one part's weight, most of them empty."""
    g = gen(3)
    for V, k in ((6200, 64), (6200, 3), (90000, 64)):
        W = 64 if V < 9000 else 20
        check(dev, torch.zeros(1, W, V, dtype=BF), torch.zeros(1, W), k)
        check(dev, torch.randint(-1, 2, (1, W, V), generator=g).to(BF), torch.zeros(1, W), k)
        check(dev, torch.arange(V).expand(1, W, V).float().contiguous(), -torch.arange(W).float()[None] / 2, k)
        s = torch.full((1, W), -INF)
        s[0, 5] = -1.0
        x = model_logits(g, 1, W, V, F32)
        check(dev, x, s, k)
        check(dev, torch.where(torch.rand(1, W, V, generator=g) < 1e-4, x, -INF), torch.zeros(1, W), k)
        check(dev, x, torch.zeros(1, W), k, torch.rand(1, W, generator=g) < 0.9, eos=2)


def test_select_nothing_to_offer(dev):
    """Scores and logits that are infinite or NaN, all finished, banned tokens, fewer candidates than places."""
    g = gen(4)
    V = 600
    x = model_logits(g, 6, 4, V, F32)
    s = falling(g, 6, 4)
    s[0] = torch.tensor([0.0, -INF, -INF, -INF])   # a first step: one beam
    s[1] = torch.tensor([NAN, INF, -INF, -3.0])
    s[2] = -INF
    x[3, 0, 5], x[3, 1, 77], x[3, 2] = NAN, INF, -INF
    x[4] = -INF
    x[4, 1, 9], x[4, 2, 3] = 1.0, -2.0             # two candidates in all
    x[5, :, :] = torch.where(torch.rand(V, generator=g) < 0.9, -INF, x[5])
    for k in (1, 4, 9, 64):
        check(dev, x, s, k)
        check(dev, x, s, k, torch.tensor([[False] * 4, [True] * 4, [True] * 4, [True, False, True, True], [True] * 4, [False, True] * 2]), eos=3)
    check(dev, x.to(BF), s, 5, torch.ones(6, 4, dtype=torch.bool), eos=V - 1)
    check(dev, torch.full((1, 1, 1), 3.0), torch.tensor([[-2.0]]), 4)


def test_select_extremes(dev):
    """Logits near the types' limits, and scores far below the logits' spacing."""
    g = gen(6)
    x = model_logits(g, 2, 4, 3001, F32)
    check(dev, x * 1e36, falling(g, 2, 4))
    check(dev, x * 1e-42, falling(g, 2, 4), 3)     # subnormals: closer than fp64 resolves beside the sum
    check(dev, x, falling(g, 2, 4) * 1e6)


def test_select_strides(dev):
    """Rows at odd addresses, beams and searches interleaved, columns strided."""
    g = gen(8)
    B, W, V = 3, 4, 5003
    s = falling(g, B, W)
    for dtype in (BF, F32):
        x = model_logits(g, B, W, V, dtype)
        check(dev, x, s, view=lambda t: torch.cat([t.new_zeros(1), t.flatten()])[1:].view(t.shape))
        check(dev, x, s, view=lambda t: torch.cat([t, t.new_full((B, W, 5), 99.0)], 2)[..., :V])
        check(dev, x, s, view=lambda t: t.transpose(0, 1).contiguous().transpose(0, 1))
        check(dev, x, s, view=lambda t: t.transpose(1, 2).contiguous().transpose(1, 2))
    one = model_logits(g, 1, 1, V)
    check(dev, one.expand(B, W, V), s, view=lambda t: one.to(dev).expand(B, W, V))
    assert ops.beam_select(torch.empty(0, 4, 10, device=dev), torch.empty(0, 4, device=dev))[0].shape == (0, 4)


def test_select_graphs(dev):
    """Two captured selections replayed in turn on two streams, eager calls between."""
    g = gen(10)
    runs = []
    for B, W, V, k in ((1, 4, 51200, 4), (3, 8, 7001, 16)):
        x, s, d = model_logits(g, B, W, V).to(dev), falling(g, B, W).to(dev), torch.zeros(B, W, dtype=torch.bool, device=dev)
        call = lambda x=x, s=s, d=d, k=k: ops.beam_select(x, s, k, done=d, eos=1)
        call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        runs.append((graph, out, call, x, s, d))
    side = [torch.cuda.Stream() for _ in runs]
    for _ in range(4):
        for _, _, _, x, s, d in runs:
            x.copy_(model_logits(g, *x.shape))
            s.copy_(falling(g, *s.shape))
            d.copy_(torch.rand(d.shape, generator=g) < 0.3)
        want = [[t.clone() for t in r[2]()] for r in runs]
        torch.cuda.synchronize()
        for st, r in zip(side, runs):
            with torch.cuda.stream(st):
                r[0].replay()
        torch.cuda.synchronize()
        for w, r in zip(want, runs):
            assert all(torch.equal(a, b) for a, b in zip(w, r[1]))


# ------------------------------------------------------------------------------------------------ slots
def moved(dev, x, parent, n=None, first=0, unit=1):
    want = ob.reorder_slots(x, parent, n, first, unit)
    y = x.to(dev)
    nd = n if n is None or isinstance(n, int) else torch.tensor(n, device=dev, dtype=torch.int32)
    assert ops.reorder_slots(y, parent.to(dev), nd, first, unit) is y
    bits = lambda t: t.contiguous().view(torch.uint8)
    assert torch.equal(bits(y.cpu()), bits(want))


@pytest.mark.parametrize("W", [1, 2, 3, 4, 5, 8, 9, 16, 17, 32, 33, 64])
def test_reorder(dev, W):
    g = gen(W)
    for G, H, T, D in ((1, 3, 37, 64), (3, 1, 5, 128), (2, 2, 1, 8)):
        x = torch.randn(2, G * W, H, T, D, generator=g).to(BF)
        parent = torch.randint(0, W, (G, W), generator=g, dtype=torch.int32)
        moved(dev, x, parent)
        moved(dev, x, parent, T // 2)
        n = torch.randint(-2, T + 3, (G * W,), generator=g).tolist()
        moved(dev, x, parent, n, first=T // 3)
        moved(dev, x, torch.arange(W, dtype=torch.int32).flip(0).expand(G, W), n)      # pairs exchange
        moved(dev, x, torch.roll(torch.arange(W, dtype=torch.int32), 1).expand(G, W))  # a cycle
        moved(dev, x, torch.zeros(G, W, dtype=torch.int32), n)                         # a fork
        odd = torch.randint(-3, W + 3, (G, W), generator=g, dtype=torch.int32)         # some slots stay
        odd[0, 0] = 2 ** 31 - 1
        moved(dev, x, odd, n, first=1)


@pytest.mark.parametrize("shape,dtype", [((2, 4, 3, 9, 5), torch.uint8), ((1, 4, 2, 11), torch.uint8), ((2, 4, 2, 7, 3), F32),
                                         ((1, 4, 2, 7, 2, 3), torch.int64), ((3, 4, 1, 6, 20), BF), ((1, 4, 2, 5, 1), BF)], ids=str)
def test_reorder_types_and_units(dev, shape, dtype):
    """Rows of any size and type; rows that stand for several tokens."""
    g = gen(len(shape))
    x = torch.randint(0, 250, shape, generator=g).to(dtype)
    parent = torch.tensor([2, 2, 0, 1], dtype=torch.int32)
    moved(dev, x, parent)
    for first, n in ((0, 3 * 7), (8, [0, 1, 7, 400]), (13, [14, 7, 8, 15])):
        moved(dev, x, parent, n, first, unit=7) if not isinstance(n, int) or n <= 7 * shape[3] else None
    moved(dev, x, parent, first=10 ** 6)
    moved(dev, x, parent, first=2 ** 32)


def test_reorder_views(dev):
    """A cache that is part of a wider buffer, slots innermost, odd addresses; what is not in the view stays."""
    g = gen(3)
    buf = torch.randn(2, 3, 6, 11, 72, generator=g).to(BF)  # (L, H, slots, T + 1, D + 8)
    parent = torch.tensor([[1, 1, 0], [2, 0, 1]], dtype=torch.int32)
    for cut in (lambda t: t[..., :10, :64].transpose(1, 2), lambda t: t[..., 1:, 3:67].transpose(1, 2)):
        want = buf.clone()
        cut(want).copy_(ob.reorder_slots(cut(buf), parent, 8))
        got = buf.to(dev)
        ops.reorder_slots(cut(got), parent.to(dev), 8)
        assert torch.equal(got.cpu(), want)
    wide = torch.stack([parent, parent * 0 - 1], 2).to(dev)[..., 0]  # parents with strides of their own
    x = torch.randn(1, 6, 2, 5, 64, generator=g).to(BF)
    y = ops.reorder_slots(x.to(dev), wide)
    assert torch.equal(y.cpu(), ob.reorder_slots(x, parent))


def test_reorder_far(dev):
    """Slots more than 2^32 bytes apart, moved in place both ways."""
    step = 2 ** 32 + 4096
    buf = torch.zeros(2 * step + 8192, device=dev, dtype=torch.uint8)
    x = buf.as_strided((1, 3, 1, 20, 64), (3 * step, step, 20 * 64, 64, 1))
    y = torch.randint(0, 256, x.shape, generator=gen(1)).to(torch.uint8)
    x.copy_(y)
    parent = torch.tensor([2, 0, 1], dtype=torch.int32)
    ops.reorder_slots(x, parent.to(dev), 17)
    assert torch.equal(x.cpu(), ob.reorder_slots(y, parent, 17))


def test_kv8_reorder(dev):
    """Slots of an 8-bit cache: what each holds is what its parent held, bit for bit; blocks before `first` and behind the
    lengths stay."""
    g = gen(5)
    c = ops.KV8Cache(4, 3, 300, 64, device=dev)
    k, v = (torch.randn(4, 3, 300, 64, generator=g).to(BF).to(dev) for _ in range(2))
    lens = torch.tensor([300, 130, 64, 201], device=dev, dtype=torch.int32)
    c.append(k, v, 0, count=lens)
    before = c.read()
    parent = torch.tensor([3, 0, 0, 1], device=dev, dtype=torch.int32)
    c.reorder(parent, lens, first=70)
    for a, b in zip(c.read(), before):
        for s, p in enumerate(parent.tolist()):
            hi = int(lens[p])
            assert torch.equal(a[s, :, 64:hi], b[p, :, 64:hi])
            assert torch.equal(a[s, :, :64], b[s, :, :64])
            rest = -(-hi // 64) * 64
            assert torch.equal(a[s, :, rest:], b[s, :, rest:])


# ------------------------------------------------------------------------------------------------ rotary embedding
@pytest.mark.parametrize("B,n,H,ctx", [(1, 1, 32, 50), (5, 1, 3, 64), (2, 7, 4, 33)])
def test_rope_kv_at(dev, B, n, H, ctx):
    """The bits of mx_rope_kv at the same positions; rows outside the cache or the table are dropped."""
    g = gen(B)
    cs = freqs_cis(32, 500).to(dev).contiguous()
    qkv = torch.randn(B, n, 3 * H * 64 + 8, generator=g).to(BF).to(dev)[..., :3 * H * 64]
    at = torch.randint(-n, ctx + 2, (B,), generator=g, dtype=torch.int32)
    at[0] = 3
    for rot0 in (0, 400, -3):
        kc, vc = (torch.full((B, H, ctx, 64), 5.0, device=dev, dtype=BF) for _ in range(2))
        q = ops.rope_kv_at(qkv, cs, kc, vc, at.to(dev), rot0)
        wk, wv = (torch.full((B, H, ctx, 64), 5.0, device=dev, dtype=BF) for _ in range(2))
        for b in range(B):
            for t in range(n):
                r = int(at[b]) + t
                if not (0 <= r < ctx and 0 <= r + rot0 < 500):
                    continue
                row = qkv[b, t].contiguous()
                k1, v1 = (torch.empty(1, H, 500, 64, device=dev, dtype=BF) for _ in range(2))
                q1 = torch.empty(1, H, 1, 64, device=dev, dtype=BF)
                _lib.call("mx_rope_kv", _lib.stream(), row.data_ptr(), row.numel(), cs.data_ptr(), q1.data_ptr(), k1.data_ptr(),
                          v1.data_ptr(), 1, 1, H, 500, r + rot0, 1, 0)
                wk[b, :, r], wv[b, :, r] = k1[0, :, r + rot0], v1[0, :, r + rot0]
                assert torch.equal(q[b, :, t], q1[0, :, 0])
        assert torch.equal(kc, wk) and torch.equal(vc, wv)
