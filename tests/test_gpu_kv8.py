"""The 8-bit KV cache and attention over it on the MI355X against the 64-bit oracle: what the cache holds bit for bit, the
attention within a bound derived from its roundings."""
import pytest
import torch

import lowbit_cases as lc
import oracle.lowbit as ol
import strix_halo_maxx_amd.ops as ops
from strix_halo_maxx_amd import _lib
from strix_halo_maxx_amd.synth import freqs_cis

pytestmark = pytest.mark.gpu
BF, F64 = torch.bfloat16, torch.float64


def gen(seed):
    return torch.Generator().manual_seed(seed)


def same(a, b):
    """bf16 a is b, a double that bf16 holds exactly (but 2^128, to which the largest bf16 rounds: infinity)."""
    a, b = a.to(F64), torch.where(b.abs() == 2.0 ** 128, b * float("inf"), b)
    return bool(((a == b) | (a.isnan() & b.isnan())).all())


def rows(g, *shape, spread=0):
    x = torch.randn(*shape, generator=g)
    if spread:
        x = x * torch.exp2(torch.randint(-spread, spread + 1, shape[:-1] + (1,), generator=g).float())
    return x.to(BF)


def i32(dev, *v):
    return torch.tensor(v, device=dev, dtype=torch.int32)


class Both:
    """A cache and its oracle, written alike."""

    def __init__(self, dev, slots, H, ctx, D):
        self.dev, self.c = dev, ops.KV8Cache(slots, H, ctx, D, device=dev)
        self.k, self.v = ol.KV8(slots, H, ctx, D), ol.KV8(slots, H, ctx, D)
        self.end = [0] * slots  # where each sequence ends: what its last block holds behind that is undefined

    def append(self, k, v, pos, counts=None, **kw):
        B = k.shape[0]
        ps = [pos] * B if isinstance(pos, int) else list(pos)
        self.c.append(k.to(self.dev), v.to(self.dev), pos if isinstance(pos, int) else i32(self.dev, *pos),
                      count=None if counts is None else i32(self.dev, *counts), **kw)
        for b in range(B):
            n = k.shape[2] if counts is None else max(0, min(counts[b], k.shape[2]))
            for slot in range(self.c.slots) if kw.get("bcast") else (b,):
                self.k.append(slot, k[b, :, :n], ps[b])
                self.v.append(slot, v[b, :, :n], ps[b])
                if n and ps[b] < self.c.ctx and ps[b] + n > 0:
                    self.end[slot] = min(ps[b] + n, self.c.ctx)

    def check(self):
        for got, want in zip(self.c.read(), (self.k, self.v)):
            for slot, n in enumerate(self.end):
                rest = -(-n // 64) * 64  # blocks that were never written
                ok = same(got[slot, :, :n].cpu(), want.val[slot, :, :n]) and same(got[slot, :, rest:].cpu(), want.val[slot, :, rest:])
                assert ok, slot


@pytest.mark.parametrize("D", [64, 128])
def test_append_fresh_and_in_steps(dev, D):
    """A prompt, then single rows with larger and smaller values across a block border: exponents rise, codes follow."""
    g = gen(D)
    c = Both(dev, 2, 3, 200, D)
    c.append(rows(g, 2, 3, 61, D, spread=3), rows(g, 2, 3, 61, D, spread=3), 0)
    c.check()
    for t, s in enumerate((0.1, 8.0, 1.0, 300.0, 0.01, 2.0 ** 20, 1.0)):
        c.append((rows(g, 2, 3, 1, D).float() * s).to(BF), (rows(g, 2, 3, 1, D).float() / s).to(BF), 61 + t)
        c.check()
    c.append(rows(g, 2, 3, 100, D, spread=5), rows(g, 2, 3, 100, D), 68)
    c.check()


@pytest.mark.parametrize("D,ctx", [(64, 1), (128, 63), (64, 64), (128, 65), (64, 300)])
def test_append_positions_on_the_device(dev, D, ctx):
    """Ragged positions and counts; rows outside the cache are dropped; zero rows; negative and far positions."""
    g = gen(ctx)
    c = Both(dev, 6, 2, ctx, D)
    n = 70
    k, v = rows(g, 6, 2, n, D), rows(g, 6, 2, n, D)
    c.append(k, v, (0, ctx // 2, ctx - 1, ctx, -5, -1000), counts=(n, 1, n, n, n, n))
    c.check()
    c.append(k * 4, v, (2 ** 31 - 1, -2 ** 31, 0, 3, 1, ctx // 3), counts=(n, n, 0, 2, -3, 2 ** 31 - 1))
    c.check()


def test_append_special_values(dev):
    """Zeros, subnormals, the largest bf16, 448 and 449 times a power of two, ties, NaN and infinities."""
    g = gen(3)
    c = Both(dev, 1, 4, 128, 64)
    k = torch.zeros(1, 4, 64, 64)
    k[0, 0, 0, :4] = torch.tensor([448.0, 17.0, 19.0, 2.0 ** -9])     # exponent 0: 17, 19 halfway
    k[0, 0, 1, :4] = torch.tensor([1.5 * 2.0 ** -10, 2.0 ** -10, 3 * 2.0 ** -10, -27.0])
    k[0, 1, 5, :2] = torch.tensor([450.0, 17.0])                      # exponent 1
    k[0, 2] = torch.randn(64, 64, generator=g) * 2.0 ** -131
    k[0, 3, 7, :3] = torch.tensor([3.3895e38, 1e38, -1e30])
    v = torch.randn(1, 4, 64, 64, generator=g)
    v[0, 1, 3, 3], v[0, 2, 9, 9], v[0, 3, 1, 1] = float("nan"), float("inf"), float("-inf")
    c.append(k[:, :, :40].to(BF), v[:, :, :40].to(BF), 0)
    c.append(k[:, :, 40:].to(BF) + 1, 100 * v[:, :, 40:].to(BF), 40)  # the kept NaN codes are rounded again
    c.check()


def test_append_strides_and_alignment(dev):
    """Views of a fused projection, odd addresses and strides, broadcast rows."""
    g = gen(5)
    H, n, D = 3, 77, 64
    qkv = rows(g, 2, n, 3 * H * D + 3)
    c = Both(dev, 2, H, 128, D)
    qd = qkv.to(dev)
    for off in (0, 3):
        part = lambda x, i: x[:, :, off + i * H * D:off + (i + 1) * H * D].unflatten(2, (H, D)).transpose(1, 2)
        c.c.append(part(qd, 1), part(qd, 2), 5 + off)
        for b in range(2):
            c.k.append(b, part(qkv, 1)[b], 5 + off)
            c.v.append(b, part(qkv, 2)[b], 5 + off)
            c.end[b] = 5 + off + n
        c.check()
    k, v = rows(g, 1, 1, n, D), rows(g, 1, H, D, n)
    c.c.append(k.to(dev).expand(2, H, n, D), v.to(dev).transpose(2, 3).expand(2, H, n, D), 0)
    for b in range(2):
        c.k.append(b, k[0].expand(H, n, D), 0)
        c.v.append(b, v[0].transpose(1, 2), 0)
        c.end[b] = n
    c.check()


def test_append_broadcast_and_rope(dev):
    """bcast writes every slot; the rotary form equals mx_rope_kv's rounded rows appended, and rotates q as it does."""
    g = gen(6)
    H, D, n, pos, ctx = 32, 64, 90, 37, 256
    cs = freqs_cis(32, ctx).to(dev)
    qkv = rows(g, n, 3 * H * D).to(dev)
    q = torch.empty(1, H, n, D, device=dev, dtype=BF)
    kc, vc = torch.zeros(2, H, ctx, D, device=dev, dtype=BF), torch.zeros(2, H, ctx, D, device=dev, dtype=BF)
    _lib.call("mx_rope_kv", _lib.stream(), qkv.data_ptr(), qkv.stride(0), cs.data_ptr(), q.data_ptr(), kc.data_ptr(),
              vc.data_ptr(), 1, n, H, ctx, pos, 2, 1)
    part = [qkv[:, i * H * D:(i + 1) * H * D].view(1, n, H, D).transpose(1, 2) for i in range(3)]
    want, got = ops.KV8Cache(2, H, ctx, D, device=dev), ops.KV8Cache(2, H, ctx, D, device=dev)
    want.append(kc[:1, :, pos:pos + n], vc[:1, :, pos:pos + n], pos, bcast=True)
    for p, b in ((pos, 0), (i32(dev, pos - 30), 30)):
        q2 = got.append(part[1], part[2], p, base=b, bcast=True, cs=cs, q=part[0])
        assert torch.equal(q2, q)
        for x, y in zip(want.read() + (want.ks, want.vs), got.read() + (got.ks, got.vs)):
            assert torch.equal(x, y)


def test_read_part(dev):
    g = gen(7)
    c = Both(dev, 2, 2, 150, 128)
    c.append(rows(g, 2, 2, 150, 128), rows(g, 2, 2, 150, 128), 0)
    for n in (1, 64, 65, 149):
        k, v = c.c.read(n)
        ok = same(k.cpu(), c.k.val[:, :, :n]) and same(v.cpu(), c.v.val[:, :, :n])
        assert ok
    assert c.c.read(0)[0].shape == (2, 2, 0, 128)


def check_sdpa(y, q, c, lens, **kw):
    """The output's rounding, 2^-8 of it; per weight 2^-8 (two e4m3 terms, half a step of 2^-4 each: 2^-4 2^-4) and the
    error of its score, taken as 2^-12 of the largest sum |q k| scale for the MFMA's sums; the product with V, 2^-12 of
    the mean |v|. A weight's error moves numerator and denominator: twice."""
    for b, n in enumerate(lens):
        ref, avg, size = ol.sdpa(q[b], c.k.val[b], c.v.val[b], n, **kw)
        out = y[b].to(F64).view(ref.shape)
        tol = 2.0 ** -8 * ref.abs() + (2.0 ** -8 + 2.0 ** -12 + 2 * 2.0 ** -12 * (1 + size)) * avg
        bad = (out - ref).abs() > tol
        assert not bool(bad.any()) and not bool(out.isnan().any()), (b, n, (out - ref).abs().max().item())


# slots' lengths, H, G, D, Tq, causal_from
SDPA = [((1,), 1, 1, 64, 1, None), ((0, 1, 63, 64, 65), 2, 1, 64, 1, None), ((130, 5, 700), 4, 4, 128, 1, None),
        ((1000,), 32, 1, 64, 1, 0), ((2100, 17), 2, 8, 128, 1, None), ((70, 3), 1, 32, 64, 1, None),
        ((40, 200), 3, 3, 64, 5, 0), ((33, 90, 0), 2, 1, 64, 40, 0), ((300, 64), 2, 4, 128, 37, 50),
        ((150,), 2, 2, 64, 150, 100), ((128, 129), 1, 7, 128, 129, 0), ((4500,), 1, 2, 64, 3, 0)]
# ways a prompt is cut: heads x rows of two workgroups per CU, of one, 64-row groups, 32-row groups, runs of keys with 64 and 128
# rows; a case for each kernel: lowbit_cases.py
CUTS = [((200,), 64, 8, 64, 130, 0), ((200,), 32, 8, 128, 130, 60), ((130,), 32, 7, 64, 120, 0), ((150,), 24, 8, 128, 128, None),
        ((200, 190), 48, 1, 64, 130, 0), ((300,), 32, 4, 128, 100, 0), ((500, 13), 8, 1, 64, 70, 0), ((700,), 4, 4, 128, 30, 0),
        ((17000,), 1, 1, 64, 50, 0), ((16700,), 1, 4, 128, 16, None), ((16500,), 1, 4, 64, 40, 100), ((16900,), 1, 8, 128, 12, 0)]


@pytest.mark.parametrize("lens,H,G,D,Tq,cf", SDPA)
def test_sdpa(dev, lens, H, G, D, Tq, cf):
    g = gen(sum(lens) + 13 * H + G + D + Tq)
    B, ctx = len(lens), max(lens) + 11
    c = Both(dev, B + 1, H, ctx, D)
    n = max(max(lens), 1)
    c.append(rows(g, B, H, n, D, spread=1), rows(g, B, H, n, D, spread=1), 0, counts=lens)
    q = rows(g, B, H * G, Tq, D)
    print("sdpa_kv8", lens, H, G, D, Tq, cf, flush=True)
    y = ops.sdpa_kv8(q.to(dev), c.c, i32(dev, *lens), causal_from=cf)
    check_sdpa(y.cpu(), q, c, lens, causal_from=cf)
    # lengths from the host, a base with the tensor, positions given
    if len(set(lens)) == 1:
        assert torch.equal(ops.sdpa_kv8(q.to(dev), c.c, lens[0], causal_from=cf), y)
        assert torch.equal(ops.sdpa_kv8(q.to(dev), c.c, lens[0], causal_from=cf, qpos0=lens[0] - Tq), y)
    assert torch.equal(ops.sdpa_kv8(q.to(dev), c.c, i32(dev, *[n - 7 for n in lens]), base=7, causal_from=cf), y)


@pytest.mark.parametrize("lens,H,G,D,Tq,cf", CUTS)
def test_sdpa_cuts(dev, lens, H, G, D, Tq, cf):
    """The bound of check_sdpa, the oracle as matrix products in 64 bits on the GPU."""
    g = torch.Generator(device=dev).manual_seed(sum(lens) + H + Tq)
    B, n = len(lens), max(lens)
    r = lambda *s: torch.randn(*s, generator=g, device=dev).to(BF)
    c = ops.KV8Cache(B, H, n, D, device=dev)
    c.append(r(B, H, n, D), r(B, H, n, D) * 3, 0, count=i32(dev, *lens))
    q = r(B, H * G, Tq, D)
    print("cut", lens, H, G, D, Tq, cf, flush=True)
    y = ops.sdpa_kv8(q, c, i32(dev, *lens), causal_from=cf).double().view(B, Tq, H, G, D)
    k, v = (x.double() for x in c.read())
    for b, t in enumerate(lens):
        j, i = torch.arange(t, device=dev)[None], torch.arange(Tq, device=dev)[:, None]
        seen = (j < t) if cf is None else (j < cf) | (j <= t - Tq + i)
        for h in range(H):
            kk, vv = k[b, h, :t], v[b, h, :t]
            qq = q[b, h * G:(h + 1) * G].double()
            s = (torch.matmul(qq, kk.t().contiguous()) * D ** -0.5).masked_fill(~seen, -float("inf"))
            size = torch.matmul(qq.abs(), kk.t().abs().contiguous()).amax(-1, keepdim=True) * D ** -0.5
            p = torch.nan_to_num(torch.softmax(s, -1))
            ref, avg = torch.matmul(p, vv), torch.matmul(p, vv.abs())
            out = y[b, :, h].transpose(0, 1)
            tol = 2.0 ** -8 * ref.abs() + (2.0 ** -8 + 2.0 ** -12 + 2 * 2.0 ** -12 * (1 + size)) * avg
            ok = bool(((out - ref).abs() <= tol).all())
            assert ok, (b, h, ((out - ref).abs() - tol).max().item())


def test_sdpa_rows_that_see_nothing_are_zero(dev):
    """Queries before the first key, empty sequences, lengths outside the cache (clamped)."""
    g = gen(11)
    c = Both(dev, 4, 2, 100, 64)
    c.append(rows(g, 4, 2, 100, 64), rows(g, 4, 2, 100, 64), 0)
    q = rows(g, 4, 2, 6, 64)
    out = torch.full((4, 6, 128), 9.0, device=dev, dtype=BF)
    y = ops.sdpa_kv8(q.to(dev), c.c, i32(dev, 0, -7, 100, 10 ** 9), qpos0=-3, causal_from=0, out=out).cpu()
    assert y is not None and bool((out[:2] == 0).all()) and bool((out[2:, :3] == 0).all())
    check_sdpa(out.cpu(), q, c, (0, 0, 100, 100), qpos0=-3, causal_from=0)


@pytest.mark.parametrize("D,Tq,cf", [(64, 1, None), (128, 20, 0), (64, 70, 64)])
def test_sdpa_masked_keys_may_hold_nan(dev, D, Tq, cf):
    """NaN keys and values behind the sequence and behind each query change nothing; a query that sees one is NaN."""
    g = gen(D + Tq)
    n, ctx, at = 150, 200, 141
    k, v, q = rows(g, 1, 2, ctx, D), rows(g, 1, 2, ctx, D), rows(g, 1, 4, Tq, D)
    clean = Both(dev, 1, 2, ctx, D)
    clean.append(k, v, 0)
    k, v = k.clone(), v.clone()
    k[:, :, n:], v[:, :, n:] = float("nan"), float("inf")
    c = Both(dev, 1, 2, ctx, D)
    c.append(k, v, 0)
    c.k.val[:, :, n:], c.v.val[:, :, n:] = 0, 0
    y = ops.sdpa_kv8(q.to(dev), c.c, n, causal_from=cf)
    check_sdpa(y.cpu(), q, c, (n,), causal_from=cf)
    if Tq == 1:
        return
    # one value at position `at` of head 1: queries at .. see it (with the mask), the others do not
    c.c.append(k[:, :, at:at + 1].to(dev), torch.full((1, 2, 1, D), float("nan"), device=dev, dtype=BF), at)
    y2 = ops.sdpa_kv8(q.to(dev), c.c, n, causal_from=cf).cpu().float()
    sees = torch.arange(Tq) + n - Tq >= at
    assert bool(y2[0, sees].isnan().all()) and not bool(y2[0, ~sees].isnan().any())
    k2 = k.clone()
    k2[:, :, at] = float("nan")
    c.c.append(k2[:, :, at:at + 1].to(dev), v[:, :, at:at + 1].to(dev), at)
    y3 = ops.sdpa_kv8(q.to(dev), c.c, n, causal_from=cf).cpu().float()
    assert bool(y3[0, sees].isnan().all()) and not bool(y3[0, ~sees].isnan().any())


def test_sdpa_non_finite_queries_and_extreme_scores(dev):
    """A NaN or infinite query gives a NaN row and no other; one key that outweighs the rest by 2^100 is its value; equal
    scores average; a long tail of small weights under one large one is kept."""
    g = gen(21)
    D, n = 64, 640
    c = Both(dev, 1, 1, n, D)
    k, v = rows(g, 1, 1, n, D) * 0.01, rows(g, 1, 1, n, D)
    k[0, 0, 77] = 0
    k[0, 0, 77, 0] = 16.0
    c.append(k, v, 0)
    q = rows(g, 1, 1, 6, D)
    q[0, 0, 1, 3], q[0, 0, 2, 5] = float("nan"), float("inf")
    q[0, 0, 3] = 0
    q[0, 0, 3, 0] = 64.0   # score 128 against about 0.08
    q[0, 0, 4] = 0         # equal scores
    q[0, 0, 5] = 0
    q[0, 0, 5, 0] = 5.5    # weight e^11 (59874) against 639 of about 1
    y = ops.sdpa_kv8(q.to(dev), c.c, n).cpu()
    assert bool(y[0, 1:3].isnan().all()) and not bool(y[0, [0, 3, 4, 5]].isnan().any())
    keep = [0, 3, 4, 5]
    check_sdpa(y[:, keep], q[:, :, keep], c, (n,))


def test_sdpa_strides_out_and_other_slots(dev):
    """q as a view of a fused projection, an output inside a larger buffer, fewer sequences than slots, unaligned q."""
    g = gen(31)
    B, H, G, D, Tq, n = 2, 2, 2, 64, 9, 100
    c = Both(dev, 3, H, 128, D)
    c.append(rows(g, 3, H, n, D), rows(g, 3, H, n, D), 0)
    fused = rows(g, B, Tq, 3 * H * G * D + 5)
    for off in (0, 3):
        q = fused[:, :, off:off + H * G * D].unflatten(2, (H * G, D)).transpose(1, 2)
        qd = fused.to(dev)[:, :, off:off + H * G * D].unflatten(2, (H * G, D)).transpose(1, 2)
        big = torch.full((B, Tq + 2, H * G * D + 12), 5.0, device=dev, dtype=BF)
        out = big[:, 1:-1, 4:4 + H * G * D]
        ops.sdpa_kv8(qd, c.c, n, out=out, causal_from=0)
        check_sdpa(out.cpu(), q, c, (n, n), causal_from=0)
        out.fill_(5.0)
        assert bool((big == 5.0).all())


@pytest.mark.parametrize("n,D,G", [(300, 64, 1), (6000, 128, 4)])
def test_step_in_a_graph(dev, n, D, G):
    """Append and attend with the position on the device: a captured graph replayed step by step equals the eager steps,
    also with two graphs of the same calls replayed in turn."""
    g = gen(n)
    H, steps, ctx = 2, 6, n + 20
    k0, v0 = rows(g, 1, H, n, D).to(dev), rows(g, 1, H, n, D).to(dev)
    ks, vs = rows(g, steps, 1, H, 1, D, spread=2).to(dev), rows(g, steps, 1, H, 1, D).to(dev)
    qs = rows(g, steps, 1, H * G, 1, D).to(dev)
    a, b = ops.KV8Cache(1, H, ctx, D, device=dev), ops.KV8Cache(1, H, ctx, D, device=dev)
    want = []
    a.append(k0, v0, 0)
    for t in range(steps):
        a.append(ks[t], vs[t], n + t)
        want.append(ops.sdpa_kv8(qs[t], a, n + t + 1))
    pos, kb, vb, qb = i32(dev, 0), ks[0].clone(), vs[0].clone(), qs[0].clone()
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            b.append(kb, vb, pos, base=n)
            y = ops.sdpa_kv8(qb, b, pos, base=n + 1)
            pos.add_(1)
        graphs.append((gr, y))
    for _ in range(2):
        b.kc.zero_(), b.vc.zero_(), b.ks.zero_(), b.vs.zero_(), pos.zero_()
        b.append(k0, v0, 0)
        for t in range(steps):
            kb.copy_(ks[t]), vb.copy_(vs[t]), qb.copy_(qs[t])
            gr, y = graphs[t % 2]
            gr.replay()
            assert torch.equal(y, want[t]), t
            torch.cuda.synchronize()
        for x, z in zip(a.read(), b.read()):
            assert torch.equal(x, z)


def test_offsets_past_32_bits(dev):
    """Codes beyond 4 GB: the last slot's last tokens are written, read by attention, and the rest stays as it was. Every
    other key is zero, so it weighs exp(0) and adds nothing; the reference counts them."""
    g = gen(41)
    H, D, n = 17, 128, 300
    ctx = (1 << 20) - 5
    c = ops.KV8Cache(2, H, ctx, D, device=dev)
    k, v, q = rows(g, 2, H, n, D), rows(g, 2, H, n, D), rows(g, 2, 2 * H, 20, D)
    c.append(k.to(dev), v.to(dev), i32(dev, 0, ctx - n))
    assert c.kc.numel() > 1 << 32
    ko, vo = ol.KV8(1, H, 320, D), ol.KV8(1, H, 320, D)
    off = (ctx - n) % 64
    ko.append(0, k[1], off), vo.append(0, v[1], off)
    kk, vv = ko.val[0, :, off:off + n].to(F64), vo.val[0, :, off:off + n].to(F64)
    for Tq in (1, 20):
        y = ops.sdpa_kv8(q[:, :, :Tq].to(dev).contiguous(), c, ctx).to(F64).view(2, Tq, 2 * H, D).cpu()
        for h in (0, 2 * H - 1):
            qq = q[1, h, :Tq].to(F64)
            s = torch.matmul(qq, kk[h // 2].t().contiguous()) * D ** -0.5
            size = (torch.matmul(qq.abs(), kk[h // 2].t().abs().contiguous()) * D ** -0.5).amax(-1, keepdim=True)
            m = s.amax(-1, keepdim=True).clamp_min(0)
            p = torch.exp(s - m)
            l = p.sum(-1, keepdim=True) + (ctx - n) * torch.exp(-m)
            ref, avg = torch.matmul(p, vv[h // 2]) / l, torch.matmul(p, vv[h // 2].abs()) / l
            tol = 2.0 ** -8 * ref.abs() + (2.0 ** -8 + 2.0 ** -12 + 2 * 2.0 ** -12 * (1 + size)) * avg
            # the fp32 running sums of a million weights: at most 2^14 terms each before they are joined
            tol = tol + 2.0 ** -10 * avg
            err = ((y[1, :, h] - ref).abs() - tol).max().item()
            assert err <= 0, (Tq, h, err)
    blk = (ctx - n) // 64
    assert not bool(c.kc[1, :, :blk].any()) and not bool(c.kc[0, :, 5:].any()) and not bool(c.ks[1, :, :blk].any())


def test_two_calls_at_once(dev):
    """Attention over one cache from two streams at the same time, each cut into runs of keys: every call has its own
    workspace."""
    g = gen(43)
    H, D, n = 4, 64, 9000
    c = ops.KV8Cache(1, H, n, D, device=dev)
    c.append(rows(g, 1, H, n, D).to(dev), rows(g, 1, H, n, D).to(dev), 0)
    qs = [rows(g, 1, H, 1, D).to(dev) for _ in range(2)]
    want = [ops.sdpa_kv8(q, c, n) for q in qs]
    torch.cuda.synchronize()
    st = [torch.cuda.Stream() for _ in qs]
    got = [[], []]
    for _ in range(20):
        for i in (0, 1):
            with torch.cuda.stream(st[i]):
                got[i].append(ops.sdpa_kv8(qs[i], c, n))
    torch.cuda.synchronize()
    for i in (0, 1):
        assert all(torch.equal(y, want[i]) for y in got[i])


def test_far_positions_and_masks(dev):
    """Mask positions beyond 32 bits mean what they say: every key, or none."""
    g = gen(44)
    c = Both(dev, 1, 2, 100, 64)
    c.append(rows(g, 1, 2, 100, 64), rows(g, 1, 2, 100, 64), 0)
    q = rows(g, 1, 2, 40, 64)
    full = ops.sdpa_kv8(q.to(dev), c.c, 100)
    for kw in (dict(causal_from=2 ** 33), dict(causal_from=0, qpos0=2 ** 32 + 5), dict(causal_from=0, qpos0=2 ** 31 - 1)):
        assert torch.equal(ops.sdpa_kv8(q.to(dev), c.c, 100, **kw), full), kw
    for q0 in (-2 ** 31, -2 ** 32 + 50):
        assert not bool(ops.sdpa_kv8(q.to(dev), c.c, 100, causal_from=0, qpos0=q0).any()), q0


# H, G, D, Tq, keys: the few-row kernel, 32-, 64- and 128-row tiles, runs of keys that are joined
BIG = [(2, 1, 64, 30, 130), (1, 4, 128, 8, 130), (2, 1, 64, 90, 130), (1, 4, 128, 40, 130), (128, 1, 64, 60, 130), (32, 8, 128, 90, 70),
       (1, 1, 64, 30, 5000), (1, 1, 128, 50, 17000)]


@pytest.mark.parametrize("H,G,D,Tq,n", BIG)
def test_sdpa_scores_up_to_the_stated_limit(dev, H, G, D, Tq, n):
    """Scores of either sign from 2^-2 to 2^29 in size, mantissas of all kinds. One column of q and k is not zero, so a score is
    one exact product and the softmax in 64 bits is known: beyond small scores it is the mean of the values at the largest.
    A weight may be off by 2^-8 and by the exponential's 2^-12 with the score's rounding (2^-23 of scores below 32, where two
    different ones both count): numerator and denominator, twice."""
    g = torch.Generator(device=dev).manual_seed(H + D + Tq + n)
    r = lambda *s: torch.rand(*s, generator=g, device=dev)
    sign = lambda *s: torch.where(r(*s) < 0.5, -1.0, 1.0)
    k = torch.zeros(1, H, n, D, device=dev)
    k[..., 5] = 13 * 2.0 ** 12 * sign(1, H, n)
    k[:, :, :64, 5] = -13 * 2.0 ** 12  # the running maximum moves
    v = torch.randn(1, H, n, D, generator=g, device=dev).to(BF)
    q = torch.zeros(1, H * G, Tq, D, device=dev)
    top = 2.0 ** 29 / (13 * 2.0 ** 12 * D ** -0.5)
    q[..., 5] = sign(1, H * G, Tq) * top * 0.99 * torch.exp2(-31 * r(1, H * G, Tq) * (r(1, H * G, Tq) < 0.7))
    q = q.to(BF)
    c = ops.KV8Cache(1, H, n, D, device=dev)
    c.append(k.to(BF), v, 0)
    print("large scores", H, G, D, Tq, n, flush=True)
    for m in (n, 1, 67):  # 1: one visible key is its value
        y = ops.sdpa_kv8(q, c, m).double().view(Tq, H, G, D)
        kk, vv = (x[0, :, :m].double() for x in c.read())
        s = (q.double().view(H, G * Tq, D)[..., 5:6] * kk[:, None, :, 5]) * D ** -0.5
        p = torch.softmax(s, -1)
        back = lambda x: x.view(H, G, Tq, D).permute(2, 0, 1, 3)
        ref, avg = back(torch.matmul(p, vv)), back(torch.matmul(p, vv.abs()))
        err = ((y - ref).abs() - 2.0 ** -8 * ref.abs() - 2 * (2.0 ** -8 + 2.0 ** -12) * avg).max().item()
        assert err <= 0, (m, err)


@pytest.mark.parametrize("D,Hq,Tq", [(64, 4, 1), (64, 4, 9), (128, 2, 1), (64, 1, 3)])
def test_sdpa_dimensions_of_size_one_carry_any_stride(dev, D, Hq, Tq):
    """One sequence, one token or one head, cut from buffers of odd pitch: strides that are never walked refuse nothing, for q and
    for out."""
    g = gen(D + Hq + Tq)
    c = Both(dev, 1, 1, 100, D)
    c.append(rows(g, 1, 1, 90, D), rows(g, 1, 1, 90, D), 0)
    q = rows(g, 1, Hq, Tq, D)
    want = ops.sdpa_kv8(q.to(dev), c.c, 90)
    check_sdpa(want.cpu(), q, c, (90,))
    W = Hq * D
    # (B, Tq, W) rows inside odd pitches: the batch's, and with one token the row's
    pitch = W + (3 if Tq == 1 else 8)
    fused = torch.empty(Tq * pitch + 8, device=dev, dtype=BF)
    view = fused.as_strided((1, Hq, Tq, D), (Tq * pitch + 3, D if Hq > 1 else 5, pitch, 1))
    view.copy_(q)
    big = torch.full((2 * (Tq * pitch + 8),), 5.0, device=dev, dtype=BF)
    out = big.as_strided((1, Tq, W), (Tq * pitch + 3, pitch, 1), 8)
    assert ops.sdpa_kv8(view, c.c, 90, out=out) is out and torch.equal(out, want)
    out.fill_(5.0)
    assert bool((big == 5.0).all())
    assert torch.equal(ops.sdpa_kv8(view, c.c, 90), want)


# more workgroups than the device holds at once: the last ones would read what the first ones have written
@pytest.mark.parametrize("B,H,G,D,Tq", [(2, 4, 2, 64, 1), (1, 4096, 1, 64, 32), (1, 32, 1, 128, 4096), (1, 64, 1, 64, 4096)])
def test_sdpa_onto_its_own_queries(dev, B, H, G, D, Tq):
    """out in q's memory: (B, Hq, Tq, D) read, (B, Tq, Hq D) written over it, and a shifted view."""
    g = torch.Generator(device=dev).manual_seed(B + H + Tq)
    r = lambda *s: torch.randn(*s, generator=g, device=dev).to(BF)
    c = ops.KV8Cache(B, H, 300, D, device=dev)
    c.append(r(B, H, 300, D), r(B, H, 300, D), 0)
    n = B * H * G * Tq * D
    mem = r(n + 8)
    q = mem[:n].view(B, H * G, Tq, D)
    want = ops.sdpa_kv8(q, c, 300, causal_from=0)
    for off in (0, 8):
        for _ in range(3):
            buf = mem.clone()
            out = buf[off:n + off].view(B, Tq, H * G * D)
            assert ops.sdpa_kv8(buf[:n].view(q.shape), c, 300, causal_from=0, out=out) is out and torch.equal(out, want), off


def exact_heads(q, k, v, n, cf, D):
    """Each (sequence, head) of q (B, H, G, Tq, D) over k, v (B, H, ctx, D) in 64 bits on the GPU: the output (G, Tq, D), the mean
    |v| under the weights, the root of the sum of squared weights times values, the largest sum |q k| scale of a row."""
    B, H, G, Tq, _ = q.shape
    for b in range(B):
        j, i = torch.arange(n[b], device=q.device)[None], torch.arange(Tq, device=q.device)[:, None]
        seen = (j < n[b]).expand(Tq, -1) if cf is None else (j < cf) | (j <= n[b] - Tq + i)
        for h in range(H):
            kk, vv, qq = k[b, h, :n[b]].double(), v[b, h, :n[b]].double(), q[b, h].double().reshape(G * Tq, D)
            s = torch.matmul(qq, kk.t().contiguous()).view(G, Tq, -1) * D ** -0.5
            size = torch.matmul(qq.abs(), kk.t().abs().contiguous()).view(G, Tq, -1) * D ** -0.5
            p = torch.nan_to_num(torch.softmax(s.masked_fill(~seen, -float("inf")), -1)).view(G * Tq, -1)
            back = lambda x: x.view(G, Tq, D)
            yield (b, h, back(torch.matmul(p, vv)), back(torch.matmul(p, vv.abs())),
                   back(torch.matmul(p * p, vv * vv)).sqrt(), size.amax(-1, keepdim=True) if n[b] else size.new_zeros(G, Tq, 1))


@pytest.mark.parametrize("lens,H,G,D,Tq,cf,ctx", lc.ATTENTION)
def test_sdpa_every_kernel(dev, lens, H, G, D, Tq, cf, ctx):
    """check_sdpa's bound on each value, and one on the whole in norm that lost bits would not pass (test_lowbit_host.py plants
    them): the output's rounding and the MFMA's sums, 2^-8 and 2^-14 of it; the weights' errors, 2^-9 each from their terms and
    2^-15 of the largest |q k| sum from their scores (the MFMA's 2^-16, twice), independent of one another, so that they add
    up in squares (spread), taken twice."""
    g = torch.Generator(device=dev).manual_seed(sum(lens) + H + Tq + D)
    r = lambda *s: torch.randn(*s, generator=g, device=dev).to(BF)
    B, n = len(lens), max(lens)
    c = ops.KV8Cache(B, H, ctx or n, D, device=dev)
    c.append(r(B, H, n, D), r(B, H, n, D) * 3, 0, count=i32(dev, *lens))
    q = r(B, H * G, Tq, D)
    print("kernel", lens, H, G, D, Tq, cf, ctx, ops.sdpa_kv8_tiling(B, H, G, Tq, c.ctx, D), flush=True)
    y = ops.sdpa_kv8(q, c, i32(dev, *lens), causal_from=cf).view(B, Tq, H, G, D)
    k, v = c.read(n)
    err2 = ref2 = spread2 = 0.0
    for b, h, ref, avg, spread, size in exact_heads(q.view(B, H, G, Tq, D), k, v, lens, cf, D):
        err = (y[b, :, h].double().transpose(0, 1) - ref).abs()
        worst = (err - 2.0 ** -8 * ref.abs() - (2.0 ** -8 + 2.0 ** -12 + 2 * 2.0 ** -12 * (1 + size)) * avg).max().item()
        assert worst <= 0, (b, h, worst)
        err2 += err.square().sum()
        ref2 += ref.square().sum()
        spread2 += ((2.0 ** -9 + 2.0 ** -15 * (1 + size)) * spread).square().sum()
    bound = (2.0 ** -8 + 2.0 ** -14) * float(ref2) ** 0.5 + 2 * float(spread2) ** 0.5
    print("norm", float(err2) ** 0.5, "bound", bound, "output", float(ref2) ** 0.5, flush=True)
    assert float(err2) ** 0.5 <= bound


@pytest.mark.parametrize("H,G,D,Tq", lc.MASKED)
def test_sdpa_masked_nan_changes_no_bit(dev, H, G, D, Tq):
    """On every kernel: keys and values of NaN behind the sequence, and behind each query, leave its bits as zeros there do (they
    do not count for a block's exponent either); queries that see one are NaN."""
    g = torch.Generator(device=dev).manual_seed(H + D + Tq)
    r = lambda *s: torch.randn(*s, generator=g, device=dev).to(BF)
    n, ctx, at = 150, 200, 141
    k, v, q = r(1, H, ctx, D), r(1, H, ctx, D), r(1, H * G, Tq, D)

    def out(fill, *rows, which="kv"):
        kk, vv = k.clone(), v.clone()
        for t in rows:
            if "k" in which:
                kk[:, :, t] = fill
            if "v" in which:
                vv[:, :, t] = fill
        c = ops.KV8Cache(1, H, ctx, D, device=dev)
        c.append(kk, vv, 0)
        return ops.sdpa_kv8(q, c, n, causal_from=0).view(Tq, -1)

    print("masked", H, G, D, Tq, ops.sdpa_kv8_tiling(1, H, G, Tq, ctx, D), flush=True)
    clean = out(0, *range(n, ctx))
    assert bool(clean.isfinite().all())
    for fill in (float("nan"), float("inf")):
        assert torch.equal(out(fill, *range(n, ctx)), clean)
    sees = torch.arange(Tq, device=dev) + n - Tq >= at
    assert bool(sees.any()) and not bool(sees.all())
    zero = out(0, at, *range(n, ctx))
    for which in ("k", "v", "kv"):
        y, z = out(float("nan"), at, *range(n, ctx), which=which), out(0, at, *range(n, ctx), which=which)
        assert bool(y[sees].isnan().all()) and torch.equal(y[~sees], z[~sees]), which
    assert torch.equal(zero[~sees], z[~sees])
