"""Host side of the MXFP4 and 8-bit cache operators, without a GPU: refusals of the C ABI before any launch and of the
Python entry points before any device work, buffer sizes, and the oracle on values worked out by hand."""
import math

import pytest
import torch

import lowbit_cases as lc
import oracle.lowbit as ol
import strix_halo_maxx_amd.ops as ops
from strix_halo_maxx_amd import _lib

A16 = 0x10000  # fake device addresses: validation never dereferences them
BF = torch.bfloat16


def test_oracle_mxfp4_by_hand():
    x = torch.zeros(1, 33)
    x[0, :8] = torch.tensor([7.0, 5.0, 2.5, 3.5, 1.25, 0.25, 0.75, -0.26])  # unit 1: saturates; ties to even
    x[0, 32] = 3.0                                                         # a block of one: unit 0.5, code 6
    assert ol.mxfp4(x)[0, [0, 1, 2, 3, 4, 5, 6, 7, 32]].tolist() == [6, 4, 2, 4, 1, 0, 1, -0.5, 3]
    assert ol.mxfp4(torch.tensor([[math.inf, 1.0]])).isnan().all()


def test_oracle_kv8_by_hand():
    c = ol.KV8(1, 1, 70, 2)
    c.append(0, torch.tensor([[[448.0, 17.0]]]), 0)       # exponent 0, 17 lies halfway between 16 and 18
    assert c.val[0, 0, 0].tolist() == [448, 16] and c.exp[0, 0, 0] == 0
    c.append(0, torch.tensor([[[449.0, 1.0]]]), 1)        # exponent 1
    assert c.val[0, 0, :2].tolist() == [[448, 16], [448, 1]] and c.exp[0, 0].tolist() == [1, -127]
    c.append(0, torch.tensor([[[2.0 ** -140, 0.0]]]), 64)
    assert c.exp[0, 0, 1] == -127


def test_mxfp4_buffer_sizes():
    lib = _lib.load()
    assert lib.mx_mxfp4_code_bytes(1, 1) == 4096 and lib.mx_mxfp4_scale_bytes(1, 1) == 256
    assert lib.mx_mxfp4_code_bytes(65, 129) == 4 * 4096 and lib.mx_mxfp4_scale_bytes(64, 513) == 5 * 256
    assert lib.mx_mxfp4_code_bytes(0, 5) == 0 and lib.mx_mxfp4_scale_bytes(5, -1) == 0
    assert lib.mx_mxfp4_code_bytes(2 ** 31 - 64, 2 ** 20) == (2 ** 31 - 64) * 2 ** 19


def test_mxfp4_refusals():
    lib = _lib.load()
    qz = lambda **kw: lib.mx_quant_mxfp4(*{**dict(st=None, x=A16, ldx=64, c=A16, s=A16, M=4, K=64), **kw}.values())
    assert qz(x=None) == -6 and qz(c=None) == -6 and qz(s=None) == -6
    assert qz(M=0) == -2 and qz(K=0) == -2 and qz(ldx=-1) == -2 and qz(M=2 ** 31 - 1, K=10 ** 6) == -2
    assert qz(x=A16 + 1) == -4 and qz(c=A16 + 8) == -4 and qz(s=A16 + 2) == -4
    vl = lambda **kw: lib.mx_mxfp4_values(*{**dict(st=None, c=A16, s=A16, y=A16, ldy=64, M=4, K=64), **kw}.values())
    assert vl(y=None) == -6 and vl(ldy=63) == -2 and vl(y=A16 + 1) == -4
    tail = dict(wc=A16, ws=A16, b=A16, R=None, ldr=0, rr=0, C=A16, ldc=64, M=4, N=64, K=64, act=0, af=0)
    gv = lambda **kw: lib.mx_gemv_mxfp4(*{**dict(st=None, x=A16, ldx=64), **tail, **kw}.values())
    gm = lambda **kw: lib.mx_gemm_mxfp4(*{**dict(st=None, xc=A16, xs=A16), **tail, **kw}.values())
    rows = lib.mx_gemv_mxfp4_rows()
    assert rows >= 1 and gv(M=rows + 1) == -2 and gv(x=None) == -6 and gv(x=A16 + 1) == -4 and gv(ldx=-8) == -2
    assert gm(xc=None) == -6 and gm(xs=None) == -6 and gm(xc=A16 + 4) == -4 and gm(xs=A16 + 1) == -4
    for f in (gv, gm):
        assert f(wc=None) == -6 and f(ws=None) == -6 and f(C=None) == -6
        assert f(act=3) == -1 and f(act=-1) == -1
        assert f(M=0) == -2 and f(N=0) == -2 and f(K=0) == -2 and f(af=-1) == -2 and f(rr=-1) == -2 and f(ldc=63) == -2
        assert f(R=A16, ldr=-1) == -2
        assert f(wc=A16 + 8) == -4 and f(ws=A16 + 2) == -4 and f(b=A16 + 2) == -4 and f(C=A16 + 1) == -4


def test_kv8_refusals():
    lib = _lib.load()
    ap = lambda **kw: lib.mx_kv8_append(*{**dict(
        st=None, k=A16, kb=64, kh=64, kt=64, v=A16, vb=64, vh=64, vt=64, kc=A16, vc=A16, ks=A16, vs=A16, B=2, H=4, n=5, D=64,
        ctx=100, slots=2, bcast=0, pos=None, pos_s=0, base=3, count=None, count_s=0, cs=None, ncs=0, q=None, qb=0, qh=0,
        qt=0, Hq=0, qo=None), **kw}.values())
    for name in ("k", "v", "kc", "vc", "ks", "vs"):
        assert ap(**{name: None}) == -6
    assert ap(D=72) == -1 and ap(D=128, cs=A16, ncs=100) == -1 and ap(cs=A16, ncs=0) == -1
    assert ap(B=3) == -2 and ap(bcast=1) == -2 and ap(n=0) == -2 and ap(H=0) == -2 and ap(H=70000) == -2
    assert ap(base=96) == -2 and ap(base=-1) == -2 and ap(ctx=0) == -2 and ap(ctx=2 ** 31 - 1) == -2
    assert ap(q=A16) == -6 and ap(q=A16, cs=A16, ncs=100, qo=None, Hq=4) == -6 and ap(q=A16, cs=A16, ncs=100, qo=A16) == -6
    assert ap(k=A16 + 1) == -4 and ap(kc=A16 + 8) == -4 and ap(pos=A16 + 2) == -4 and ap(count=A16 + 1) == -4
    rd = lambda **kw: lib.mx_kv8_read(*{**dict(st=None, kc=A16, vc=A16, ks=A16, vs=A16, k=A16, v=A16, slots=1, H=1, n=10,
                                               D=64, ctx=10), **kw}.values())
    assert rd(k=None) == -6 and rd(D=96) == -1 and rd(n=11) == -2 and rd(n=0) == -2 and rd(v=A16 + 8) == -4
    sd = lambda **kw: lib.mx_kv8_sdpa(*{**dict(
        st=None, q=A16, qb=64, qh=64, qt=64, kc=A16, vc=A16, ks=A16, vs=A16, o=A16, ob=64, ot=64, B=1, H=1, G=1, Tq=1, D=64,
        ctx=100, len=None, len_s=0, base=50, qpos=0, qend=1, cf=0, scale=0.125, part=None, pe=0), **kw}.values())
    for name in ("q", "kc", "vc", "ks", "vs", "o"):
        assert sd(**{name: None}) == -6
    assert sd(D=72) == -1
    assert sd(B=0) == -2 and sd(G=0) == -2 and sd(Tq=0) == -2 and sd(ctx=0) == -2 and sd(cf=-1) == -2
    assert sd(Tq=2 ** 30, G=4) == -2 and sd(scale=0.0) == -2 and sd(scale=float("nan")) == -2 and sd(scale=math.inf) == -2
    assert sd(qt=4) == -2 and sd(ot=2) == -2 and sd(q=A16 + 8) == -4 and sd(o=A16 + 4) == -4 and sd(len=A16 + 2) == -4
    need = lib.mx_kv8_sdpa_ws(1, 1, 1, 1, 10 ** 6, 64)
    assert need > 0 and lib.mx_kv8_sdpa_ws(1, 1, 1, 1, 64, 64) == 0 and lib.mx_kv8_sdpa_ws(0, 1, 1, 1, 64, 64) == 0
    assert sd(ctx=10 ** 6) == -3 and sd(ctx=10 ** 6, part=A16, pe=need - 1) == -3 and sd(ctx=10 ** 6, part=A16 + 4, pe=need) == -3


def raises(match, f, *a, **kw):
    with pytest.raises(ValueError, match=match):
        f(*a, **kw)


def test_python_refusals():
    x = torch.zeros(3, 64, dtype=BF)
    raises("bfloat16", ops.quant_mxfp4, x.float())
    raises("GPU", ops.quant_mxfp4, x)
    raises("column", ops.quant_mxfp4, torch.zeros(3, 0, dtype=BF))
    raises("bf16", ops.MxFp4Lin, x, None, torch.float16)
    w = ops.MxFp4(torch.zeros(4352, dtype=torch.uint8), 10, 64)
    lin = ops.MxFp4Lin.from_quantized(w, None)
    raises("bias", ops.MxFp4Lin.from_quantized, w, torch.zeros(11))
    raises("width 32", lin, x[:, :32])
    raises("gated", lin, x, act="glu")
    raises("act_from", lin, x, act_from=-1)
    raises("float32", lin, x.float())
    raises("out must", lin, x, out=torch.zeros(3, 9, dtype=BF))
    raises("residual width", lin, x, res=torch.zeros(3, 9, dtype=BF))
    raises("residual rows", lin, x, res=torch.zeros(2, 10, dtype=BF))
    raises("different rows", lin, x, pre=ops.MxFp4(w.data, 4, 64))
    raises("width 32", lin, None, pre=ops.MxFp4(w.data, 4, 32))
    raises("GPU", lin, x)
    raises("out must", w.values, out=torch.zeros(10, 65, dtype=BF))
    for a in ((0, 1, 8, 64), (1, 1, 0, 64), (1, 1, 8, 72)):
        raises("must be positive", ops.KV8Cache, *a, device="cpu")
    z = lambda *s: torch.zeros(*s, dtype=torch.uint8)
    assert ops.KV8Cache.over(z(2, 2, 2, 4096), z(2, 2, 2, 4096), z(2, 2, 2), z(2, 2, 2), 100).hd == 64
    raises("do not hold", ops.KV8Cache.over, z(2, 2, 2, 4096), z(2, 2, 2, 4096), z(2, 2, 2), z(2, 2, 2), 129)
    raises("do not hold", ops.KV8Cache.over, z(2, 2, 2, 4608), z(2, 2, 2, 4608), z(2, 2, 2), z(2, 2, 2), 100)
    raises("storage", ops.KV8Cache.over, z(2, 2, 2, 4096), z(2, 2, 2, 4096), z(2, 2, 3), z(2, 2, 2), 100)
    c = ops.KV8Cache(2, 2, 100, 64, device="cpu")
    k = torch.zeros(2, 2, 5, 64, dtype=BF)
    i = lambda *v: torch.tensor(v, dtype=torch.int32)
    raises("k, v must", c.append, k, k[:, :, :4])
    raises("k, v must", c.append, k[:, :1], k[:, :1])
    raises("sequences", c.append, k, k, bcast=True)
    raises("sequences", c.append, k.repeat(2, 1, 1, 1), k.repeat(2, 1, 1, 1))
    raises("outside", c.append, k, k, 96)
    raises("outside", c.append, k, k, -1)
    raises("2 values", c.append, k, k, i(1))
    raises("int32", c.append, k, k, i(1, 2).long())
    raises("count", c.append, k, k, count=3)
    raises("q goes", c.append, k, k, q=k)
    raises("rotary table", c.append, k, k, 3, cs=torch.zeros(7, 16, 2))
    raises("cs must", c.append, k, k, 3, cs=torch.zeros(70, 32, 2))
    raises("q must", c.append, k, k, cs=torch.zeros(100, 16, 2), q=k[:, :, :3])
    raises("float32", c.append, k.float(), k.float())
    raises("GPU", c.append, k, k)
    raises("outside", c.read, 101)
    q = torch.zeros(2, 4, 3, 64, dtype=BF)
    raises("does not fit", ops.sdpa_kv8, q[:, :3], c, 5)
    raises("does not fit", ops.sdpa_kv8, q.repeat(2, 1, 1, 1), c, 5)
    raises("does not fit", ops.sdpa_kv8, q[..., :32], c, 5)
    raises("bfloat16", ops.sdpa_kv8, q.half(), c, 5)
    raises("outside", ops.sdpa_kv8, q, c, 101)
    raises("2 values", ops.sdpa_kv8, q, c, i(1, 2, 3))
    raises("positive and finite", ops.sdpa_kv8, q, c, 5, scale=0.0)
    raises("causal_from", ops.sdpa_kv8, q, c, 5, causal_from=-1)
    raises("out must", ops.sdpa_kv8, q, c, 5, out=torch.zeros(2, 3, 255, dtype=BF))
    raises("GPU", ops.sdpa_kv8, q, c, 5)
    assert c.append(k[:, :, :0], k[:, :, :0], 100) is None and ops.sdpa_kv8(q[:, :, :0], c, 5).shape == (2, 0, 256)


def test_buffers_that_do_not_hold_the_matrix():
    z = lambda n, dt=torch.uint8: torch.zeros(n, dtype=dt)
    assert ops.MxFp4(z(4352), 64, 128).K == 128
    raises("takes 4352", ops.MxFp4, z(4351), 10, 64)
    raises("takes 8704", ops.MxFp4, z(4352), 65, 64)
    raises("takes 8704", ops.MxFp4, z(4352), 3, 129)
    raises("takes 4352", ops.MxFp4, z(4352, torch.int8), 10, 64)
    raises("takes 4352", ops.MxFp4, z(8704)[::2], 10, 64)
    raises("in MXFP4", ops.MxFp4, z(4352), 10, 0)
    raises("in MXFP4", ops.MxFp4, z(4352), -1, 64)
    raises("aligned", ops.MxFp4, z(4400)[3:], 10, 64)
    raises("weight must", ops.MxFp4Lin, torch.zeros(64, dtype=BF), None)
    raises("weight must", ops.MxFp4Lin, torch.zeros(2, 3, 64, dtype=BF), None)


def test_values_past_32_bits():
    c = ops.KV8Cache(1, 1, 100, 64, device="cpu")
    k, p = torch.zeros(1, 1, 5, 64, dtype=BF), torch.zeros(1, dtype=torch.int32)
    raises("32 bits", c.append, k, k, p, base=2 ** 32)
    raises("32 bits", c.append, k, k, 2 ** 31)
    raises("32 bits", ops.sdpa_kv8, k, c, p, base=-2 ** 31 - 1)
    lib = _lib.load()
    tail = dict(wc=A16, ws=A16, b=None, R=None, ldr=0, rr=0, C=A16, ldc=2 ** 28, M=4, N=2 ** 27 + 1, K=64, act=0, af=0)
    assert lib.mx_gemv_mxfp4(*{**dict(st=None, x=A16, ldx=64), **tail}.values()) == -2  # 2^32 threads in a grid
    assert lib.mx_gemm_mxfp4(*{**dict(st=None, xc=A16, xs=A16), **tail}.values()) == -2


def test_widths_that_the_linear_takes():
    lin = ops.MxFp4Lin.from_quantized(ops.MxFp4(torch.zeros(5 * 4352, dtype=torch.uint8), 10, 588), None)
    assert lin.Kp == 592
    x = torch.zeros(3, 600, dtype=BF)
    raises("GPU", lin, x[:, :588])
    raises("GPU", lin, x[:, :592])
    raises("width 600", lin, x)
    raises("width 590", lin, x[:, :590])


def test_layernorm_linear_refusals():
    lib = _lib.load()
    f = lambda **kw: lib.mx_ln_gemv_mxfp4(*{**dict(st=None, x=A16, g=A16, be=A16, eps=1e-5, wc=A16, ws=A16, b=None, C=A16, N=64,
                                                   K=64, act=0, af=0), **kw}.values())
    for name in ("x", "g", "be", "wc", "ws", "C"):
        assert f(**{name: None}) == -6
    assert f(K=60) == -2 and f(K=lib.mx_ln_gemv_mxfp4_cols() + 8) == -2 and f(K=0) == -2 and f(N=0) == -2 and f(act=3) == -1
    assert f(x=A16 + 1) == -4 and f(g=A16 + 1) == -4 and f(af=-1) == -2 and f(N=2 ** 27 + 1) == -2
    lin = ops.MxFp4Lin.from_quantized(ops.MxFp4(torch.zeros(4352, dtype=torch.uint8), 10, 64), None)
    x, v = torch.zeros(1, 64, dtype=BF), torch.ones(64, dtype=BF)
    raises("GPU", lin.ln, x, (v, v))
    raises("GPU", lin.ln, x.expand(3, -1), (v, v))
    raises("contiguous", lin.ln, x[:, :32], (v, v))
    raises("contiguous", lin.ln, x, (v[:32], v))
    raises("contiguous", lin.ln, x, (v, torch.ones(128, dtype=BF)[::2]))
    raises("float32", lin.ln, x, (v.float(), v))
    raises("gated", lin.ln, x, (v, v), act="glu")
    raises("out must", lin.ln, x, (v, v), out=torch.zeros(1, 9, dtype=BF))


def test_scale_whose_product_overflows():
    """scale log2(e) is what the kernel multiplies by: infinite, it would make 0 times it NaN."""
    lib = _lib.load()
    sd = lambda scale: lib.mx_kv8_sdpa(None, A16, 64, 64, 64, A16, A16, A16, A16, A16, 64, 64, 1, 1, 1, 1, 64, 100, None, 0, 50, 0,
                                       1, 0, scale, None, 0)
    assert sd(3e38) == -2 and sd(math.inf) == -2
    raises("at most 2", ops.sdpa_kv8, torch.zeros(1, 1, 1, 64, dtype=BF), ops.KV8Cache(1, 1, 9, 64, device="cpu"), 5, scale=3e38)


def test_strides_of_size_one_are_not_looked_at():
    c = ops.KV8Cache(1, 1, 100, 64, device="cpu")
    q = torch.zeros(1, 2, 1, 64, dtype=BF)
    raises("GPU", ops.sdpa_kv8, q, c, 5, out=torch.zeros(400, dtype=BF).as_strided((1, 1, 128), (131, 129, 1)))
    raises("out must", ops.sdpa_kv8, torch.zeros(1, 2, 2, 64, dtype=BF), c, 5,
           out=torch.zeros(400, dtype=BF).as_strided((1, 2, 128), (1, 129, 1)))
    w = ops.MxFp4(torch.zeros(4352, dtype=torch.uint8), 10, 1)
    raises("GPU", w.values, out=torch.zeros(1, 10, dtype=BF).t())


def test_every_mxfp4_kernel_has_its_cases():
    """The kernels that mx_gemm_mxfp4 takes over a sweep of shapes, tiles with and without 16-byte stores, against those that the
    GPU tests check values of; and the forms of the launch that quantises its rows."""
    sizes = sorted({s * m // 8 for s in (16, 64, 256, 1024, 4096, 16384) for m in range(4, 17)})
    swept = {ops.mxfp4_tiling(m, n, k) for m in sizes for n in sizes for k in (64, 256, 257, 512, 513, 2048, 2049, 8192)}
    assert len(swept) == 11
    assert {ops.mxfp4_tiling(*s) for s in lc.ROWS} == {t for t in swept if not t[2]}
    got = {(ops.mxfp4_tiling(*s), s[1] % 8 == 0) for s in lc.TILES}
    assert got == {(t, v) for t in swept if t[2] for v in (True, False)}
    form = lambda m, k: (8 if k % 8 or m > 4 else 1 if m == 1 else 4, k % 8 == 0, k > 2048)
    assert {form(m, k) for m, n, k in lc.FEW} == {form(m, k) for m in range(1, 9) for k in (8, 9, 2048, 2049, 2056)}
    assert all(m <= _lib.load().mx_gemv_mxfp4_rows() for m, n, k in lc.FEW)
    assert ops.mxfp4_tiling(0, 5, 5) == ops.mxfp4_tiling(5, -1, 5) == (0, 0, 0, 0)


def attention_kernel(B, H, G, Tq, ctx, D):
    rows, waves, runs, chunk = ops.sdpa_kv8_tiling(B, H, G, Tq, ctx, D)
    return D, rows, waves, runs > 1


def test_every_attention_kernel_has_its_cases():
    """The same for sdpa_kv8: each kernel with and without a join, each that reloads scales, each over masked NaN."""
    swept = {attention_kernel(B, H, 1, Tq, ctx, D) for B in (1, 4, 32) for H in (1, 3, 8, 32, 64, 100, 200, 600)
             for Tq in (1, 16, 17, 33, 60, 70, 129, 300, 1000, 4000) for ctx in (1, 500, 1600, 4000, 16000, 17000, 200000)
             for D in (64, 128)}
    assert len(swept) == 22
    full = lambda c: (len(c[0]), c[1], c[2], c[4], c[6] or max(c[0]), c[3])
    assert {attention_kernel(*full(c)) for c in lc.ATTENTION} == swept
    long_runs = {attention_kernel(*full(c))[:3] for c in lc.ATTENTION if ops.sdpa_kv8_tiling(*full(c))[3] > 64}
    assert long_runs >= {k[:3] for k in swept if k[1] > 16}
    assert {attention_kernel(1, H, G, Tq, 200, D)[:3] for H, G, D, Tq in lc.MASKED} == {k[:3] for k in swept}
    assert ops.sdpa_kv8_tiling(0, 1, 1, 1, 64, 64) == ops.sdpa_kv8_tiling(1, 1, 1, 1, 64, 72) == (0, 0, 0, 0)


def test_norm_bound_tells_lost_bits():
    """The bound in norm that the attention's GPU tests use, on the formula with its roundings planted: two e4m3 terms per weight
    pass with room; a weight or a query without its low term does not."""
    g = torch.Generator().manual_seed(0)
    n, D, T = 1000, 64, 24
    q, k, v = (torch.randn(s, D, generator=g).to(BF).double() for s in (T, n, n))
    v = 3 * v
    e4m3 = lambda x: ol.nearest(x, ol.E4M3)

    def terms(x, low):  # relative to a power of two just above the row's largest, as e4m3 terms of up to 256
        unit = torch.exp2(torch.ceil(torch.log2(x.abs().amax(-1, keepdim=True)))) / 256
        hi = e4m3(x / unit)
        return unit * (hi + (e4m3((x / unit - hi) * 16) / 16 if low else 0))

    def attend(q, p_terms):
        w = torch.exp(q @ k.t() * D ** -0.5 - 8)
        return (p_terms(w) @ v) / w.sum(-1, keepdim=True), w / w.sum(-1, keepdim=True)

    ref, p = attend(q, lambda w: w)
    size = (q.abs() @ k.t().abs()).amax(-1, keepdim=True) * D ** -0.5
    spread = ((p * p) @ (v * v)).sqrt()
    bound = (2.0 ** -8 + 2.0 ** -14) * ref.norm() + 2 * ((2.0 ** -9 + 2.0 ** -15 * (1 + size)) * spread).norm()
    off = lambda y: float((y.to(BF).double() - ref).norm() / bound)
    assert torch.equal(terms(q, True), q)  # two terms hold a bf16
    assert off(attend(q, lambda w: terms(w, True))[0]) < 0.5
    assert off(attend(q, lambda w: terms(w, False))[0]) > 2
    assert off(attend(terms(q, False), lambda w: terms(w, True))[0]) > 2


def test_counts_that_wrap():
    """Sequences times heads past any grid: refused before the products of such counts wrap (to a division by zero, or to a few
    workgroups over memory that nobody has)."""
    lib, big = _lib.load(), 2 ** 30
    assert lib.mx_kv8_sdpa_ws(big, big, 1, 2048, 64, 64) == 0 and ops.sdpa_kv8_tiling(big, big, 1, 2048, 64, 64) == (0, 0, 0, 0)
    assert lib.mx_kv8_sdpa_ws(1, 1, 2 ** 16, 2 ** 16, 64, 64) == 0
    sd = lambda B, H, Tq: lib.mx_kv8_sdpa(None, A16, 64, 64, 64, A16, A16, A16, A16, A16, 64, 64, B, H, 1, Tq, 64, 64, None, 0, 50, 0,
                                          1, 0, 0.125, None, 0)
    assert sd(big, big, 2048) == -2 and sd(2 ** 23, 1, 1) == -2
    assert lib.mx_kv8_read(None, A16, A16, A16, A16, A16, A16, 2 ** 31 - 1, 2 ** 31 - 1, 256, 64, 256) == -2
    assert lib.mx_kv8_read(None, A16, A16, A16, A16, A16, A16, big, big, 1024, 64, 1024) == -2


def test_what_lies_apart():
    """_apart against the addresses themselves: blocks, columns of one buffer, heads of a fused projection, expanded rows."""
    buf = torch.zeros(4000, dtype=BF)
    views = [buf.as_strided(*v) for v in (
        ((3, 20), (50, 1), 0), ((3, 20), (50, 1), 20), ((3, 20), (50, 1), 30), ((3, 20), (50, 1), 31), ((3, 20), (50, 1), 45),
        ((3, 20), (60, 1), 20), ((1, 20), (50, 1), 70), ((1, 20), (50, 1), 60), ((3, 20), (0, 1), 20), ((3, 50), (50, 1), 150),
        ((3, 50), (50, 1), 149), ((2, 2, 3, 10), (150, 10, 50, 1), 0), ((2, 3, 20), (150, 50, 1), 20), ((2, 3, 20), (150, 50, 1), 19),
        ((2, 2, 3, 10), (150, 20, 50, 1), 5), ((2, 3, 20), (1000, 50, 1), 36), ((20,), (1,), 25))]
    cells = [set((torch.arange(4000).as_strided(v.shape, v.stride(), v.storage_offset())).flatten().tolist()) for v in views]
    sure = 0
    for a, x in zip(views, cells):
        for b, y in zip(views, cells):
            if ops._apart(a, b):
                assert not x & y, (a.shape, a.stride(), a.storage_offset(), b.shape, b.stride(), b.storage_offset())
                sure += 1
    assert ops._apart(views[0], views[1]) and ops._apart(views[0], views[2]) and not ops._apart(views[0], views[3])
    assert ops._apart(views[11], views[12]) and not ops._apart(views[11], views[13]) and ops._apart(views[0], views[9])
    assert sure >= 40
