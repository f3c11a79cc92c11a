"""MXFP4 quantisation and Linear on the MI355X against the 64-bit oracle: the quantised values bit for bit (every step but
the rounding of the code is exact), the Linear within its one bf16 rounding plus that of an fp32 sum."""
import pytest
import torch

import lowbit_cases as lc
import oracle.lowbit as ol
import strix_halo_maxx_amd.ops as ops

pytestmark = pytest.mark.gpu
BF, F64 = torch.bfloat16, torch.float64


def gen(seed):
    return torch.Generator().manual_seed(seed)


def same(a, b):
    """Equal values, NaN where NaN."""
    a, b = a.to(F64), b.to(F64)
    return bool(((a == b) | (a.isnan() & b.isnan())).all())


@pytest.mark.parametrize("M,K", [(1, 1), (1, 2048), (3, 31), (17, 32), (5, 33), (16, 128), (15, 129), (33, 700), (130, 2055)])
def test_quantised_values_are_exact(dev, M, K):
    g = gen(M * 10007 + K)
    x = (torch.randn(M, K, generator=g) * torch.exp2(torch.randint(-20, 20, (M, K), generator=g).float())).to(BF)
    q = ops.quant_mxfp4(x.to(dev))
    ok = same(q.values().cpu(), ol.mxfp4(x))
    assert ok


def test_quantised_special_values(dev):
    """Ties, the saturation between 6 and 8 units, zeros, subnormals, the largest bf16, blocks with NaN and infinities."""
    rows = torch.zeros(9, 64)
    rows[0, :12] = torch.tensor([4.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.25, -5.0, -2.5, 4.5])
    rows[1, :6] = torch.tensor([7.96875, 6.5, 5.0, 6.0, -7.0, 0.2])
    rows[3] = torch.randn(64, generator=gen(1)) * 2.0 ** -130
    rows[4, ::2] = 2.0 ** -133
    rows[5, :3] = torch.tensor([3.3895e38, -1e38, 1e37])
    rows[6, 3], rows[6, 40] = float("nan"), 1.0
    rows[7, 3], rows[7, 40] = 1.0, float("-inf")
    rows[8, :2] = torch.tensor([2.0 ** -126, 2.0 ** -125])
    x = rows.to(BF)
    y = ops.quant_mxfp4(x.to(dev)).values().cpu()
    assert same(y, ol.mxfp4(x))
    assert y[0, :12].tolist() == [4.0, 0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, 0.0, -4.0, -2.0, 4.0]
    assert y[6, :32].isnan().all() and not y[6, 32:].isnan().any() and y[7, 32:].isnan().all()


def test_quant_reads_any_rows(dev):
    """Unaligned starts, odd row strides, a transposed input, repeated rows, more than two dimensions, no rows."""
    g = gen(4)
    big = torch.randn(40, 301, generator=g).to(BF)
    d = big.to(dev)
    for a, b in ((big[:, 1:290], d[:, 1:290]), (big[3:20, 8:264], d[3:20, 8:264]), (big.t(), d.t()),
                 (big[:1].expand(20, -1), d[:1].expand(20, -1))):
        assert same(ops.quant_mxfp4(b).values().cpu(), ol.mxfp4(a.reshape(-1, a.shape[-1])))
    q = ops.quant_mxfp4(d.view(4, 10, 301))
    assert (q.rows, q.K) == (40, 301) and same(q.values().cpu(), ol.mxfp4(big))
    assert ops.quant_mxfp4(d[:0]).values().shape == (0, 301)
    out = torch.full((42, 310), 7.0, device=dev, dtype=BF)
    ops.quant_mxfp4(d).values(out=out[1:41, 3:304])
    assert same(out[1:41, 3:304].cpu(), ol.mxfp4(big))
    out[1:41, 3:304] = 7.0
    assert bool((out == 7.0).all())


def close(y, ref, mag, act=None):
    """One rounding to bf16 (2^-8 of the value), the fp32 sum of at most 2^14 exact products (2^-24 of the magnitude for
    each of the sum's steps, 2^-10 steps' worth: 2^-14 with room to spare over any order), the activation's slope (at
    most 1.13) and its own few fp32 roundings, 2^-20 of the value and of 1."""
    err = (y.to(F64) - ref).abs()
    tol = 2.0 ** -8 * ref.abs() + 1.13 * 2.0 ** -14 * mag + (2.0 ** -20 * (1 + ref.abs()) if act else 0)
    assert bool((err <= tol).all()), (err - tol).max().item()


SHAPES = [(1, 1, 1), (1, 8192, 2048), (1, 2048, 8192), (2, 100, 4304), (7, 37, 100), (16, 64, 129), (17, 768, 768),
          (33, 130, 1000), (64, 260, 512), (65, 129, 640), (128, 128, 128), (130, 259, 1152), (300, 1000, 385),
          (520, 516, 2304)]
# more workgroups than fit at once, or more tiles than workgroups (128 x 128), K whole and just past a step, ragged edges; which
# shape takes which kernel: lowbit_cases.py
LARGE = [(2100, 4304, 128), (1800, 5000, 257), (2600, 3333, 384), (1500, 6144, 513), (2049, 4100, 1152)]


@pytest.mark.parametrize("M,N,K", SHAPES)
def test_linear(dev, M, N, K):
    g = gen(M + 3 * N + 7 * K)
    x, w = torch.randn(M, K, generator=g).to(BF), (torch.randn(N, K, generator=g) * 0.05).to(BF)
    b, r = (torch.randn(N, generator=g) * 0.1).to(BF), torch.randn(M, N, generator=g).to(BF)
    lin, plain = ops.MxFp4Lin(w, b, device=dev), ops.MxFp4Lin(w, None, device=dev)
    xd, rd = x.to(dev), r.to(dev)
    print(f"mxfp4 linear {M} x {N} x {K}", flush=True)
    close(plain(xd).cpu(), *ol.mxfp4_linear(x, w))
    for act in ("tanh", "erf"):
        close(lin(xd, act=act).cpu(), *ol.mxfp4_linear(x, w, b, act), act=act)
    close(lin(xd, res=rd).cpu(), *ol.mxfp4_linear(x, w, b, res=r))
    f = N // 2 + 1
    close(lin(xd, gelu=True, res=rd, act_from=f).cpu(), *ol.mxfp4_linear(x, w, b, "tanh", r, f), act="tanh")
    # quantised beforehand: the same codes, another order of the sum at most
    close(lin(None, pre=lin.quant(xd)).cpu(), *ol.mxfp4_linear(x, w, b))


@pytest.mark.parametrize("M,N,K", LARGE)
def test_linear_many_tiles(dev, M, N, K):
    """Against the fp32 product of the quantised values (exact products; its sum's error is covered like the kernel's)."""
    g = torch.Generator(device=dev).manual_seed(M)
    x, w = torch.randn(M, K, generator=g, device=dev).to(BF), torch.randn(N, K, generator=g, device=dev).to(BF)
    b, r = torch.randn(N, generator=g, device=dev).to(BF), torch.randn(M, N, generator=g, device=dev).to(BF)
    lin = ops.MxFp4Lin(w, b, device=dev)
    xq, wq = lin.quant(x).values().float(), lin.wq.values().float()
    y = torch.matmul(xq, wq.t().contiguous()) + b.float()
    mag = torch.matmul(xq.abs(), wq.t().abs().contiguous()) + b.float().abs()
    close(lin(x), y.double(), mag.double())
    close(lin(x, res=r, act="tanh"), ol.gelu(y.double(), "tanh") + r.double(), mag.double(), act="tanh")


def test_linear_views_and_leading_dims(dev):
    """Leading dimensions, rows at odd strides and addresses, residual rows that repeat, an output inside a larger buffer
    whose rest stays."""
    g = gen(9)
    w, b = (torch.randn(100, 96, generator=g) * 0.1).to(BF), torch.randn(100, generator=g).to(BF)
    lin = ops.MxFp4Lin(w, b, device=dev)
    for M in (6, 150):
        x = torch.randn(M, 131, generator=g).to(BF)
        xd = x.to(dev)[:, 5:101]
        xs = x[:, 5:101]
        ref, mag = ol.mxfp4_linear(xs, w, b)
        close(lin(xd).cpu(), ref, mag)
        assert lin(xd.reshape(2, M // 2, 96)).shape == (2, M // 2, 100)
        r = torch.randn(3, 100, generator=g).to(BF)
        close(lin(xd, res=r.to(dev)).cpu(), ref + r.to(F64).repeat(M // 3, 1), mag)
        for c0 in (4, 7):
            out = torch.full((M + 2, 120), 3.0, device=dev, dtype=BF)
            assert lin(xd, out=out[1:-1, c0:c0 + 100]) is not None
            close(out[1:-1, c0:c0 + 100].cpu(), ref, mag)
            out[1:-1, c0:c0 + 100] = 3.0
            assert bool((out == 3.0).all())
    assert lin(xd[:0]).shape == (0, 100)
    assert lin(xd[:1].expand(20, -1)).shape == (20, 100)


@pytest.mark.parametrize("M", [3, 40, 200])
def test_linear_nan_stays_in_its_row(dev, M):
    g = gen(M)
    x, w = torch.randn(M, 256, generator=g).to(BF), torch.randn(50, 256, generator=g).to(BF)
    x[1, 70], x[2, 200] = float("nan"), float("inf")
    y = ops.MxFp4Lin(w, None, device=dev)(x.to(dev)).cpu()
    bad = y.isnan().any(1)
    assert bad.nonzero().flatten().tolist() == [1, 2] and bool(y[1:3].isnan().all())
    keep = [m for m in range(M) if m not in (1, 2)]
    ref, mag = ol.mxfp4_linear(x[keep], w)
    close(y[keep], ref, mag)


@pytest.mark.parametrize("M", [1, 16, 48, 200])
def test_linear_in_a_graph_and_on_a_side_stream(dev, M):
    g = gen(M)
    w, b = torch.randn(96, 320, generator=g).to(BF), torch.randn(96, generator=g).to(BF)
    lin = ops.MxFp4Lin(w, b, device=dev)
    x = torch.randn(M, 320, generator=g).to(BF).to(dev)
    want = [lin(x * s, act="tanh") for s in (1, 2, 3)]
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        side = lin(x, act="tanh")
    torch.cuda.current_stream().wait_stream(st)
    assert torch.equal(side, want[0])
    buf = x.clone()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        y = lin(buf, act="tanh")
    for s in (1, 2, 3, 1, 2, 3):
        buf.copy_(x * s)
        gr.replay()
        assert torch.equal(y, want[s - 1])
        torch.cuda.synchronize()


@pytest.mark.parametrize("M", [3, 200])
def test_linear_onto_its_own_input_and_residual(dev, M):
    """out may be x (few rows: every workgroup reads all of x, so the product must not write it) or res."""
    g = gen(M + 1)
    w = (torch.randn(512, 512, generator=g) * 0.1).to(BF)
    lin = ops.MxFp4Lin(w, None, device=dev)
    x = torch.randn(M, 512, generator=g).to(BF).to(dev)
    want, add = lin(x), lin(x, res=x)
    buf = x.clone()
    assert lin(buf, out=buf) is buf and torch.equal(buf, want)
    buf = x.clone()
    lin(x, res=buf, out=buf)
    assert torch.equal(buf, add)
    row = torch.zeros(M, 1024, device=dev, dtype=BF)  # x and out side by side in the rows of one buffer
    row[:, :512] = x
    lin(row[:, :512], out=row[:, 512:])
    assert torch.equal(row[:, 512:], want) and torch.equal(row[:, :512], x)


def test_vision_tower_takes_it(dev):
    """The Linear as the tower's lin_cls: the patch embedding (588 columns, read from rows padded to 592, its residual the
    positions) against the formula, and a block."""
    import strix_halo_maxx_amd.md2 as md2
    import strix_halo_maxx_amd.synth as S
    w = S.vision_weights(0, layers=1)
    vt = md2.VisionTower(w, lin_cls=ops.MxFp4Lin)
    img = S.images_u8(3, 2).to(dev)
    a = ops.patchify(img, vt.P, mode=0, ldo=592)
    emb = vt.embed(img)
    ref, mag = ol.mxfp4_linear(a[:, :588].cpu(), w["patch_emb.weight"].to(BF), w["patch_emb.bias"].to(BF))
    close(emb.cpu(), ref + w["pos_emb"].to(BF).view(-1, ref.shape[1]).to(F64).repeat(2, 1), mag)
    y = vt(img)
    assert y.shape == (2, 729, 1152) and bool(y.isfinite().all())


def test_offsets_past_32_bits(dev):
    """Inputs, codes and outputs beyond 4 GB: the last rows are those of a short call."""
    M, K = 300_017, 8192
    x = torch.zeros(M, K, device=dev, dtype=BF)
    x[-70:] = torch.randn(70, K, generator=gen(5)).to(BF).to(dev)
    q = ops.quant_mxfp4(x)
    y = q.values(out=x)  # 4.9 GB
    tail = ops.quant_mxfp4(y[-70:].contiguous()).values()
    assert torch.equal(y[-70:], tail) and not bool(y[:1000].any())
    del q, y, x
    w = (torch.randn(8192, 640, generator=gen(6)) * 0.1).to(BF)
    lin = ops.MxFp4Lin(w, None, device=dev)
    x = torch.zeros(M, 640, device=dev, dtype=BF)
    x[-70:] = torch.randn(70, 640, generator=gen(7)).to(BF).to(dev)
    ref, mag = ol.mxfp4_linear(x[-70:].cpu(), w)
    y = lin(x)
    close(y[-70:].cpu(), ref, mag)
    assert not bool(y[:1000].any()) and not bool(y[150_000:151_000].any())


@pytest.mark.parametrize("K", [8, 520, 1152, 2040, 2048, 2056])
def test_linear_of_a_layernorm(dev, K):
    """LayerNorm and Linear in one launch (one row, K up to 2048; beyond, two calls) give the bits of the two operators: rows
    with a large mean, a constant row, a NaN, an infinity, a row of zeros; outputs in place and inside a buffer."""
    g = gen(K)
    N = 300
    lin = ops.MxFp4Lin((torch.randn(N, K, generator=g) * 0.1).to(BF), torch.randn(N, generator=g), device=dev)
    ln = [(torch.randn(K, generator=g) * s + m).to(BF).to(dev) for s, m in ((0.2, 1.0), (0.1, 0.0))]
    x = torch.randn(7, K, generator=g)
    x[1] += 100.0
    x[2], x[3] = 3.25, 0.0
    x[4, K // 2], x[5, K - 1] = float("nan"), float("inf")
    x = x.to(BF).to(dev)
    for r in range(7):
        for eps, kw in ((1e-5, {}), (1e-3, dict(act="tanh", act_from=133)), (1e-5, dict(act="erf"))):
            got, want = lin.ln(x[r:r + 1], ln, eps=eps, **kw), lin(ops.layernorm(x[r:r + 1], *ln, eps=eps), **kw)
            assert same(got.cpu(), want.cpu()), (r, kw)
    want = lin(ops.layernorm(x, *ln))
    assert same(lin.ln(x, ln).cpu(), want.cpu())
    assert lin.ln(x[0], ln).shape == (N,) and torch.equal(lin.ln(x[0], ln), want[0])
    buf = torch.full((3, N + 9), 5.0, device=dev, dtype=BF)
    lin.ln(x[:1], ln, out=buf[1:2, 3:N + 3])
    assert torch.equal(buf[1, 3:N + 3], want[0])
    buf[1, 3:N + 3] = 5.0
    assert bool((buf == 5.0).all())
    row, gr = x[:1].clone(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        y = lin.ln(row, ln)
    for r in (0, 1, 6, 0):
        row.copy_(x[r:r + 1])
        gr.replay()
        assert torch.equal(y[0], want[r])
        torch.cuda.synchronize()


def test_linear_of_a_layernorm_onto_its_input(dev):
    g = gen(77)
    lin = ops.MxFp4Lin((torch.randn(512, 512, generator=g) * 0.1).to(BF), None, device=dev)
    ln = [torch.randn(512, generator=g).to(BF).to(dev) for _ in range(2)]
    x = torch.randn(1, 512, generator=g).to(BF).to(dev)
    want = lin.ln(x, ln)
    lin.ln(x, ln, out=x)
    assert torch.equal(x, want)


@pytest.mark.parametrize("M,N,K", [(4, 96, 256), (12, 512, 512), (60, 1000, 320), (768, 2048, 640)])
def test_residual_that_overlaps_the_output(dev, M, N, K):
    """A residual in the output's memory, other than as the output itself: rows that repeat, rows or columns further on, one row
    for all, another pitch. Each result takes the residual as it was before the call."""
    g = gen(M + N + K)
    lin = ops.MxFp4Lin((torch.randn(N, K, generator=g) * 0.1).to(BF), torch.randn(N, generator=g), device=dev)
    x = torch.randn(M, K, generator=g).to(BF).to(dev)
    buf0 = torch.randn((M + 3) * (N + 16), generator=g).to(BF).to(dev)
    at = lambda b, rows, ld, off=0, step=1: b.as_strided((rows, N), (ld, step), off)
    ld = N + 16
    views = [(at(buf0, M // 2, ld), 0), (at(buf0, 1, ld), 0), (at(buf0, M, ld, ld), 0), (at(buf0, M, ld, 8), 0), (at(buf0, M, ld), 8),
             (at(buf0, M, 0, 2 * ld), 0), (at(buf0, M, N), 0), (at(buf0, M // 4, ld, ld), 0)]
    for r0, off in views:
        want = lin(x, res=r0.clone())
        for _ in range(3):
            buf = buf0.clone()
            res = buf.as_strided(r0.shape, r0.stride(), r0.storage_offset())
            y = at(buf, M, ld, off)
            assert lin(x, res=res, out=y) is y and torch.equal(y, want), (r0.shape, r0.stride(), r0.storage_offset(), off)
    # as the output itself nothing is copied, and a single row's pitch does not matter
    buf = buf0.clone()
    want = lin(x, res=at(buf0, M, ld).clone())
    lin(x, res=at(buf, M, ld), out=at(buf, M, ld))
    assert torch.equal(at(buf, M, ld), want)


def product(x, w):
    """The product of the quantised values in 64 bits, and that of their sizes (x, w on the GPU)."""
    xq, wt = ops.quant_mxfp4(x).values().double(), ops.quant_mxfp4(w).values().double().t().contiguous()
    return torch.matmul(xq, wt), torch.matmul(xq.abs(), wt.abs())


@pytest.mark.parametrize("M,N,K", lc.ROWS + lc.TILES + lc.FEW)
def test_every_kernel_against_64_bits(dev, M, N, K):
    """Each kernel that the product takes, with what its write-out can do: bias, both activations from the first column or a later
    one, a residual of as many rows, of fewer, and one row for all, an output inside a larger buffer (16-byte aligned, and not)."""
    g = torch.Generator(device=dev).manual_seed(M + 3 * N + 7 * K)
    r = lambda *s: torch.randn(*s, generator=g, device=dev)
    x, w, b, res = r(M, K).to(BF), (r(N, K) * 0.05).to(BF), r(N).to(BF), r(M, N).to(BF)
    x[M // 2] *= 50
    w[N // 3] *= 7
    lin, plain = ops.MxFp4Lin(w, b, device=dev), ops.MxFp4Lin(w, None, device=dev)
    print(f"mxfp4 kernel {M} x {N} x {K}", flush=True)
    y0, mag = product(x, w)
    yb, magb = y0 + b.double(), mag + b.double().abs()
    close(plain(x), y0, mag)
    for act, f in (("tanh", 0), ("erf", N // 2 + 1), ("erf", 0), ("tanh", 8)):
        ref = torch.cat([yb[:, :f], ol.gelu(yb[:, f:], act)], 1)
        close(lin(x, act=act, act_from=f), ref, magb, act=act)
        close(lin(x, act=act, act_from=f, res=res), ref + res.double(), magb, act=act)
    close(lin(x, res=res[:1].expand(M, N)), yb + res[:1].double(), magb)
    if M % 2 == 0:
        close(lin(x, res=res[:M // 2]), yb + res[:M // 2].double().repeat(2, 1), magb)
    buf = torch.full((M + 1, N + 24), 3.0, device=dev, dtype=BF)
    for c0 in (8, 5):
        out = buf[:-1, c0:c0 + N]
        lin(x, res=res, out=out)
        close(out, yb + res.double(), magb)
        out.fill_(3.0)
        assert bool((buf == 3.0).all())
