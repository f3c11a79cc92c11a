"""Host side of the shared-prefix attention, beam selection and slot reordering, without a GPU: refusals of the C ABI before any
launch and of the Python entry points before any device work, workspace sizes, and the oracle on values worked out by hand."""
import math

import pytest
import torch

import oracle.beams as ob
import strix_halo_maxx_amd.ops as ops
from beam_cases import ATTENTION, MASKED
from strix_halo_maxx_amd import _lib

A16 = 0x10000  # fake device addresses: validation never dereferences them
BF = torch.bfloat16
INF = math.inf


def test_oracle_prefix_by_hand():
    q = torch.zeros(1, 1, 2, 1)
    pk, pv = torch.zeros(1, 1, 2, 1), torch.tensor([2.0, 4.0]).view(1, 1, 2, 1)
    k, v = torch.zeros(1, 1, 3, 1), torch.tensor([9.0, 30.0, INF]).view(1, 1, 3, 1)
    see = lambda **kw: ob.sdpa_prefix(q, pk, pv, k, v, scale=1.0, **kw)[0].flatten().tolist()
    assert see(kv_len=[2]) == [5.0, 11.25]             # query 0: 2, 4, 9; query 1: and 30
    assert see(kv_len=[2], prefix_len=[0]) == [9.0, 19.5]
    assert see(kv_len=[1]) == [3.0, 5.0]               # the first query comes before the only own key
    assert see(kv_len=[0], prefix_len=[0]) == [0.0, 0.0]
    assert see(kv_len=[1], causal=False) == [5.0, 5.0] and see(kv_len=[3])[1] == INF


def test_oracle_select_by_hand():
    x = torch.log(torch.tensor([[[1.0, 2, 1], [4, 2, 2]]]))  # shares 1/4 1/2 1/4 and 1/2 1/4 1/4
    s = torch.tensor([[0.0, 0.0]])
    v, p, t, _ = ob.beam_select(x, s, 4)
    assert p.tolist() == [[0, 1, 0, 0]] and t.tolist() == [[1, 0, 0, 2]]
    assert torch.allclose(v.exp(), torch.tensor([[0.5, 0.5, 0.25, 0.25]], dtype=torch.float64))
    v, p, t, d = ob.beam_select(x, torch.tensor([[-INF, -1.5]]), 3, torch.tensor([[False, True]]), 2)
    assert v.tolist() == [[-1.5, -INF, -INF]] and p.tolist() == [[1, 0, 0]] and t.tolist() == [[2, 2, 2]] and bool(d.all())


def test_oracle_reorder_by_hand():
    x = torch.arange(6.0).view(1, 3, 1, 2)  # slots 01 23 45
    r = lambda *a, **kw: ob.reorder_slots(x, torch.tensor(a), **kw).flatten().tolist()
    assert r(1, 2, 0) == [2, 3, 4, 5, 0, 1] and r(0, 0, 7) == [0, 1, 0, 1, 4, 5]
    assert r(1, 2, 0, n=[2, 1, 0]) == [2, 1, 2, 3, 0, 1] and r(1, 1, 1, first=1) == [0, 3, 2, 3, 4, 3]
    assert r(1, 1, 1, n=5, first=5, unit=4) == [0, 3, 2, 3, 4, 3]


def prefix(strides=None, **kw):
    import ctypes
    st = {**{n: 64 for n in ("qb", "qh", "qt", "pkn", "pkh", "pkt", "pvn", "pvh", "pvt", "kb", "kh", "kt", "vb", "vh", "vt")}, **(strides or {})}
    return _lib.load().mx_sdpa_prefix(*{**dict(
        st=None, q=A16, pk=A16, pv=A16, k=A16, v=A16, o=A16, strides=(ctypes.c_long * 15)(*st.values()), ob=64, ot=64, N=1, S=100, H=1,
        G=1, Tq=1, D=64, P=500, T=9, plen=None, ps=0, pbase=500, len=None, ls=0, base=9, causal=1, scale=1.0, part=A16,
        pe=10 ** 9), **kw}.values())


def test_prefix_refusals():
    for n in ("q", "o", "pk", "pv", "k", "v"):
        assert prefix(**{n: None}) == -6
    assert _lib.load().mx_sdpa_prefix(None, A16, A16, A16, A16, A16, A16, None, 64, 64, 1, 1, 1, 1, 1, 64, 1, 1, None, 0, 1, None, 0, 1, 1,
                                      1.0, A16, 10 ** 9) == -6
    assert prefix(D=72) == -1
    for n in ("N", "S", "H", "G", "Tq"):
        assert prefix(**{n: 0}) == -2 and prefix(**{n: 2 ** 31 - 1}) == -2
    assert prefix(P=-1) == -2 and prefix(T=-1) == -2 and prefix(P=2 ** 31 - 1) == -2
    for s in (0.0, -1.0, INF, math.nan, 3e38):
        assert prefix(scale=s) == -2
    for n in ("qb", "qh", "qt", "pkn", "pkh", "pkt", "pvn", "pvh", "pvt", "kb", "kh", "kt", "vb", "vh", "vt"):
        assert prefix({n: 68}) == -2
    for n in ("pkt", "pvt", "kt", "vt"):
        assert prefix({n: -8}) == -2 and prefix({n: 2 ** 23}) == -2
    assert prefix(ob=62) == -2 and prefix(ot=62) == -2
    for n in ("q", "pk", "pv", "k", "v"):
        assert prefix(**{n: A16 + 8}) == -4
    assert prefix(o=A16 + 4) == -4 and prefix(plen=A16 + 2) == -4 and prefix(len=A16 + 1) == -4
    need = _lib.load().mx_sdpa_prefix_ws(1, 100, 1, 1, 1, 5000, 9, 64)
    assert need > 0 and prefix(P=5000, pe=need - 1) == -3 and prefix(P=5000, part=None) == -3 and prefix(P=5000, part=A16 + 8) == -3


def test_prefix_cases_take_every_kernel():
    """The GPU tests' shapes: each kernel of each head dim, with one run of keys and with several where it can have them, and each
    under masks."""
    def kernel(N, S, H, G, D, Tq, P, T):
        kind, q, k, ra, rows, rb = ops.sdpa_prefix_tiling(N, S, H, G, Tq, P, T, D)
        return (D, kind) + ((rows,) if kind == 0 else (q, k))

    def runs(N, S, H, G, D, Tq, P, T):
        t = ops.sdpa_prefix_tiling(N, S, H, G, Tq, P, T, D)
        return max(t[3], t[5]) > 1
    forms = [(0, 16), (0, 32), (1, 2, 4), (1, 4, 1), (2, 1, 4), (2, 2, 4), (2, 4, 1), (2, 4, 2), (2, 8, 1)]
    want = {(D, *f) for D in (64, 128) for f in forms}
    assert {kernel(*c) for c, _, _ in ATTENTION} == want
    assert {kernel(*c) for c in MASKED} == want
    split = {kernel(*c) for c, _, _ in ATTENTION if runs(*c)}
    assert split >= {(D, *f) for D in (64, 128) for f in forms if f not in ((2, 4, 1), (2, 1, 4))}
    whole = {kernel(*c)[1:] for c, _, _ in ATTENTION if not runs(*c)}
    assert whole >= {f for f in forms if f[0] != 1}


def test_prefix_workspace():
    ws = _lib.load().mx_sdpa_prefix_ws
    assert ws(1, 1, 1, 1, 1, 0, 1, 72) == 0 and ws(0, 1, 1, 1, 1, 0, 1, 64) == 0 and ws(1, 1, 1, 1, 1, -1, 1, 64) == 0
    assert ws(1, 1, 1, 1, 1, 64, 64, 64) == 0 and ws(1, 4, 32, 1, 1, 794, 64, 64) == 0  # one run
    assert ws(1, 64, 8, 4, 1, 2 ** 31 - 256, 2 ** 31 - 256, 128) > 0


def select(**kw):
    return _lib.load().mx_beam_select(*{**dict(
        st=None, x=A16, fp32=0, sb=4000, sw=1000, score=A16, done=None, eos=-1, B=2, W=4, V=1000, k=4, os=A16, op=A16, ot=A16, od=None,
        ws=A16, wb=10 ** 6), **kw}.values())


def test_select_refusals():
    for n in ("x", "score", "os", "op", "ot"):
        assert select(**{n: None}) == -6
    for n in ("B", "W", "V", "k"):
        assert select(**{n: 0}) == -2
    assert select(W=65) == -2 and select(k=65) == -2 and select(V=2 ** 31 - 1) == -2 and select(B=2 ** 23) == -2
    assert select(eos=1000) == -2 and select(done=A16) == -2
    assert select(B=1, W=64, V=2 * 10 ** 7, wb=2 ** 40) == -2  # the merge's lists do not fit
    assert select(x=A16 + 1) == -4 and select(x=A16 + 2, fp32=1) == -4 and select(score=A16 + 2) == -4 and select(ot=A16 + 1) == -4
    need = _lib.load().mx_beam_select_ws(2, 4, 1000, 4)
    assert need > 0 and select(wb=need - 1) == -3 and select(ws=None) == -3 and select(ws=A16 + 4) == -3
    assert _lib.load().mx_beam_select_ws(1, 65, 10, 1) == 0 and _lib.load().mx_beam_select_ws(0, 1, 10, 1) == 0


def test_reorder_refusals():
    mv = lambda **kw: _lib.load().mx_reorder_slots(*{**dict(
        st=None, x=A16, sn=1024, ss=512, sh=128, stt=64, N=1, G=1, W=2, H=4, T=2, rb=64, par=A16, pg=2, pw=1, len=None, ls=0, base=2,
        unit=1, first=0), **kw}.values())
    assert mv(x=None) == -6 and mv(par=None) == -6
    for n in ("N", "G", "W", "H", "T", "rb", "unit"):
        assert mv(**{n: 0}) == -2
    assert mv(W=65) == -2 and mv(first=-1) == -2 and mv(N=2 ** 20, H=2 ** 12) == -2
    assert mv(par=A16 + 2) == -4 and mv(len=A16 + 1) == -4
    assert mv(W=1) == 0 and mv(first=2) == 0  # nothing moves: nothing is launched


def test_rope_at_refusals():
    rp = lambda **kw: _lib.load().mx_rope_kv_at(*{**dict(
        st=None, qkv=A16, ldq=192, cs=A16, ncs=9, q=A16, kc=A16, vc=A16, B=1, n=1, H=1, ctx=5, at=A16, ats=1, rot0=0), **kw}.values())
    for n in ("qkv", "cs", "q", "kc", "vc", "at"):
        assert rp(**{n: None}) == -6
    for n in ("B", "n", "H", "ctx", "ncs"):
        assert rp(**{n: 0}) == -2
    assert rp(ldq=184) == -2 and rp(B=2 ** 20, n=2 ** 10) == -2
    assert rp(ldq=196) == -4 and rp(qkv=A16 + 8) == -4 and rp(kc=A16 + 8) == -4 and rp(at=A16 + 2) == -4


def z(*s, dtype=BF):
    return torch.zeros(*s, dtype=dtype)


def test_python_refusals_prefix():
    ok = dict(q=z(4, 6, 1, 64), pk=z(2, 3, 10, 64), pv=z(2, 3, 10, 64), k=z(4, 3, 5, 64), v=z(4, 3, 5, 64))
    bad = [dict(q=z(4, 6, 64)), dict(q=z(3, 6, 1, 64)), dict(q=z(4, 7, 1, 64)), dict(q=z(4, 6, 1, 72)), dict(pk=z(2, 3, 9, 64)),
           dict(pv=z(2, 3, 10, 128)), dict(k=z(4, 3, 6, 64)), dict(k=z(4, 2, 5, 64), v=z(4, 2, 5, 64)),
           dict(k=z(2, 3, 5, 64), v=z(2, 3, 5, 64)), dict(q=z(4, 6, 1, 64, dtype=torch.float16)), dict(pk=z(2, 3, 10, 64).float()),
           dict(pk=z(0, 3, 10, 64), pv=z(0, 3, 10, 64)), dict(kv_len=6), dict(kv_len=-1), dict(prefix_len=11),
           dict(kv_len=z(3, dtype=torch.int32)), dict(kv_len=z(4, dtype=torch.int64)), dict(prefix_len=z(4, dtype=torch.int32)),
           dict(scale=0.0), dict(scale=INF), dict(out=z(4, 1, 383)), dict(out=z(4, 1, 384).float()),
           dict(out=z(4, 384, 1).transpose(1, 2)[:, :, ::2])]
    for b in bad:
        with pytest.raises(ValueError):
            ops.sdpa_prefix(**{**ok, **b})
    with pytest.raises(ValueError, match="GPU"):
        ops.sdpa_prefix(**ok)
    assert ops.sdpa_prefix(**{**ok, "q": z(4, 6, 0, 64)}).shape == (4, 0, 384)


def test_python_refusals_select():
    ok = dict(logits=z(2, 3, 10), scores=z(2, 3, dtype=torch.float32), k=3, done=z(2, 3, dtype=torch.bool), eos=1)
    bad = [dict(logits=z(2, 3)), dict(logits=z(2, 3, 10, dtype=torch.float16)), dict(scores=z(2, 3)), dict(scores=z(2, 4, dtype=torch.float32)),
           dict(k=0), dict(k=65), dict(eos=10), dict(eos=-1), dict(eos=None), dict(done=z(2, 3, dtype=torch.uint8)),
           dict(done=z(3, dtype=torch.bool)), dict(logits=z(1, 65, 10), scores=z(1, 65, dtype=torch.float32), done=None), dict(logits=z(2, 3, 0)),
           dict(logits=z(1, 1, 1).expand(1, 64, 4 * 10 ** 8), scores=z(1, 64, dtype=torch.float32), done=None)]
    for b in bad:
        with pytest.raises(ValueError):
            ops.beam_select(**{**ok, **b})
    with pytest.raises(ValueError, match="GPU"):
        ops.beam_select(**ok)


def test_python_refusals_reorder():
    x, p = z(1, 4, 2, 5, 8), z(2, 2, dtype=torch.int32)
    for kw in (dict(x=z(4, 2, 5)), dict(parent=p.long()), dict(parent=z(3, dtype=torch.int32)), dict(parent=z(2, 2, 1, dtype=torch.int32)),
               dict(n=6), dict(n=-1), dict(n=z(2, dtype=torch.int32)), dict(first=-1), dict(unit=0), dict(unit=2 ** 31, n=3),
               dict(x=z(1, 1, 2, 5, 8).expand(1, 4, 2, 5, 8)), dict(x=z(1, 4, 2, 8, 5).transpose(3, 4)),
               dict(x=z(1, 65, 1, 1, 8), parent=z(65, dtype=torch.int32))):
        with pytest.raises(ValueError):
            ops.reorder_slots(**{**dict(x=x, parent=p), **kw})
    with pytest.raises(ValueError, match="GPU"):
        ops.reorder_slots(x, p)


def test_python_refusals_rope():
    ok = dict(qkv=z(2, 1, 192), cs=z(9, 16, 2, dtype=torch.float32), kc=z(2, 1, 5, 64), vc=z(2, 1, 5, 64), at=z(2, dtype=torch.int32))
    for kw in (dict(rot0=2 ** 31), dict(qkv=z(1, 1, 192)), dict(qkv=z(2, 1, 191)), dict(cs=z(9, 16, 2)), dict(cs=z(9, 32, dtype=torch.float32)),
               dict(kc=z(2, 1, 5, 128)), dict(vc=z(2, 1, 6, 64)), dict(at=z(1, dtype=torch.int32)), dict(at=z(2, dtype=torch.int64)),
               dict(kc=z(2, 5, 1, 64).transpose(1, 2)[:, :, ::2], vc=z(2, 5, 1, 64).transpose(1, 2)[:, :, ::2])):
        with pytest.raises(ValueError):
            ops.rope_kv_at(**{**ok, **kw})
    with pytest.raises(ValueError, match="GPU"):
        ops.rope_kv_at(**ok)


def test_outgrown_workspace_stays(monkeypatch):
    """A search of many beams follows a captured query, and needs more split-K scratch: what the graph writes to stays its own."""
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    ws = ops.Workspace(torch.device("cpu"))
    sizes = []
    for n in (100, 50, 2000, 9000):
        ws.reserve(n, 0)
        sizes.append(ws.ws)
    assert sizes[0] is sizes[1] and sizes[3] is ws.ws and all(any(t is o for o in ws.outgrown) for t in sizes[:3])
