"""The text decoder with MXFP4 Linears and / or the 8-bit cache: it is the public operators, composed (bit for bit: the same
kernels on the same values, whether positions come from the host or the device); it stays near the bf16 decoder by as much
as the formats allow; captured graphs equal the eager calls; a query finds the same prefix whatever was asked before."""
import pytest
import torch

import strix_halo_maxx_amd.md2text as mt
import strix_halo_maxx_amd.ops as ops
import strix_halo_maxx_amd.synth as S
from strix_halo_maxx_amd import _lib

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
D, H, HD, FF = 2048, 32, 64, 8192
FORMS = [dict(mxfp4=True), dict(kv8=True), dict(mxfp4=True, kv8=True), dict(w8a8=True, kv8=True)]


def name(f):
    return "+".join(f)


def inputs(dev, n_img=70, n_ids=25):
    return S.activations(7, (n_img, D), "img").to(dev), S.prompt_ids(8, n_ids).to(dev)


class Composed:
    """Two MXFP4 layers over 8-bit caches from the public operators alone."""

    def __init__(self, w, dev, ctx):
        self.dev, self.layers = dev, []
        g = lambda n: w[n].to(dev, BF).contiguous()
        for i in range(2):
            p = f"blocks.{i}."
            qf = ops.MxFp4Lin(torch.cat([w[p + "attn.qkv.weight"], w[p + "mlp.fc1.weight"]]),
                              torch.cat([w[p + "attn.qkv.bias"], w[p + "mlp.fc1.bias"]]), device=dev)
            out = ops.MxFp4Lin(torch.cat([w[p + "mlp.fc2.weight"], w[p + "attn.proj.weight"]], 1),
                               w[p + "mlp.fc2.bias"].float() + w[p + "attn.proj.bias"].float(), device=dev)
            self.layers.append(dict(ln=(g(p + "ln.weight"), g(p + "ln.bias")), qf=qf, out=out,
                                    kv=ops.KV8Cache(1, H, ctx, HD, device=dev)))
        self.post = (g("post_ln.weight"), g("post_ln.bias"))
        self.cs = S.freqs_cis(32, 2048).to(dev)

    def run(self, x, pos, causal_from):
        n = x.shape[0]
        for L in self.layers:
            h = ops.layernorm(x, *L["ln"])
            y = L["qf"](h, act="tanh", act_from=3 * D)
            q, k, v = y[:, :3 * D].reshape(n, 3, H, HD).permute(1, 2, 0, 3)[:, None]
            q = L["kv"].append(k, v, pos, cs=self.cs, q=q)
            a = ops.sdpa_kv8(q, L["kv"], pos + n, causal_from=causal_from)
            x = L["out"](torch.cat([y[:, 3 * D:], a[0]], 1), res=x)
        return x


def test_prefill_and_decode_are_the_operators_composed(dev):
    w = S.text_weights(3, layers=2)
    dec = mt.TextDecoder(w, ctx=256, mxfp4=True, kv8=True)
    assert not dec.use_mk and dec.kc is None and "wqf" not in dec.blocks[0]
    img, ids = inputs(dev)
    ref = Composed(w, dev, 256)
    x = torch.cat([dec.wte[mt.BOS:mt.BOS + 1], img.to(BF), dec.wte[ids]])
    want = ref.run(x, 0, 71)[71:]
    got = dec.prefill(img, ids)
    assert torch.equal(got, want)
    for L, kv in zip(ref.layers, dec.kv):
        assert all(torch.equal(a, b) for a, b in zip(L["kv"].read(96), kv.read(96)))
    dec.start_decode()
    for t in range(40):  # across a block border at 128
        row = dec.xd[0].clone()[None]
        dec.decode_step(logits=True)
        want = ref.run(row, 96 + t, None)
        lm = torch.empty(dec.V, device=dev, dtype=BF)
        part = torch.zeros_like(dec.part)
        _lib.call("mx_ln_gemv_argmax", _lib.stream(), want.data_ptr(), dec.post_ln[0].data_ptr(), dec.post_ln[1].data_ptr(),
                  1e-5, dec.w_lm.data_ptr(), dec.w_lm.stride(0), dec.b_lm.data_ptr(), dec.V, D, lm.data_ptr(),
                  part.data_ptr(), dec.nparts)
        assert torch.equal(dec.logits, lm), t


@pytest.mark.parametrize("form", FORMS, ids=name)
def test_near_the_bf16_decoder(dev, form):
    """The last layer's output against the bf16 decoder's. MXFP4: a code is off by at most a quarter of a value above half a
    unit, about an eighth in the root mean square of a normal block, for weights and activations, so a Linear's output by
    about 0.18 and the residual sum of two layers by less than 0.35. The cache: e4m3 is off by at most 2^-4 of a value.
    W8A8: by 2^-7 of the largest, below that."""
    w = S.text_weights(4, layers=2)
    img, ids = inputs(dev, 200, 30)
    ref = mt.TextDecoder(w, ctx=512).prefill(img, ids).float()
    got = mt.TextDecoder(w, ctx=512, **form).prefill(img, ids).float()
    r = float((got - ref).norm() / ref.norm())
    print(name(form), "rel-L2 vs bf16", r, flush=True)
    assert r < (0.35 if form.get("mxfp4") else 2.0 ** -4)


@pytest.mark.parametrize("form", FORMS, ids=name)
def test_generate_graph_equals_eager(dev, form):
    """Prefill and 60 greedy tokens, eager and as captured graphs (prefill and step), twice in a row on one decoder."""
    w = S.text_weights(5, layers=2)
    img, ids = inputs(dev)
    dec = mt.TextDecoder(w, ctx=192, **form)
    eager = dec.generate(img, ids, 60, use_graph=False).tolist()
    dec.capture_prefill(img.shape[0], ids.shape[0])
    for _ in range(2):
        assert dec.generate(img, ids, 60).tolist() == eager
    with pytest.raises(ValueError):
        dec.generate(img, ids, 98)


@pytest.mark.parametrize("form", FORMS, ids=name)
def test_query_finds_the_same_prefix_again(dev, form):
    """Question A, then B, then A again: A's logits are the same bits, eager and as a graph, and after a prefill with
    decoded tokens over the same slots the prefix is again what encode() left."""
    w = S.text_weights(6, layers=2)
    dec = mt.TextDecoder(w, ctx=256, nq=2, L=16, yes_ids=[11, 222, 3333, 44444], no_ids=[55, 666, 7777, 50000], **form)
    img, _ = inputs(dev, 70)
    ask = lambda s: dec.set_questions([S.prompt_ids(s, 9).tolist(), S.prompt_ids(s + 1, 16).tolist()])
    dec.encode(img)
    ask(1)
    a = dec.query().clone()
    ask(30)
    b = dec.query().clone()
    ask(1)
    assert torch.equal(dec.query(), a) and not torch.equal(a, b)
    dec.capture_query()
    for s, want in ((30, b), (1, a), (1, a), (30, b)):
        ask(s)
        assert torch.equal(dec.query(), want)
    dec.generate(img, S.prompt_ids(9, 16), 10, use_graph=False)
    dec.encode(img)
    ask(1)
    assert torch.equal(dec.query(), a)


def test_formats_that_exclude_each_other(dev):
    w = S.text_weights(2, layers=1)
    with pytest.raises(ValueError, match="either"):
        mt.TextDecoder(w, mxfp4=True, w8a8=True)
    with pytest.raises(ValueError, match="Linear class"):
        mt.TextDecoder(w, lin_cls=ops.MxI8Lin, mxfp4=True)
    assert mt.TextDecoder(w, lin_cls=ops.MxFp4Lin, ctx=64).mxfp4


def questions(dev, **kw):
    w = S.text_weights(6, layers=kw.pop("layers", 2))
    return mt.TextDecoder(w, ctx=256, nq=2, yes_ids=[11, 222, 3333, 44444], no_ids=[55, 666, 7777, 50000], **kw)


def cached(dec, n):
    """What the caches hold of positions 0 .. n - 1 of each slot (n: a length for each)."""
    return [x[s, :, :m].clone() for kv in dec.kv for x in kv.read() for s, m in enumerate(n)]


def scales(dec, n):
    return [x[s, :, :-(-m // 64)].clone() for kv in dec.kv for x in (kv.ks, kv.vs) for s, m in enumerate(n)]


def equal(a, b):
    return len(a) == len(b) and all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("form", [f for f in FORMS if f.get("kv8")], ids=name)
def test_question_does_not_depend_on_its_padding(dev, form):
    """Rows behind a question's end leave its logits, its cached rows and the exponents of their blocks alone: other embeddings of
    the padding id change nothing, eager and captured; and the ids of one question nothing in the other."""
    dec = questions(dev, L=24, **form)
    img, _ = inputs(dev, 70)
    dec.encode(img)
    q = [S.prompt_ids(1, 9).tolist(), S.prompt_ids(2, 14).tolist()]
    dec.set_questions(q)
    n = [71 + len(x) for x in q]
    want = dec.query().clone(), cached(dec, n), scales(dec, n)
    pads = S.activations(3, (4, D), "pad").to(dev)
    pads[2, 7], pads[3] = 300.0, 0
    for pad in pads:
        dec.wte[0] = pad
        assert torch.equal(dec.query(), want[0]) and equal(cached(dec, n), want[1]) and equal(scales(dec, n), want[2])
    dec.capture_query()
    for pad in pads:
        dec.wte[0] = pad
        assert torch.equal(dec.query(), want[0]) and equal(cached(dec, n), want[1]) and equal(scales(dec, n), want[2])
    dec.set_questions([q[0], S.prompt_ids(5, 24).tolist()])  # longer: the replayed graph follows the lengths
    got = dec.query().clone()
    assert torch.equal(got[0], want[0][0]) and not torch.equal(got[1], want[0][1])
    dec.query_graph = None
    assert torch.equal(dec.query(), got)


def test_question_does_not_depend_on_the_rows_it_is_padded_to(dev):
    """MXFP4 products give a row the same bits whatever the number of rows up to 32: L = 10 and L = 16 agree."""
    img, _ = inputs(dev, 70)
    q = [S.prompt_ids(1, 9).tolist(), S.prompt_ids(2, 10).tolist()]
    n, out = [71 + len(x) for x in q], []
    for L in (10, 16):
        dec = questions(dev, L=L, mxfp4=True, kv8=True)
        dec.wte[0] = 0
        dec.wte[0, 7] = 300.0
        dec.encode(img)
        dec.set_questions(q)
        out.append((dec.query().clone(), cached(dec, n), scales(dec, n)))
    assert torch.equal(out[0][0], out[1][0]) and equal(out[0][1], out[1][1]) and equal(out[0][2], out[1][2])


@pytest.mark.parametrize("form", [dict(mxfp4=True, kv8=True), dict(w8a8=True, kv8=True)], ids=name)
@pytest.mark.parametrize("n_img", [70, 63, 126])  # the prefix ends inside a block, with it, and on a block's last row but one
def test_query_after_prefill_and_after_encode(dev, form, n_img):
    """One layer, Linears that give a row the same bits in both passes: the prompt behind the prefix leaves the prefix that query()
    reads as encode() leaves it, whatever the prompt, eager and captured, and so the logits."""
    dec = questions(dev, L=16, layers=1, **form)
    img, _ = inputs(dev, n_img)
    q = [S.prompt_ids(1, 9).tolist(), S.prompt_ids(2, 16).tolist()]
    dec.set_questions(q)
    dec.encode(img)
    n = [n_img + 1 + len(x) for x in q]
    want = dec.query().clone(), cached(dec, n), scales(dec, n)
    for graph in (False, True):
        if graph:
            dec.capture_prefill(n_img, 40)
        for seed in (21, 22, 23):
            hidden = dec.prefill(img, S.prompt_ids(seed, 40).to(dev)).clone()
            assert torch.equal(dec.query(), want[0]) and equal(cached(dec, n), want[1]) and equal(scales(dec, n), want[2]), seed
            assert torch.equal(dec.prefill(img, S.prompt_ids(seed, 40).to(dev)), hidden)
            dec.start_decode()
            for _ in range(3):
                dec.decode_step()
            assert torch.equal(dec.query(), want[0]) and equal(cached(dec, n), want[1]) and equal(scales(dec, n), want[2]), seed
