"""The text decoder's beam search: every selection is the 64-bit oracle's on the logits it was made from, the logits are those of
the hypotheses (so their rows were moved with them), captured steps equal eager ones, and a query over one shared copy of the
prefix is the query over one per slot up to roundings."""
import pytest
import torch

import oracle.beams as ob
import oracle.md2_text as ot
import strix_halo_maxx_amd.md2text as mt
import strix_halo_maxx_amd.synth as S

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
FORMS = [dict(), dict(w8a8=True), dict(mxfp4=True), dict(kv8=True), dict(mxfp4=True, kv8=True)]


def name(f):
    return "+".join(f) or "bf16"


def rel(a, b):
    a, b = a.float().cpu(), b.float().cpu()
    return float((a - b).norm() / b.norm())


def image(dev, seed=7, n=70):
    return S.activations(seed, (n, 2048), "img").to(dev)


class Record:
    """The selections of a search: logits, scores and finished beams before, what was chosen."""

    def __init__(self, monkeypatch):
        self.steps = []
        real = mt.ops.beam_select

        def select(logits, scores, k=None, done=None, eos=None):
            out = real(logits, scores, k, done=done, eos=eos)
            self.steps.append(tuple(None if t is None else t.cpu().clone() for t in (logits, scores, done, *out)))
            return out
        monkeypatch.setattr(mt.ops, "beam_select", select)

    def check(self, W, eos):
        """Each choice is the oracle's; returns the hypotheses (groups, W) of tokens at every step."""
        hyps, history = None, []
        for logits, scores, done, score, parent, token, fin in self.steps:
            want = ob.beam_select(logits, scores, W, done, eos)
            assert torch.equal(parent, want[1]) and torch.equal(token, want[2]) and (eos is None or torch.equal(fin, want[3]))
            assert bool(((score.double() - want[0]).abs() <= 2.0 ** -17 + 2.0 ** -24 * want[0].abs()).all())
            old = hyps or [[[]] for _ in range(logits.shape[0])]
            hyps = [[old[b][int(parent[b, w])] + [int(token[b, w])] for w in range(W)] for b in range(logits.shape[0])]
            history.append(hyps)
        return history


def decoder(form, layers=2, seed=3, **kw):
    w = S.text_weights(seed, layers=layers)
    return w, mt.TextDecoder(w, ctx=256, **form, **kw)


@pytest.mark.parametrize("form", FORMS, ids=name)
def test_generate_beams(dev, monkeypatch, form):
    """Six tokens by four beams behind a 71-row prefix and a 25-id prompt. The logits of a hypothesis against a pass over all its
    tokens: bf16 roundings and W8A8's (which falls with them) 2 %; MXFP4: bf16 roundings carry less than 1/16 of the values
    over a code's border, by a quarter of themselves, below 0.2 over two layers; the 8-bit cache: 2^-4 of a value, as the
    blocks' exponents come out."""
    w, dec = decoder(form)
    img, ids = image(dev), S.prompt_ids(8, 25)
    rec = Record(monkeypatch)
    tokens, scores = dec.generate_beams(img, ids, 6, beams=4, use_graph=False)
    assert tokens.shape == (4, 6) and scores.shape == (4,)
    history = rec.check(4, None)
    assert tokens.tolist() == history[-1][0] and torch.equal(scores.cpu(), rec.steps[-1][3][0])
    assert all(len({tuple(h) for h in step[0]}) == 4 for step in history)
    tol = 0.2 if form.get("mxfp4") else 2.0 ** -4 if form.get("kv8") else 2e-2
    for t in (1, 3, 5):
        for b, h in enumerate(history[t - 1][0]):
            dec.prefill(img, torch.cat([ids, torch.tensor(h)]))
            assert rel(rec.steps[t][0][0, b], dec.logits) < tol, (t, b)


def test_generate_beams_against_the_oracle(dev, monkeypatch):
    """The same against the oracle's decoder, teacher-forced on every hypothesis (rel-L2 1e-2, as its greedy steps)."""
    w, dec = decoder({})
    img, ids = image(dev), S.prompt_ids(8, 25)
    rec = Record(monkeypatch)
    dec.generate_beams(img, ids, 4, beams=3, use_graph=False)
    history = rec.check(3, None)
    ora = ot.Text(w, 256, S.freqs_cis(32, 2048))
    assert rel(rec.steps[0][0], ora.prefill(img.cpu(), ids)) < 1e-2
    for t in (1, 2, 3):
        for b, h in enumerate(history[t - 1][0]):
            ora.prefill(img.cpu(), ids)
            for tok in h:
                lg = ora.step(tok)
            assert rel(rec.steps[t][0][0, b], lg) < 1e-2, (t, b)


@pytest.mark.parametrize("form", [dict(), dict(shared_prefix=True), dict(w8a8=True), dict(kv8=True)], ids=name)
def test_answer(dev, monkeypatch, form):
    """Three questions of unlike lengths, three beams each: every question's logits against a decoder that is asked it alone."""
    w, dec = decoder(form, nq=3, L=16)
    img = image(dev)
    qs = [S.prompt_ids(20, 9).tolist(), S.prompt_ids(21, 16).tolist(), S.prompt_ids(22, 1).tolist()]
    dec.encode(img)
    dec.set_questions(qs)
    dec.full_logits = True
    first = dec.query().clone()
    rec = Record(monkeypatch)
    tokens, scores = dec.answer(5, beams=3, use_graph=False)
    assert tokens.shape == (3, 3, 5) and scores.shape == (3, 3)
    history = rec.check(3, None)
    assert torch.equal(rec.steps[0][0][:, 0], first.cpu()) and tokens.tolist() == history[-1]
    assert torch.equal(dec.query(), first)  # the search leaves the prefix and the questions as they were
    tol = 2.0 ** -4 if form.get("kv8") else 2e-2
    one = mt.TextDecoder(w, ctx=256, **{k: v for k, v in form.items() if k != "shared_prefix"})
    for t in (1, 4):
        for q in range(3):
            for b, h in enumerate(history[t - 1][q]):
                one.prefill(img, torch.tensor(qs[q] + h))
                assert rel(rec.steps[t][0][q, b], one.logits) < tol, (t, q, b)


@pytest.mark.parametrize("form", FORMS, ids=name)
def test_graph_equals_eager(dev, form):
    """Searches by eager steps and by the captured step, on one decoder in turn, on other inputs between: the same bits."""
    w, dec = decoder(form, nq=2, L=12)
    img, img2, ids = image(dev), image(dev, 9), S.prompt_ids(8, 25)
    qs = [S.prompt_ids(20, 9).tolist(), S.prompt_ids(21, 12).tolist()]

    def run(graph):
        out = [*dec.generate_beams(img, ids, 12, beams=3, use_graph=graph)]
        dec.encode(img)
        dec.set_questions(qs)
        out += [*dec.answer(9, beams=2, eos=11, use_graph=graph)]
        out += [*dec.answer(9, use_graph=graph)]
        return [t.cpu() for t in out]
    want = run(False)
    for other in range(3):
        got = run(True)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), other
        dec.generate_beams(img2, ids, 12, beams=3)
    assert all(torch.equal(a, b) for a, b in zip(run(False), want))


def test_eos_and_length(dev, monkeypatch):
    """A token that ends hypotheses: they keep their scores, the rest is eos, and a search whose beams have all ended stops."""
    w, dec = decoder({})
    img, ids = image(dev), S.prompt_ids(8, 25)
    free, _ = dec.generate_beams(img, ids, 6, beams=4)
    eos = int(free[0, 2])
    rec = Record(monkeypatch)
    tokens, scores = dec.generate_beams(img, ids, 6, beams=4, eos=eos, use_graph=False)
    history = rec.check(4, eos)
    assert tokens.tolist() == history[-1][0]
    ended = [h for h in tokens.tolist() if eos in h]
    assert ended and all(set(h[h.index(eos):]) == {eos} for h in ended)
    by_len, s2 = dec.generate_beams(img, ids, 6, beams=4, eos=eos, length_penalty=2.0, use_graph=False)
    n = [h.index(eos) + 1 if eos in h else 6 for h in tokens.tolist()]
    want = sorted(zip([float(s) / m ** 2 for s, m in zip(scores, n)], tokens.tolist()), key=lambda x: -x[0])
    assert by_len.tolist() == [h for _, h in want]
    assert all(abs(a - float(b)) < 1e-5 * abs(a) for (a, _), b in zip(want, s2))
    dec.b_lm[eos] += 100.0
    dec.lm_full = None
    steps = len(rec.steps)
    tokens, _ = dec.generate_beams(img, ids, 60, beams=4, eos=eos, use_graph=False)
    assert len(rec.steps) - steps < 20 and tokens.shape == (4, 60) and bool((tokens[:, 2:] == eos).all())


def test_shared_prefix_query(dev):
    """One copy of the prefix for the questions: logits as near the copies' as two bf16 attentions of two layers are, and the
    other slots hold no prefix."""
    yn = dict(yes_ids=[11, 222, 3333, 44444], no_ids=[55, 666, 7777, 50000])
    w, dec = decoder({}, nq=4, L=16, **yn)
    _, one = decoder(dict(shared_prefix=True), nq=4, L=16, **yn)
    img = image(dev, n=129)
    qs = [S.prompt_ids(30 + i, n).tolist() for i, n in enumerate((16, 3, 9, 1))]
    for d in (dec, one):
        d.encode(img)
        d.set_questions(qs)
    a, b = dec.query(), one.query()
    print("shared prefix, rel-L2 of the logits", rel(b, a), flush=True)
    assert rel(b, a) < 1e-2
    assert all(not bool(k[1:, :, :130].any()) and not bool(v[1:, :, :130].any()) for k, v in zip(one.kc, one.vc))
    one.capture_query()
    assert torch.equal(one.query(), b)
    ids = S.prompt_ids(8, 20)
    assert torch.equal(one.generate(img, ids, 5), dec.generate(img, ids, 5))  # slot 0 is what it was
    one.query()


def test_captured_query_after_a_wide_search(dev):
    """A captured query and a captured step stay what they were when wider products have come between, replayed over again."""
    w, dec = decoder({}, nq=2, L=12)
    img = image(dev)
    dec.full_logits = True
    dec.encode(img)
    dec.set_questions([S.prompt_ids(20, 9).tolist(), S.prompt_ids(21, 12).tolist()])
    dec.capture_query()
    first = dec.query().clone()
    few = dec.answer(6, beams=2)
    for beams in (16, 64):
        dec.answer(4, beams=beams)
        mine = [torch.full((1 << e,), 7.0, device=dev) for e in range(10, 23)]  # memory that something else holds now
        again = dec.answer(6, beams=2)
        assert torch.equal(dec.query(), first) and all(torch.equal(a, b) for a, b in zip(again, few))
        assert all(bool((t == 7.0).all()) for t in mine)


def test_refusals(dev):
    w, dec = decoder({}, nq=2, L=8)
    img, ids = image(dev), S.prompt_ids(8, 25)
    with pytest.raises(RuntimeError):
        dec.answer(3)
    for kw in (dict(n_tokens=0), dict(n_tokens=3, beams=0), dict(n_tokens=3, beams=65), dict(n_tokens=3, eos=51200),
               dict(n_tokens=3, eos=-1), dict(n_tokens=2000)):
        with pytest.raises(ValueError):
            dec.generate_beams(img, ids, **kw)
    with pytest.raises(ValueError):
        mt.TextDecoder(w, ctx=256, kv8=True, shared_prefix=True)
