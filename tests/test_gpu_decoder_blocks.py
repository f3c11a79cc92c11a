"""Beam search over the 8-bit cache past a border of its blocks of 64 tokens: a step that moves two blocks of a beam, a fresh block
in a beam's slot, and buffers whose later blocks still hold another search's codes and exponents."""
import pytest
import torch

import strix_halo_maxx_amd.md2text as mt
import strix_halo_maxx_amd.synth as S
from test_gpu_decoder_beams import Record, decoder, image, name, rel

pytestmark = pytest.mark.gpu
KV8 = [dict(kv8=True), dict(mxfp4=True, kv8=True)]


def another_search(dec):
    """What a kept search's buffers may hold: the largest codes under large exponents, in every block."""
    assert len(dec.beam_states) == 1
    for c in next(iter(dec.beam_states.values())).kv:
        for t, x in ((c.kc, 0x7e), (c.vc, 0xfe), (c.ks, 190), (c.vs, 190)):
            t.fill_(x)


@pytest.mark.parametrize("form", KV8, ids=name)
def test_generate_past_a_block(dev, monkeypatch, form):
    """From row 121 to row 135. The logits of a hypothesis against a pass over all its tokens, before and behind the border, as in the
    searches inside one block: 2^-4 of a value for the 8-bit cache, MXFP4's below 0.2."""
    w, dec = decoder(form)
    img, other, ids = image(dev), image(dev, 9), S.prompt_ids(8, 50)
    rec = Record(monkeypatch)
    first = dec.generate_beams(img, ids, 16, beams=4, use_graph=False)
    history, steps = rec.check(4, None), rec.steps
    monkeypatch.undo()  # captured steps take no records
    tol = 0.2 if form.get("mxfp4") else 2.0 ** -4
    for t in (6, 7, 8, 9, 15):
        for b, h in enumerate(history[t - 1][0]):
            dec.prefill(img, torch.cat([ids, torch.tensor(h)]))
            assert rel(steps[t][0][0, b], dec.logits) < tol, (t, b)
    for graph in (False, True, True):
        dec.generate_beams(other, ids, 16, beams=4, use_graph=graph)
        another_search(dec)
        again = dec.generate_beams(img, ids, 16, beams=4, use_graph=graph)
        assert all(torch.equal(a, b) for a, b in zip(first, again)), graph


@pytest.mark.parametrize("form", KV8, ids=name)
def test_answer_past_a_block(dev, monkeypatch, form):
    """Questions that end at rows 120, 127 and 112, three beams each, 18 tokens: some cross the border, some start at it."""
    w, dec = decoder(form, nq=3, L=16)
    img, other = image(dev, n=110), image(dev, 9, n=110)
    qs = [S.prompt_ids(20, 9).tolist(), S.prompt_ids(21, 16).tolist(), S.prompt_ids(22, 1).tolist()]
    dec.set_questions(qs)
    dec.encode(img)
    rec = Record(monkeypatch)
    first = dec.answer(18, beams=3, use_graph=False)
    history, steps = rec.check(3, None), rec.steps
    monkeypatch.undo()  # captured steps take no records
    for graph in (False, True, True):
        dec.encode(other)
        dec.answer(18, beams=3, use_graph=graph)
        another_search(dec)
        dec.encode(img)
        again = dec.answer(18, beams=3, use_graph=graph)
        assert all(torch.equal(a, b) for a, b in zip(first, again)), graph
    tol = 0.2 if form.get("mxfp4") else 2.0 ** -4
    one = mt.TextDecoder(w, ctx=256, **form)
    for t in (2, 9, 17):
        for q in range(3):
            for b, h in enumerate(history[t - 1][q]):
                one.prefill(img, torch.tensor(qs[q] + h))
                assert rel(steps[t][0][q, b], one.logits) < tol, (t, q, b)
