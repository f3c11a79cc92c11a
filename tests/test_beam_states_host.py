"""What a text decoder keeps of its beam searches, without a GPU: the buffers on the CPU, no layer run."""
import torch

import strix_halo_maxx_amd.md2text as mt


def decoder(layers=2, H=2, hd=64, kv8=False):
    dec = object.__new__(mt.TextDecoder)
    dec.dev, dec.V, dec.H, dec.hd, dec.kv8, dec.blocks, dec.cs = torch.device("cpu"), 100, H, hd, kv8, [None] * layers, torch.zeros(4000, 16, 2)
    dec.beam_states, dec.logits = {}, torch.zeros(100)
    dec.prefill = lambda *a: None
    return dec


def test_searches_by_numbers():
    """Sizes and the end token in tensors: a search is that of their values at the call."""
    dec, seen = decoder(), []
    dec._beam_search = lambda st, logits, n_tokens, eos, *a: seen.append((st, n_tokens, eos)) or (torch.zeros(1), torch.zeros(1))
    img, ids = torch.zeros(5, 8), torch.zeros(3)
    n, beams, eos = torch.tensor(6), torch.tensor(2), torch.tensor(7)
    dec.generate_beams(img, ids, n, beams=beams, eos=eos)
    n.fill_(9), beams.fill_(3), eos.fill_(8)
    dec.generate_beams(img, ids, n, beams=beams, eos=eos)
    (a, *x), (b, *y) = seen
    assert x == [6, 7] and y == [9, 8] and all(type(v) is int for v in x + y)
    assert a.W == 2 and b.W == 3 and b.hist.shape[1] >= 9 and b.T == 8


def test_the_search_in_use_stays():
    """Searches of ever new lengths between do not take the buffers and the graph of the one that comes again."""
    dec = decoder()
    first = dec._beam_state(1, 4, 9, 0, 30, None)
    for prefix in range(40, 60):
        other = dec._beam_state(1, 4, 9, 0, prefix, None)
        assert dec._beam_state(1, 4, 9, 0, prefix, None) is other
        assert dec._beam_state(1, 4, 9, 0, 30, None) is first
        assert len(dec.beam_states) <= 4
    for prefix in range(40, 44):
        dec._beam_state(1, 4, 9, 0, prefix, None)
    assert dec._beam_state(1, 4, 9, 0, 30, None) is not first


def test_bytes_of_kept_searches(monkeypatch):
    """The buffers of earlier searches go where they would hold more than BEAM_BYTES with the new one's."""
    for kv8 in (False, True):
        dec = decoder(kv8=kv8)
        a = dec._beam_state(1, 4, 9, 0, 100, None)
        held = [a.own] if not kv8 else [t for c in a.kv for t in (c.kc, c.vc)]
        size = sum(t.numel() * t.element_size() for t in held)
        assert a.kept == size
        monkeypatch.setattr(mt, "BEAM_BYTES", 2 * size)
        b = dec._beam_state(1, 4, 9, 0, 101, None)
        assert list(dec.beam_states.values()) == [a, b]
        dec._beam_state(1, 4, 9, 0, 102, None)
        assert list(dec.beam_states.values())[0] is b and len(dec.beam_states) == 2
        big = dec._beam_state(1, 64, 9, 0, 102, None)  # more than the bound for itself
        assert list(dec.beam_states.values()) == [big]
