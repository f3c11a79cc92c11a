"""The checks of prefix_needles.py against a plain attention on the CPU: they pass it, and see every single key that it is made to
lose, to count twice or to take for its neighbour."""
import math

import pytest
import torch

from prefix_needles import counts, needles

CASES = [((1, 3, 2, 2, 64, 1, 70, 40), (40, 0, 7), None), ((2, 2, 1, 2, 128, 5, 33, 20), (20, 3, 0, 5), (33, 0)), ((1, 1, 1, 1, 64, 70, 0, 90), None, None),
         ((3, 1, 1, 1, 64, 2, 40, 0), None, (40, 39, 1))]


def plain(q, pk, pv, k, v, kv_len, prefix_len, prefix=lambda i: i, own=lambda i: i):
    """In fp32; prefix, own: what is done to the lists of keys that a row sees."""
    B, Hq, Tq, D = q.shape
    N, H, P = pk.shape[:3]
    S, G, out = B // N, Hq // H, torch.zeros(B, Tq, Hq, D)
    for b in range(B):
        p = P if prefix_len is None else int(prefix_len[b // S])
        t = k.shape[2] if kv_len is None else int(kv_len[b])
        for i in range(Tq):
            a, o = prefix(list(range(p))), own(list(range(min(max(t - Tq + 1 + i, 0), t))))
            for h in range(H):
                kk, vv = torch.cat([pk[b // S, h, a], k[b, h, o]]).float(), torch.cat([pv[b // S, h, a], v[b, h, o]]).float()
                if len(kk):
                    w = torch.softmax(q[b, h * G:(h + 1) * G, i].float() @ kk.t() / math.sqrt(D), 1)
                    out[b, i, h * G:(h + 1) * G] = w @ vv
    return out.flatten(2).to(torch.bfloat16)


@pytest.mark.parametrize("case", CASES, ids=str)
def test_the_formula_passes(case):
    counts(plain, *case)
    needles(plain, *case)


LOST = [lambda i: i[1:], lambda i: i[:-1], lambda i: i[:17] + i[18:], lambda i: i + i[-1:], lambda i: i[:33] + i[32:],
        lambda i: i[:-1] + i[-2:-1]]


@pytest.mark.parametrize("where", ["prefix", "own"])
@pytest.mark.parametrize("lost", range(len(LOST)))
def test_a_key_lost_or_doubled_is_seen(where, lost):
    bad = lambda *a: plain(*a, **{where: LOST[lost]})
    with pytest.raises(AssertionError):
        counts(bad, *CASES[0])


@pytest.mark.parametrize("where", ["prefix", "own"])
def test_a_key_taken_for_another_is_seen(where):
    """The last key's value with its neighbour's place, as a wrong row of V would give it."""
    def bad(q, pk, pv, k, v, kv_len, prefix_len):
        pv, v = (t.clone() for t in (pv, v))
        x = pv if where == "prefix" else v
        x[:, :, -1] = x[:, :, -2]
        return plain(q, pk, pv, k, v, kv_len, prefix_len)
    with pytest.raises(AssertionError):
        needles(bad, *CASES[0])
