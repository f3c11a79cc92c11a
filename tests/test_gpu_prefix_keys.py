"""Attention over shared prefixes on the MI355X, key by key (prefix_needles.py), and infinite values whose weight is 0 in fp32."""
import math

import pytest
import torch

import strix_halo_maxx_amd.ops as ops
from beam_cases import ATTENTION, MASKED
from prefix_needles import counts, needles

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.mark.parametrize("case", ATTENTION, ids=str)
def test_every_key_once(dev, case):
    counts(ops.sdpa_prefix, *case, dev=dev)


@pytest.mark.parametrize("case", ATTENTION, ids=str)
def test_keys_are_themselves(dev, case):
    """Both sides of every 32nd key of the prefixes, and the last own keys that each query sees."""
    needles(ops.sdpa_prefix, *case, dev=dev)


@pytest.mark.parametrize("case", MASKED, ids=str)
def test_infinite_values_without_weight(dev, case):
    """One key of the prefix has all the weight, the others' underflow to 0. An infinite value of such a key makes its column of the
    rows that see it infinite or NaN (the formula's product with a weight above 0, or fp32's with 0), and nothing else."""
    N, S, H, G, D, Tq, P, T = case
    B = N * S
    g = torch.Generator().manual_seed(P)
    rnd = lambda *s: torch.randn(*s, generator=g).to(BF)
    lens = [(T - 5 * b) % (T + 1) for b in range(B)]  # sequence 0 has all T
    plens = [max(P - 13 * n, 0) for n in range(N)]
    big = 128.0  # its score: 128^2 D^-1/2 >= 1448, in base 2 more than 2000 above the others' 0
    q, pk, pv, k, v = rnd(B, H * G, Tq, D), torch.zeros(N, H, P, D).to(BF), rnd(N, H, P, D), torch.zeros(B, H, T, D).to(BF), rnd(B, H, T, D)
    q[..., 0] = big
    for n in range(N):
        pk[n, :, plens[n] // 2, 0] = big
    pv[0, :, 0, 3], pv[0, :, plens[0] - 1, 4] = math.inf, -math.inf
    v[0, :, 0, 5], v[0, :, T - 1, 6] = math.inf, math.inf
    i32 = lambda x: torch.tensor(x, device=dev, dtype=torch.int32)
    got = ops.sdpa_prefix(*(t.to(dev) for t in (q, pk, pv, k, v)), i32(lens), i32(plens)).cpu().view(B, Tq, H, G, D)
    want = torch.stack([pv[n, :, plens[n] // 2] for n in range(N)]).repeat_interleave(S, 0)[:, None, :, None].expand(B, Tq, H, G, D)
    odd = torch.zeros(B, Tq, H, G, D, dtype=torch.bool)
    odd[:S, ..., 3] = odd[:S, ..., 4] = True
    odd[0, max(Tq - T, 0):, ..., 5] = True  # the queries that see its first own key; the last alone sees the last
    odd[0, Tq - 1, ..., 6] = True
    assert not bool(torch.isfinite(got[odd]).any())
    assert torch.equal(got[~odd], want[~odd])
