"""Sizes and arguments of the shared-prefix attention, beam selection and slot reordering that no call on real memory reaches: what
the C entries cannot hold is refused, nothing of an earlier call is taken for a later one. Without a GPU: the tensors have no
memory, or the call stops before the library."""
import pytest
import torch

import strix_halo_maxx_amd.ops as ops
from strix_halo_maxx_amd import _lib

BF, F32, I32, U8 = torch.bfloat16, torch.float32, torch.int32, torch.uint8
FAR = 2 ** 32 + 64  # 64 to whoever keeps the lower 32 bits


def no(*s, dtype=BF):
    """A tensor without memory."""
    return torch.empty(*s, dtype=dtype, device="meta")


def test_reorder_sizes_past_31_bits():
    p, n = no(1, 2, dtype=I32), no(2, dtype=I32)
    for x in (no(1, 2, 1, 1, FAR, dtype=U8), no(1, 2, 1, 1, 2 ** 31, dtype=U8), no(1, 2, 1, 1, 2 ** 29, dtype=F32),
              no(1, 2, 1, FAR, 16), no(1, 2, FAR, 1, 16), no(FAR, 2, 1, 1, 16)):
        with pytest.raises(ValueError, match="32 bits"):
            ops.reorder_slots(x, p, n)
    for x in (no(1, 2, 1, 1, 2 ** 31 - 16, dtype=U8), no(1, 2, 1, 2 ** 31 - 1, 16)):  # these reach the library
        with pytest.raises(ValueError, match="GPU"):
            ops.reorder_slots(x, p, n)
    with pytest.raises(ValueError, match="32 bits"):
        ops.reorder_slots(no(1, FAR, 1, 1, 16), no(FAR // 2, 2, dtype=I32))


def test_select_sizes_past_31_bits():
    for B, V in ((1, FAR), (FAR, 10), (1, 2 ** 31)):
        with pytest.raises(ValueError, match="32 bits"):
            ops.beam_select(no(B, 1, V), no(B, 1, dtype=F32), 1)


def test_prefix_sizes_past_31_bits():
    for P, T, Tq, N in ((FAR, 3, 1, 1), (3, FAR, 1, 1), (3, 3, FAR, 1), (2 ** 31, 3, 1, 1), (3, 3, 1, FAR)):
        q, pk, k = no(N, 1, Tq, 64), no(N, 1, P, 64), no(N, 1, T, 64)
        with pytest.raises(ValueError, match="32 bits"):
            ops.sdpa_prefix(q, pk, pk, k, k)
    for i in range(7):
        with pytest.raises(ValueError, match="32 bits"):
            ops.sdpa_prefix_tiling(*(FAR if i == j else 1 for j in range(7)), 64)


def test_rope_sizes_past_31_bits():
    for ctx, n, pos, B in ((FAR, 1, 9, 1), (5, FAR, 9, 1), (5, 1, FAR, 1), (5, 1, 9, FAR)):
        kc = no(B, 1, ctx, 64)
        with pytest.raises(ValueError, match="32 bits"):
            ops.rope_kv_at(no(B, n, 192), no(pos, 16, 2, dtype=F32), kc, kc, no(B, dtype=I32))


def test_select_searches_of_one_grid():
    """The merge has 1024 threads for each search: 2^32 and more are no grid."""
    ws = _lib.load().mx_beam_select_ws
    assert ws(2 ** 22 - 1, 1, 10, 1) == (2 ** 22 - 1) * 16 and ws(2 ** 22, 1, 10, 1) == 0 and ws(5000000, 1, 10, 1) == 0
    a = 0x10000  # never dereferenced: refused before any launch
    assert _lib.load().mx_beam_select(None, a, 0, 10, 10, a, None, -1, 2 ** 22, 1, 10, 1, a, a, a, None, a, 2 ** 40) == -2
    with pytest.raises(ValueError, match="too many"):
        ops.beam_select(no(2 ** 22, 1, 10), no(2 ** 22, 1, dtype=F32), 1)


def test_select_count_in_a_tensor(monkeypatch):
    """How many to select may be any number, also one that changes its value between calls."""
    monkeypatch.setattr(ops, "_call_on", lambda *a: None)
    x, s, k = torch.zeros(1, 3, 10), torch.zeros(1, 3), torch.tensor(2)
    assert ops.beam_select(x, s, k)[0].shape == (1, 2)
    k.fill_(3)
    assert ops.beam_select(x, s, k)[0].shape == (1, 3)


def test_prefix_copies_what_it_has_to(monkeypatch):
    """Where one tensor has strides or an address that the kernel does not take, that one is copied: not a prefix of gigabytes for
    a query at an odd address."""
    seen = []
    monkeypatch.setattr(ops, "_call_on", lambda dev, name, *a: seen.append(a[:5]))
    x = [torch.zeros(4, 2, 3, 64, dtype=BF)] + [torch.zeros(2, 2, 10, 64, dtype=BF) for _ in range(2)] + \
        [torch.zeros(4, 2, 5, 64, dtype=BF) for _ in range(2)]
    shift = lambda t: torch.cat([t.new_zeros(1), t.flatten()])[1:].view(t.shape)
    wide = lambda t: torch.cat([t, t.new_zeros(*t.shape[:3], 3)], 3)[..., :t.shape[3]]
    cols = lambda t: t.transpose(2, 3).contiguous().transpose(2, 3)
    for f in (shift, wide, cols):
        for i in range(5):
            y = [f(t) if i == j else t for j, t in enumerate(x)]
            ops.sdpa_prefix(*y)
            assert [p != t.data_ptr() for p, t in zip(seen[-1], y)] == [i == j for j in range(5)], (f, i)
            assert seen[-1][i] % 16 == 0
