"""The workspace of packed linear attention: states between the segments of one sequence, whatever the number of sequences."""

from __future__ import annotations

import ctypes
import random

import pytest

from causal_conv1d_amd import _lib


def floats(L, seqs, heads, dk, dv, batch=1, backward=False):
    lib, b = _lib.load(), _lib.AttnBwdParams()
    p = b.fwd
    p.batch, p.seqlen, p.heads, p.key_heads, p.dk, p.dv, p.scale, p.dtype = batch, L, heads, heads, dk, dv, 1.0, 1
    if seqs:
        p.cu_seqlens, p.num_seqs = 16, seqs
    n = lib.cc1d_attn_bwd_workspace_floats(ctypes.byref(b)) if backward else lib.cc1d_attn_workspace_floats(ctypes.byref(p))
    assert n >= 0
    return n


@pytest.mark.parametrize("L,heads,dk,dv", [(8192, 32, 128, 128), (65536, 40, 128, 128), (8192, 32, 64, 64), (1000, 3, 17, 5)])
@pytest.mark.parametrize("backward", [False, True])
def test_it_does_not_grow_with_the_sequences(L, heads, dk, dv, backward):
    one = floats(L, 1, heads, dk, dv, backward=backward)
    for seqs in (2, 13, 256, 2048):
        assert floats(L, seqs, heads, dk, dv, backward=backward) == one
    # packed or not, a state lies between neighbouring segments of at least 128 positions, and a position has three sums
    states = (L // 128) * heads * (dk * dv + 1) * (2 if backward else 1) + 16
    assert one <= states + (3 * (L + 4) * heads if backward else 0)


def test_large_packing_is_small():
    # 65536 positions of 40 heads of 128 x 128 in 2048 sequences: 2.7 GB of q, k, v and outputs in 16 bits
    assert floats(65536, 2048, 40, 128, 128) * 4 < 60e6
    assert floats(65536, 2048, 40, 128, 128, backward=True) * 4 < 140e6


def test_states_between_segments_have_places_of_their_own():
    """The numbering of the kernels, on the CPU: distinct, and below (seqlen - 1) / seg, for any boundaries."""
    rng = random.Random(0)
    for _ in range(300):
        L, seg = rng.randint(1, 5000), 64 * rng.randint(1, 6)
        ends = sorted(rng.randint(0, L) for _ in range(rng.randint(1, 60)))
        seen = set()
        for first, end in zip(ends, ends[1:]):
            segs = -(-(end - first) // seg)
            for p in range(1, segs):
                place = first // seg + p - 1
                assert 0 <= place < (L - 1) // seg and place not in seen
                seen.add(place)
