"""Packed linear attention: sequences of many segments between short and empty ones, and many sequences."""

from __future__ import annotations

import pytest
import torch

from test_attn_gpu import BF16, DEV, FP32, check_packed, compare, make, own

pytestmark = pytest.mark.gpu

ENDS = {
    "long between short": [0, 5, 5, 1300, 1301, 1364, 2600, 2600, 2792, 2800],
    "on the segments' grid": [0, 192, 384, 384, 1152, 1153, 2304, 2496],
    "one position beyond": [1, 194, 387, 388, 965, 1158, 1160, 2313],
}


@pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("which", ENDS)
def test_sequences_of_many_segments(which, dtype):
    ends = ENDS[which]
    check_packed(make(1, ends[-1] + (3 if ends[0] else 0), 2, 1, 48, 40, dtype, True, True, len(ends) - 1), ends)


def test_hundreds_of_sequences():
    """Some of several segments; a few of them are held to the definition."""
    lengths = [3 * (i % 7) + (900 if i % 40 == 39 else 0) for i in range(200)]
    ends = [0]
    for n in lengths:
        ends.append(ends[-1] + n)
    p = make(1, ends[-1], 2, 2, 64, 64, BF16, True, True, len(lengths))
    got = own(p, torch.tensor(ends, dtype=torch.int32, device=DEV))
    for i in (0, 1, 38, 39, 79, 80, 198, 199):
        a, b = ends[i], ends[i + 1]
        one = {n: None if t is None else (t[i:i + 1] if n in ("init", "dfinal") else t[:, a:b]) for n, t in p.items()}
        part = {n: t[i:i + 1] if n in ("final", "dinit") else t[:, a:b] for n, t in got.items()}
        compare(part, one, name=f"sequence {i} ")
