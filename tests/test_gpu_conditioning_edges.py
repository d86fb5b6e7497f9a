"""Conditioning calls at the edges of their work units (B200 only).

Values are held to the bounds of ``test_gpu_conditioning``, whose plain
restatements in 64 bits are used here too; bitwise comparisons are between
calls of the same sizes, which the operators answer alike.
"""
import pytest

import test_gpu_conditioning as base

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,S,N,H,lens", [
    # more units than SMs; blocks of 8, 160, 224 and 129 rows are some units' last,
    # and the unit after one of them has a member without keys
    (2, 520, 512, 40, [512, 0]), (2, 416, 300, 80, [300, 77]), (2, 480, 128, 80, [0, 128]), (3, 385, 640, 50, [640, 0, 5]),
], ids=lambda x: "-".join(map(str, x)) if isinstance(x, list) else str(x))
def test_dense_rows_beside_units_of_part_tiles(gpu, B, S, N, H, lens):
    """A unit whose last rows leave some of a tile's warps without any must not
    touch what the unit before it is still writing out."""
    import torch

    q, k, v, _ = base._inputs(B, S, N, H, H, 70)
    first = base._run_cross(q, k, v, lens)
    base._check_attention(q, k, v, lens, first)
    for _ in range(30):
        again = base._run_cross(q, k, v, lens)
        assert torch.equal(again["out"], first["out"]) and torch.equal(again["lse"], first["lse"])
