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


@pytest.mark.parametrize("N", [1, 77, 128, 129, 600])
@pytest.mark.parametrize("std", [1.0, 4.0])
def test_gradient_of_a_lone_key_is_zero(gpu, N, std):
    """The softmax over one key is 1 whatever its logit: dq and dk are 0 to the
    last bit, dv is the sum of do.  q_len * heads large enough that a key tile
    of the member is cut among blocks, too."""
    import torch

    for seed in range(90, 94):
        B, S, H, Hk = 3, 700, 6, 2
        lens = [1, N, 1]
        q, k, v, do = base._inputs(B, S, N, H, Hk, seed, std=std)
        got = base._run_cross(q, k, v, lens, do)
        base._check_attention(q, k, v, lens, got, do, one_block=N <= 128)
        for b in (0, 2):
            assert (got["dq"][b] == 0).all(), (seed, b, got["dq"][b].abs().max().item())
            assert (got["dk"][b] == 0).all(), (seed, b, got["dk"][b].abs().max().item())


@pytest.mark.parametrize("N", [1, 200])
def test_gradient_of_a_lone_key_is_zero_in_millions_of_rows(gpu, N):
    """P dP / P is dP in all but a few rows in a million, whose dS is a last
    bit of dP: those too come out as 0."""
    q, k, v, do = base._inputs(1, 65536, N, 40, 40, 3, std=4.0)
    got = base._run_cross(q, k, v, [1], do)
    assert (got["dq"] == 0).all() and (got["dk"] == 0).all()


@pytest.mark.parametrize("N", [128, 300])
def test_gradient_of_rows_with_one_key_of_weight(gpu, N):
    """Rows whose every other weight is 0 in fp32, with logits of 5,792 to 11,585:
    lse is off by 2^-24 of that, so the one weight by up to 2^-9, but dS is 0.  With up to
    128 keys delta is P dP / P, two roundings from dP: dS is at most 2^-22 |dP| then.
    dk takes dP from a product of its own: its 128 additions are off by at most
    2^-23 of the sum of magnitudes each, 2^-16 in all, as is the first one's."""
    import torch

    lens, S, H = [128, 100, 65, 64, 20], 200, 2
    B = len(lens)
    _, _, v, do = base._inputs(B, S, N, H, H, 95)
    g = base._gen(96)
    k = torch.where(torch.rand(B, N, H, base.D, device="cuda", generator=g) < 0.5, -32.0, 32.0).to(torch.bfloat16)
    at = torch.stack([torch.randint(0, n, (S,), device="cuda", generator=g) for n in lens])
    member = torch.arange(B, device="cuda")[:, None]
    size = torch.randint(64, 129, (B, S, H, 1), device="cuda", generator=g) / 128
    q, hot = (k[member, at] * size).to(torch.bfloat16), v[member, at]
    got = base._run_cross(q, k, v, lens, do)
    assert torch.equal(got["out"], hot)
    dp, mag = (do.double() * hot.double()).sum(-1), (do.double().abs() * hot.double().abs()).sum(-1)
    bound = 32 * base.SCALE * (2.0 ** -22 * dp.abs())[..., None]
    over = (got["dq"].double().abs() - bound).amax((1, 2, 3))
    assert (over <= 0).all(), over.tolist()
    rows = torch.zeros(B, N, H, device="cuda", dtype=torch.float64)
    for b in range(B):
        rows[b].index_add_(0, at[b], 2.0 ** -22 * dp[b].abs() + 2.0 ** -15 * mag[b])
    over = (got["dk"].double().abs() - 32 * base.SCALE * rows[..., None]).amax((1, 2, 3))
    assert (over <= 0).all(), over.tolist()
