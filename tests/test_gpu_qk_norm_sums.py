"""The weights' gradients of the q/k norm over many rows (B200 only): sums that
run over tokens, members and blocks, held tightly enough to miss a row.

A term g x r is off by 2^-20 of the magnitudes that enter it (as in
``test_gpu_conditioning``).  The kernel chains its additions: the rows of one
group of eight threads (a warp's runs of 4 << shift rows, shift <= 3, spread over
at most 2 x 148 blocks of 8 warps), the 32 groups of a block, every eighth block
and those eight.  Each addition is off by at most 2^-24 of the sum of magnitudes.
"""
import pytest

import test_gpu_conditioning as base

pytestmark = pytest.mark.gpu


def _depth(rows):
    """Additions on the way of a row to its sum, at most."""
    return 8 * -(-rows // (2 * 148 * 8 * 4 * 8)) + 8 + 32 + 37 + 8


def _contributions(x, w, table, eps, grad):
    """Every row's share of dw and its magnitude, [B, S, H, 128] in 64 bits."""
    x, g = x.double(), grad.double()
    unit = x / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    mag = g.abs()
    if table is not None:
        t = table.double()[None, :, None]
        h = t.shape[-2]
        a, b = g[..., :h].clone(), g[..., h:2 * h].clone()
        g, mag = g.clone(), mag.clone()
        g[..., :h], g[..., h:2 * h] = t[..., 0] * a + t[..., 2] * b, t[..., 1] * a + t[..., 3] * b
        t, a, b = t.abs(), a.abs(), b.abs()
        mag[..., :h], mag[..., h:2 * h] = t[..., 0] * a + t[..., 2] * b, t[..., 1] * a + t[..., 3] * b
    return g * unit, mag * unit.abs()


# (batch, tokens, heads, half): rows a warp of 4, 8, 16 and 32, the last runs cut
SIZES = [(3, 601, 5, 64), (3, 6001, 5, 64), (20001, 1, 1, 64), (2, 40001, 1, 48), (2, 9001, 5, 33), (1, 32768, 40, None)]


@pytest.mark.parametrize("B,S,H,half", SIZES, ids=lambda x: str(x))
def test_weight_gradients_hold_every_row(gpu, B, S, H, half):
    import torch

    g = base._gen(97)
    x, grad = base._normal(g, B, S, H, base.D), base._normal(g, B, S, H, base.D)
    w = base._normal(g, base.D, mean=1.0, std=0.5)
    tab = None if half is None else base._rope(S, half, 98)
    dx, dw, dwk = torch.empty_like(x), torch.empty(base.D, device="cuda"), torch.empty(base.D, device="cuda")
    terms, mags = _contributions(x, w, tab, 1e-5, grad)
    terms, mags = terms.reshape(-1, base.D), mags.reshape(-1, base.D)
    rows = terms.shape[0]

    def run(grad):
        base._rt().qk_norm_rope_bwd(q=x, k=x, q_grad=grad, k_grad=grad, q_norm=w, k_norm=w, dq=dx, dk=dx.clone(),
                                    dq_norm=dw, dk_norm=dwk, eps=1e-5, q_rope=tab, k_rope=tab)
        assert torch.equal(dw, dwk)

    run(grad)
    tol = (2.0 ** -20 + 2.0 ** -24 * _depth(rows)) * mags.sum(0)
    if rows < 200000:  # the bound sees a row that is left out, in a tenth of the channels at least
        assert (terms.abs() > tol).double().mean() > 0.1
    base._assert_within("dw", dw, terms.sum(0), tol)
    # one row alone, at the ends of runs, tokens, members and the operand: a
    # gradient of 0 elsewhere adds nothing, so it is held to its own 2^-20
    lone = torch.zeros_like(grad)
    flat, given = lone.view(-1, base.D), grad.view(-1, base.D)
    for row in sorted({r for at in (0, 32, 32 * 2368, S * H, rows) for r in (at - 33, at - 5, at - 4, at - 1, at, at + 3)
                       if 0 <= r < rows}):
        flat[row] = given[row]
        run(lone)
        flat[row] = 0
        base._assert_within(f"dw of row {row}", dw, terms[row], 2.0 ** -20 * mags[row] + 1e-38)
