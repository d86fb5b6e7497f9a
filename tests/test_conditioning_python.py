"""Refusals of the Python forms of the conditioning calls that need no device."""
import pytest


def _operands(d=128):
    import torch

    return [torch.zeros(n, 2, d, dtype=torch.bfloat16) for n in (3, 5, 5)]


@pytest.mark.parametrize("which", [0, 1, 2])
def test_cross_sdpa_refuses_to_lose_a_gradient(which):
    import torch

    from h3attention import cross_sdpa

    x = _operands()
    x[which].requires_grad_()
    with pytest.raises(ValueError, match="gives no gradients"):
        cross_sdpa(*x, 128)
    with torch.no_grad(), pytest.raises(ValueError, match="must be a CUDA tensor"):
        cross_sdpa(*x, 128)


def test_cross_sdpa_refuses_another_head_dim():
    """The scale follows from head_dim: one that is not the operands' would scale wrongly."""
    from h3attention import cross_sdpa

    with pytest.raises(ValueError, match="head_dim 64, got 128"):
        cross_sdpa(*_operands(), 64)
