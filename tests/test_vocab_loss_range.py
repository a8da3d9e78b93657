"""Losses over a vocabulary on CPU tensors (ops/vocab_loss.py) where there are no rows, where values are infinite, and at the
ends of the arguments' ranges."""
import math

import pytest
import torch

from determined_1_amd.ops.vocab_loss import linear_cross_entropy, linear_topk_distill, topk_distill


def _head(n=7, d=5, v=11, dtype=torch.float64):
    g = torch.Generator().manual_seed(n * 100 + v)
    return tuple(torch.randn(*s, generator=g, dtype=torch.float64).to(dtype) for s in ((n, d), (v, d), (v,)))


@pytest.mark.parametrize("junk", [math.inf, math.nan])
def test_no_rows_are_zero_whatever_the_weights_hold(junk):
    x, w, b = _head()
    w[3], b[2] = junk, -math.inf
    leaves = [x[:0].requires_grad_(True), w.requires_grad_(True), b.requires_grad_(True)]
    none = torch.zeros(0, dtype=torch.long)
    for loss in (linear_cross_entropy(leaves[0], w, none, b), linear_topk_distill(leaves[0], w, torch.zeros(0, 2), none[:, None].expand(0, 2), b)):
        assert loss.item() == 0.0 and loss.dtype == torch.float64
        for leaf, grad in zip(leaves, torch.autograd.grad(loss, leaves)):
            assert torch.equal(grad, torch.zeros_like(leaf))
    assert linear_cross_entropy(x[:0].bfloat16(), w.detach().bfloat16(), none).dtype == torch.float32
    assert topk_distill(x[:0].bfloat16(), x[:0, :2], none[:, None].expand(0, 2)).dtype == torch.float32


def test_a_masked_target_that_does_not_count():
    """With a label smoothing of 1 the target has no share, so a masked one makes the loss infinite as any masked word
    does, and not NaN; one outside the vocabulary is NaN all the same."""
    x, w, b = _head()
    b[4] = -math.inf
    t = torch.tensor([4, 1, 2, 4, 11, 5, 6])
    loss = linear_cross_entropy(x, w, t, b, label_smoothing=1.0, reduction="none")
    assert loss.isnan().tolist() == [False] * 4 + [True] + [False] * 2 and (loss[:4] == math.inf).all()


@pytest.mark.parametrize("ignore", [2 ** 63, -2 ** 63 - 1, 2 ** 64 - 100])
def test_an_index_that_no_target_can_hold_is_refused(ignore):
    x, w, _ = _head()
    with pytest.raises(ValueError, match="linear_cross_entropy"):
        linear_cross_entropy(x, w, torch.arange(7), ignore_index=ignore)
    assert linear_cross_entropy(x, w, torch.arange(7), ignore_index=-2 ** 63).item() > 0
