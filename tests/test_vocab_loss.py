"""Losses over a vocabulary (ops/vocab_loss.py) on CPU tensors: values and gradients against torch's own
losses and against differences, and the refusals."""
import math

import pytest
import torch
import torch.nn.functional as F

from determined_1_amd.ops.vocab_loss import linear_cross_entropy, linear_topk_distill, topk_distill


def _head(n=7, d=5, v=11, dtype=torch.float64):
    g = torch.Generator().manual_seed(n * 100 + v)
    x, w, b = (torch.randn(*s, generator=g, dtype=torch.float64).to(dtype) for s in ((n, d), (v, d), (v,)))
    return x, w, b, g


def _lists(n, v, k, g):
    index = torch.stack([torch.randperm(v, generator=g)[:k] for _ in range(n)])
    return torch.randn(n, k, generator=g, dtype=torch.float64), index


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("smooth", [0.0, 0.2, 1.0])
def test_cross_entropy_is_torchs(reduction, smooth):
    x, w, b, g = _head()
    t = torch.randint(0, 11, (7,), generator=g)
    t[2] = -100
    got = linear_cross_entropy(x, w, t, b, label_smoothing=smooth, reduction=reduction)
    ref = F.cross_entropy(F.linear(x, w, b), t, label_smoothing=smooth, reduction=reduction)
    torch.testing.assert_close(got, ref)


@pytest.mark.parametrize("heat", [1.0, 2.5])
def test_distill_is_torchs_divergence(heat):
    x, w, b, g = _head()
    teacher, index = _lists(7, 11, 4, g)
    q = torch.zeros(7, 11, dtype=torch.float64).scatter_(1, index, torch.softmax(teacher / heat, 1))
    z = F.linear(x, w, b)
    ref = heat * heat * F.kl_div(F.log_softmax(z / heat, 1), q, reduction="none").sum(1)
    for got in (topk_distill(z, teacher, index, temperature=heat, reduction="none"),
                linear_topk_distill(x, w, teacher, index, b, temperature=heat, reduction="none")):
        torch.testing.assert_close(got, ref)
    torch.testing.assert_close(topk_distill(z, teacher, index.int(), temperature=heat), ref.mean())


def test_gradients_against_differences():
    x, w, b, g = _head(4, 3, 6)
    t = torch.tensor([5, -100, 0, 2])
    teacher, index = _lists(4, 6, 3, g)
    index[1, 1:] = -1
    index[2] = -1
    teacher[3, 0] = -math.inf
    leaves = [a.requires_grad_(True) for a in (x, w, b)]
    for red in ("mean", "sum", "none"):
        assert torch.autograd.gradcheck(lambda x, w, b: linear_cross_entropy(x, w, t, b, label_smoothing=0.1, reduction=red), leaves)
        assert torch.autograd.gradcheck(lambda x, w, b: linear_topk_distill(x, w, teacher, index, b, temperature=2.0, reduction=red),
                                        leaves)
        assert torch.autograd.gradcheck(lambda z: topk_distill(z, teacher, index, temperature=2.0, reduction=red),
                                        [F.linear(x, w, b).detach().requires_grad_(True)])


def test_rows_without_a_target():
    x, w, b, g = _head()
    x.requires_grad_(True)
    t = torch.full((7,), -1)
    loss = linear_cross_entropy(x, w, t, ignore_index=-1)
    assert loss.item() == 0.0
    loss.backward()
    assert torch.equal(x.grad, torch.zeros_like(x))
    teacher, index = _lists(7, 11, 3, g)
    assert linear_topk_distill(x, w, teacher, index * 0 - 1).item() == 0.0
    assert linear_topk_distill(x, w, torch.full_like(teacher, -math.inf), index).item() == 0.0
    # an ignored row's values do not matter, whatever they are
    with torch.no_grad():
        x[3] = math.nan
    w.requires_grad_(True)
    index[3] = -1
    for loss in (linear_cross_entropy(x, w, torch.tensor([1, 2, 3, -100, 5, 6, 7])), linear_topk_distill(x, w, teacher, index)):
        assert math.isfinite(loss.item())
        assert all(torch.isfinite(g).all() for g in torch.autograd.grad(loss, [x, w]))


def test_words_outside_the_vocabulary_are_nan():
    x, w, b, g = _head()
    t = torch.tensor([0, 1, 11, 3, -7, 5, 6])
    rows = linear_cross_entropy(x, w, t, reduction="none")
    assert rows.isnan().tolist() == [False, False, True, False, True, False, False]
    teacher, index = _lists(7, 11, 3, g)
    index[4, 1] = 11
    assert topk_distill(F.linear(x, w), teacher, index, reduction="none").isnan().tolist() == [False] * 4 + [True] + [False] * 2


def test_a_word_twice_adds_up():
    x, w, _, g = _head()
    z = F.linear(x, w)
    teacher = torch.tensor([[1.0, 2.0, 2.0]], dtype=torch.float64).expand(7, 3)
    index = torch.tensor([[4, 9, 9]]).expand(7, 3)
    once = topk_distill(z, torch.tensor([[1.0, 2.0 + math.log(2.0)]], dtype=torch.float64).expand(7, 2), index[:, :2], reduction="none")
    got = topk_distill(z, teacher, index, reduction="none")
    q = torch.softmax(teacher[0], 0)  # two entries of q / 2 each: the entropy of the split is log 2 less
    torch.testing.assert_close(got + 2 * q[1] * math.log(2.0), once)


def test_empty_batch_and_leading_shapes():
    x, w, b, _ = _head()
    w.requires_grad_(True)
    loss = linear_cross_entropy(x[:0], w, torch.zeros(0, dtype=torch.long))
    loss.backward()
    assert loss.item() == 0.0 and torch.equal(w.grad, torch.zeros_like(w))
    assert linear_cross_entropy(x[:0], w, torch.zeros(0, dtype=torch.long), reduction="none").shape == (0,)
    assert topk_distill(x[:0], x[:0, :2], torch.zeros(0, 2, dtype=torch.long)).item() == 0.0
    t = torch.arange(6).reshape(2, 3)
    assert linear_cross_entropy(x[:6].reshape(2, 3, 5), w, t, reduction="none").shape == (2, 3)
    assert linear_cross_entropy(x[0], w, torch.tensor(3), reduction="none").shape == ()
    lists = torch.zeros(2, 3, 4), torch.arange(4).expand(2, 3, 4)
    assert linear_topk_distill(x[:6].reshape(2, 3, 5), w, *lists, reduction="none").shape == (2, 3)
    assert topk_distill(torch.zeros(2, 3, 8), *lists, reduction="none").shape == (2, 3)


def test_losses_of_half_types_are_fp32():
    x, w, b, g = _head(dtype=torch.bfloat16)
    assert linear_cross_entropy(x, w, torch.arange(7), b.float()).dtype == torch.float32


@pytest.mark.parametrize("error,change", [
    (ValueError, dict(reduction="average")),
    (ValueError, dict(label_smoothing=1.5)),
    (ValueError, dict(hold_bytes=-1)),
    (ValueError, dict(hold_bytes=0.5)),
    (ValueError, dict(target=torch.zeros(6, dtype=torch.long))),
    (ValueError, dict(target=torch.zeros(7, 1, dtype=torch.long))),
    (TypeError, dict(target=torch.zeros(7))),
    (ValueError, dict(weight=torch.zeros(11, 4))),
    (ValueError, dict(weight=torch.zeros(0, 5))),
    (ValueError, dict(weight=torch.zeros(11, 5, 1))),
    (TypeError, dict(weight=torch.zeros(11, 5, dtype=torch.bfloat16))),
    (TypeError, dict(x=torch.zeros(7, 5, dtype=torch.long))),
    (ValueError, dict(bias=torch.zeros(10))),
    (TypeError, dict(bias=torch.zeros(11, dtype=torch.bfloat16))),
    (ValueError, dict(weight=torch.zeros(11, 5, device="meta"))),
])
def test_cross_entropy_refuses(error, change):
    args = dict(x=torch.zeros(7, 5), weight=torch.zeros(11, 5), target=torch.zeros(7, dtype=torch.long), bias=None)
    args.update(change)
    with pytest.raises(error, match="linear_cross_entropy"):
        linear_cross_entropy(**args)


@pytest.mark.parametrize("error,change", [
    (ValueError, dict(reduction="batchmean")),
    (ValueError, dict(temperature=0.0)),
    (ValueError, dict(temperature=math.inf)),
    (ValueError, dict(temperature=math.nan)),
    (ValueError, dict(teacher_index=torch.zeros(7, 2, dtype=torch.long))),
    (ValueError, dict(teacher_index=torch.zeros(7, 0, dtype=torch.long), teacher_logits=torch.zeros(7, 0))),
    (ValueError, dict(teacher_index=torch.zeros(6, 3, dtype=torch.long), teacher_logits=torch.zeros(6, 3))),
    (TypeError, dict(teacher_index=torch.zeros(7, 3, dtype=torch.int16))),
    (TypeError, dict(teacher_logits=torch.zeros(7, 3, dtype=torch.long))),
])
def test_distill_refuses(error, change):
    args = dict(teacher_logits=torch.zeros(7, 3), teacher_index=torch.zeros(7, 3, dtype=torch.long))
    args.update(change)
    with pytest.raises(error, match="topk_distill"):
        topk_distill(torch.zeros(7, 11), **args)
    with pytest.raises(error, match="linear_topk_distill"):
        linear_topk_distill(torch.zeros(7, 5), torch.zeros(11, 5), **args)
    with pytest.raises(TypeError, match="topk_distill"):
        topk_distill(torch.zeros(7, 11, dtype=torch.long), torch.zeros(7, 3), torch.zeros(7, 3, dtype=torch.long))
