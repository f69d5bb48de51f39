"""norm.residual_modulate's gradients where only some of the rows' are asked for: the same bits, None for the others."""

import itertools

import pytest
import torch

from flicker_amd import autograd, norm
from tests.test_gpu_residual import _operands

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("width", [5, 40, 1000, 2000, 9000])
@pytest.mark.parametrize("wanted", list(itertools.product((False, True), repeat=3)))
def test_wanted(device, width, wanted):
    x, branch, dr, dy, rows = _operands(1, 2, 37, width, "bf16", "fp32", device)
    every = norm.residual_modulate_backward(dr, dy, x, branch, *rows)
    some = norm.residual_modulate_backward(dr, dy, x, branch, *rows, wanted=wanted)
    assert torch.equal(some[0], every[0]) and torch.equal(some[1], every[1])
    for got, want, asked in zip(some[2:], every[2:], wanted, strict=True):
        assert (got is None) == (not asked) and (got is None or torch.equal(got, want))
    none = norm.residual_modulate_backward(dr[:, :0], dy[:, :0], x[:, :0], branch[:, :0], *rows, wanted=wanted)
    assert [t is not None for t in none[2:]] == list(wanted) and not any(t.any() for t in none[2:] if t is not None)


@pytest.mark.parametrize("wanted", list(itertools.product((False, True), repeat=3)))
def test_autograd_asks_for_what_it_needs(device, monkeypatch, wanted):
    x, branch, dr, dy, rows = _operands(2, 2, 9, 64, "fp32", "fp32", device)
    asked = []
    backward = norm.residual_modulate_backward
    monkeypatch.setattr(norm, "residual_modulate_backward", lambda *a, **kw: (asked.append(kw["wanted"]), backward(*a, **kw))[1])
    want = backward(dr, dy, x, branch, *rows)
    leaves = [x.clone().requires_grad_(), branch.clone(), *(t.clone().requires_grad_(w) for t, w in zip(rows, wanted))]
    r, y = autograd.residual_modulate(*leaves)
    torch.autograd.backward((r, y), (dr, dy))
    assert asked == [wanted]
    for leaf, grad in zip(leaves, want):
        assert leaf.grad is None if not leaf.requires_grad else torch.equal(leaf.grad, grad)


def test_wanted_takes_three(device):
    x, branch, dr, dy, rows = _operands(3, 1, 4, 64, "bf16", "bf16", device)
    with pytest.raises(ValueError):
        norm.residual_modulate_backward(dr, dy, x, branch, *rows, wanted=(True, False))
