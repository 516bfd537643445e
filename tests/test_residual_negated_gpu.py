"""Tensors whose memory holds the negatives of their values: the imaginary part of a
conjugate, which of one value is contiguous, and torch's view of that kind."""

import pytest
import torch

import ngdn_residual_oracle as oracle
from nested_recurrent_memory_amd.model_ops import dropout, residual_norm, sample_tokens
from test_residual_gpu import NAMES, TYPES, close, make

pytestmark = pytest.mark.gpu


def negated(t):
    n = torch._neg_view((-t).cuda())
    assert n.is_neg() and torch.equal(n.cpu(), t)
    return n


def test_dropout_of_negated_views():
    one = torch.tensor([3 + 4j], device="cuda").conj().imag
    assert one.is_neg() and one.is_contiguous()
    assert dropout(one, 2.0 ** -32, 3).item() == -4.0
    x, dy = torch.randn(5, 7), torch.randn(5, 7)
    assert torch.equal(dropout(negated(x), 0.4, 3), dropout(x.cuda(), 0.4, 3))
    xg = x.cuda().requires_grad_(True)
    for g in (negated(dy), dy.cuda()):
        dx, = torch.autograd.grad(dropout(xg, 0.4, 3), xg, g)
        assert torch.equal(dx, dropout(dy.cuda(), 0.4, 3))


def test_residual_norm_of_negated_views():
    a, dh, dy = make((3, 4, 40), TYPES[0], "full")
    leaf = {n: negated(a[n]).requires_grad_(True) for n in NAMES}
    h, y = residual_norm(**leaf)
    want = oracle.residual_norm(**a, dh=dh, dy=dy)
    close("h", h, want["h"], torch.float32)
    close("y", y, want["y"], torch.float32)
    for n, t in zip(NAMES, torch.autograd.grad([h, y], list(leaf.values()), [negated(dh), negated(dy)])):
        close("d" + n, t, want["d" + n], torch.float32)
    with torch.no_grad():
        assert torch.equal(residual_norm(**leaf)[1], y)


def test_sample_tokens_of_negated_views():
    g = torch.Generator().manual_seed(1)
    l, u, t, p = torch.randn(4, 300, generator=g), torch.rand(4, generator=g), 0.5 + torch.rand(4), torch.rand(4)
    want = sample_tokens(l.cuda(), u.cuda(), t.cuda(), 40, p.cuda())
    assert torch.equal(sample_tokens(negated(l), negated(u), negated(t), 40, negated(p)), want)
    assert torch.equal(sample_tokens(negated(l)[:, 3:], u.cuda()), sample_tokens(l[:, 3:].cuda(), u.cuda()))
