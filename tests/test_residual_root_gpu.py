"""The reciprocal root of a row's mean square, where every step before it is exact."""

import pytest
import torch

from nested_recurrent_memory_amd.model_ops import residual_norm

pytestmark = pytest.mark.gpu


def test_reciprocal_roots_are_rounded_once():
    """Rows of one value of 12 bits, eps 0: its square and the root of that are exact
    in fp32, so 1 / sqrt is the value's reciprocal, rounded once, and y = h times that
    one rounding more. Each way: the norm of the sum, and the norm of the branch."""
    x = torch.cat([(torch.arange(2048, 4096) * 2.0 ** e) for e in (-20, -11, 3)]).float().reshape(-1, 1)
    want = x * (1 / x.double()).float()
    one, zero = torch.ones(1, device="cuda"), torch.zeros_like(x).cuda()
    h, y = residual_norm(x.cuda(), zero, one, eps=0.0)
    assert torch.equal(h.cpu(), x) and torch.equal(y.cpu(), want)
    assert torch.equal(residual_norm(zero, x.cuda(), post_weight=one, eps=0.0).cpu(), want)


def test_rows_whose_mean_square_has_no_root():
    """Zeros with eps 0 (1 / 0 is infinite, times 0 is NaN) and squares beyond fp32
    (their mean is infinite, its reciprocal root 0), as the formula in fp32 gives them."""
    x = torch.tensor([[0.0, 0.0], [3e38, 0.0], [1e-30, 0.0], [1.0, 1.0]])
    want = x * torch.rsqrt((x * x).mean(-1, keepdim=True))
    one = torch.ones(2, device="cuda")
    y = residual_norm(x.cuda(), torch.zeros_like(x).cuda(), one, eps=0.0)[1].cpu()
    assert torch.equal(torch.isnan(y), torch.isnan(want)) and torch.equal(y[1], torch.zeros(2))
    assert torch.equal(torch.isinf(y), torch.isinf(want)) and torch.equal(y[3], torch.ones(2))
