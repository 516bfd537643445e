"""The sampler where top_k is more than its lists hold, on rows of mostly distinct
logits: the last one kept is found in its bin by a list, then top_p's among the bins,
then the token by both and min_p. Against sorting in float64; tokens are equal.

A weight is rounded to a unit of 2^-s, s = 62 - log2 V (V up to a power of two), the
largest being 1: a sum before a border is off by at most V 2^-(s+1), 2^-29 at 131072.
A random number lies that near one of the row's V borders with a probability below
V 2^-28 / (the row's sum): 10^-6 a row for the 131072 normal logits here, whose sum is
in the hundreds and more, 3 10^-4 for the peaked ones, whose sum is 1 to 5, if every
rounding fell to one side (sqrt(V) times less if not). None of the fixed seeds here is
such a one."""

import pytest
import torch

from nested_recurrent_memory_amd.model_ops import sample_tokens
from test_sample_gpu import BF16, F32, check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["normal", "peaked", "masked"])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V", [1000, 8193, 32001, 131072])
def test_more_kept_than_a_list_holds(V, dtype, kind):
    for j, k in enumerate((256, 257, 300, 1000, V - 1)):
        for i, kw in enumerate((dict(), dict(top_p=0.95), dict(top_p=0.995, min_p=1e-4), dict(min_p=1e-5),
                                dict(temperature=3.0, top_p=0.999, min_p=1e-3))):
            l, u = make(3, V, dtype, kind, seed=10 * j + i)
            check(l, u, top_k=k, **kw)


def test_fewer_logits_than_top_k():
    """Rows masked down to fewer than top_k, to one and to a few equal ones."""
    for dtype in (F32, BF16):
        l, u = make(5, 20000, dtype)
        order = torch.rand(5, 20000, generator=torch.Generator().manual_seed(1)).argsort(1)
        for row, n in enumerate((1, 200, 299, 1500, 19999)):
            l[row, order[row, n:]] = -float("inf")
        l[1][l[1] > -float("inf")] = 0.5
        for k in (300, 2000, 19998):
            for kw in (dict(), dict(top_p=0.9), dict(top_p=0.97, min_p=1e-3)):
                check(l, u, top_k=k, **kw)


def test_more_than_256_pass_min_p_behind_a_cut():
    """Both borders inside what is kept: the oracle's count of it says so."""
    l, u = make(4, 32001, F32, "normal", seed=4)
    w = (l.double() - l.double().max(1, keepdim=True).values).exp().sort(1, descending=True).values
    assert (w[:, 999] > 2e-3).all() and ((w[:, :1500] >= 0.05).sum(1) > 256).all()
    for k in (300, 1000, 1500):
        for floor in (0.02, 0.05, 0.06):
            for top_p in (1.0, 0.999, 0.9):
                check(l, u, top_k=k, top_p=top_p, min_p=floor)


@pytest.mark.parametrize("V,s", [(131072, 45), (131073, 44), (2048, 51), (9, 51)])
def test_a_weight_is_rounded_to_its_unit(V, s):
    """The random number 0 takes the first token that weighs anything: one of 0.6 units
    weighs one, one of 0.4 none (a logit near -30 in fp32 holds its weight to 2^-19)."""
    l = torch.full((2, V), -float("inf"), dtype=torch.float64)
    l[:, 8] = 0.0
    l[:, 3] = torch.tensor([0.6, 0.4], dtype=torch.float64).log() - s * torch.tensor(2.0, dtype=torch.float64).log()
    got = sample_tokens(l.float().cuda(), torch.zeros(2, device="cuda"))
    assert got.tolist() == [3, 8]
