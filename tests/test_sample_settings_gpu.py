"""Settings a row outside their ranges."""

import pytest
import torch

from nested_recurrent_memory_amd.model_ops import sample_tokens

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name,bad", [("temperature", (-0.5, float("inf"), float("nan"))),
                                      ("top_p", (-0.1, 1.5, float("inf"), float("nan"))),
                                      ("min_p", (-0.1, 1.5, float("inf"), float("nan")))])
def test_values_outside_their_ranges_give_no_token(name, bad):
    """Of a tensor; the same values as numbers are refused."""
    l = torch.randn(len(bad) + 2, 300, generator=torch.Generator().manual_seed(2)).cuda()
    u = torch.full((len(bad) + 2,), 0.4, device="cuda")
    v = torch.tensor((0.0, *bad, 1.0), device="cuda")
    for kw in (dict(), dict(top_k=20)):
        got = sample_tokens(l, u, **{name: v}, **kw).tolist()
        assert got[1:-1] == [-1] * len(bad) and got[0] >= 0 and got[-1] >= 0
    for b in bad:
        with pytest.raises(ValueError, match=name):
            sample_tokens(l, u, **{name: b})
