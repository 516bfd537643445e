"""Settings of the sampler that are neither numbers nor tensors, on the CPU."""

import numpy as np
import pytest
import torch

from nested_recurrent_memory_amd.model_ops import sample_tokens


class Raises:
    def __index__(self):
        raise KeyError("of its own")


def test_a_top_k_that_is_no_integer_raises_its_own_error():
    """An array of several has __index__, which raises; the call must not go on."""
    l, u = torch.randn(2, 5), torch.rand(2)
    with pytest.raises(TypeError, match="integer"):
        sample_tokens(l, u, 1.0, np.array([1, 2]))
    with pytest.raises(KeyError, match="of its own"):
        sample_tokens(l, u, 1.0, Raises())
    for k in (3, np.int64(3), np.array(3), True, -2 ** 70, 2 ** 70):        # integers: on to the next check
        with pytest.raises(ValueError, match="no CPU path"):
            sample_tokens(l, u, 1.0, k)
    for bad in (np.array([0.5, 0.5]), "0.5", None):
        with pytest.raises(TypeError):
            sample_tokens(l, u, bad)
