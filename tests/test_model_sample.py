"""What the model's sample() does around the model and the sampler, on the CPU: both
are stand-ins that say what they were given."""

import types

import pytest
import torch
import torch.nn as nn

from nested_recurrent_memory_amd import model as model_module
from nested_recurrent_memory_amd.model import NestedGDN2Config, NestedGDN2ForCausalLM


class Stand(nn.Module):
    def __init__(self):
        super().__init__()
        self.given = []

    def forward(self, input_ids, **kw):
        self.given.append(input_ids.clone())
        return types.SimpleNamespace(last_hidden_state=torch.zeros(*input_ids.shape, 64), past_key_values=None)


@pytest.fixture
def stand(monkeypatch):
    """(a model, what its layers were given, tokens [steps][B] for the sampler to give)"""
    m = NestedGDN2ForCausalLM(NestedGDN2Config(vocab_size=64, hidden_size=64, num_hidden_layers=1, num_heads=1,
                                               head_dim=64, n_queries_per_level=(16,)))
    m.model = Stand()
    tokens = []
    monkeypatch.setattr(model_module, "sample_tokens", lambda *a: torch.tensor(tokens.pop(0)))
    return m, m.model.given, tokens


@pytest.mark.parametrize("eos", [None, 9])
def test_a_sequence_without_a_token_goes_on_with_minus_one(stand, eos):
    """And the model is given ids of its vocabulary alone: what a lookup of another
    reads is not said, and outside the table's memory."""
    m, given, tokens = stand
    tokens += [[5, -1, 6], [9, 7, -1], [3, -1, 8], [4, 2, 1]]
    ids = torch.tensor([[1, 2], [3, 4], [5, 6]])
    got = m.sample(ids, 4, u=torch.rand(3, 4), eos_token_id=eos)
    want = [[5, 9, 3, 4] if eos is None else [5, 9, 9, 9], [-1, -1, -1, -1], [6, -1, -1, -1]]
    assert got[:, :2].tolist() == ids.tolist() and got[:, 2:].tolist() == want
    assert len(given) == 4 and torch.equal(given[0], ids)
    assert all(t.shape == (3, 1) and (t >= 0).all() and (t < 64).all() for t in given[1:])
    assert [t[0].item() for t in given[1:]] == want[0][:3]


def test_sampling_in_training_mode_is_refused_where_it_would_drop(stand):
    """With dropout the same u would not give the same tokens, and checkpointing's
    layers keep no cache. Without either, and in evaluation, the mode is no matter."""
    m, given, tokens = stand
    ids, u = torch.tensor([[1, 2]]), torch.rand(1, 1)

    def tokens_of(**kw):
        tokens[:] = [[5]]
        return m.sample(ids, 1, u=u, **kw).tolist()

    assert m.train() and tokens_of() == [[1, 2, 5]]
    m.model.layers = nn.ModuleList([model_module.NestedGDN2Block(NestedGDN2Config(
        vocab_size=64, hidden_size=64, num_hidden_layers=1, num_heads=1, head_dim=64, n_queries_per_level=(16,),
        resid_dropout=0.1), 0)])
    for mode in (m, m.model.layers[0]):
        mode.train()
        state = torch.get_rng_state()
        with pytest.raises(RuntimeError, match="eval"):
            tokens_of()
        assert torch.equal(state, torch.get_rng_state()) and m.model.layers[0].training
        m.eval()
        assert tokens_of() == [[1, 2, 5]]
    m.train()
    m.model.layers[0].eval()
    assert tokens_of() == [[1, 2, 5]]
    m.model.layers[0].resid_dropout = 0.0
    m.train()
    assert tokens_of() == [[1, 2, 5]]
    m.model.layers[0].gradient_checkpointing = True
    with pytest.raises(RuntimeError, match="eval"):
        tokens_of()
    m.eval()
    assert tokens_of() == [[1, 2, 5]]
