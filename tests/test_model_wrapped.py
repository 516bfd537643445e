"""Layers of the model that are not its blocks themselves, on the CPU: a replacement
with the signature that a block had before it could do more with its output than add
it, in a model none of whose layers does."""

import pytest
import torch
import torch.nn as nn

from nested_recurrent_memory_amd.model import NestedGDN2Config, NestedGDN2Model


class Replacement(nn.Module):
    def __init__(self, scale):
        super().__init__()
        self.scale = scale

    def forward(self, hidden_states, residual=None, past_key_values=None, use_cache=False, defer_residual=False):
        assert defer_residual
        if residual is not None:
            hidden_states = hidden_states + residual
        return hidden_states, self.scale * hidden_states, past_key_values


@pytest.mark.parametrize("output_hidden_states", [False, True])
def test_replacement_layers(output_hidden_states):
    m = NestedGDN2Model(NestedGDN2Config(vocab_size=64, hidden_size=64, num_hidden_layers=3, num_heads=1, head_dim=64,
                                         n_queries_per_level=(16,), fuse_norm=False))
    for i, scale in enumerate((0.5, -0.25, 2.0)):       # 1 + scale: sums without rounding of few bits
        m.layers[i] = Replacement(scale)
    x = torch.randint(-8, 9, (2, 5, 64)).float()
    out = m(inputs_embeds=x, use_cache=False, output_hidden_states=output_hidden_states, return_dict=True)
    want = [x, 1.5 * x, 1.125 * x, 3.375 * x]
    assert torch.equal(out.last_hidden_state, m.norm(want[-1]))
    if output_hidden_states:
        assert all(torch.equal(a, b) for a, b in zip(out.hidden_states, want[:3]))


NEW = ("post_norm", "layer_scale", "branch_scale", "resid_dropout")


def test_a_config_without_the_options():
    """The reference's config, or one pickled before this package had them."""
    cfg = NestedGDN2Config(vocab_size=64, hidden_size=64, num_hidden_layers=1, num_heads=1, head_dim=64,
                           n_queries_per_level=(16,))
    want = set(NestedGDN2Model(cfg).state_dict())
    for n in NEW:
        delattr(cfg, n)
    m = NestedGDN2Model(cfg)
    assert set(m.state_dict()) == want
    assert m.layers[0].branch("attn") == m.layers[0].branch("mlp") == (None, None)
    x, y = torch.randn(2, 3, 64), torch.randn(2, 3, 64)
    assert torch.equal(m.layers[0].join(x, y, (None, None)), x + y)


def test_a_model_pickled_before_the_options(tmp_path):
    """Its blocks have none of their attributes."""
    m = NestedGDN2Model(NestedGDN2Config(vocab_size=64, hidden_size=64, num_hidden_layers=1, num_heads=1, head_dim=64,
                                         n_queries_per_level=(16,)))
    for n in ("plain", "branch_scale", "resid_dropout"):
        del m.layers[0].__dict__[n]
    torch.save(m, tmp_path / "model.pt")
    block = torch.load(tmp_path / "model.pt", weights_only=False).layers[0]
    x, y = torch.randn(2, 3, 64), torch.randn(2, 3, 64)
    assert torch.equal(block.join(x, y, block.branch("mlp")), x + y)
