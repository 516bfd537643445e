"""The model's options for its residual path, and its sampling, on the CPU: what
the config refuses, the parameters they add, and that they survive a checkpoint."""

import pytest
import torch

from nested_recurrent_memory_amd.model import NestedGDN2Config, NestedGDN2ForCausalLM


def _config(**kw):
    return NestedGDN2Config(**dict(dict(vocab_size=64, hidden_size=64, num_hidden_layers=2, num_heads=1, head_dim=64,
                                        n_queries_per_level=(16,)), **kw))


def test_config_refuses():
    for p in (-0.1, 1.5):
        with pytest.raises(ValueError, match="resid_dropout"):
            _config(resid_dropout=p)
    for kw in (dict(post_norm=True), dict(layer_scale=0.1), dict(branch_scale=0.5), dict(resid_dropout=0.1)):
        with pytest.raises(ValueError, match="need fuse_norm"):
            _config(fuse_norm=False, **kw)
    assert _config(fuse_norm=False).fuse_norm is False


def test_parameters_and_round_trip(tmp_path):
    plain = set(NestedGDN2ForCausalLM(_config()).state_dict())
    cfg = _config(post_norm=True, layer_scale=0.25, branch_scale=0.5, resid_dropout=0.1)
    m = NestedGDN2ForCausalLM(cfg)
    new = {f"model.layers.{i}.{n}" for i in range(2)
           for n in ("attn_post_norm.weight", "mlp_post_norm.weight", "attn_gate", "mlp_gate")}
    assert set(m.state_dict()) == plain | new
    assert all((p == 0.25).all() for n, p in m.named_parameters() if n.endswith("_gate"))
    with torch.no_grad():
        for p in m.parameters():
            p.add_(0.01 * torch.randn_like(p))
    m.save_pretrained(tmp_path)
    again = NestedGDN2ForCausalLM.from_pretrained(tmp_path)
    for n in ("post_norm", "layer_scale", "branch_scale", "resid_dropout"):
        assert getattr(again.config, n) == getattr(cfg, n)
    for n, t in m.state_dict().items():
        assert torch.equal(again.state_dict()[n], t), n


def test_sample_refuses_other_numbers_of_random_numbers():
    m = NestedGDN2ForCausalLM(_config())
    with pytest.raises(ValueError, match="sample: u"):
        m.sample(torch.zeros(2, 3, dtype=torch.long), 4, u=torch.rand(2, 3))
