"""Blocks inside a module that wraps them (as timing, logging and offloading do), and
blocks of two kinds in one model."""

import pytest
import torch
import torch.nn as nn

from nested_recurrent_memory_amd.model_ops import add_rms_norm
from test_model_residual_gpu import DEV, EVERY, make, step

pytestmark = pytest.mark.gpu


class Wrapper(nn.Module):
    def __init__(self, inner):
        super().__init__()
        self.inner = inner

    def forward(self, *args, **kw):
        return self.inner(*args, **kw)


@pytest.mark.parametrize("kw", [dict(), EVERY, dict(EVERY, resid_dropout=0.2)], ids=["plain", "options", "dropout"])
def test_wrapped_blocks(kw):
    """The same calls in the same order: the same bits."""
    m = make(num_hidden_layers=3, **kw).train()
    ids = torch.randint(0, 512, (2, 128), device=DEV)
    loss, grads = step(m, ids)
    with torch.no_grad():
        want = m.eval()(ids, output_hidden_states=True)
    for i in (0, 2):
        m.model.layers[i] = Wrapper(m.model.layers[i])
    again, got = step(m.train(), ids)
    got = {n.replace(".inner.", "."): g for n, g in got.items()}
    assert torch.equal(loss, again) and set(got) == set(grads)
    assert all((grads[n] is None and g is None) or torch.equal(grads[n], g) for n, g in got.items())
    with torch.no_grad():
        out = m.eval()(ids, output_hidden_states=True)
    assert torch.equal(out.logits, want.logits)
    assert all(torch.equal(a, b) for a, b in zip(out.hidden_states, want.hidden_states))


@pytest.mark.parametrize("first", [True, False])
def test_blocks_of_two_kinds(first):
    """Each output is added as its own block says, whatever the next one does: the
    blocks one after another, each called alone (fp32; a norm that is formed from the
    sum as it is written, or before: the same up to fp32 roundings)."""
    m, other = make(**EVERY).eval(), make(seed=1, branch_scale=0.3).eval()
    plain = make(seed=2).eval()
    m.model.layers[0 if first else 1] = plain.model.layers[0]
    m.model.layers.append(other.model.layers[1])
    ids = torch.randint(0, 512, (1, 70), device=DEV)
    with torch.no_grad():
        got = m.model(ids, use_cache=False, return_dict=True).last_hidden_state
        h = m.model.embeddings(ids)
        for layer in m.model.layers:
            h, _ = layer(h)
        _, want = add_rms_norm(h, torch.zeros_like(h), m.model.norm.weight, m.model.norm.eps)
    torch.testing.assert_close(got, want, rtol=1e-4, atol=1e-5)
