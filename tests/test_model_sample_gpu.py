"""The model's sample() where a sequence's logits have no answer."""

import pytest
import torch
import torch.nn as nn

from test_model_residual_gpu import DEV, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("table", ["own", "torch"])
def test_a_sequence_without_a_token_leaves_the_others(table):
    m = make().eval()
    if table == "torch":
        new = nn.Embedding(512, 128, device=DEV)
        new.weight.data.copy_(m.model.embeddings.weight)
        m.set_input_embeddings(new)
    g = torch.Generator(DEV).manual_seed(3)
    ids = torch.randint(8, 512, (3, 11), device=DEV, generator=g)
    u = torch.rand(3, 6, device=DEV, generator=g)
    want = m.sample(ids, 6, u=u, top_k=40)
    with torch.no_grad():
        m.get_input_embeddings().weight[7] = float("inf")
    assert not (want[:, 11:] == 7).any()          # the others read another row
    ids[1, 4] = 7
    got = m.sample(ids, 6, u=u, top_k=40)
    assert torch.equal(got[[0, 2]], want[[0, 2]])
    assert got[1].tolist() == ids[1].tolist() + [-1] * 6
