"""The model with norms after its blocks, gates, scales and dropout, and its
sampling. The same model with the residual path in plain torch gives the same loss
and gradients (fp32, norm-wise 1e-5, the bar of the fused norms' test: a model of
two layers whose other kernels are the same)."""

import pytest
import torch

import ngdn_residual_oracle as oracle
from nested_recurrent_memory_amd import model as model_module
from nested_recurrent_memory_amd.model import NestedGDN2Config, NestedGDN2ForCausalLM
from nested_recurrent_memory_amd.model_ops import dropout

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
EVERY = dict(post_norm=True, layer_scale=0.5, branch_scale=0.7)


def make(seed=0, **kw):
    torch.manual_seed(seed)
    m = NestedGDN2ForCausalLM(NestedGDN2Config(
        **dict(dict(vocab_size=512, hidden_size=128, num_hidden_layers=2, num_heads=2, head_dim=64, num_levels=2,
                    firing_intervals=(1, 2), n_queries_per_level=(16,)), **kw))).to(DEV)
    with torch.no_grad():
        for p in m.parameters():
            p.add_(0.01 * torch.randn_like(p))
    return m


def plain_residual_norm(x, branch, weight=None, post_weight=None, gate=None, residual_scale=1.0, branch_scale=1.0,
                        p=0.0, seed=0, offset=0, eps=1e-5, out_dtype=None):
    norm = lambda v, w: v * torch.rsqrt(v.square().mean(-1, keepdim=True) + eps) * w  # noqa: E731
    z = branch.float()
    if post_weight is not None:
        z = norm(z, post_weight)
    if gate is not None:
        z = z * gate
    if p:
        z = torch.where(dropout(torch.ones_like(z), p, seed, offset) != 0, z / (1 - p), 0.0)
    h = residual_scale * x + branch_scale * z
    return h if weight is None else (h, norm(h, weight).to(out_dtype or h.dtype))


def step(m, ids, seed=5, **kw):
    torch.manual_seed(seed)
    loss = m(input_ids=ids, labels=ids, **kw).loss
    names = [n for n, p in m.named_parameters() if p.requires_grad]
    grads = torch.autograd.grad(loss, [p for p in m.parameters() if p.requires_grad], allow_unused=True)
    return loss.detach(), dict(zip(names, grads))


def rel(a, b):
    return ((a.double() - b.double()).norm() / b.double().norm().clamp_min(1e-30)).item()


@pytest.mark.parametrize("kw", [dict(post_norm=True), dict(layer_scale=0.3), dict(branch_scale=0.5),
                                dict(resid_dropout=0.2), dict(EVERY, resid_dropout=0.1)],
                         ids=["post", "gate", "scale", "dropout", "all"])
def test_against_the_path_in_plain_torch(kw, monkeypatch):
    m = make(**kw).train()
    ids = torch.randint(0, 512, (2, 192), device=DEV, generator=torch.Generator(DEV).manual_seed(1))
    loss, grads = step(m, ids)
    monkeypatch.setattr(model_module, "residual_norm", plain_residual_norm)
    want, wgrads = step(m, ids)
    assert abs(loss.item() - want.item()) <= 1e-5 * abs(want.item())
    for n, g in wgrads.items():
        assert (g is None) == (grads[n] is None), n
        if g is not None:
            assert rel(grads[n], g) <= 1e-5, (n, rel(grads[n], g))
    if "layer_scale" in kw:
        assert grads["model.layers.1.mlp_gate"].abs().max() > 0


def test_dropout_in_training_only():
    ids = torch.randint(0, 512, (2, 128), device=DEV)
    m, base = make(**EVERY, resid_dropout=0.3), make(**EVERY)
    base.load_state_dict(m.state_dict())
    a, b, c = (step(m.train(), ids, seed=s)[0] for s in (1, 1, 2))
    assert torch.equal(a, b) and not torch.equal(a, c)
    with torch.no_grad():
        assert torch.equal(m.eval()(ids).logits, base.eval()(ids).logits)


@pytest.mark.parametrize("reentrant", [False, True])
def test_gradient_checkpointing_drops_the_same(reentrant):
    m = make(**EVERY, resid_dropout=0.2).train()
    ids = torch.randint(0, 512, (2, 128), device=DEV)

    def grads():
        torch.manual_seed(3)
        m.zero_grad()
        loss = m(input_ids=ids, labels=ids).loss
        loss.backward()
        return loss.detach(), {n: p.grad.clone() for n, p in m.named_parameters() if p.grad is not None}

    loss, want = grads()
    m.gradient_checkpointing_enable(dict(use_reentrant=reentrant))
    m.model.embeddings.weight.requires_grad_(True)
    again, got = grads()
    assert torch.equal(loss, again) and set(got) == set(want)
    for n in want:
        assert rel(got[n], want[n]) <= 1e-5, n


def test_a_captured_join_drops_other_values_on_each_replay():
    block = make(resid_dropout=0.25).train().model.layers[0]
    x, out = torch.zeros(64, 128, device=DEV), torch.ones(64, 128, device=DEV)
    params = block.branch("attn")

    def work():
        with torch.no_grad():
            return block.join(x, out, params, block.mlp_norm)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        h, y = work()
    seen = []
    for _ in range(4):
        g.replay()
        torch.cuda.synchronize()
        kept = h != 0
        assert torch.equal(h[kept], torch.full_like(h[kept], 1 / 0.75))
        # 8192 draws: five standard deviations are 0.024
        assert abs(kept.double().mean().item() - 0.75) < 0.024
        seen.append(kept.clone())
        work()
    assert all(not torch.equal(a, b) for i, a in enumerate(seen) for b in seen[:i])


@pytest.mark.parametrize("autocast", [False, True])
def test_bf16(autocast):
    """Autocast (an fp32 stream) and a bf16 model: a finite loss, close to fp32's."""
    m = make(**EVERY, resid_dropout=0.1).train()
    ids = torch.randint(0, 512, (2, 128), device=DEV)
    want, _ = step(m, ids)
    if autocast:
        with torch.autocast("cuda", dtype=torch.bfloat16):
            got, grads = step(m, ids)
    else:
        got, grads = step(m.to(torch.bfloat16), ids)
    assert abs(got.item() - want.item()) <= 2e-2 * want.item()
    assert all(torch.isfinite(g).all() for g in grads.values() if g is not None)


def test_hidden_states_are_the_stream():
    m = make(**EVERY).eval()
    ids = torch.randint(0, 512, (1, 70), device=DEV)
    with torch.no_grad():
        out = m(ids, output_hidden_states=True)
        # fused into the next norm or not: y may be formed from a sum that was not rounded
        # (fp32: the same up to an fp32 rounding)
        torch.testing.assert_close(out.logits, m(ids).logits, rtol=1e-4, atol=1e-5)
        h, cache = m.model.layers[0](out.hidden_states[0])
        torch.testing.assert_close(out.hidden_states[1], h, rtol=1e-5, atol=1e-6)


def test_a_block_called_alone():
    m = make(**EVERY).eval()
    x = torch.randn(1, 64, 128, device=DEV)
    with torch.no_grad():
        h, mlp, _ = m.model.layers[0](x, defer_residual=True)
        want, _ = m.model.layers[0](x)
        got = plain_residual_norm(h, mlp, None, *m.model.layers[0].branch("mlp"), branch_scale=0.7)
    torch.testing.assert_close(got, want, rtol=1e-5, atol=1e-6)


# ---------------------------------------------------------------- sampling

@pytest.mark.parametrize("kw", [dict(), EVERY], ids=["plain", "all"])
def test_greedy_is_generate(kw):
    m = make(**kw).eval()
    ids = torch.randint(0, 512, (1, 37), device=DEV)
    got = m.sample(ids, 12, temperature=0.0)
    want = m.generate(ids, max_new_tokens=12, do_sample=False, use_cache=True, pad_token_id=0)
    assert torch.equal(got, want)


def test_sample_draws_what_the_sampler_draws():
    """Step by step: each token is the sampler's of that step's logits, each
    request with its own settings; the same numbers give the same tokens."""
    m = make(**EVERY).eval()
    g = torch.Generator(DEV).manual_seed(4)
    ids = torch.randint(0, 512, (3, 20), device=DEV, generator=g)
    u = torch.rand(3, 8, device=DEV, generator=g)
    kw = dict(temperature=torch.tensor([0.0, 0.8, 1.5], device=DEV), top_k=torch.tensor([0, 40, 5], device=DEV),
              top_p=0.95, min_p=0.001)
    got = m.sample(ids, 8, u=u, **kw)
    assert torch.equal(got, m.sample(ids, 8, u=u, **kw)) and got.shape == (3, 28)
    seen, cache = ids, None
    with torch.no_grad():
        for i in range(8):
            out = m(seen if cache is None else seen[:, -1:], past_key_values=cache, use_cache=True)
            cache = out.past_key_values
            token = oracle.sample(out.logits[:, -1].cpu(), u[:, i].cpu(),
                                  **{k: v.cpu() if torch.is_tensor(v) else v for k, v in kw.items()})
            seen = torch.cat((seen, token.to(DEV)[:, None]), 1)
    assert torch.equal(got, seen)


def test_sample_ends():
    m = make().eval()
    ids = torch.randint(0, 512, (2, 9), device=DEV)
    u = torch.rand(2, 30, device=DEV, generator=torch.Generator(DEV).manual_seed(1))
    free = m.sample(ids, 30, u=u, top_k=3)
    eos = free[0, 12].item()
    got = m.sample(ids, 30, u=u, top_k=3, eos_token_id=eos)
    for b in range(2):
        new = free[b, 9:].tolist()
        n = new.index(eos) + 1 if eos in new else 30
        row = got[b, 9:].tolist()
        assert row[:n] == new[:n] and all(t == eos for t in row[n:])
    a = m.sample(ids, 5, generator=torch.Generator(DEV).manual_seed(7))
    assert torch.equal(a, m.sample(ids, 5, generator=torch.Generator(DEV).manual_seed(7)))
    assert m.sample(ids, 0).shape == (2, 9)
