"""The sampler against sorting in float64: tokens are equal. The two sums differ
by less than 2^-40 of the whole (weights in units of 2^-42 at least, sums of V
roundings in float64), so a random number lies between their borders with a
probability below V 2^-40 a row: none of the fixed seeds here does."""

import pytest
import torch

import ngdn_residual_oracle as oracle
from nested_recurrent_memory_amd.model_ops import residual_norm, sample_tokens

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def make(B, V, dtype=F32, kind="normal", seed=0):
    g = torch.Generator().manual_seed(seed * 31 + B * 7 + V)
    l = torch.randn(B, V, generator=g)
    if kind == "peaked":
        l = 12 - 1.6 * (torch.rand(B, V, generator=g).argsort(1) + 1.0).log() + l
    elif kind == "ties":
        l = (2 * l).round()
    elif kind == "equal":
        l = torch.full((B, V), 3.25)
    elif kind == "wide":
        l = 1e4 * l
    elif kind == "narrow":
        l = 1e-4 * l + 5
    elif kind == "masked":
        l = torch.where(torch.rand(B, V, generator=g) < 0.9, -float("inf"), l)
    elif kind == "lowest":
        l = torch.where(torch.rand(B, V, generator=g) < 0.5, torch.finfo(dtype).min, l)
    return l.to(dtype), torch.rand(B, generator=g)


def check(l, u, **kw):
    got = sample_tokens(l.cuda(), u.cuda(), **{k: v.cuda() if torch.is_tensor(v) else v for k, v in kw.items()})
    assert got.dtype == torch.int64 and got.shape == u.shape
    want = oracle.sample(l.reshape(-1, l.shape[-1]), u.reshape(-1), **kw).view(u.shape)
    assert torch.equal(got.cpu(), want), (got.cpu()[got.cpu() != want], want[got.cpu() != want])
    return got


SETTINGS = [dict(), dict(temperature=0.0), dict(temperature=0.7, top_k=1), dict(top_k=5), dict(top_k=50, top_p=0.9),
            dict(temperature=1.3, top_p=0.95), dict(top_p=0.3), dict(top_p=0.0), dict(min_p=0.1), dict(min_p=1.0),
            dict(temperature=0.8, top_k=40, top_p=0.95, min_p=0.05), dict(top_k=10 ** 12, top_p=1.0),
            dict(temperature=1e-30), dict(temperature=1e30, top_k=7, top_p=0.5)]
KINDS = ["normal", "peaked", "ties", "equal", "wide", "narrow", "masked", "lowest"]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("V", [1, 2, 7, 8, 9, 64, 1000, 8191, 8192, 8193, 32001])
def test_settings(V, dtype, kind):
    if kind == "wide" and dtype == F16:
        kind = "normal"
    B = 6 if V < 5000 else 3
    for i, kw in enumerate(SETTINGS):
        l, u = make(B, V, dtype, kind, seed=i)
        check(l, u, **kw)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V", [65536, 131072, 200003, 1 << 20])
def test_large_vocabularies(V, dtype):
    for i, kw in enumerate(SETTINGS[3:6] + SETTINGS[10:11]):
        l, u = make(2, V, dtype, "peaked" if i % 2 else "normal", seed=i)
        check(l, u, **kw)


@pytest.mark.parametrize("kind", ["normal", "peaked", "ties", "equal"])
def test_every_place_is_reached(kind):
    """Random numbers over the whole interval on one row: its ends, and the first
    and the last token."""
    l, _ = make(1, 300, F32, kind)
    u = torch.cat((torch.linspace(0, 1, 2000)[:-1], torch.tensor([1 - 2.0 ** -24]))).float()
    for kw in SETTINGS[:6]:
        check(l.expand(2000, 300), u, **kw)
    d = torch.linspace(0, 1, 999, dtype=torch.float64)
    check(l.expand(999, 300), d, top_p=0.9)


def test_settings_of_each_request():
    B, V = 200, 5000
    g = torch.Generator().manual_seed(5)
    for dtype, kint in ((BF16, torch.int32), (F32, torch.int64)):
        l, u = make(B, V, dtype, "peaked")
        t = torch.rand(B, generator=g) * 1.5
        t[::7] = 0
        k = torch.randint(-3, 100, (B,), generator=g).to(kint)
        p = torch.rand(B, generator=g)
        p[::3] = 1
        m = torch.rand(B, generator=g) * 0.2
        m[::2] = 0
        want = check(l, u, temperature=t, top_k=k, top_p=p, min_p=m)
        # one row at a time: the same tokens, whatever the others are
        one = [sample_tokens(l[i:i + 1].cuda(), u[i:i + 1].cuda(), t[i].item(), int(k[i]), p[i].item(), m[i].item())
               for i in range(0, B, 17)]
        assert torch.equal(torch.cat(one), want[::17])
        # other types of settings, and one for all
        check(l, u, temperature=t.double().float(), top_k=torch.tensor(30), top_p=torch.tensor(0.75))


def test_rows_without_an_answer():
    inf, nan = float("inf"), float("nan")
    l = torch.zeros(6, 40)
    l[0] = -inf
    l[1, 5] = inf
    l[2, 39] = nan
    l[3, :39] = -inf
    l[4, 0] = -nan
    u = torch.full((6,), 0.5)
    for kw in SETTINGS:
        got = check(l, u, **kw).tolist()
        assert got[:3] == [-1, -1, -1] and got[3] == 39 and got[4] == -1 and got[5] >= 0
    for bad in (-1.0, inf, nan):
        t = torch.ones(6)
        t[5] = bad
        assert check(l, u, temperature=t)[5] == -1
    for name, bad in (("top_p", -0.1), ("top_p", nan), ("min_p", -0.1), ("min_p", 1.5), ("min_p", nan)):
        v = torch.ones(6)
        v[5] = bad
        assert check(l, u, **{name: v})[5] == -1
    for bad in (-0.1, 1.5, nan):
        u[5] = bad
        assert check(l, u)[5] == -1


def test_zeros_of_both_signs_are_equal():
    l = torch.zeros(4, 20)
    l[:, ::2] = -0.0
    for kw in (dict(top_k=3), dict(top_p=0.25), dict(temperature=0.0)):
        check(l, torch.tensor([0.0, 0.3, 0.6, 0.99]), **kw)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_many_equal_logits_of_both_signs(dtype):
    """More equal ones than a list holds in the bin where the last one kept is, on
    either side of zero, and few values in all."""
    g = torch.Generator().manual_seed(9)
    for V in (3000, 40000):
        l = (1e-3 * torch.randint(-3, 4, (5, V), generator=g)).to(dtype)
        l[3] = l[3].abs()
        l[4] = -l[4].abs() - 1
        for kw in (dict(top_k=V // 3), dict(top_k=V // 2), dict(top_k=6 * V // 7), dict(top_p=0.1), dict(top_p=0.45),
                   dict(top_p=0.6), dict(top_p=0.95), dict(top_k=V // 2, top_p=0.9), dict(temperature=0.0)):
            for u in (torch.rand(5, generator=g), torch.zeros(5), torch.full((5,), 1 - 2.0 ** -24)):
                check(l, u, **kw)


def test_strided_rows():
    """The last position of prompts, a vocabulary padded in memory, a row that
    starts at an odd value, columns, more dimensions, none."""
    l, u = make(12, 777, BF16, "peaked")
    kw = dict(top_k=20, top_p=0.9)
    want = check(l, u, **kw)
    x = torch.full((12, 5, 777), 60.0, dtype=BF16, device="cuda")
    x[:, -1] = l.cuda()
    assert torch.equal(sample_tokens(x[:, -1], u.cuda(), **kw), want)
    x = torch.full((12, 1001), 60.0, dtype=BF16, device="cuda")
    x[:, 3:780] = l.cuda()
    assert torch.equal(sample_tokens(x[:, 3:780], u.cuda(), **kw), want)
    assert torch.equal(sample_tokens(l.cuda().t().contiguous().t(), u.cuda(), **kw), want)
    assert torch.equal(sample_tokens(l.cuda().view(3, 4, 777), u.cuda().view(3, 4), **kw), want.view(3, 4))
    assert torch.equal(sample_tokens(l[5].cuda(), u[5].cuda(), **kw), want[5])
    assert torch.equal(sample_tokens(l[:1].cuda().expand(9, 777), u[:1].cuda().expand(9), **kw), want[:1].expand(9))
    assert sample_tokens(l[:0].cuda(), u[:0].cuda()).shape == (0,)


def test_frequencies():
    """200000 draws of 12 tokens: each count within five standard deviations of
    its expectation (of 12 counts, one outside has a probability of 7e-6; the
    seed is fixed)."""
    l = torch.tensor([0.0, 1.0, -1.0, 2.0, 0.5, -3.0, 1.5, 0.1, 0.2, -0.5, 2.5, -2.0])
    n = 200000
    u = torch.rand(n, generator=torch.Generator().manual_seed(3))
    got = torch.bincount(sample_tokens(l.cuda().expand(n, 12), u.cuda(), 0.9).cpu(), minlength=12).double()
    p = torch.softmax(l.double() / 0.9, 0)
    assert ((got - n * p).abs() <= 5 * (n * p * (1 - p)).sqrt()).all()


def test_captured_in_a_graph_and_on_another_stream():
    l, u = make(9, 4000, BF16, "peaked")
    sl, su = l.cuda(), u.cuda()
    t = torch.full((9,), 0.8, device="cuda")
    work = lambda: sample_tokens(sl, su, t, 30, 0.9)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = work()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, work())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = work()
    for i in range(4):
        l, u = make(9, 4000, BF16, "peaked", seed=i + 1)
        sl.copy_(l)
        su.copy_(u)
        t.fill_(0.5 + 0.2 * i)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, work())
        assert torch.equal(out.cpu(), oracle.sample(l, u, temperature=t.cpu(), top_k=30, top_p=0.9))


def test_a_token_after_a_block():
    """The last residual norm of a model, its logits, and the token, for each of a
    batch: what a generated token passes behind the mixer, in one captured graph."""
    g = torch.Generator().manual_seed(2)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    x, b, w, pw, gate, head = r(5, 64), r(5, 64), 1 + 0.1 * r(64), 1 + 0.1 * r(64), r(64), r(500, 64)
    cu = [t.cuda() for t in (x, b, w, pw, gate, head)]
    u = torch.rand(5, generator=g)
    su = u.cuda()

    def work():
        h, y = residual_norm(cu[0], cu[1], cu[2], post_weight=cu[3], gate=cu[4])
        logits = y @ cu[5].t()
        return logits, sample_tokens(logits, su, 0.8, 40, 0.9)

    work()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        logits, token = work()
    for i in range(3):
        su.copy_(torch.rand(5, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(token, work()[1])
        assert torch.equal(token.cpu(), oracle.sample(logits.cpu(), su.cpu(), temperature=0.8, top_k=40, top_p=0.9))
    y = oracle.residual_norm(x, b, w, pw, gate)["y"][0]
    # a dot product of 64 fp32 terms and the norm's own error, on logits of order 10
    assert (logits.cpu().double() - y @ head.double().t()).abs().max() < 1e-3


def test_rows_far_apart():
    """Rows 2^31 values and more from each other."""
    l, u = make(3, 1000, BF16, "peaked")
    x = torch.empty(2 * ((1 << 31) + 77) + 1000, dtype=BF16, device="cuda")
    rows = x.as_strided((3, 1000), ((1 << 31) + 77, 1))
    rows.copy_(l)
    assert torch.equal(sample_tokens(rows, u.cuda(), top_k=30, top_p=0.9).cpu(), oracle.sample(l, u, top_k=30, top_p=0.9))


def test_tensors_of_transforms_are_refused():
    l, u = torch.randn(3, 40, device="cuda"), torch.rand(3, device="cuda")
    with pytest.raises((RuntimeError, ValueError)):
        torch.func.vmap(lambda a, b: sample_tokens(a, b))(l, u)
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode() as mode:
        with pytest.raises(RuntimeError):
            sample_tokens(mode.from_tensor(l), mode.from_tensor(u))
        with pytest.raises((RuntimeError, AssertionError)):           # the mode's own for tensors not of it
            sample_tokens(l, u)


def test_logits_that_require_a_gradient():
    l, u = make(4, 300)
    x = l.cuda().requires_grad_(True)
    token = sample_tokens(x, u.cuda())
    assert not token.requires_grad and torch.equal(token.cpu(), oracle.sample(l, u))
