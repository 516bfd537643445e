"""Dropout and the residual norm against float64. Dropout's bits are compared
exactly where the arithmetic is one product; the residual norm's values within
the oracle's count of fp32 roundings and the one to their type."""

import math

import pytest
import torch

import ngdn_residual_oracle as oracle
from nested_recurrent_memory_amd.model_ops import dropout, residual_norm

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def half(dtype):
    return torch.finfo(dtype).eps / 2


def least(dtype):
    # half a step below the smallest normal number
    return {F16: 2.0 ** -25, BF16: 2.0 ** -134, F32: 2.0 ** -149}[dtype]


# ---------------------------------------------------------------- dropout

def drop_want(x, p, seed, offset):
    keep = oracle.kept(x.shape, p, seed, offset)
    return keep, torch.where(keep, x.double() / (1 - p) if p < 1 else 0 * x.double(), 0.0)


def check_drop(y, x, p, seed, offset):
    keep, want = drop_want(x, p, seed, offset)
    y = y.detach()
    assert y.dtype == x.dtype and y.shape == x.shape
    got = y.double().cpu()
    assert (got[~keep] == 0).all()
    # the factor's rounding, the product's, and the one to the type
    tol = (half(x.dtype) + 2 * 2.0 ** -24) * want.abs() + least(x.dtype)
    assert ((got - want).abs() <= tol).all()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("n", [1, 3, 4, 7, 8, 9, 255, 2047, 2048, 2050, 100003])
def test_dropout(n, dtype):
    x = torch.randn(n, generator=torch.Generator().manual_seed(n)).to(dtype)
    for p, seed, offset in ((0.1, 0, 0), (0.5, 12345678901, 1), (0.9, -1, 2 ** 40 + 3), (2.0 ** -32, 5, -7)):
        xg = x.cuda().requires_grad_(True)
        y = dropout(xg, p, seed, offset)
        check_drop(y, x, p, seed % 2 ** 64, offset % 2 ** 64)
        dy = torch.randn(n).to(dtype)
        dx, = torch.autograd.grad(y, xg, dy.cuda())
        check_drop(dx, dy, p, seed % 2 ** 64, offset % 2 ** 64)


def test_dropout_probabilities_at_the_ends():
    x = torch.tensor([1.0, float("inf"), float("nan"), -3.0], device="cuda")
    assert dropout(x, 0.0, 3) is x
    assert dropout(x, 2.0 ** -34, 3) is x
    assert torch.equal(dropout(x, 1.0, 3), torch.zeros(4, device="cuda"))
    xg = x.clone().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(dropout(xg, 1.0, 3), xg, x)[0], torch.zeros(4, device="cuda"))


def test_dropped_infinities_and_nan_are_zero():
    x = torch.full((4096,), float("nan"))
    x[::2] = float("inf")
    keep = oracle.kept(x.shape, 0.5, 9, 0)
    y = dropout(x.cuda(), 0.5, 9).cpu()
    assert (y[~keep] == 0).all() and not torch.isfinite(y[keep]).any()


def test_dropout_of_views():
    """Strided inputs and gradients, and rows that start at any value."""
    big = torch.randn(61, 34)
    for dtype in (F32, BF16):
        for view in (lambda t: t.t(), lambda t: t[1:, 3:20], lambda t: t.reshape(-1)[1:], lambda t: t[:, :1].expand(61, 9),
                     lambda t: t.reshape(-1)[5:6]):
            x = big.to(dtype)
            xg = x.cuda()
            check_drop(dropout(view(xg), 0.3, 4, 2), view(x), 0.3, 4, 2)
    assert dropout(big.cuda()[:0], 0.3, 4).shape == (0, 34)


def test_dropout_differentiated_again():
    x = torch.randn(5, 9, device="cuda", requires_grad=True)
    v = torch.randn(5, 9, device="cuda", requires_grad=True)
    t = torch.randn(5, 9, device="cuda")
    dx, = torch.autograd.grad(dropout(x, 0.4, 8), x, v, create_graph=True)
    dv, = torch.autograd.grad(dx, v, t)
    assert torch.equal(dv, dropout(t, 0.4, 8))


def test_dropout_seed_on_the_gpu_and_refusals():
    x = torch.randn(33, 10, device="cuda")
    s = torch.tensor([2 ** 62 + 9], device="cuda")
    assert torch.equal(dropout(x, 0.3, s, 5), dropout(x, 0.3, 2 ** 62 + 9, 5))
    xg = x.clone().requires_grad_(True)
    y = dropout(xg, 0.3, s)
    s.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, xg, x)
    with pytest.raises(ValueError, match="no CPU path"):
        dropout(x, 0.3, torch.tensor([3]))
    y = dropout(xg, 0.3, 1)
    with pytest.raises(RuntimeError, match="not supported"):
        torch.autograd.grad(y, xg, torch.ones(2, 33, 10, device="cuda"), is_grads_batched=True)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, x)
        with pytest.raises((RuntimeError, NotImplementedError)):
            dropout(dual, 0.3, 1)


def test_dropout_captured_with_a_seed_that_changes():
    x, dy = torch.randn(77, 30), torch.randn(77, 30)
    sx, sdy, seed = x.cuda(), dy.cuda(), torch.zeros(1, dtype=torch.long, device="cuda")

    def work():
        xg = sx.detach().requires_grad_(True)
        y = dropout(xg, 0.25, seed, 6)
        return y.detach(), torch.autograd.grad(y, xg, sdy)[0]

    g, out = captured(work)
    for i in range(4):
        seed.fill_(i * 1000003)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, work()))
        check_drop(out[0], x, 0.25, i * 1000003, 6)
        check_drop(out[1], dy, 0.25, i * 1000003, 6)


def captured(work):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = work()
    return g, out


# ---------------------------------------------------------------- the residual norm

GATES = [None, "channel", "sequence", "token", "full"]
NAMES = ("x", "branch", "weight", "post_weight", "gate")


def make(shape, types, gate=None, pre=True, post=True, params=F32, seed=0):
    g = torch.Generator().manual_seed(seed * 7919 + math.prod(shape) + shape[-1])
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    xd, rd, yd = types
    D = shape[-1]
    a = dict(x=r(*shape).to(xd), branch=(0.5 * r(*shape)).to(rd), weight=(1 + 0.1 * r(D)).to(params) if pre else None,
             post_weight=(1 + 0.1 * r(D)).to(params) if post else None, gate=None)
    gs = {None: None, "channel": (D,), "sequence": (shape[0],) + (1,) * (len(shape) - 2) + (D,),
          "token": shape[:-1] + (1,), "full": shape}[gate]
    if gs:
        a["gate"] = r(*gs).to(params if gate == "channel" else rd)
    return a, r(*shape).to(xd), r(*shape).to(yd)


def close(name, got, want, dtype):
    value, bound = want
    assert got.dtype == dtype and got.shape == value.shape, (name, got.dtype, got.shape)
    err = (got.detach().double().cpu() - value).abs()
    tol = bound * (1 + 2 * half(dtype)) + half(dtype) * value.abs() + least(dtype)
    assert (err <= tol).all(), (name, (err / tol.clamp(min=1e-300)).max().item(), err.max().item())


def check(a, dh, dy, types, with_dh=True, with_dy=True, **kw):
    pre = a["weight"] is not None
    yd = types[2]
    cu = {n: t.cuda().requires_grad_(True) if t is not None else None for n, t in a.items()}
    out = residual_norm(**cu, **kw, out_dtype=yd)
    h, y = out if pre else (out, None)
    want = oracle.residual_norm(**a, **kw, dh=dh if with_dh else None, dy=dy if with_dy and pre else None)
    close("h", h, want["h"], types[0])
    if pre:
        close("y", y, want["y"], yd)
    # without a gradient: the same bits
    with torch.no_grad():
        again = residual_norm(**cu, **kw, out_dtype=yd)
        assert torch.equal(h, again[0] if pre else again) and (not pre or torch.equal(y, again[1]))
    outs, grads = ([h] if with_dh else []) + ([y] if pre and with_dy else []), \
        ([dh.cuda()] if with_dh else []) + ([dy.cuda()] if pre and with_dy else [])
    names = [n for n in NAMES if a[n] is not None]
    got = torch.autograd.grad(outs, [cu[n] for n in names], grads)
    for n, t in zip(names, got):
        close("d" + n, t, want["d" + n], a[n].dtype)
    return got


TYPES = [(F32, F32, F32), (BF16, BF16, BF16), (F32, BF16, BF16), (F32, BF16, F32), (F32, F32, BF16)]


@pytest.mark.parametrize("types", TYPES, ids=["fff", "bbb", "fbb", "fbf", "ffb"])
@pytest.mark.parametrize("D", [1, 2, 5, 7, 8, 9, 12, 15, 64, 65, 100, 128, 200, 256, 260, 512, 515, 1001, 1024])
def test_widths(D, types):
    a, dh, dy = make((2, 3, D), types, "channel")
    check(a, dh, dy, types, residual_scale=0.7, branch_scale=1.3, p=0.2, seed=D, offset=3)


@pytest.mark.parametrize("types", [TYPES[0], TYPES[1]], ids=["fff", "bbb"])
@pytest.mark.parametrize("D", [2047, 2048, 4100, 8192, 8193, 10000, 16384])
def test_wide_rows(D, types):
    a, dh, dy = make((3, D), types, "token")
    check(a, dh, dy, types, p=0.1, seed=1)


@pytest.mark.parametrize("p", [0.0, 0.3])
@pytest.mark.parametrize("pre,post", [(True, True), (True, False), (False, True), (False, False)])
@pytest.mark.parametrize("gate", GATES)
@pytest.mark.parametrize("shape", [(3, 5, 36), (2, 7, 321), (1, 1, 1024), (2, 1, 515), (4, 2, 3, 20), (6, 40)])
def test_gates_and_norms(shape, gate, pre, post, p):
    types = TYPES[(len(shape) + pre + 2 * post) % len(TYPES)]
    a, dh, dy = make(shape, types, gate, pre, post)
    check(a, dh, dy, types, p=p, seed=11, offset=2 ** 33, branch_scale=0.5)


@pytest.mark.parametrize("which", ["dh", "dy"])
@pytest.mark.parametrize("gate", [None, "channel", "token"])
def test_one_output_differentiated(gate, which):
    """The other's gradient is none at all, not a tensor of zeros."""
    types = TYPES[0]
    a, dh, dy = make((2, 9, 40), types, gate)
    check(a, dh, dy, types, with_dh=which == "dh", with_dy=which == "dy")


@pytest.mark.parametrize("params", [BF16, F16])
def test_parameters_of_other_types(params):
    for types in (TYPES[0], TYPES[1]):
        a, dh, dy = make((4, 6, 72), types, "channel", params=params)
        check(a, dh, dy, types, p=0.1)


@pytest.mark.parametrize("types", [(F16, F16, F16), (F16, F32, BF16), (BF16, F32, BF16), (BF16, BF16, F32),
                                   (F32, F16, F16), (BF16, F16, F16)],
                         ids=lambda t: "-".join(str(d)[6:] for d in t))
def test_other_types(types):
    """fp16 and mixed types run in fp32: a value may be rounded twice on its way
    to its type, the first time to fp32 (which the bound counts)."""
    a, dh, dy = make((3, 4, 50), types, "full")
    check(a, dh, dy, types)


@pytest.mark.parametrize("rows,T", [(1, 1), (3000, 1), (1, 3000), (40, 75), (700, 4)])
def test_many_rows(rows, T):
    """More rows than the backward's workgroups take at once; sequences of few
    rows and many."""
    a, dh, dy = make((rows, T, 64), TYPES[2], "sequence")
    check(a, dh, dy, TYPES[2], p=0.1)
    a, dh, dy = make((rows, T, 520), TYPES[1], "channel")
    check(a, dh, dy, TYPES[1])


def test_strided_and_unaligned_inputs():
    types = TYPES[1]
    a, dh, dy = make((4, 6, 40), types, "full")
    for cut in (lambda t: t.transpose(0, 1), lambda t: t[:, 1:, 3:], lambda t: t[1:2]):
        b = {n: (cut(t) if t.dim() == 3 else t[:cut(a["x"]).shape[-1]]) if t is not None else None for n, t in a.items()}
        check(b, cut(dh), cut(dy), types, p=0.2, seed=5)
    # rows that start at an odd value of a buffer
    flat = torch.randn(1 + 3 * 40).to(BF16)
    b = dict(a, x=flat[1:].view(3, 40), branch=flat[:-1].view(3, 40), gate=None)
    cu = flat.cuda()
    h, y = residual_norm(cu[1:].view(3, 40), cu[:-1].view(3, 40), b["weight"].cuda(), b["post_weight"].cuda())
    want = oracle.residual_norm(**b)
    close("h", h, want["h"], BF16)
    close("y", y, want["y"], BF16)


def test_no_rows():
    for gate in GATES:
        a, dh, dy = make((2, 0, 24), TYPES[0], gate)
        cu = {n: t.cuda().requires_grad_(True) if t is not None else None for n, t in a.items()}
        h, y = residual_norm(**cu)
        assert h.shape == y.shape == (2, 0, 24)
        names = [n for n in NAMES if a[n] is not None]
        for n, t in zip(names, torch.autograd.grad([h, y], [cu[n] for n in names], [dh.cuda(), dy.cuda()])):
            assert t.shape == a[n].shape and (t == 0).all(), n


def test_infinities_and_nan():
    """A row's NaN stays in the row (and in the sums over rows); a dropped one
    without a norm on the branch reaches nothing."""
    a, _, _ = make((5, 64), TYPES[0], post=False)
    keep = oracle.kept((5, 64), 0.5, 2, 0)
    clean = a["branch"].clone()
    a["branch"][~keep] = float("nan")
    a["branch"][1][keep[1]] = clean[1][keep[1]]
    got = [residual_norm(a["x"].cuda(), b.cuda(), a["weight"].cuda(), p=0.5, seed=2) for b in (a["branch"], clean)]
    for t, w in zip(*got):
        assert torch.equal(t, w)
    a["x"][2, 7] = float("inf")
    a["x"][3, 1] = float("nan")
    h, y = residual_norm(a["x"].cuda(), clean.cuda(), a["weight"].cuda())
    ok = [0, 1, 4]
    assert torch.isfinite(h[ok]).all() and torch.isfinite(y[ok]).all()
    assert torch.isnan(y[3]).all() and h[2, 7] == float("inf")


def test_zero_rows_and_all_dropped():
    a, dh, dy = make((4, 48), TYPES[0], "channel")
    a["branch"][1] = 0
    a["x"][2] = 0
    a["branch"][2] = 0
    check(a, dh, dy, TYPES[0])
    a, dh, dy = make((4, 48), TYPES[0], "full")
    check(a, dh, dy, TYPES[0], p=1.0)


def test_unwanted_gradients_are_not_formed():
    a, dh, dy = make((3, 5, 33), TYPES[0], "channel")
    every = check(a, dh, dy, TYPES[0])
    for only in range(5):
        cu = {n: a[n].cuda().requires_grad_(i == only) for i, n in enumerate(NAMES)}
        h, y = residual_norm(**cu)
        t, = torch.autograd.grad([h, y], [cu[NAMES[only]]], [dh.cuda(), dy.cuda()])
        assert torch.equal(t, every[only]), NAMES[only]


def test_gradient_twice_and_other_transforms_are_refused():
    a, dh, dy = make((3, 20), TYPES[0])
    x = a["x"].cuda().requires_grad_(True)
    h, y = residual_norm(x, a["branch"].cuda(), a["weight"].cuda())
    dx, = torch.autograd.grad(y, x, dy.cuda(), create_graph=True)
    with pytest.raises(RuntimeError, match="cannot be differentiated again"):
        dx.sum().backward()
    h, y = residual_norm(x, a["branch"].cuda(), a["weight"].cuda())
    with pytest.raises(RuntimeError, match="not supported"):
        torch.autograd.grad(y, x, torch.ones(2, 3, 20, device="cuda"), is_grads_batched=True)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x.detach(), x.detach())
        with pytest.raises((RuntimeError, NotImplementedError)):
            residual_norm(dual, a["branch"].cuda(), a["weight"].cuda())


def test_inputs_changed_between_the_passes_are_noticed():
    a, dh, dy = make((3, 20), TYPES[0])
    x = a["x"].cuda()
    b = a["branch"].cuda().requires_grad_(True)
    h, y = residual_norm(x, b, a["weight"].cuda())
    x.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, b, dy.cuda())


def test_same_bits_every_run():
    a, dh, dy = make((7, 300, 515), TYPES[2], "channel")
    runs = []
    for _ in range(3):
        cu = {n: t.cuda().requires_grad_(True) for n, t in a.items()}
        h, y = residual_norm(**cu, p=0.1, seed=3, out_dtype=BF16)
        runs.append([h, y, *torch.autograd.grad([h, y], list(cu.values()), [dh.cuda(), dy.cuda()])])
    assert all(torch.equal(s, t) for r in runs[1:] for s, t in zip(runs[0], r))


@pytest.mark.parametrize("shape,gate", [((1, 1024), "channel"), ((5, 33, 100), "sequence"), ((300, 515), "full")])
def test_captured_in_a_graph(shape, gate):
    """Both passes captured, replayed on new values with eager work between."""
    a, dh, dy = make(shape, TYPES[1], gate)
    s = {n: t.cuda() for n, t in a.items()}
    sdh, sdy, seed = dh.cuda(), dy.cuda(), torch.zeros(1, dtype=torch.long, device="cuda")

    def work():
        leaf = {n: t.detach().requires_grad_(True) for n, t in s.items()}
        h, y = residual_norm(**leaf, p=0.1, seed=seed)
        return [h.detach(), y.detach(), *torch.autograd.grad([h, y], list(leaf.values()), [sdh, sdy])]

    g, out = captured(work)
    for i in range(4):
        new, dh, dy = make(shape, TYPES[1], gate, seed=i + 1)
        for n in NAMES:
            s[n].copy_(new[n])
        sdh.copy_(dh)
        sdy.copy_(dy)
        seed.fill_(i)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, work())), i
        want = oracle.residual_norm(**new, p=0.1, seed=i, dh=dh, dy=dy)
        for n, t in zip(("h", "y", "dx", "dbranch", "dweight", "dpost_weight", "dgate"), out):
            close(n, t, want[n], t.dtype)


def test_on_another_stream():
    a, dh, dy = make((40, 700), TYPES[0], "channel")
    want = check(a, dh, dy, TYPES[0])
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        cu = {n: t.cuda().requires_grad_(True) for n, t in a.items()}
        h, y = residual_norm(**cu)
        got = torch.autograd.grad([h, y], list(cu.values()), [dh.cuda(), dy.cuda()])
    side.synchronize()
    assert all(torch.equal(s, t) for s, t in zip(got, want))


def test_the_gradient_is_the_differences():
    """Of the fp32 kernel itself: a central difference over 2e-2 of the mean
    output times a fixed direction, in float64 sums. Its own error: second order,
    (1e-2)^2 / 6 of the third derivative (of order one of the value), plus rounding
    u sqrt(n) / 1e-2 of it: 1e-2 relative to the gradient's scale."""
    a, dh, dy = make((2, 3, 24), TYPES[0], "channel")
    cu = {n: t.cuda() for n, t in a.items()}

    def loss(c):
        h, y = residual_norm(**c, p=0.2, seed=4)
        return ((h.double().cpu() * dh.double()).sum() + (y.double().cpu() * dy.double()).sum()).item()

    leaf = {n: t.clone().requires_grad_(True) for n, t in cu.items()}
    h, y = residual_norm(**leaf, p=0.2, seed=4)
    grads = torch.autograd.grad([h, y], list(leaf.values()), [dh.cuda(), dy.cuda()])
    for (n, t), g in zip(cu.items(), grads):
        v = torch.randn(t.shape, generator=torch.Generator().manual_seed(1)).cuda()
        up, down = (loss(dict(cu, **{n: t + s * 1e-2 * v})) for s in (1, -1))
        want = (g.double() * v.double()).sum().item()
        scale = (g.double().norm() * v.double().norm()).item()
        assert abs((up - down) / 2e-2 - want) <= 1e-2 * scale, n


def test_function_transforms_fake_tensors_and_subclasses_are_refused():
    a, _, _ = make((3, 20), TYPES[0])
    x, b, w = a["x"].cuda(), a["branch"].cuda(), a["weight"].cuda()
    for f in (lambda t: residual_norm(t, b, w)[1], lambda t: dropout(t, 0.3, 1)):
        with pytest.raises(RuntimeError):
            torch.func.grad(lambda t: f(t).sum())(x)
        with pytest.raises(RuntimeError):
            torch.func.vmap(lambda t: f(t))(torch.stack((x, x)))
        with pytest.raises(RuntimeError):
            torch.func.jvp(f, (x,), (x,))
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode() as mode:
        fake = mode.from_tensor(x)
        for f in (lambda: residual_norm(fake, fake), lambda: dropout(fake, 0.3, 1), lambda: residual_norm(x, b, w),
                  lambda: dropout(x, 0.3, 1)):
            with pytest.raises((RuntimeError, AssertionError)):       # the mode's own for tensors not of it
                f()


def test_more_than_2_to_31_values():
    """The last rows of 2^31 values and more: places, and the generator's blocks."""
    rows, D = (1 << 20) + 3, 2048
    x = torch.zeros(rows, D, dtype=BF16, device="cuda")
    b = torch.zeros(rows, D, dtype=BF16, device="cuda")
    g = torch.Generator().manual_seed(0)
    tx, tb, w = (torch.randn(s, generator=g) for s in ((3, D), (3, D), (D,)))
    x[-3:], b[-3:] = tx.cuda(), tb.cuda()
    first = (rows - 3) * D
    keep = torch.tensor(oracle.words(first, 3 * D, 77, 5), dtype=torch.int64).view(3, D) >= round(0.25 * 2 ** 32)
    h, y = residual_norm(x, b, w.cuda(), p=0.25, seed=77, offset=5)
    tx, tb = tx.to(BF16), tb.to(BF16)
    want = oracle.residual_norm(tx, torch.where(keep, tb.double() / 0.75, 0.0), w)
    for n, t in (("h", h), ("y", y)):
        value, bound = want[n]
        # the branch's factor rounds once more than the oracle knows of
        close(n, t[-3:], (value, bound + 4 * 2.0 ** -24 * value.abs()), BF16)
    assert (h[:-3] == 0).all()
    del h, y
    got = dropout(x, 0.25, 77, 5)[-3:]
    assert torch.equal(got.cpu(), torch.where(keep, tx.float() * (1 / 0.75), 0.0).to(BF16))
    xg = x.requires_grad_(True)
    h, y = residual_norm(xg, b, w.cuda(), p=0.25, seed=77, offset=5)
    dy = torch.zeros_like(b)
    dy[-3:] = tb.cuda()
    dx, = torch.autograd.grad(y, xg, dy)
    want = oracle.residual_norm(tx, torch.where(keep, tb.double() / 0.75, 0.0), w, dy=tb)["dx"]
    close("dx", dx[-3:], (want[0], 1.01 * want[1] + 2.0 ** -20 * want[0].abs().max()), BF16)


def test_threads_and_streams_at_once():
    """Four threads, a stream each, both passes: the bits of one alone."""
    import threading
    cases = [make((50 + i, 640), TYPES[1], "channel", seed=i) for i in range(4)]

    def work(a, dh, dy):
        cu = {n: t.cuda().requires_grad_(True) for n, t in a.items()}
        h, y = residual_norm(**cu, p=0.1, seed=2)
        return [h, y, *torch.autograd.grad([h, y], list(cu.values()), [dh.cuda(), dy.cuda()])]

    want = [work(*c) for c in cases]
    got = [None] * 4

    def run(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got[i] = work(*cases[i])
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=run, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert all(torch.equal(p, q) for a, b in zip(got, want) for p, q in zip(a, b))


def test_one_tensor_in_several_places():
    """x as the branch too, one weight for both norms: their gradients add."""
    a, dh, dy = make((4, 56), TYPES[0], post=False)
    x, w = a["x"].cuda().requires_grad_(True), a["weight"].cuda().requires_grad_(True)
    h, y = residual_norm(x, x, w, post_weight=w, gate=x)
    dx, dw = torch.autograd.grad([h, y], [x, w], [dh.cuda(), dy.cuda()])
    o = oracle.residual_norm(a["x"], a["x"], a["weight"], a["weight"], a["x"], dh=dh, dy=dy)
    add = lambda *n: tuple(sum(o[k][j] for k in n) for j in (0, 1))  # noqa: E731
    # autograd adds them in fp32: a rounding each
    for got, names in ((dx, ("dx", "dbranch", "dgate")), (dw, ("dweight", "dpost_weight"))):
        value, bound = add(*names)
        close(names[0], got, (value, bound + 2 * 2.0 ** -24 * sum(o[k][0].abs() for k in names)), F32)


def test_backward_twice_expanded_gradients_and_inference_mode():
    a, dh, dy = make((3, 7, 30), TYPES[1], "channel")
    cu = {n: t.cuda().requires_grad_(True) for n, t in a.items()}
    h, y = residual_norm(**cu, p=0.2, seed=6)
    one = torch.ones(1, dtype=BF16)
    grads = [torch.autograd.grad([h, y], list(cu.values()), [one.cuda().expand(3, 7, 30)] * 2, retain_graph=i == 0)
             for i in range(2)]
    assert all(torch.equal(p, q) for p, q in zip(*grads))
    want = oracle.residual_norm(**a, p=0.2, seed=6, dh=one.expand(3, 7, 30), dy=one.expand(3, 7, 30))
    for n, t in zip(NAMES, grads[0]):
        close("d" + n, t, want["d" + n], a[n].dtype)
    with torch.inference_mode():
        again = residual_norm(**{n: t.cuda() for n, t in a.items()}, p=0.2, seed=6)
        assert torch.equal(h, again[0]) and torch.equal(y, again[1])
        assert torch.equal(dropout(again[0], 0.3, 2), dropout(h.detach(), 0.3, 2))


def test_tensors_whose_memory_was_released_are_refused():
    """As sharded training leaves a parameter between its uses."""
    a, _, _ = make((4, 56), TYPES[0])
    x, b, w = a["x"].cuda(), a["branch"].cuda(), a["weight"].cuda()
    big = torch.ones(200, device="cuda")
    part = big[100:156]
    big.untyped_storage().resize_(0)
    for f in (lambda: residual_norm(x, b, part), lambda: residual_norm(x, b, w, gate=part), lambda: dropout(part, 0.5, 1)):
        with pytest.raises(RuntimeError, match="memory does not hold it"):
            f()
