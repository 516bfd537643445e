"""gated_recurrence and step_gated_recurrence against the float64 oracle.

The bar of every element is the oracle's bound on the fp32 error (derived
there) plus, where the result is rounded to a narrower type, half a step of
that type; plus 1e-30 for what flushes to zero."""

import pytest
import torch

import ngdn_recurrence_oracle as oracle
from nested_recurrent_memory_amd import gated_recurrence, step_gated_recurrence

pytestmark = pytest.mark.gpu

NAMES = ("x", "f", "wz", "A_log", "dt_bias", "initial_state")


def make(B, T, D, H, dtype, rows=None, seed=0, state=True, spread=1.0):
    g = torch.Generator().manual_seed(seed * 7919 + B * 104729 + T * 1009 + D)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    rows = B if rows is None else rows
    dt = torch.exp(torch.rand(D, generator=g) * 4.6 - 6.9)
    p = dict(x=r(B, T, D).to(dtype), f=(r(B, T, D) * spread).to(dtype), wz=(r(B, T, D) * spread).to(dtype),
             A_log=torch.log(1 + 15 * torch.rand(H, generator=g)), dt_bias=dt + torch.log(-torch.expm1(-dt)),
             initial_state=r(rows, D) if state else None)
    return p, r(B, T, D).to(dtype), r(rows, D)


def gpu(p, grad=True):
    return {n: (t.cuda().requires_grad_(grad) if t is not None else None) for n, t in p.items()}


def check(name, got, want, dtype):
    value, bound = want
    got = got.detach().double().cpu()
    half = torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0
    # below its smallest normal number 2^-14 fp16 has steps of 2^-24: half of one is 2^-25
    least = 2.0 ** -25 if dtype == torch.float16 else 1e-30
    tol = bound * (1 + half) + half * value.abs() + least
    err = (got - value).abs()
    bad = ~(err <= tol)
    assert not bad.any(), (f"{name}: {int(bad.sum())} of {bad.numel()} outside, worst "
                           f"{(err / tol)[bad].max().item():.3g} times the bound")


def run_and_check(p, dy, dfinal, cu=None, on_gpu=None):
    q = on_gpu or gpu(p)
    cu_gpu = torch.tensor(cu, device="cuda", dtype=torch.int32) if cu is not None else None
    y, final = gated_recurrence(q["x"], q["f"], q["wz"], q["A_log"], q["dt_bias"], q["initial_state"],
                                output_final_state=True, cu_seqlens=cu_gpu)
    want = oracle.recurrence(*(p[n] for n in NAMES[:5]), p["initial_state"], cu, dy, dfinal)
    dtype = p["x"].dtype
    assert y.dtype == dtype and final.dtype == torch.float32
    names = [n for n in NAMES if q[n] is not None]
    grads = torch.autograd.grad([y, final], [q[n] for n in names], [dy.cuda(), dfinal.cuda()])
    check("y", y, want["y"], dtype)
    check("final", final, want["final"], torch.float32)
    for n, g in zip(names, grads):
        assert g.dtype == p[n].dtype and g.shape == p[n].shape
        check("d" + n, g, want["d" + n], p[n].dtype)
    return y, final, dict(zip(names, grads))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,T,D,H", [
    (1, 1, 1, 1), (2, 1, 64, 4), (1, 2, 3, 3), (3, 15, 2, 1), (2, 16, 65, 5), (1, 17, 128, 8),
    (2, 63, 130, 2), (1, 64, 66, 66), (1, 65, 64, 1), (2, 127, 129, 3), (1, 128, 256, 4),
    (1, 129, 515, 515), (3, 300, 36, 4), (1, 1000, 66, 6), (1, 2100, 8, 2)])
def test_sizes(B, T, D, H, dtype):
    p, dy, dfinal = make(B, T, D, H, dtype)
    run_and_check(p, dy, dfinal)


def test_no_initial_state_no_final_gradient():
    p, dy, _ = make(2, 70, 64, 4, torch.bfloat16, state=False)
    q = gpu(p)
    y, final = gated_recurrence(*(q[n] for n in NAMES[:5]))
    assert final is None
    want = oracle.recurrence(*(p[n] for n in NAMES[:5]), None, None, dy, None)
    grads = torch.autograd.grad(y, [q[n] for n in NAMES[:5]], dy.cuda())
    check("y", y, want["y"], torch.bfloat16)
    for n, g in zip(NAMES, grads):
        check("d" + n, g, want["d" + n], p[n].dtype)


def test_gradient_through_the_final_state_alone():
    p, dy, dfinal = make(2, 70, 64, 4, torch.float32)
    q = gpu(p)
    _, final = gated_recurrence(*(q[n] for n in NAMES[:5]), q["initial_state"], True)
    want = oracle.recurrence(*(p[n] for n in NAMES[:5]), p["initial_state"], None, dy * 0, dfinal)
    for n, g in zip(NAMES, torch.autograd.grad(final, [q[n] for n in NAMES], dfinal.cuda())):
        check("d" + n, g, want["d" + n], p[n].dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("cu", [
    [0, 200], [0, 0, 200], [0, 200, 200], [0, 1, 2, 3, 200], [0, 16, 32, 48, 200], [0, 15, 17, 64, 65, 128, 190],
    [3, 3, 3, 20, 140, 140, 140, 199], [0, 0, 0], [200, 200], [7, 8], [0, 64, 128, 129, 129, 130, 180],
    list(range(0, 201))], ids=str)
def test_packed_sequences(cu, dtype):
    """Boundaries at, before and behind the ends of runs, empty sequences first,
    last and together, tokens before the first and behind the last, whose
    values are NaN: nothing of them may reach anything."""
    p, dy, dfinal = make(1, 200, 66, 6, dtype, rows=len(cu) - 1)
    used = torch.zeros(200, dtype=torch.bool)
    used[cu[0]:cu[-1]] = True
    poisoned = {n: (torch.where(used[None, :, None], t, float("nan")) if n in ("x", "f", "wz") else t)
                for n, t in p.items()}
    clean = {n: (torch.where(used[None, :, None], t, 0.0).to(t.dtype) if n in ("x", "f", "wz") else t)
             for n, t in p.items()}
    dyp = torch.where(used[None, :, None], dy, float("nan"))
    q = gpu(poisoned)
    cu_gpu = torch.tensor(cu, device="cuda")                       # int64
    y, final = gated_recurrence(*(q[n] for n in NAMES[:5]), q["initial_state"], True, cu_gpu)
    want = oracle.recurrence(*(clean[n] for n in NAMES[:5]), p["initial_state"], cu, dy, dfinal)
    grads = torch.autograd.grad([y, final], [q[n] for n in NAMES], [dyp.cuda(), dfinal.cuda()])
    check("y", y, want["y"], dtype)
    check("final", final, want["final"], torch.float32)
    for n, g in zip(NAMES, grads):
        check("d" + n, g, want["d" + n], p[n].dtype)
    assert not y[0][~used].any() and not grads[0][0][~used].any()


def test_packed_equals_padded():
    """Sequences packed and as rows of a batch: the same tokens."""
    p, dy, dfinal = make(3, 50, 64, 4, torch.float32)
    q = gpu(p)
    y, final = gated_recurrence(*(q[n] for n in NAMES[:5]), q["initial_state"], True)
    cu = torch.tensor([0, 50, 100, 150], device="cuda")
    flat = {n: q[n].detach().reshape(1, 150, 64) for n in NAMES[:3]}
    yp, fp = gated_recurrence(*flat.values(), q["A_log"].detach(), q["dt_bias"].detach(),
                              q["initial_state"].detach(), True, cu)
    want = oracle.recurrence(*(p[n] for n in NAMES[:5]), p["initial_state"])
    for got in (y, yp.reshape(3, 50, 64)):
        check("y", got, want["y"], torch.float32)
    for got in (final, fp):
        check("final", got, want["final"], torch.float32)


@pytest.mark.parametrize("D,width", [(64, 192), (65, 200), (66, 199), (64, 193)])
def test_column_slices_and_strides(D, width):
    """x, f and wz as column slices of one tensor at any offset, a transposed
    (time-major) batch, an expanded row, and a gradient with strides."""
    dtype = torch.bfloat16
    p, dy, dfinal = make(2, 40, D, 1, dtype)
    joint = torch.zeros(40, 2, width, dtype=dtype)          # time-major
    at = [0, D, width - D]
    for n, o in zip(("x", "f", "wz"), at):
        joint[..., o:o + D] = p[n].transpose(0, 1)
    if width < 3 * D:                                       # the slices overlap
        p = dict(p, **{n: joint[..., o:o + D].transpose(0, 1).contiguous() for n, o in zip(("x", "f", "wz"), at)})
    jg = joint.cuda()
    q = gpu(p)
    for n, o in zip(("x", "f", "wz"), at):
        q[n] = jg[..., o:o + D].transpose(0, 1).requires_grad_(True)
    run_and_check(p, dy.transpose(0, 1).contiguous().transpose(0, 1), dfinal, on_gpu=q)
    # one row for the whole batch, and one gradient value for every channel
    e = {n: (p[n][:1] if n in ("x", "f", "wz") else p[n]) for n in NAMES}
    q = gpu(e)
    big = [q[n].expand(2, 40, D) for n in ("x", "f", "wz")]
    y, _ = gated_recurrence(*big, q["A_log"], q["dt_bias"], q["initial_state"])
    one = dy[..., :1]
    g = torch.autograd.grad(y, [q["x"]], one.cuda().expand(2, 40, D))[0]
    want = oracle.recurrence(*(e[n].expand(2, 40, D) for n in ("x", "f", "wz")), p["A_log"], p["dt_bias"],
                             p["initial_state"], None, one.expand(2, 40, D))
    check("y", y, want["y"], dtype)
    # each row's gradient is rounded to bf16 before torch adds the two
    v, b = (t.sum(0, keepdim=True) for t in want["dx"])
    half = torch.finfo(dtype).eps / 2
    tol = b + half * want["dx"][0].abs().sum(0, keepdim=True) * 1.01 + half * v.abs()
    assert ((g.double().cpu() - v).abs() <= tol * 1.01 + 1e-30).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_extreme_gates(dtype):
    """Decays of exactly 1 and 0, gates shut and open, and all between: the
    gradient of sqrt(1 - a^2) has a pole where a = 1, which the decay's own
    derivative cancels."""
    p, dy, dfinal = make(1, 90, 64, 64, dtype, spread=1.0)
    f = torch.linspace(-110, 110, 64).repeat(90, 1)
    p["f"] = f[None].to(dtype)
    p["wz"] = torch.linspace(90, -90, 64).roll(17).repeat(90, 1)[None].to(dtype)
    p["A_log"] = torch.linspace(-12, 6, 64).roll(29)
    q = gpu(p)
    y, final = gated_recurrence(*(q[n] for n in NAMES[:5]), q["initial_state"], True)
    grads = torch.autograd.grad([y, final], [q[n] for n in NAMES], [dy.cuda(), dfinal.cuda()])
    want = oracle.recurrence(*(p[n] for n in NAMES[:5]), p["initial_state"], None, dy, dfinal)
    for n, got in [("y", y), ("final", final)] + [("d" + n, g) for n, g in zip(NAMES, grads)]:
        assert torch.isfinite(got).all(), n
        # decays and gates below the smallest normal number flush to 0: up to 1e-17 each
        # (the root of 1e-34) times what they multiply, 2^10 at most in these sums
        v, b = want[n]
        check(n, got, (v, b + 1e-14), got.dtype)


def test_nan_and_inf_stay_in_their_channel_and_sequence():
    p, _, _ = make(2, 100, 64, 4, torch.float32)
    q = gpu(p, grad=False)
    ref, fref = gated_recurrence(*(q[n] for n in NAMES[:5]), q["initial_state"], True)
    x = q["x"].clone()
    x[0, 37, 5], x[1, 80, 9] = float("nan"), float("inf")
    y, final = gated_recurrence(x, *(q[n] for n in NAMES[1:5]), q["initial_state"], True)
    bad = torch.zeros_like(y, dtype=torch.bool)
    bad[0, 37:, 5] = True
    bad[1, 80:, 9] = True
    assert torch.equal(y[~bad], ref[~bad]) and not torch.isfinite(y[bad]).any()
    assert torch.isnan(final[0, 5]) and not torch.isfinite(final[1, 9])
    # a NaN of every bit set, as memory that was never written can hold
    x = q["x"].clone()
    x[0, 37:90, 5] = torch.tensor(-1, dtype=torch.int32).view(torch.float32).item()
    x.view(torch.int32)[0, 37:90, 5] = -1
    y, final = gated_recurrence(x, *(q[n] for n in NAMES[1:5]), q["initial_state"], True)
    assert torch.isnan(y[0, 37:, 5]).all() and torch.isnan(final[0, 5])


def test_no_tokens():
    z = torch.zeros(2, 0, 8, device="cuda", requires_grad=True)
    A, dt = torch.zeros(2, device="cuda"), torch.zeros(8, device="cuda")
    h = torch.randn(2, 8, device="cuda", requires_grad=True)
    y, final = gated_recurrence(z, z, z, A, dt, h, True)
    assert y.shape == (2, 0, 8) and torch.equal(final, h)
    assert torch.equal(torch.autograd.grad(final, h, torch.ones_like(h))[0], torch.ones_like(h))
    y, final = gated_recurrence(z[:0], z[:0], z[:0], A, dt, h[:0], True)
    assert y.shape == (0, 0, 8) and final.shape == (0, 8)
    x = torch.randn(1, 6, 8, device="cuda")
    y, final = gated_recurrence(x, x, x, A, dt, None, True, torch.zeros(1, device="cuda", dtype=torch.int32))
    assert not y.any() and final.shape == (0, 8)


def test_unsorted_boundaries_read_nothing_outside():
    """Boundaries that are not sorted, or outside the row, give some result."""
    p, dy, _ = make(1, 100, 66, 6, torch.float32, rows=4)
    q = gpu(p)
    for cu in ([0, 70, 30, 100, 100], [-5, 10, 20, 400, 500], [90, 0, 0, 0, 100], [50, 50, 3, 2, 1]):
        y, _ = gated_recurrence(*(q[n] for n in NAMES[:5]), q["initial_state"], True,
                                torch.tensor(cu, device="cuda"))
        torch.autograd.grad(y, [q[n] for n in NAMES], dy.cuda())
    torch.cuda.synchronize()


def test_same_bits_every_run():
    p, dy, dfinal = make(2, 3000, 256, 4, torch.bfloat16)
    runs = []
    for _ in range(3):
        q = gpu(p)
        y, final = gated_recurrence(*(q[n] for n in NAMES[:5]), q["initial_state"], True)
        runs.append((y, final, *torch.autograd.grad([y, final], [q[n] for n in NAMES],
                                                    [dy.cuda(), dfinal.cuda()])))
    for r in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(r, runs[0]))


def test_long_row_in_two_calls():
    """A state carried from one call to the next continues the row, over many
    workgroups: both within the oracle's bound of the whole row."""
    p, dy, dfinal = make(1, 5000, 10, 2, torch.float32)
    q = gpu(p, grad=False)
    whole, end = gated_recurrence(*(q[n] for n in NAMES[:5]), q["initial_state"], True)
    a, s = gated_recurrence(*(q[n][:, :2345] for n in NAMES[:3]), q["A_log"], q["dt_bias"],
                            q["initial_state"], True)
    b, s = gated_recurrence(*(q[n][:, 2345:] for n in NAMES[:3]), q["A_log"], q["dt_bias"], s, True)
    want = oracle.recurrence(*(p[n] for n in NAMES[:5]), p["initial_state"])
    for y, f in ((whole, end), (torch.cat((a, b), 1), s)):
        check("y", y, want["y"], torch.float32)
        check("final", f, want["final"], torch.float32)


def test_gradients_are_differences_of_the_outputs():
    """fp32 central differences along a random direction. Step e = 2^-6: the
    second-order error is e^2 of the third derivative's scale (2e-4), the
    rounding error 2^-24 / e of the sum of the terms' sizes (4e-6)."""
    p, dy, dfinal = make(2, 200, 64, 4, torch.float32)
    q = gpu(p)
    dy, dfinal = dy.cuda(), dfinal.cuda()

    def loss(s, name, v):
        t = {n: q[n].detach() + (s * v if n == name else 0) for n in NAMES}
        y, f = gated_recurrence(*(t[n] for n in NAMES[:5]), t["initial_state"], True)
        return ((y.double() * dy).sum() + (f.double() * dfinal).sum()).item()

    y, f = gated_recurrence(*(q[n] for n in NAMES[:5]), q["initial_state"], True)
    size = ((y.detach() * dy).abs().sum() + (f.detach() * dfinal).abs().sum()).item()
    for n, g in zip(NAMES, torch.autograd.grad([y, f], [q[n] for n in NAMES], [dy, dfinal])):
        v = torch.randn_like(g)
        e = 2.0 ** -6
        got, want = (loss(e, n, v) - loss(-e, n, v)) / (2 * e), (g.double() * v).sum().item()
        assert abs(got - want) <= 1e-3 * size, (n, got, want, size)


def test_differentiating_twice_raises():
    p, dy, _ = make(1, 20, 8, 2, torch.float32, state=False)
    q = gpu(p)
    y, _ = gated_recurrence(*(q[n] for n in NAMES[:5]))
    g, = torch.autograd.grad(y.sum(), q["x"], create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), q["x"])


def test_captured_in_a_graph_and_on_another_stream():
    """Forward and backward captured together, replayed with new inputs between
    eager work, against the eager results, bit for bit; two graphs at once."""
    p, dy, dfinal = make(1, 700, 66, 6, torch.bfloat16, rows=3)
    cu = torch.tensor([0, 100, 100, 650], device="cuda", dtype=torch.int32)
    dy, dfinal = dy.cuda(), dfinal.cuda()

    def work(s):
        q = {n: s[n].detach().requires_grad_(True) for n in NAMES}
        y, f = gated_recurrence(*(q[n] for n in NAMES[:5]), q["initial_state"], True, cu)
        return (y.detach(), f.detach(), *torch.autograd.grad([y, f], [q[n] for n in NAMES], [dy, dfinal]))

    static = [gpu(p, grad=False) for _ in range(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work(static[0])
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for s in static:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(work(s))
        graphs.append(g)
    for i in range(4):
        new = [make(1, 700, 66, 6, torch.bfloat16, rows=3, seed=10 + 2 * i + k)[0] for k in range(2)]
        for s, n in zip(static, new):
            for name in NAMES:
                s[name].copy_(n[name])
        streams = [torch.cuda.Stream() for _ in graphs]
        for g, st in zip(graphs, streams):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                g.replay()
        for st in streams:
            torch.cuda.current_stream().wait_stream(st)
        torch.cuda.synchronize()
        for s, o in zip(static, outs):
            assert all(torch.equal(a, b) for a, b in zip(o, work(s))), i


# ---------------------------------------------------------------- one token

@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,D,H", [(1, 1, 1), (1, 1024, 16), (3, 515, 5), (256, 64, 64), (7, 130, 2)])
@pytest.mark.parametrize("inplace", [False, True])
def test_step(B, D, H, dtype, inplace):
    p, _, _ = make(B, 1, D, H, dtype)
    q = gpu(p, grad=False)
    tok = [q[n][:, 0] for n in NAMES[:3]] + [q["A_log"], q["dt_bias"]]
    want = oracle.step(*(p[n][:, 0] for n in NAMES[:3]), p["A_log"], p["dt_bias"], p["initial_state"])
    state = q["initial_state"].clone()
    y, new = step_gated_recurrence(*tok, state, inplace=inplace)
    assert y.dtype == dtype and new.dtype == torch.float32
    assert (new is state) if inplace else torch.equal(state, q["initial_state"])
    check("state", new, want, torch.float32)
    check("y", y, want, dtype)


def test_step_strides_and_refusals():
    p, _, _ = make(4, 1, 64, 4, torch.bfloat16)
    joint = torch.cat([p[n][:, 0] for n in NAMES[:3]], -1).cuda()
    q = gpu(p, grad=False)
    tok = list(joint.split(64, -1)) + [q["A_log"], q["dt_bias"]]
    want = oracle.step(*(p[n][:, 0] for n in NAMES[:3]), p["A_log"], p["dt_bias"], p["initial_state"])
    check("state", step_gated_recurrence(*tok, q["initial_state"])[1], want, torch.float32)
    with pytest.raises(ValueError, match="inplace"):
        step_gated_recurrence(*tok, q["initial_state"].bfloat16(), inplace=True)
    with pytest.raises(ValueError, match="inplace"):
        step_gated_recurrence(*tok, torch.zeros(64, 4, device="cuda").t(), inplace=True)
    with pytest.raises(RuntimeError, match="forward-only"):
        step_gated_recurrence(*tok, q["initial_state"].requires_grad_(True))
    e = [t[:0] for t in tok[:3]] + tok[3:]
    y, s = step_gated_recurrence(*e, torch.zeros(0, 64, device="cuda"))
    assert y.shape == (0, 64) and s.shape == (0, 64)


def test_prompt_then_tokens():
    """A prompt through the whole-sequence form, then the step token by token in
    a captured graph, is the whole row at once."""
    p, _, _ = make(2, 120, 64, 4, torch.float32)
    q = gpu(p, grad=False)
    want = oracle.recurrence(*(p[n] for n in NAMES[:5]), p["initial_state"])
    y, state = gated_recurrence(*(q[n][:, :100] for n in NAMES[:3]), q["A_log"], q["dt_bias"],
                                q["initial_state"], True)
    tok = [torch.empty(2, 64, device="cuda") for _ in range(3)]
    keep = state.clone()
    step_gated_recurrence(*tok, q["A_log"], q["dt_bias"], state, inplace=True)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out, _ = step_gated_recurrence(*tok, q["A_log"], q["dt_bias"], state, inplace=True)
    state.copy_(keep)
    ys = [y]
    for t in range(100, 120):
        for dst, n in zip(tok, NAMES):
            dst.copy_(q[n][:, t])
        g.replay()
        ys.append(out.clone()[:, None])
    check("y", torch.cat(ys, 1), want["y"], torch.float32)
    check("final", state, want["final"], torch.float32)


# ---------------------------------------------------------------- rows of many tiles, types, streams

@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,D,H,S", [(3100, 70, 7, 60), (2500, 130, 2, 3), (4000, 9, 9, 900)])
def test_long_packed_rows(T, D, H, S, dtype):
    """Sequences over many workgroups' tiles, some empty, tokens before the first
    and behind the last."""
    g = torch.Generator().manual_seed(T + S)
    cu = torch.sort(torch.randint(5, T - 40, (S + 1,), generator=g)).values
    cu[S // 2] = cu[S // 2 - 1]
    p, dy, dfinal = make(1, T, D, H, dtype, rows=S)
    run_and_check(p, dy, dfinal, cu=cu.tolist())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,T,D,H", [(2, 5000, 66, 3), (1, 1024, 128, 1), (1, 1025, 64, 64)])
def test_long_rows(B, T, D, H, dtype):
    p, dy, dfinal = make(B, T, D, H, dtype)
    run_and_check(p, dy, dfinal)


@pytest.mark.parametrize("types", [(torch.bfloat16, torch.float32, torch.float32),
                                   (torch.float32, torch.bfloat16, torch.float16),
                                   (torch.float16, torch.bfloat16, torch.bfloat16)])
def test_mixed_types_lose_nothing(types):
    p, dy, dfinal = make(2, 150, 64, 4, torch.float32)
    for n, t in zip(("x", "f", "wz"), types):
        p[n] = p[n].to(t)
    run_and_check(p, dy.to(types[0]), dfinal)
    want = oracle.recurrence(*(p[n][:, :1] for n in NAMES[:3]), p["A_log"], p["dt_bias"], p["initial_state"])
    s = gpu(p, grad=False)
    y, state = step_gated_recurrence(*(s[n][:, 0] for n in NAMES[:3]), s["A_log"], s["dt_bias"],
                                     s["initial_state"])
    check("y", y[:, None], want["y"], types[0])
    check("state", state, want["final"], torch.float32)


def test_without_gradients_the_same_bits():
    """Under no_grad (parameters that require it) and in inference mode."""
    p, _, _ = make(2, 700, 66, 6, torch.bfloat16)
    q = gpu(p)
    args = [q[n] for n in NAMES]
    y, f = gated_recurrence(*args, output_final_state=True)
    with torch.no_grad():
        y1, f1 = gated_recurrence(*args, output_final_state=True)
    with torch.inference_mode():
        y2, f2 = gated_recurrence(*args, output_final_state=True)
        s = torch.zeros(2, 66, device="cuda")
        step_gated_recurrence(*(q[n][:, 0] for n in NAMES[:3]), q["A_log"], q["dt_bias"], s, inplace=True)
    assert y.requires_grad and not y1.requires_grad
    assert torch.equal(y, y1) and torch.equal(f, f1) and torch.equal(y, y2) and torch.equal(f, f2)


def test_calls_on_two_streams_at_once():
    """Two long rows whose tiles wait for one another, each on a stream of its
    own, forward and backward, against the same calls alone."""
    def work(q, dy):
        y, f = gated_recurrence(*(q[n] for n in NAMES), output_final_state=True)
        return (y.detach(), f.detach(), *torch.autograd.grad([y, f], [q[n] for n in NAMES], [dy, torch.ones_like(f)]))

    qs, dys = [], []
    for k in range(2):
        p, dy, _ = make(1, 20000, 512, 8, torch.bfloat16, seed=k)
        qs.append(gpu(p))
        dys.append(dy.cuda())
    alone = [work(q, dy) for q, dy in zip(qs, dys)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in qs]
    outs = [None, None]
    for _ in range(4):
        for k, st in enumerate(streams):
            with torch.cuda.stream(st):
                outs[k] = work(qs[k], dys[k])
    torch.cuda.synchronize()
    for a, b in zip(alone, outs):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_a_state_saved_by_a_graph_is_not_updated_behind_it():
    p, _, _ = make(2, 1, 64, 4, torch.float32)
    s = gpu(p, grad=False)
    state = s["initial_state"]
    w = torch.ones_like(state).requires_grad_()
    out = (w * state).sum()
    step_gated_recurrence(*(s[n][:, 0] for n in NAMES[:3]), s["A_log"], s["dt_bias"], state, inplace=True)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.backward()


def test_a_long_row_captured_in_a_graph():
    """More tiles than a link of the chain joins; replays with new inputs between
    eager calls, each against the eager result."""
    p, dy, dfinal = make(1, 4500, 130, 2, torch.bfloat16)
    s = gpu(p, grad=False)
    dy, dfinal = dy.cuda(), dfinal.cuda()

    def work():
        q = [s[n].detach().requires_grad_(True) for n in NAMES]
        y, f = gated_recurrence(*q, output_final_state=True)
        return (y.detach(), f.detach(), *torch.autograd.grad([y, f], q, [dy, dfinal]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = work()
    for i in range(4):
        for name, t in make(1, 4500, 130, 2, torch.bfloat16, seed=20 + i)[0].items():
            s[name].copy_(t)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, work())), i


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,T,D,H", [(1, 256, 70, 7), (3, 257, 64, 1), (2, 250, 9, 9), (4, 300, 4096, 64),
                                     (4, 512, 4095, 5), (5, 513, 3333, 1)])
def test_rows_of_few_tiles(B, T, D, H, dtype):
    """Around the sizes of one, two and a few tiles, with many strips too."""
    p, dy, dfinal = make(B, T, D, H, dtype)
    run_and_check(p, dy, dfinal)


def test_open_write_gates():
    """Where the gate is open 1 - sigmoid(wz) is small and keeps its relative
    precision: sigmoid(-wz), with the oracle's error of a sigmoid."""
    p, dy, dfinal = make(1, 40, 64, 4, torch.float32)
    p["wz"] = torch.linspace(-100, 80, 64).repeat(40, 1)[None]
    q = gpu(p)
    y, _ = gated_recurrence(*(q[n] for n in NAMES))
    dx, dw = torch.autograd.grad(y, [q["x"], q["wz"]], dy.cuda())
    v, b = oracle.recurrence(*(p[n] for n in NAMES[:5]), p["initial_state"], None, dy)["dx"]
    k = p["x"].double() * torch.sigmoid(-p["wz"].double())
    rel = (10 + 2 * p["wz"].double().abs()) * oracle.U
    err = (dw.double().cpu() - v * k).abs()
    assert (err <= b * k.abs() + rel * (v * k).abs() + 1e-37).all(), (err / (v * k).abs()).max()


def test_as_many_decays_as_a_grid_has_no_room_for():
    """2^24 heads of one channel: a workgroup each would be 2^32 work-items. Channels
    do not meet, so every part has the bits of a call of its own."""
    D = (1 << 24) + 5
    g = torch.Generator(device="cuda").manual_seed(3)
    r = lambda: torch.randn(D, generator=g, device="cuda")  # noqa: E731
    t = [r().view(1, 1, D) for _ in range(3)] + [r() * 0.1, r() - 3]

    def grads(lo, hi):
        q = [v[..., lo:hi].detach().requires_grad_(True) for v in t]
        y, f = gated_recurrence(*q, output_final_state=True)
        return [v.reshape(-1) for v in (y.detach(), *torch.autograd.grad(f.sum(), q))]

    whole = grads(0, D)
    for lo in (0, 1 << 22, (1 << 22) * 3 - 512, D - 1003):
        for a, b in zip(whole, grads(lo, lo + 1003)):
            assert torch.equal(a[lo:lo + 1003], b), lo
    assert all(torch.isfinite(v).all() for v in whole)


@pytest.mark.parametrize("B,T,D,H", [(5, 513, 3333, 1), (4, 512, 4095, 5), (1, 40, 200, 2)])
def test_a_wide_heads_decay_gradient_is_its_channels(B, T, D, H):
    """dA_log of a head against the float64 sum of the same channels' as heads of
    their own, which are the same bits up to that sum: at most D / (64 H) + 16
    fp32 roundings in a row."""
    p, dy, dfinal = make(B, T, D, H, torch.bfloat16)

    def grad(A_log):
        q = gpu(dict(p, A_log=A_log))
        y, f = gated_recurrence(*(q[n] for n in NAMES), output_final_state=True)
        return torch.autograd.grad([y, f], q["A_log"], [dy.cuda(), dfinal.cuda()])[0].double().view(H, -1)

    got, each = grad(p["A_log"])[:, 0], grad(p["A_log"].repeat_interleave(D // H))
    assert ((got - each.sum(1)).abs() <= (D / (64 * H) + 16) * oracle.U * each.abs().sum(1)).all()


def test_thousands_of_packed_sequences():
    """More boundaries than the first launch keeps in shared memory, some together."""
    T, S = 9000, 5000
    g = torch.Generator().manual_seed(5)
    cu = torch.sort(torch.randint(3, T - 10, (S + 1,), generator=g)).values
    p, dy, dfinal = make(1, T, 6, 2, torch.float32, rows=S)
    run_and_check(p, dy, dfinal, cu=cu.tolist())
