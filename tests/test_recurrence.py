"""The gated linear recurrence's oracle and the refusals of its entry points
and of the embedding's, on the CPU."""

import ctypes

import pytest
import torch

import ngdn_recurrence_oracle as oracle
from nested_recurrent_memory_amd import _lib, gated_recurrence, step_gated_recurrence
from nested_recurrent_memory_amd.model_ops import Embedding, embedding


def _inputs(B=2, T=5, D=4, H=2, dtype=torch.float64):
    g = torch.Generator().manual_seed(B * 1000 + T * 10 + D)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    return dict(x=r(B, T, D).to(dtype), f=r(B, T, D).to(dtype), wz=r(B, T, D).to(dtype),
                A_log=r(H).to(dtype), dt_bias=(r(D) - 2).to(dtype))


def _loss(p, h0, cu, dy, dfinal):
    o = oracle.recurrence(p["x"], p["f"], p["wz"], p["A_log"], p["dt_bias"], h0, cu)
    return (o["y"][0] * dy).sum() + (o["final"][0] * dfinal).sum()


@pytest.mark.parametrize("cu", [None, [0, 0, 3, 3, 4], [1, 2, 5]])
def test_oracle_gradients_are_differences(cu):
    """Central differences of the float64 forward: step 1e-5, whose own error
    is of the order of 1e-10 of the third derivatives plus 1e-11 of rounding."""
    p = _inputs(B=1 if cu else 2)
    rows = len(cu) - 1 if cu else 2
    g = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    h0, dfinal, dy = r(rows, 4), r(rows, 4), r(*p["x"].shape)
    o = oracle.recurrence(*(p[n] for n in ("x", "f", "wz", "A_log", "dt_bias")), h0, cu, dy, dfinal)
    for name, t in [*p.items(), ("initial_state", h0)]:
        want = o["d" + name][0]
        for i in range(t.numel()):
            flat, keep = t.view(-1), t.view(-1)[i].item()
            flat[i] = keep + 1e-5
            up = _loss(p, h0, cu, dy, dfinal)
            flat[i] = keep - 1e-5
            down = _loss(p, h0, cu, dy, dfinal)
            flat[i] = keep
            assert abs((up - down) / 2e-5 - want.view(-1)[i]) < 1e-6, (name, i)


def test_shapes_and_types_are_refused():
    p = _inputs(dtype=torch.float32)
    args = [p[n] for n in ("x", "f", "wz", "A_log", "dt_bias")]

    def bad(match, i=None, t=None, fn=gated_recurrence, **kw):
        a = list(args)
        if i is not None:
            a[i] = t
        with pytest.raises(ValueError, match=match):
            fn(*a, **kw)

    bad("x ", 0, p["x"][:, 0])
    bad("x ", 1, p["f"][:, :3])
    bad("x ", 2, p["wz"][..., :2])
    bad("A_log", 3, torch.zeros(3))
    bad("A_log", 3, torch.zeros(2, 2))
    bad("dt_bias", 4, torch.zeros(5))
    bad("f is", 1, p["f"].double())
    bad("x is", 0, p["x"].long())
    bad("initial_state", initial_state=torch.zeros(3, 4))
    bad("cu_seqlens", cu_seqlens=torch.tensor([0, 5]))                     # B = 2
    one = [p[n][:1] for n in ("x", "f", "wz")] + args[3:]
    for cu in (torch.tensor([0.0, 5.0]), torch.tensor([[0, 5]]), torch.zeros(0, dtype=torch.int32)):
        with pytest.raises(ValueError, match="cu_seqlens"):
            gated_recurrence(*one, cu_seqlens=cu)
    with pytest.raises(ValueError, match="initial_state"):
        gated_recurrence(*one, cu_seqlens=torch.tensor([0, 2, 5]), initial_state=torch.zeros(1, 4))
    bad("no CPU path")
    tok = [t[:, 0] for t in args[:3]] + args[3:]
    with pytest.raises(ValueError, match="state"):
        step_gated_recurrence(*tok, torch.zeros(2, 3))
    with pytest.raises(ValueError, match="no CPU path"):
        step_gated_recurrence(*tok, torch.zeros(2, 4))
    with pytest.raises(ValueError, match="x "):
        step_gated_recurrence(*args, torch.zeros(2, 4))


def test_embedding_arguments_are_refused():
    w, ids = torch.zeros(5, 4), torch.tensor([0, 1])
    for bad in (dict(ids=ids.float()), dict(ids=ids.to(torch.int16)), dict(weight=w[0]),
                dict(weight=w.double()), dict(weight=w.long()), dict(padding_idx=5),
                dict(padding_idx=-6), dict(out_dtype=torch.float64), dict(weight=w[:0]),
                dict(weight=w[:, :0])):
        with pytest.raises(ValueError, match="embedding:"):
            embedding(**{"ids": ids, "weight": w, **bad})
    with pytest.raises(ValueError, match="no CPU path"):
        embedding(ids, w)


def test_embedding_module_off_the_gpu_is_torchs():
    """The module in place of nn.Embedding keeps what nn.Embedding does off the
    GPU, gradients included, and its state dict."""
    m = Embedding(6, 3, padding_idx=2)
    ref = torch.nn.Embedding(6, 3, padding_idx=2)
    ref.load_state_dict(m.state_dict())
    ids = torch.tensor([[0, 2, 5], [5, 1, 2]])
    (m(ids) ** 2).sum().backward()
    (ref(ids) ** 2).sum().backward()
    assert torch.equal(m(ids), ref(ids)) and torch.equal(m.weight.grad, ref.weight.grad)


FAKE = [ctypes.c_void_p(4096 * (i + 1)) for i in range(8)]


def _args(**kw):
    a = _lib.RecurrenceArgs()
    a.B, a.T, a.D, a.H = 1, 16, 8, 2
    for n in ("x", "f", "wz", "A_log", "dt_bias", "h0", "y", "final_state", "hs", "dy", "dx", "df", "dwz",
              "dA_log", "ddt_bias", "ws"):
        setattr(a, n, 4096)
    for n, v in kw.items():
        setattr(a, n, v)
    return a


@pytest.mark.parametrize("kw,word", [
    (dict(D=0), "D=0"), (dict(H=3), "multiple of H"), (dict(B=0), "B=0"), (dict(T=0), "T=0"),
    (dict(x=None), "NULL"), (dict(hs=None), "NULL"), (dict(ws=None), "NULL"),
    (dict(S=2), "packed"), (dict(cu=4096), "packed"), (dict(cu=4096, S=2, B=2), "packed"),
    (dict(B=2, D=1 << 30, H=1), "exceeds"), (dict(cu=4096, S=1 << 30), "exceeds"),
    (dict(B=1, T=1 << 30, D=1 << 20, H=1), "workgroups"),
])
def test_recurrence_entry_points_refuse_before_any_launch(kw, word):
    so = _lib.lib()
    a = _args(**kw)
    for name in ("ngdn_recurrence_fwd", "ngdn_recurrence_bwd")[kw == dict(hs=None):]:
        assert getattr(so, name)(1, ctypes.byref(a), None) == 1
        assert word.encode() in so.ngdn_last_error(), so.ngdn_last_error()
    assert so.ngdn_recurrence_fwd(7, ctypes.byref(a), None) == 1
    assert so.ngdn_recurrence_fwd(1, None, None) == 1 and b"NULL" in so.ngdn_last_error()


def test_step_and_embedding_entry_points_refuse_before_any_launch():
    so = _lib.lib()
    a = _args(h0=None)
    assert so.ngdn_recurrence_step(1, ctypes.byref(a), None) == 1 and b"NULL" in so.ngdn_last_error()
    p = FAKE
    for N, V, D, t in ((-1, 4, 4, 0), (4, 0, 4, 0), (4, 4, 0, 0), (4, 4, 4, 3), ((1 << 24) + 1, 4, 4, 0),
                       (4, 1 << 24, 4, 0)):
        assert so.ngdn_embedding_fwd(t, 0, N, V, D, 1.0, p[0], p[1], p[2], None) == 1
        assert so.ngdn_embedding_bwd(t, 0, N, V, D, 1.0, -1, p[0], p[1], p[2], p[3], None) == 1
    assert so.ngdn_embedding_fwd(0, 0, 4, 4, 4, 1.0, None, p[1], p[2], None) == 1
    assert b"NULL" in so.ngdn_last_error()
    assert so.ngdn_embedding_bwd(0, 0, 4, 4, 4, 1.0, -1, p[0], p[1], p[2], None, None) == 1


def test_recurrence_struct_matches_header():
    """The ctypes mirror of ngdn_recurrence_args has the header's fields, in
    order and with the header's types."""
    import os
    import re
    text = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include",
                             "ngdn.h")).read()
    body = re.search(r"typedef struct ngdn_recurrence_args \{(.*?)\}", text, re.S).group(1)
    fields = []
    for decl in filter(None, (d.strip() for d in body.split(";"))):
        ty, names = re.match(r"((?:const )?\w+)\s*(.*)", decl, re.S).groups()
        for n in names.split(","):
            n = n.strip()
            fields.append((n.lstrip("* "), "ptr" if n.startswith("*") else ty))
    ct = {"int32_t": ctypes.c_int32, "int64_t": ctypes.c_int64, "ptr": ctypes.c_void_p}
    assert [(n, ct[t]) for n, t in fields] == list(_lib.RecurrenceArgs._fields_)
    assert int(re.search(r"#define NGDN_REC_RUN (\d+)", text).group(1)) == _lib.REC_RUN


def test_sizes_beyond_the_library_are_refused():
    """Sizes are 32 bits in the library: a larger one must not wrap on its way."""
    e = torch.zeros(1)
    x = e.expand(1, 1 << 31, 1)
    with pytest.raises(ValueError, match="sizes up to"):
        gated_recurrence(x, x, x, e, e)
    with pytest.raises(ValueError, match="sizes up to"):
        step_gated_recurrence(x[0], x[0], x[0], e, e, x[0])
    with pytest.raises(ValueError, match="cu_seqlens"):
        gated_recurrence(e.view(1, 1, 1), e.view(1, 1, 1), e.view(1, 1, 1), e, e,
                         cu_seqlens=torch.zeros(1, dtype=torch.int32).expand((1 << 31) + 5))
    with pytest.raises(ValueError, match="sizes up to"):
        embedding(torch.zeros(1, dtype=torch.long), e.expand(1, (1 << 31) + 5))


def test_recurrence_workspace_alignment_is_refused():
    so = _lib.lib()
    for name in ("ngdn_recurrence_fwd", "ngdn_recurrence_bwd"):
        assert getattr(so, name)(1, ctypes.byref(_args(ws=4100)), None) == 1
        assert b"aligned" in so.ngdn_last_error()


def test_embedding_module_is_traced_as_torchs():
    m = torch.nn.Sequential(Embedding(7, 3))
    ids = torch.tensor([1, 6])
    assert torch.equal(torch.fx.symbolic_trace(m)(ids), m(ids))


def test_states_of_other_types_are_refused():
    x, h = torch.zeros(1, 2, 4), torch.zeros(1, 4)
    for bad in (h.double(), h.long()):
        with pytest.raises(ValueError, match="the state is"):
            gated_recurrence(x, x, x, h[0, :2], h[0], initial_state=bad)
        with pytest.raises(ValueError, match="the state is"):
            step_gated_recurrence(h, h, h, h[0, :2], h[0], bad)


def test_import_without_torchs_gpu_names():
    """A torch built without a GPU has none of the names that read its streams:
    the package (schedules, the layer's configuration, modules on the CPU) imports."""
    import os
    import subprocess
    import sys
    code = ("import torch\n"
            "del torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice\n"
            "from nested_recurrent_memory_amd import NestedGDN2LayerConfig, n_firings\n"
            "from nested_recurrent_memory_amd.model_ops import Embedding\n"
            "NestedGDN2LayerConfig()\n"
            "assert Embedding(3, 2)(torch.tensor([1])).shape == (1, 2)\n")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr


def test_step_refuses_forward_mode():
    """Forward-mode tangents have no way through the step: refused, not dropped.
    A dual level without tangents changes nothing."""
    from torch.autograd import forward_ad
    x, A, h = torch.zeros(1, 4), torch.zeros(2), torch.zeros(1, 4)
    args = [x, x, x, A, h[0], h]
    with forward_ad.dual_level():
        for i in range(6):
            a = list(args)
            a[i] = forward_ad.make_dual(a[i], torch.ones_like(a[i]))
            with pytest.raises(RuntimeError, match="forward-only"):
                step_gated_recurrence(*a)
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-only"):
                step_gated_recurrence(*a)
        with pytest.raises(ValueError, match="no CPU path"):
            step_gated_recurrence(*args)


def test_a_node_of_another_interface_is_refused(monkeypatch):
    """The C++ node describes one interface, as the library does; without it the
    message says what to build."""
    import sys
    import nested_recurrent_memory_amd as package
    _lib.node()
    monkeypatch.setattr(_lib, "_nodes", None)
    with monkeypatch.context() as m:
        m.setattr(_lib, "VERSION", 1)
        with pytest.raises(_lib.NgdnError, match="rebuild"):
            _lib.node()
    monkeypatch.delattr(package, "_node")
    monkeypatch.setitem(sys.modules, package.__name__ + "._node", None)
    with pytest.raises(_lib.NgdnError, match="build it"):
        _lib.node()
