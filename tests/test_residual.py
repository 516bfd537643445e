"""Dropout, the residual norm and the sampler on the CPU: their oracle, and what
their entry points refuse."""

import ctypes

import pytest
import torch

import ngdn_residual_oracle as oracle
from nested_recurrent_memory_amd import _lib
from nested_recurrent_memory_amd.model_ops import dropout, residual_norm, sample_tokens


def test_generator_gives_the_published_words():
    """Known answers of Philox4x32 with seven rounds, and that the two forms of
    the oracle agree beyond 32 bits of seed and offset."""
    assert oracle.words(0, 4, 0, 0) == [0x5f6fb709, 0x0d893f64, 0x4f121f81, 0x4f730a48]
    for seed, offset in ((0, 0), (2 ** 63 + 12345, 2 ** 40 + 1), (2 ** 64 - 1, 2 ** 64 - 1)):
        assert oracle.words(0, 11, seed, offset) == oracle.words_np(11, seed, offset).tolist()
    assert oracle.words(3, 6, 7, 9) == oracle.words_np(9, 7, 9)[3:].tolist()


def _args(gate, B=2, T=3, D=5, post=True):
    g = torch.Generator().manual_seed(D + 10 * T)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    a = dict(x=r(B, T, D), branch=r(B, T, D), weight=1 + 0.1 * r(D), post_weight=1 + 0.1 * r(D) if post else None,
             gate=None)
    if gate:
        a["gate"] = r(*{"channel": (D,), "sequence": (B, 1, D), "token": (B, T, 1), "full": (B, T, D)}[gate])
    return a, r(B, T, D), r(B, T, D)


@pytest.mark.parametrize("p", [0.0, 0.3])
@pytest.mark.parametrize("gate", [None, "channel", "sequence", "token", "full"])
def test_oracle_gradients_are_differences(gate, p):
    """Central differences in float64 with a step of 1e-5: their own error is of
    the order of 1e-10 of the third derivatives plus 1e-11 of rounding."""
    a, dh, dy = _args(gate, post=p == 0)
    kw = dict(residual_scale=0.7, branch_scale=1.5, p=p, seed=3, offset=1)
    o = oracle.residual_norm(**a, **kw, dh=dh, dy=dy)

    def loss():
        v = oracle.residual_norm(**a, **kw)
        return ((v["h"][0] * dh).sum() + (v["y"][0] * dy).sum()).item()

    for name, t in a.items():
        if t is None:
            continue
        want, flat = o["d" + name][0], t.view(-1)
        assert want.shape == t.shape
        for i in range(t.numel()):
            keep = flat[i].item()
            flat[i] = keep + 1e-5
            up = loss()
            flat[i] = keep - 1e-5
            down = loss()
            flat[i] = keep
            assert abs((up - down) / 2e-5 - want.reshape(-1)[i].item()) < 1e-6, (name, i)


def test_oracle_sampler():
    """By hand: weights 1, 1/2, 1/4, 1/8 at places 2, 0, 3, 1."""
    l = torch.log(torch.tensor([[0.5, 0.125, 1.0, 0.25]], dtype=torch.float64))
    pick = lambda u, **kw: oracle.sample(l, [u], **kw).item()  # noqa: E731
    assert [pick(u) for u in (0.0, 0.26, 0.27, 0.33, 0.34, 0.86, 0.87, 0.99)] == [0, 0, 1, 1, 2, 2, 3, 3]
    assert [pick(u, top_k=2) for u in (0.3, 0.34)] == [0, 2]
    assert [pick(u, top_p=0.5) for u in (0.0, 0.99)] == [2, 2]
    assert [pick(u, top_p=0.54) for u in (0.3, 0.34)] == [0, 2]
    assert [pick(u, min_p=0.3) for u in (0.3, 0.34)] == [0, 2]
    assert pick(0.9, temperature=0.0) == 2


def refused(match, fn, *args, **kw):
    with pytest.raises(ValueError, match=match):
        fn(*args, **kw)


def test_dropout_refuses():
    x = torch.randn(3, 4)
    refused("no CPU path", dropout, x, 0.1, 0)
    refused("no CPU path", dropout, x.to("meta"), 0.1, 0)
    refused("no CPU path", dropout, x, 0.1, torch.zeros(1, dtype=torch.long))
    refused("x is Double", dropout, x.double(), 0.1, 0)
    refused("x is Long", dropout, x.long(), 0.1, 0)
    for p in (-0.1, 1.1, float("nan")):
        refused("p .* outside", dropout, x, p, 0)
    refused("seed must be an integer", dropout, x, 0.1, 0.5)
    refused("seed must be an integer", dropout, x, 0.1, True)
    refused("offset must be an integer", dropout, x, 0.1, 0, "1")
    refused("one int64", dropout, x, 0.1, torch.zeros(2, dtype=torch.long))
    refused("one int64", dropout, x, 0.1, torch.zeros(1))


def test_residual_norm_refuses():
    x, w = torch.randn(2, 3, 4), torch.randn(4)
    refused("no CPU path", residual_norm, x, x)
    refused("no CPU path", residual_norm, x.to("meta"), x.to("meta"), w.to("meta"))
    refused("one shape", residual_norm, x, x[:, :2])
    refused("one shape", residual_norm, x[0, 0, 0], x[0, 0, 0])
    refused("rows of 16385", residual_norm, torch.zeros(1, 16385), torch.zeros(1, 16385))
    refused("rows of 0", residual_norm, x[..., :0], x[..., :0])
    refused("x is Double", residual_norm, x.double(), x)
    refused("branch is Double", residual_norm, x, x.double())
    refused("weight \\(3", residual_norm, x, x, w[:3])
    refused("weight is Double", residual_norm, x, x, w.double())
    refused("post_weight \\(1, 4", residual_norm, x, x, w, post_weight=w[None])
    for bad in (w[:3], x[:, :, :2], x[:, :1, :1], x[:1, :, :], x[0], x[0, :, :1], x[..., None], w[0], torch.ones(1, 1, 1)):
        refused("gate .* for x", residual_norm, x, x, w, gate=bad)
    refused("gate is Double", residual_norm, x, x, w, gate=w.double())
    refused("p .* outside", residual_norm, x, x, w, p=1.5)
    refused("seed must be", residual_norm, x, x, w, p=0.5, seed=None)
    refused("eps", residual_norm, x, x, w, eps=-1.0)
    refused("eps", residual_norm, x, x, w, eps=float("nan"))
    refused("out_dtype Double", residual_norm, x, x, w, out_dtype=torch.float64)


def test_sample_tokens_refuses():
    l, u = torch.randn(2, 5), torch.rand(2)
    refused("no CPU path", sample_tokens, l, u)
    refused("no CPU path", sample_tokens, l.to("meta"), u.to("meta"))
    refused("logits is Double", sample_tokens, l.double(), u)
    refused("u ", sample_tokens, l, u[:1])
    refused("u is BFloat16", sample_tokens, l, u.bfloat16())
    refused("2\\^20", sample_tokens, torch.zeros(1, (1 << 20) + 1), u[:1])
    refused("logits \\(2, 0\\)", sample_tokens, l[:, :0], u)
    for bad in (-0.5, float("inf"), float("nan")):
        refused("temperature", sample_tokens, l, u, bad)
    for bad in (-0.1, 1.1, float("nan")):
        refused("top_p", sample_tokens, l, u, 1.0, 0, bad)
        refused("min_p", sample_tokens, l, u, min_p=bad)
    refused("top_k must be an integer", sample_tokens, l, u, top_k=2.5)
    refused("top_k is Float", sample_tokens, l, u, top_k=u)
    refused("temperature is Long", sample_tokens, l, u, u.long())
    refused("top_p \\(1\\)", sample_tokens, l, u, top_p=u[:1])
    refused("no CPU path", sample_tokens, l, u, u)


class Residual(ctypes.Structure):
    """ngdn_residual_args of include/ngdn.h."""
    _fields_ = ([(n, ctypes.c_int64) for n in ("rows", "seq")] +
                [(n, ctypes.c_int32) for n in ("D", "gate_kind", "x_dtype", "branch_dtype", "y_dtype", "w_dtype",
                                               "pw_dtype", "gate_dtype")] +
                [(n, ctypes.c_float) for n in ("residual_scale", "branch_scale", "eps", "keep")] +
                [(n, ctypes.c_int64) for n in ("threshold", "seed", "offset")] +
                [(n, ctypes.c_void_p) for n in ("seed_ptr", "x", "branch", "weight", "post_weight", "gate", "h", "y",
                                                "rstd_h", "rstd_b", "dh", "dy", "dx", "dbranch", "dweight",
                                                "dpost_weight", "dgate", "ws")])


class Sample(ctypes.Structure):
    """ngdn_sample_args of include/ngdn.h."""
    _fields_ = ([(n, ctypes.c_int64) for n in ("rows", "stride")] +
                [(n, ctypes.c_int32) for n in ("V", "u_wide", "top_k_wide")] +
                [(n, ctypes.c_float) for n in ("temperature", "top_p", "min_p")] + [("top_k", ctypes.c_int64)] +
                [(n, ctypes.c_void_p) for n in ("logits", "u", "temperature_ptr", "top_p_ptr", "min_p_ptr",
                                                "top_k_ptr", "token")])


def test_entry_points_refuse_before_any_launch():
    so = _lib.lib()
    said = lambda text: text in so.ngdn_last_error()  # noqa: E731
    x = ctypes.c_void_p(4096)           # never dereferenced
    assert so.ngdn_dropout(2, 8, 1, 1.0, 0, None, 0, x, x, None) == 1 and said(b"dtype 2")
    assert so.ngdn_dropout(0, 8, 0, 1.0, 0, None, 0, x, x, None) == 1 and said(b"threshold 0")
    assert so.ngdn_dropout(0, 8, 2 ** 32 + 1, 1.0, 0, None, 0, x, x, None) == 1 and said(b"threshold")
    assert so.ngdn_dropout(0, -1, 1, 1.0, 0, None, 0, x, x, None) == 1 and said(b"n=-1")
    assert so.ngdn_dropout(0, 8, 1, 1.0, 0, None, 0, None, x, None) == 1 and said(b"NULL")
    assert so.ngdn_dropout(0, 0, 1, 1.0, 0, None, 0, None, None, None) == 0      # nothing to do

    def norm(fn="ngdn_residual_norm_fwd", **kw):
        a = Residual(rows=4, D=8, branch_scale=1, residual_scale=1, eps=1e-5, x=4096, branch=4096, h=4096, ws=4096)
        for n, v in kw.items():
            setattr(a, n, v)
        return getattr(so, fn)(ctypes.byref(a), None)

    for kw, text in ((dict(D=0), b"D=0"), (dict(D=16385), b"D=16385"), (dict(rows=-1), b"rows=-1"),
                     (dict(x_dtype=1), b"dtypes 1, 0, 0"), (dict(y_dtype=3), b"dtypes 0, 0, 3"),
                     (dict(w_dtype=7), b"parameter dtype 7"), (dict(gate_kind=5), b"gate_kind 5"),
                     (dict(gate_kind=1), b"NULL"), (dict(gate_kind=2, gate=4096, seq=3), b"seq=3"),
                     (dict(gate_kind=2, gate=4096, seq=0), b"seq=0"), (dict(threshold=-1), b"threshold -1"),
                     (dict(weight=4096), b"NULL"), (dict(branch=None), b"NULL")):
        assert norm(**kw) == 1 and said(text), (kw, so.ngdn_last_error())
    for kw, text in ((dict(dy=4096), b"without its parameter"), (dict(dpost_weight=4096), b"without its parameter"),
                     (dict(dgate=4096), b"without its parameter"), (dict(weight=4096, dy=4096), b"NULL"),
                     (dict(post_weight=4096), b"NULL"), (dict(ws=None), b"NULL")):
        assert norm("ngdn_residual_norm_bwd", **kw) == 1 and said(text), (kw, so.ngdn_last_error())
    assert norm(rows=0, x=None, branch=None, h=None) == 0
    assert so.ngdn_residual_norm_ws(ctypes.byref(Residual(rows=4, D=0))) == -1

    def sample(dtype=0, **kw):
        a = Sample(rows=2, V=5, stride=5, temperature=1, top_p=1, logits=4096, u=4096, token=4096)
        for n, v in kw.items():
            setattr(a, n, v)
        return so.ngdn_sample(dtype, ctypes.byref(a), None)

    for kw, text in ((dict(dtype=3), b"dtype 3"), (dict(V=0), b"V=0"), (dict(V=(1 << 20) + 1), b"V=1048577"),
                     (dict(rows=1 << 22), b"rows="), (dict(u=None), b"NULL"), (dict(token=None), b"NULL")):
        assert sample(**kw) == 1 and said(text), (kw, so.ngdn_last_error())
    assert sample(rows=0, logits=None) == 0
    assert so.ngdn_sample(0, None, None) == 1 and said(b"args is NULL")
