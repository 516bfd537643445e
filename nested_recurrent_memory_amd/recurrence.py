"""A gated linear recurrence with a vector state, on the HIP kernels of
libngdn.so (csrc/recurrence.hip, entry points in include/ngdn.h).

Beside ``chunk_nested_gdn2`` (a matrix state a head, a delta rule, levels)
the plain form of such a memory: one state value a channel, a decay and a
write gate from the token. With the decay parameters of the layer's gate
prologue (``NestedGDN2Attention.A_log``, ``dt_bias``):

    g_t = -exp(A_log) softplus(f_t + dt_bias)            log decay, <= 0
    h_t = exp(g_t) h_(t-1) + sqrt(1 - exp(2 g_t)) sigmoid(wz_t) x_t
    y_t = h_t

* ``gated_recurrence``: whole sequences, forward and backward, rows of one
  length (the padding of a shorter one is tokens like the others) or packed
  sequences, a state in and out.
* ``step_gated_recurrence``: one token, for decoding. Forward only.

Inputs all in bfloat16 or all in float32 run on the kernels as they are, float16
and mixed types in float32; states and the decay parameters are float32 in the kernels. There is
no fallback: without the library (or on tensors off the GPU) the calls raise.
"""

from __future__ import annotations

import ctypes

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib

__all__ = ["gated_recurrence", "step_gated_recurrence"]


def _code(dtype):
    return _lib.NGDN_BF16 if dtype == torch.bfloat16 else _lib.NGDN_F32


def _on_gpu(name, *ts):
    # the kernels take raw device pointers: a host tensor must never reach them
    dev = ts[0].device
    for t in ts:
        if t is not None and (not t.is_cuda or t.device != dev):
            raise ValueError(f"{name}: every tensor must be on one GPU (got {t.device}); "
                             "there is no CPU path")


def _rows(t, dtype):
    """t in dtype with its last dimension consecutive: the kernels take any
    other strides."""
    if t.dtype != dtype:
        t = t.to(dtype)
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _f32(t):
    if t is None:
        return None
    if t.dtype != torch.float32:
        t = t.to(torch.float32)
    return t if t.is_contiguous() else t.contiguous()


_TYPES = (torch.bfloat16, torch.float16, torch.float32)
_MOST = (1 << 31) - 1           # of any size, which the library takes in 32 bits


def _work_type(x, f, wz):
    """The kernels' type: a narrower one than a tensor's own would lose its bits."""
    same = x.dtype == f.dtype == wz.dtype == torch.bfloat16
    return torch.bfloat16 if same else torch.float32


def _token_args(B, T, D, x, f, wz, A_log, dt_bias):
    a = _lib.RecurrenceArgs()
    a.B, a.T, a.D, a.H = B, T, D, A_log.shape[0]
    a.x, a.f, a.wz = x.data_ptr(), f.data_ptr(), wz.data_ptr()
    a.A_log, a.dt_bias = A_log.data_ptr(), dt_bias.data_ptr()
    a.x_b, a.f_b, a.w_b = x.stride(0), f.stride(0), wz.stride(0)
    return a


def _sequence_args(x, f, wz, A_log, dt_bias, h0, cu):
    a = _token_args(*x.shape, x, f, wz, A_log, dt_bias)
    a.x_t, a.f_t, a.w_t = x.stride(1), f.stride(1), wz.stride(1)
    if cu is not None:
        a.S, a.cu = cu.shape[0] - 1, cu.data_ptr()
    if h0 is not None:
        a.h0 = h0.data_ptr()
    return a


def _forward(x, f, wz, A_log, dt_bias, h0, cu, want_final, train):
    """y in the work type, the final state, and what the backward reads."""
    B, T, D = x.shape
    wd = _work_type(x, f, wz)
    xw, fw, ww = _rows(x, wd), _rows(f, wd), _rows(wz, wd)
    A, dt, h = _f32(A_log), _f32(dt_bias), _f32(h0)
    if cu is not None:
        cu = cu.to(torch.int32).contiguous()
    rows = B if cu is None else cu.shape[0] - 1
    dev = x.device
    y = torch.empty((B, T, D), device=dev, dtype=wd)
    final = torch.empty((rows, D), device=dev, dtype=torch.float32) if want_final else None
    hs = None
    if y.numel() == 0 or rows == 0:       # no token: the states stay
        y.zero_()
        if want_final:
            final.copy_(h) if h is not None else final.zero_()
    else:
        a = _sequence_args(xw, fw, ww, A, dt, h, cu)
        ws = torch.empty(_lib.lib().ngdn_recurrence_ws(B, T, D, 0), device=dev, dtype=torch.float32)
        a.y, a.final_state, a.ws = y.data_ptr(), _lib.ptr(final), ws.data_ptr()
        if train:
            hs = torch.empty((B, -(-T // _lib.REC_RUN), D), device=dev, dtype=torch.float32)
            a.hs = hs.data_ptr()
        _lib.on_device(y, "ngdn_recurrence_fwd", _code(wd), ctypes.byref(a))
    return y, final, (xw, fw, ww, A, dt, h, cu, hs)


class _RecurrenceFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, f, wz, A_log, dt_bias, h0, cu, want_final):
        y, final, saved = _forward(x, f, wz, A_log, dt_bias, h0, cu, want_final, True)
        ctx.save_for_backward(*saved)
        wd, f32 = y.dtype, torch.float32
        types = (x.dtype, f.dtype, wz.dtype, A_log.dtype, dt_bias.dtype, f32 if h0 is None else h0.dtype)
        ctx.dtypes = None if types == (wd, wd, wd, f32, f32, f32) else types
        ctx.set_materialize_grads(False)
        return y if y.dtype == x.dtype else y.to(x.dtype), final

    @staticmethod
    def backward(ctx, dy, dfinal):
        # once_differentiable's wrapping costs 3 us and is for a backward that a graph is made of
        return (_backward_once if torch.is_grad_enabled() else _backward)(ctx, dy, dfinal)


def _backward(ctx, dy, dfinal):
    xw, fw, ww, A, dt, h, cu, hs = ctx.saved_tensors
    B, T, D = xw.shape
    wd, dev = xw.dtype, xw.device
    rows = B if cu is None else cu.shape[0] - 1
    dh0 = torch.empty((rows, D), device=dev, dtype=torch.float32) if ctx.needs_input_grad[5] else None
    dx = torch.empty((B, T, D), device=dev, dtype=wd)
    df, dw = torch.empty_like(dx), torch.empty_like(dx)
    dA, ddt = torch.empty_like(A), torch.empty_like(dt)
    dfinal = _f32(dfinal)
    if hs is None:
        for t in (dx, df, dw, dA, ddt):
            t.zero_()
        if dh0 is not None:
            dh0.copy_(dfinal) if dfinal is not None else dh0.zero_()
    else:
        dyw = _rows(dy, wd) if dy is not None else torch.zeros_like(dx)
        a = _sequence_args(xw, fw, ww, A, dt, h, cu)
        ws = torch.empty(_lib.lib().ngdn_recurrence_ws(B, T, D, 1), device=dev, dtype=torch.float32)
        a.hs, a.ws, a.dy, a.dfinal = hs.data_ptr(), ws.data_ptr(), dyw.data_ptr(), _lib.ptr(dfinal)
        a.dy_b, a.dy_t = dyw.stride(0), dyw.stride(1)
        a.dx, a.df, a.dwz = dx.data_ptr(), df.data_ptr(), dw.data_ptr()
        a.dA_log, a.ddt_bias, a.dh0 = dA.data_ptr(), ddt.data_ptr(), _lib.ptr(dh0)
        _lib.on_device(dx, "ngdn_recurrence_bwd", _code(wd), ctypes.byref(a))
    grads = (dx, df, dw, dA, ddt, dh0)
    if ctx.dtypes:
        grads = (g if g is None else g.to(d) for g, d in zip(grads, ctx.dtypes))
    return *grads, None, None


_backward_once = once_differentiable(_backward)


def _check(name, x, f, wz, A_log, dt_bias, state, dims):
    if x.dim() != dims or f.shape != x.shape or wz.shape != x.shape:
        want = "[B,T,D]" if dims == 3 else "[B,D]"
        raise ValueError(f"{name}: x {tuple(x.shape)}, f {tuple(f.shape)}, wz {tuple(wz.shape)} "
                         f"(all {want})")
    D = x.shape[-1]
    if D < 1 or dt_bias.shape != (D,) or A_log.dim() != 1 or A_log.shape[0] < 1 or D % A_log.shape[0]:
        raise ValueError(f"{name}: dt_bias {tuple(dt_bias.shape)}, A_log {tuple(A_log.shape)} for "
                         f"D={D} (dt_bias [D], A_log [H] with D a multiple of H)")
    if max(x.shape) > _MOST:
        raise ValueError(f"{name}: x {tuple(x.shape)} (sizes up to {_MOST})")
    for n, t in (("x", x), ("f", f), ("wz", wz), ("A_log", A_log), ("dt_bias", dt_bias), ("the state", state)):
        if t is not None and t.dtype not in _TYPES:
            raise ValueError(f"{name}: {n} is {t.dtype} (bf16, fp16 or fp32)")


def gated_recurrence(x, f, wz, A_log, dt_bias, initial_state=None, output_final_state=False,
                     cu_seqlens=None):
    """x, f, wz [B,T,D] (the values, the decay and the write gate before their
    softplus and sigmoid; column slices of one projection are read as they
    are); dt_bias [D]; A_log [H] with D a multiple of H, head h having the
    channels h D/H .. (h + 1) D/H - 1 (H = D: a decay for every channel).
    Returns (y [B,T,D] in x's dtype, the final state fp32 or None).

    Without cu_seqlens every row of the batch is a sequence of all T tokens (one
    padded behind its end has a final state behind the padding); initial_state
    and the final state are [B,D]. With cu_seqlens (int tensor [S+1] on the GPU,
    0 <= cu_seqlens[0] <= ... <= cu_seqlens[S] <= T; its values are not
    checked) B is 1 and tokens cu_seqlens[s] .. cu_seqlens[s+1] - 1 are
    sequence s; the states are [S,D], and an empty sequence keeps its state.
    Tokens in no sequence have y = 0 and no effect on anything.

    Differentiable once in every tensor (not forward-mode); gradients have the
    bits of every other run on the same inputs. To capture the backward into a
    graph, let no eager graph of the same leaves live: autograd would then
    leave the captured stream."""
    _check("gated_recurrence", x, f, wz, A_log, dt_bias, initial_state, 3)
    B, T, D = x.shape
    rows = B
    if cu_seqlens is not None:
        if (B != 1 or cu_seqlens.dim() != 1 or not 1 <= cu_seqlens.shape[0] <= _MOST
                or cu_seqlens.dtype not in (torch.int32, torch.int64)):
            raise ValueError(f"gated_recurrence: cu_seqlens {cu_seqlens.dtype} {tuple(cu_seqlens.shape)} "
                             f"with B={B} (int32 or int64 [S+1], B = 1)")
        rows = cu_seqlens.shape[0] - 1
    if initial_state is not None and tuple(initial_state.shape) != (rows, D):
        raise ValueError(f"gated_recurrence: initial_state {tuple(initial_state.shape)}, expected "
                         f"{(rows, D)}")
    _on_gpu("gated_recurrence", x, f, wz, A_log, dt_bias, initial_state, cu_seqlens)
    args = (x, f, wz, A_log, dt_bias, initial_state, cu_seqlens, bool(output_final_state))
    if forward_ad._current_level < 0 and not (torch.is_grad_enabled() and any(
            t is not None and t.requires_grad for t in args[:6])):
        y, final, _ = _forward(*args, False)
        return y if y.dtype == x.dtype else y.to(x.dtype), final
    return _RecurrenceFn.apply(*args)


def step_gated_recurrence(x, f, wz, A_log, dt_bias, state, *, inplace=False):
    """One token of B sequences: x, f, wz [B,D], state [B,D]. Returns (y [B,D]
    in x's dtype, the new state [B,D] fp32). The state passed in is not
    modified, or with ``inplace=True`` (fp32, contiguous) updated and
    returned, which keeps the buffer fixed for graph capture. Forward only: inputs
    that want a gradient or carry a forward-mode tangent are refused."""
    name = "step_gated_recurrence"
    _check(name, x, f, wz, A_log, dt_bias, state, 2)
    B, D = x.shape
    if tuple(state.shape) != (B, D):
        raise ValueError(f"{name}: state {tuple(state.shape)}, expected {(B, D)}")
    if forward_ad._current_level >= 0 and any(
            forward_ad.unpack_dual(t).tangent is not None for t in (x, f, wz, A_log, dt_bias, state)):
        raise RuntimeError(f"{name} is forward-only (decoding): no tangent goes through it")
    _on_gpu(name, x, f, wz, A_log, dt_bias, state)
    if torch.is_grad_enabled() and any(t.requires_grad for t in (x, f, wz, A_log, dt_bias, state)):
        raise RuntimeError(f"{name} is forward-only (decoding); call it under torch.no_grad() or on "
                           "tensors that do not require grad")
    wd = _work_type(x, f, wz)
    xw, fw, ww = _rows(x, wd), _rows(f, wd), _rows(wz, wd)
    A, dt = _f32(A_log), _f32(dt_bias)
    if inplace:
        if state.dtype != torch.float32 or not state.is_contiguous():
            raise ValueError(f"{name}: inplace=True needs a contiguous fp32 state")
        s_in = s_out = state
        if not state.is_inference():        # a graph that saved it must not use the new values
            torch.autograd.graph.increment_version(state)
    else:
        s_in = _f32(state)
        s_out = torch.empty_like(s_in)
    y = torch.empty((B, D), device=x.device, dtype=wd)
    if B:
        a = _token_args(B, 1, D, xw, fw, ww, A, dt)
        a.h0, a.final_state, a.y = s_in.data_ptr(), s_out.data_ptr(), y.data_ptr()
        _lib.on_device(y, "ngdn_recurrence_step", _code(wd), ctypes.byref(a))
    return y if y.dtype == x.dtype else y.to(x.dtype), s_out
