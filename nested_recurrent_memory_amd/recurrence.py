"""A gated linear recurrence with a vector state, on the HIP kernels of
libngdn.so (csrc/recurrence.hip, entry points in include/ngdn.h).

Beside ``chunk_nested_gdn2`` (a matrix state a head, a delta rule, levels)
the plain form of such a memory: one state value a channel, a decay and a
write gate from the token. With the decay parameters of the layer's gate
prologue (``NestedGDN2Attention.A_log``, ``dt_bias``):

    g_t = -exp(A_log) softplus(f_t + dt_bias)            log decay, <= 0
    h_t = exp(g_t) h_(t-1) + sqrt(1 - exp(2 g_t)) sigmoid(wz_t) x_t
    y_t = h_t

* ``gated_recurrence``: whole sequences, forward and backward, padded batches
  or packed sequences, a state in and out.
* ``step_gated_recurrence``: one token, for decoding. Forward only.

Inputs in bfloat16 or float32 run on the kernels as they are, float16 in
float32; states and the decay parameters are float32 in the kernels. There is
no fallback: without the library (or on tensors off the GPU) the calls raise.
"""

from __future__ import annotations

import ctypes

import torch
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


def _call(name, dtype, args, t):
    # on t's device, whichever is current: a launch needs its stream's device
    if t.device.index == torch.cuda.current_device():
        _lib.call(name, _code(dtype), ctypes.byref(args), _lib.stream_of(t))
    else:
        with torch.cuda.device(t.device):
            _lib.call(name, _code(dtype), ctypes.byref(args), _lib.stream_of(t))


def _rows(t, dtype):
    """t in dtype with its last dimension consecutive: the kernels take any
    other strides."""
    t = t.to(dtype)
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _f32(t):
    return None if t is None else t.to(torch.float32).contiguous()


def _fill(args, B, T, D, x, f, wz, A_log, dt_bias):
    args.B, args.T, args.D, args.H = B, T, D, A_log.shape[0]
    args.x, args.f, args.wz = x.data_ptr(), f.data_ptr(), wz.data_ptr()
    args.A_log, args.dt_bias = A_log.data_ptr(), dt_bias.data_ptr()
    args.x_b, args.f_b, args.w_b = x.stride(0), f.stride(0), wz.stride(0)
    return args


def _sequence_args(x, f, wz, A_log, dt_bias, h0, cu):
    B, T, D = x.shape
    a = _fill(_lib.RecurrenceArgs(), B, T, D, x, f, wz, A_log, dt_bias)
    a.x_t, a.f_t, a.w_t = x.stride(1), f.stride(1), wz.stride(1)
    if cu is not None:
        a.S, a.cu = cu.shape[0] - 1, cu.data_ptr()
    a.h0 = _lib.ptr(h0)
    return a


class _RecurrenceFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, f, wz, A_log, dt_bias, h0, cu, want_final):
        B, T, D = x.shape
        wd = x.dtype if x.dtype in (torch.bfloat16, torch.float32) else torch.float32
        xw, fw, ww = (_rows(t, wd) for t in (x, f, wz))
        A, dt, h = _f32(A_log), _f32(dt_bias), _f32(h0)
        cu = cu.to(torch.int32).contiguous() if cu is not None else None
        rows = B if cu is None else cu.shape[0] - 1
        y = torch.empty(B, T, D, device=x.device, dtype=wd)
        final = torch.empty(rows, D, device=x.device, dtype=torch.float32) if want_final else None
        hs = None
        if y.numel() == 0 or rows == 0:       # no token: the states stay
            y.zero_()
            if want_final:
                final.copy_(h) if h is not None else final.zero_()
        else:
            a = _sequence_args(xw, fw, ww, A, dt, h, cu)
            nseg = -(-T // _lib.REC_RUN)
            hs = torch.empty(B, nseg, D, device=x.device, dtype=torch.float32)
            ws = torch.empty(_lib.lib().ngdn_recurrence_ws(B, T, D, 0), device=x.device,
                             dtype=torch.float32)
            a.y, a.final_state, a.hs, a.ws = y.data_ptr(), _lib.ptr(final), hs.data_ptr(), ws.data_ptr()
            _call("ngdn_recurrence_fwd", wd, a, x)
        ctx.save_for_backward(xw, fw, ww, A, dt, h, cu, hs)
        ctx.dtypes = tuple(t.dtype if t is not None else None for t in (x, f, wz, A_log, dt_bias, h0))
        ctx.set_materialize_grads(False)
        return y.to(x.dtype), final

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dfinal):
        xw, fw, ww, A, dt, h, cu, hs = ctx.saved_tensors
        B, T, D = xw.shape
        wd, dev = xw.dtype, xw.device
        rows = B if cu is None else cu.shape[0] - 1
        dh0 = torch.empty(rows, D, device=dev, dtype=torch.float32) if ctx.needs_input_grad[5] else None
        dx, df, dw = (torch.empty(B, T, D, device=dev, dtype=wd) for _ in range(3))
        dA, ddt = torch.empty_like(A), torch.empty_like(dt)
        dfinal = _f32(dfinal)
        if hs is None:
            for t in (dx, df, dw, dA, ddt):
                t.zero_()
            if dh0 is not None:
                dh0.copy_(dfinal) if dfinal is not None else dh0.zero_()
        else:
            dyw = _rows(dy, wd) if dy is not None else torch.zeros(B, T, D, device=dev, dtype=wd)
            a = _sequence_args(xw, fw, ww, A, dt, h, cu)
            ws = torch.empty(_lib.lib().ngdn_recurrence_ws(B, T, D, 1), device=dev, dtype=torch.float32)
            a.hs, a.ws, a.dy, a.dfinal = hs.data_ptr(), ws.data_ptr(), dyw.data_ptr(), _lib.ptr(dfinal)
            a.dy_b, a.dy_t = dyw.stride(0), dyw.stride(1)
            a.dx, a.df, a.dwz = dx.data_ptr(), df.data_ptr(), dw.data_ptr()
            a.dA_log, a.ddt_bias, a.dh0 = dA.data_ptr(), ddt.data_ptr(), _lib.ptr(dh0)
            _call("ngdn_recurrence_bwd", wd, a, xw)
        return tuple(g.to(d) if g is not None else None
                     for g, d in zip((dx, df, dw, dA, ddt, dh0), ctx.dtypes)) + (None, None)


def _check(name, x, f, wz, A_log, dt_bias, dims):
    if x.dim() != dims or f.shape != x.shape or wz.shape != x.shape:
        want = "[B,T,D]" if dims == 3 else "[B,D]"
        raise ValueError(f"{name}: x {tuple(x.shape)}, f {tuple(f.shape)}, wz {tuple(wz.shape)} "
                         f"(all {want})")
    D = x.shape[-1]
    if D < 1 or dt_bias.shape != (D,) or A_log.dim() != 1 or A_log.shape[0] < 1 or D % A_log.shape[0]:
        raise ValueError(f"{name}: dt_bias {tuple(dt_bias.shape)}, A_log {tuple(A_log.shape)} for "
                         f"D={D} (dt_bias [D], A_log [H] with D a multiple of H)")
    for n, t in (("x", x), ("f", f), ("wz", wz), ("A_log", A_log), ("dt_bias", dt_bias)):
        if t.dtype not in (torch.bfloat16, torch.float16, torch.float32):
            raise ValueError(f"{name}: {n} is {t.dtype} (bf16, fp16 or fp32)")


def gated_recurrence(x, f, wz, A_log, dt_bias, initial_state=None, output_final_state=False,
                     cu_seqlens=None):
    """x, f, wz [B,T,D] (the values, the decay and the write gate before their
    softplus and sigmoid; column slices of one projection are read as they
    are); dt_bias [D]; A_log [H] with D a multiple of H, head h having the
    channels h D/H .. (h + 1) D/H - 1 (H = D: a decay for every channel).
    Returns (y [B,T,D] in x's dtype, the final state fp32 or None).

    Without cu_seqlens every row of the batch is a sequence; initial_state and
    the final state are [B,D]. With cu_seqlens (int tensor [S+1] on the GPU,
    0 <= cu_seqlens[0] <= ... <= cu_seqlens[S] <= T; its values are not
    checked) B is 1 and tokens cu_seqlens[s] .. cu_seqlens[s+1] - 1 are
    sequence s; the states are [S,D], and an empty sequence keeps its state.
    Tokens in no sequence have y = 0 and no effect on anything.

    Differentiable once in every tensor; gradients have the bits of every
    other run on the same inputs."""
    _check("gated_recurrence", x, f, wz, A_log, dt_bias, 3)
    B, T, D = x.shape
    rows = B
    if cu_seqlens is not None:
        if (B != 1 or cu_seqlens.dim() != 1 or cu_seqlens.shape[0] < 1
                or cu_seqlens.dtype not in (torch.int32, torch.int64)):
            raise ValueError(f"gated_recurrence: cu_seqlens {cu_seqlens.dtype} {tuple(cu_seqlens.shape)} "
                             f"with B={B} (int32 or int64 [S+1], B = 1)")
        rows = cu_seqlens.shape[0] - 1
    if initial_state is not None and tuple(initial_state.shape) != (rows, D):
        raise ValueError(f"gated_recurrence: initial_state {tuple(initial_state.shape)}, expected "
                         f"{(rows, D)}")
    _on_gpu("gated_recurrence", x, f, wz, A_log, dt_bias, initial_state, cu_seqlens)
    return _RecurrenceFn.apply(x, f, wz, A_log, dt_bias, initial_state, cu_seqlens,
                               bool(output_final_state))


def step_gated_recurrence(x, f, wz, A_log, dt_bias, state, *, inplace=False):
    """One token of B sequences: x, f, wz [B,D], state [B,D]. Returns (y [B,D]
    in x's dtype, the new state [B,D] fp32). The state passed in is not
    modified, or with ``inplace=True`` (fp32, contiguous) updated and
    returned, which keeps the buffer fixed for graph capture. Forward only."""
    name = "step_gated_recurrence"
    _check(name, x, f, wz, A_log, dt_bias, 2)
    B, D = x.shape
    if tuple(state.shape) != (B, D):
        raise ValueError(f"{name}: state {tuple(state.shape)}, expected {(B, D)}")
    _on_gpu(name, x, f, wz, A_log, dt_bias, state)
    if torch.is_grad_enabled() and any(t.requires_grad for t in (x, f, wz, A_log, dt_bias, state)):
        raise RuntimeError(f"{name} is forward-only (decoding); call it under torch.no_grad() or on "
                           "tensors that do not require grad")
    wd = x.dtype if x.dtype in (torch.bfloat16, torch.float32) else torch.float32
    xw, fw, ww = (_rows(t, wd) for t in (x, f, wz))
    A, dt = _f32(A_log), _f32(dt_bias)
    if inplace:
        if state.dtype != torch.float32 or not state.is_contiguous():
            raise ValueError(f"{name}: inplace=True needs a contiguous fp32 state")
        s_in = s_out = state
    else:
        s_in = _f32(state)
        s_out = torch.empty_like(s_in)
    y = torch.empty(B, D, device=x.device, dtype=wd)
    if B:
        a = _fill(_lib.RecurrenceArgs(), B, 1, D, xw, fw, ww, A, dt)
        a.h0, a.final_state, a.y = s_in.data_ptr(), s_out.data_ptr(), y.data_ptr()
        _call("ngdn_recurrence_step", wd, a, x)
    return y.to(x.dtype), s_out
