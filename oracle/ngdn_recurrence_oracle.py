"""The gated linear recurrence and the embedding in float64 on the CPU, token
by token, with the errors that fp32 kernels may make.

``recurrence`` returns the outputs and gradients (the formulas written out)
and, for each, a bound on the fp32 error of any evaluation that

* forms z, softplus, e^g, 1 - e^2g and the sigmoid with the relative errors
  below (u = 2^-24, one fp32 rounding; the hardware exp2, reciprocal and
  reciprocal root are within 2 u),
* and joins tokens in any order (a product or sum a token, so a rounding each).

  z = f + bias: 3 u |z| + 3 u (two products with log2(e), a sum);
  softplus: relative error that of its polynomial, 5 u, 4 u of roundings, and
    the error of z (|d log softplus / dz| <= 1): r_g = 14 u + 3 u |z|, two
    more for exp(A_log), whose argument has u |A_log|;
  a = e^g: 2 u + |g| r_g;   1 - a: relative error 16 u r (the subtraction, from
    -g = 1/16) or r_g (the series): q = (1 - a)(1 + a): r_q = 20 u + r_g;
  beta and 1 / beta: half of it and 3 u;  sigmoid: 4 u + 2 u |w|, and so is
    1 - sigmoid(w) = sigmoid(-w), which no subtraction may form.
"""

import torch

U = 2.0 ** -24


def _gates(x, f, wz, A_log, dt_bias):
    x, f, wz, A_log, dt_bias = (t.detach().double().cpu() for t in (x, f, wz, A_log, dt_bias))
    D, H = dt_bias.shape[0], A_log.shape[0]
    la = A_log.repeat_interleave(D // H)
    z = f + dt_bias
    sp = torch.logaddexp(z, torch.zeros_like(z))
    g = -la.exp() * sp
    a = g.exp()
    q = -(2 * g).expm1()
    beta, s, sz = q.sqrt(), torch.sigmoid(wz), torch.sigmoid(z)
    rg = (16 + 3 * z.abs().clamp(max=200) + la.abs()) * U
    ra = 2 * U + g.abs().clamp(max=200) * rg
    rb = 13 * U + rg / 2
    ru = rb + (6 + 2 * wz.abs().clamp(max=200)) * U
    return x, la, z, g, a, q, beta, s, sz, rg, ra, rb, ru


def sequences(B, T, cu):
    """(row, first, stop, state index) of every sequence."""
    if cu is None:
        return [(b, 0, T, b) for b in range(B)]
    return [(0, int(cu[i]), int(cu[i + 1]), i) for i in range(len(cu) - 1)]


def recurrence(x, f, wz, A_log, dt_bias, h0=None, cu=None, dy=None, dfinal=None):
    """{name: (value, bound)} with y, final and, with dy, dx, df, dwz, dA_log,
    ddt_bias, dinitial_state."""
    B, T, D = x.shape
    xx, la, z, g, a, q, beta, s, sz, rg, ra, rb, ru = _gates(x, f, wz, A_log, dt_bias)
    used = torch.zeros(B, T, 1, dtype=torch.bool)
    seqs = sequences(B, T, cu)
    for b, lo, hi, _ in seqs:
        used[b, lo:hi] = True
    xx = torch.where(used, xx, 0.0)
    u = beta * s * xx
    rows = len(seqs)
    h0 = torch.zeros(rows, D, dtype=torch.float64) if h0 is None else h0.detach().double().cpu()
    y, prev, ey, eprev = (torch.zeros(B, T, D, dtype=torch.float64) for _ in range(4))
    final, efinal = h0.clone(), torch.zeros_like(h0)
    for b, lo, hi, i in seqs:
        h, m, e = h0[i], h0[i].abs(), torch.zeros(D, dtype=torch.float64)
        for t in range(lo, hi):
            prev[b, t], eprev[b, t] = h, e
            # m bounds what is summed, e its error: the decay's own, the new term's, a
            # rounding each for the product, the sum and the joining of runs
            e = a[b, t] * (e + (ra[b, t] + 3 * U) * m) + (ru[b, t] + 3 * U) * u[b, t].abs()
            h = a[b, t] * h + u[b, t]
            m = a[b, t] * m + u[b, t].abs()
            e = e + 3 * U * m
            y[b, t], ey[b, t] = h, e
        final[i], efinal[i] = h, e
    out = {"y": (y, ey), "final": (final, efinal)}
    if dy is None:
        return out
    dy = torch.where(used, dy.detach().double().cpu(), 0.0)
    dfinal = torch.zeros_like(h0) if dfinal is None else dfinal.detach().double().cpu()
    lam, elam = torch.zeros_like(y), torch.zeros_like(y)
    dh0, edh0 = dfinal.clone(), torch.zeros_like(dfinal)
    for b, lo, hi, i in seqs:
        c, m, e = dfinal[i], dfinal[i].abs(), torch.zeros(D, dtype=torch.float64)
        for t in reversed(range(lo, hi)):
            lt, m = dy[b, t] + c, dy[b, t].abs() + m
            e = e + 3 * U * m
            lam[b, t], elam[b, t] = lt, e
            e = a[b, t] * (e + (ra[b, t] + 3 * U) * m)
            c, m = a[b, t] * lt, a[b, t] * m
        dh0[i], edh0[i] = c, e
    bs = beta * s
    dx = lam * bs
    edx = elam * bs + (ru + 3 * U) * dx.abs()
    w = wz.detach().double().cpu()
    k = xx * torch.sigmoid(-w)
    dw = dx * k
    edw = edx * k.abs() + dw.abs() * (10 + 2 * w.abs().clamp(max=200)) * U
    safe = torch.where(beta > 0, a * a / beta, 0.0)
    p1, p2 = a * prev, safe * s * xx
    inner = p1 - p2
    dg = lam * inner
    edg = (elam * inner.abs() + lam.abs() * ((ra + 3 * U) * p1.abs() + a * eprev
                                             + (2 * ra + rb + ru + 6 * U) * p2.abs()))
    df = -la.exp() * sz * dg
    rs = (10 + 3 * z.abs().clamp(max=200) + la.abs()) * U
    edf = la.exp() * sz * edg + rs * df.abs()
    zero = lambda v: torch.where(used, v, 0.0)  # noqa: E731
    df, edf, dg, edg = zero(df), zero(edf), zero(dg), zero(edg)
    # sums over B T tokens: at most 64 + (tokens / 512) roundings in a row
    deep = (64 + B * T / 512) * U
    H = A_log.shape[0]
    dA, eA = dg * g, edg * g.abs() + (rg + 2 * U) * (dg * g).abs()
    heads = lambda v: v.sum((0, 1)).view(H, -1).sum(1)  # noqa: E731
    out.update(dx=(dx, edx), df=(df, edf), dwz=(dw, edw),
               ddt_bias=(df.sum((0, 1)), (edf + deep * df.abs()).sum((0, 1))),
               dA_log=(heads(dA), heads(eA + deep * dA.abs())), dinitial_state=(dh0, edh0))
    return out


def step(x, f, wz, A_log, dt_bias, state):
    """(new state, bound)."""
    o = recurrence(x[:, None], f[:, None], wz[:, None], A_log, dt_bias, state)
    return o["final"]


def embedding(ids, weight, scale=1.0):
    ids, w = ids.cpu(), weight.detach().double().cpu()
    ok = (ids >= 0) & (ids < w.shape[0])
    y = w[ids.clamp(0, w.shape[0] - 1)] * scale
    return torch.where(ok.unsqueeze(-1), y, float("nan"))


def embedding_grad(ids, dy, V, scale=1.0, padding_idx=None):
    """(dw, bound): a row of m terms has at most m + 2 roundings in fp32."""
    ids, dy = ids.cpu().reshape(-1), dy.detach().double().cpu()
    dy = dy.reshape(ids.numel(), -1)
    keep = (ids >= 0) & (ids < V)
    if padding_idx is not None:
        keep &= ids != padding_idx
    dw = torch.zeros(V, dy.shape[1], dtype=torch.float64)
    mag, n = torch.zeros_like(dw), torch.zeros(V, 1, dtype=torch.float64)
    dw.index_add_(0, ids[keep], dy[keep])
    mag.index_add_(0, ids[keep], dy[keep].abs())
    n.index_add_(0, ids[keep], torch.ones(int(keep.sum()), 1, dtype=torch.float64))
    return dw * scale, (n + 2) * U * mag * abs(scale)
