"""Dropout, the residual norm and the sampler in float64, with bounds on the
error of a computation in fp32. Used only by the tests.

The bounds count roundings of u = 2^-24 each. A sum over a row of D values takes
at most SUM of them on any value's way (eight or sixteen values a lane, six steps
of a wave, up to sixteen waves); 1 / sqrt of its mean halves the relative error and
adds five (mean, eps, root, quotient, reciprocal of D), and the hardware's own root
and quotient are within one unit each.
"""

import numpy as np
import torch

U = 2.0 ** -24
SUM = 16 + 6 + 16
STAT = SUM / 2 + 8          # relative roundings of rstd
M0, M1, W0, W1, LOW = 0xD2511F53, 0xCD9E8D57, 0x9E3779B9, 0xBB67AE85, 0xFFFFFFFF


def words(first, n, seed, offset):
    """Words first ... first + n - 1 of Philox4x32-7, by Python's integers."""
    out = []
    for block in range(first // 4, (first + n + 3) // 4):
        c = [block & LOW, block >> 32, offset & LOW, offset >> 32 & LOW]
        k0, k1 = seed & LOW, seed >> 32 & LOW
        for _ in range(7):
            a, b = M0 * c[0], M1 * c[2]
            c = [b >> 32 ^ c[1] ^ k0, b & LOW, a >> 32 ^ c[3] ^ k1, a & LOW]
            k0, k1 = k0 + W0 & LOW, k1 + W1 & LOW
        out += c
    return out[first % 4:first % 4 + n]


def words_np(n, seed, offset):
    """The same from word 0, by numpy (64-bit products)."""
    block = np.arange((n + 3) // 4, dtype=np.uint64)
    low, sh, zero = np.uint64(LOW), np.uint64(32), np.zeros_like(block)
    c = [block & low, block >> sh, zero + np.uint64(offset & LOW), zero + np.uint64(offset >> 32 & LOW)]
    k0, k1 = seed & LOW, seed >> 32 & LOW
    for _ in range(7):
        a, b = c[0] * np.uint64(M0), c[2] * np.uint64(M1)
        c = [b >> sh ^ c[1] ^ np.uint64(k0), b & low, a >> sh ^ c[3] ^ np.uint64(k1), a & low]
        k0, k1 = k0 + W0 & LOW, k1 + W1 & LOW
    return np.stack(c, 1).reshape(-1)[:n]


def kept(shape, p, seed, offset):
    n = int(np.prod(shape, dtype=np.int64))
    return torch.from_numpy(words_np(n, seed, offset) >= np.uint64(round(p * 2 ** 32))).view(shape)


def _rows(t, x):
    """A gate over all of x."""
    return t.double().expand(x.shape) if t is not None else torch.ones(x.shape, dtype=torch.float64)


def _fold(v, like):
    """v summed over what ``like`` was broadcast over, and how many values a sum has."""
    count = 1
    if like.dim() == 1 and v.dim() > 1:
        count = v.numel() // v.shape[-1]
        return v.reshape(-1, v.shape[-1]).sum(0), count
    for d in range(v.dim()):
        if like.shape[d] == 1 and v.shape[d] > 1:
            count *= v.shape[d]
            v = v.sum(d, keepdim=True)
    return v, count


def residual_norm(x, branch, weight=None, post_weight=None, gate=None, residual_scale=1.0, branch_scale=1.0,
                  p=0.0, seed=0, offset=0, eps=1e-5, dh=None, dy=None):
    """name -> (value, bound) of h, y and, with dh or dy, of every gradient.
    Bounds are of the fp32 values, before an output is rounded to its type."""
    f = lambda t: t.double() if t is not None else None  # noqa: E731
    x, branch, weight, post_weight = f(x), f(branch), f(weight), f(post_weight)
    D = x.shape[-1]
    mean = lambda v: v.sum(-1, keepdim=True) / D  # noqa: E731
    g = _rows(gate, x)
    keep = kept(x.shape, p, seed, offset) if p else torch.ones(x.shape, dtype=torch.bool)
    factor = branch_scale / (1 - p) if p < 1 else 0.0
    z, ez = branch, 0 * branch
    if post_weight is not None:
        sb = (mean(branch * branch) + eps).rsqrt()
        bn = branch * sb
        z = bn * post_weight
        ez = z.abs() * (STAT + 3) * U
    drop = lambda v: torch.where(keep, v * factor, 0)  # noqa: E731
    u = drop(z * g)
    eu = drop(ez * g).abs() + u.abs() * 5 * U
    h = residual_scale * x + u
    eh = eu + ((residual_scale * x).abs() * 2 + u.abs()) * U
    out = {"h": (h, eh)}
    norm = weight is not None
    if norm:
        sh = (mean(h * h) + eps).rsqrt()
        n = h * sh
        # a relative change of the root mean square is at most |eh| / |h| over the row
        rel = (mean(eh * eh) / (mean(h * h) + eps)).sqrt() + STAT * U
        en = sh * eh + n.abs() * (rel + 2 * U)
        out["y"] = (n * weight, weight.abs() * en + (n * weight).abs() * 2 * U)
    if dh is None and dy is None:
        return out
    d, ed = torch.zeros_like(x), torch.zeros_like(x)
    if dy is not None and norm:
        dy = dy.double()
        q = dy * weight
        m = mean(q * n)
        em = mean(q.abs() * en + (q * n).abs() * (SUM + 4) * U)
        d = sh * (q - n * m)
        ed = sh * ((q.abs() + (n * m).abs()) * (rel + 5 * U) + en * m.abs() + n.abs() * em)
        dw, c = _fold(dy * n, weight)
        out["dweight"] = (dw, _fold((dy.abs() * en), weight)[0] + _fold((dy * n).abs(), weight)[0] * (c + 8) * U)
    elif norm:
        out["dweight"] = (torch.zeros_like(weight), torch.zeros_like(weight))
    if dh is not None:
        d = d + dh.double()
        ed = ed + d.abs() * U
    out["dx"] = (residual_scale * d, abs(residual_scale) * (ed + d.abs() * 2 * U))
    du = drop(d)
    edu = drop(ed).abs() + du.abs() * 4 * U
    if gate is not None:
        v, c = _fold(du * z, gate)
        out["dgate"] = (v, _fold(edu * z.abs() + du.abs() * ez, gate)[0] + _fold((du * z).abs(), gate)[0] * (c + 8) * U)
    dz = du * g
    edz = edu * g.abs() + dz.abs() * 2 * U
    if post_weight is not None:
        ebn = bn.abs() * (STAT + 2) * U
        dp, c = _fold(dz * bn, post_weight)
        out["dpost_weight"] = (dp, _fold(edz * bn.abs() + dz.abs() * ebn, post_weight)[0]
                               + _fold((dz * bn).abs(), post_weight)[0] * (c + 8) * U)
        q, eq = dz * post_weight, edz * post_weight.abs() + (dz * post_weight).abs() * 2 * U
        m = mean(q * bn)
        em = mean(eq * bn.abs() + q.abs() * ebn + (q * bn).abs() * (SUM + 4) * U)
        dz = sb * (q - bn * m)
        edz = sb * (eq + (q.abs() + (bn * m).abs()) * (STAT + 5) * U + ebn * m.abs() + bn.abs() * em)
    out["dbranch"] = (dz, edz)
    return out


def sample(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """Tokens [rows] of logits [rows, V], by sorting."""
    l = logits.double().cpu().numpy()
    rows, V = l.shape

    def each(v, dtype):
        v = np.asarray(v.cpu().numpy() if torch.is_tensor(v) else v, dtype=dtype)
        return np.broadcast_to(v, (rows,))

    T, P, least = (each(v, np.float32).astype(np.float64) for v in (temperature, top_p, min_p))
    K, U01 = each(top_k, np.int64), each(u, np.float64)
    token = np.full(rows, -1, dtype=np.int64)
    for i in range(rows):
        top = l[i].max()
        if not np.isfinite(top):            # NaN too
            continue
        if not (0 <= T[i] < np.inf and 0 <= P[i] <= 1 and 0 <= least[i] <= 1 and 0 <= U01[i] <= 1):
            continue
        if T[i] == 0:
            token[i] = int(np.argmax(l[i]))
            continue
        w = np.exp((l[i] - top) / T[i])
        order = np.argsort(-l[i], kind="stable")
        if K[i] > 0:
            order = order[:K[i]]
        if P[i] < 1:
            c = np.cumsum(w[order])
            order = order[(c - w[order] < P[i] * c[-1]) | (np.arange(len(order)) == 0)]
        order = np.sort(order[w[order] >= least[i]])
        c = np.cumsum(w[order])
        over = np.nonzero(c > U01[i] * c[-1])[0]
        token[i] = order[over[0]] if len(over) else order[np.nonzero(w[order])[0][-1]]
    return torch.from_numpy(token)
