"""Timed cases of dropout, of the residual norm and of the sampler.

Paths (``case["path"]``):
  drop     model_ops.dropout forward and its gradient
  norm     model_ops.residual_norm forward alone (generation, prompts)
  train    model_ops.residual_norm forward and every gradient
  sample   model_ops.sample_tokens, a token a row of logits

``run`` computes each in plain torch, or with ``own`` through the package's
entry points. ``exact`` restates each in float64.

Dropout: element i of a tensor (in row-major order) is kept where word i % 4 of
the generator's block i // 4 is at least round(p 2^32), and then divided by
1 - p. The generator is Philox4x32 with seven rounds (Salmon, Moraes, Dror, Shaw:
Parallel random numbers: as easy as 1, 2, 3; SC11), its counter (block, offset)
and its key the seed, each as two 32-bit words, low word first.

Residual norm, over rows of D (N(v, w) = v / sqrt(mean(v^2) + eps) w):
  h = residual_scale x + branch_scale dropout(gate N(branch, post_weight))
  y = N(h, weight)

Sampler, per row with l its logits, t its temperature, w_i = exp((l_i - max l) / t):
the top_k largest, of those (largest first, lower index first among equals) the
ones before which less than top_p of their sum lies, of those the ones with
w_i >= min_p. The token is the first in index order with the kept weights up to
and with it above u times their sum. t = 0 takes the first of the largest. A row
whose largest logit is not finite (all masked by -inf) gives -1.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
EPS = 1e-5


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # a short sequence's hidden states between two layers
        _drop("drop_short", rows=256, width=1024, dtype="bf16", p=0.1),
        # a batch's gated MLP activations at the default model's intermediate size
        _drop("drop_mlp", rows=16384, width=2816, dtype="bf16", p=0.1),
        # fp32 training, a ragged batch of odd width, a strong rate
        _drop("drop_odd_fp32", rows=5003, width=515, dtype="fp32", p=0.5),
        # one sequence being generated: one token of the default model
        _norm("norm", "norm_token", B=1, T=1, D=1024, stream="bf16", branch="bf16", gate="channel"),
        # a serving batch, gates that each sequence's conditioning gives
        _norm("norm", "norm_tokens", B=128, T=1, D=2048, stream="bf16", branch="bf16", gate="sequence"),
        # prompts on an fp32 stream under bf16 autocast
        _norm("norm", "norm_prompts", B=4, T=4096, D=2048, stream="fp32", branch="bf16", gate="none"),
        # the benchmark's batch and length, a layer scale and dropout
        _norm("train", "train_batch", B=4, T=8192, D=2048, stream="bf16", branch="bf16", gate="channel",
              p=0.1),
        # an fp32 stream, no norm after the branch, a gate for each value, sequences of odd length
        _norm("train", "train_gated_fp32", B=3, T=1333, D=1024, stream="fp32", branch="bf16", gate="full",
              post=False, out="bf16"),
        # a small batch of odd width in fp32, a gate a token, h alone (the last block)
        _norm("train", "train_odd_fp32", B=2, T=777, D=1001, stream="fp32", branch="fp32", gate="token",
              p=0.1, pre=False),
        # the next token of one sequence
        _sample("sample_one", B=1, V=32000, dtype="bf16", temperature=0.8, top_p=0.9),
        # a serving batch on a vocabulary padded in memory, each request with its own settings
        _sample("sample_requests", B=64, V=32001, dtype="bf16", requests=True, padded=True, masked=0.1),
        # a large batch and vocabulary in fp32
        _sample("sample_large", B=256, V=131072, dtype="fp32", temperature=1.0, top_k=50, top_p=0.95,
                min_p=0.01),
    ]


def _drop(name, *, rows, width, dtype, p):
    c = dict(path="drop", rows=rows, width=width, dtype=dtype, p=p)
    return dict(c, name=name) if name else c


def _norm(path, name, *, B, T, D, stream, branch, gate, out=None, post=True, pre=True, p=0.0,
          residual_scale=1.0, branch_scale=1.0):
    c = dict(path=path, B=B, T=T, D=D, stream=stream, branch=branch, gate=gate, out=out or branch,
             post=post, pre=pre, p=p, residual_scale=residual_scale, branch_scale=branch_scale)
    return dict(c, name=name) if name else c


def _sample(name, *, B, V, dtype, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, requests=False,
            padded=False, masked=0.0):
    c = dict(path="sample", B=B, V=V, dtype=dtype, temperature=temperature, top_k=top_k, top_p=top_p,
             min_p=min_p, requests=requests, padded=padded, masked=masked)
    return dict(c, name=name) if name else c


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


WIDTHS = [64, 100, 128, 256, 512, 515, 768, 1000, 1001, 1024, 1536, 2048, 2816, 4096, 4100]


def draw(rng):
    path = rng.choice(["drop", "norm", "norm", "train", "train", "train", "sample", "sample", "sample"])
    if path == "drop":
        width = rng.choice(WIDTHS)
        dtype = rng.choice(["bf16", "fp32"])
        most = 16384 * 2816 // (1 if dtype == "bf16" else 2)
        return _drop(None, rows=_log_int(rng, 1, most // width), width=width, dtype=dtype,
                     p=rng.choice([0.05, 0.1, 0.2, 0.5]))
    if path == "sample":
        V = rng.choice([1000, 8000, 8003, 32000, 32001, 65536, 100000, 131072])
        return _sample(None, B=_log_int(rng, 1, min(512, 256 * 131072 // V)), V=V,
                       dtype=rng.choice(["bf16", "fp32"]), temperature=rng.choice([0.0, 0.6, 0.8, 1.0, 1.3]),
                       top_k=rng.choice([0, 0, 1, 20, 50, 1000]), top_p=rng.choice([1.0, 0.8, 0.9, 0.95]),
                       min_p=rng.choice([0.0, 0.0, 0.01, 0.1]), requests=rng.random() < 0.4,
                       padded=rng.random() < 0.3, masked=rng.choice([0.0, 0.0, 0.1, 0.999]))
    stream, branch, out = rng.choice([("bf16", "bf16", "bf16"), ("bf16", "bf16", "bf16"),
                                      ("fp32", "bf16", "bf16"), ("fp32", "fp32", "fp32")])
    D = rng.choice(WIDTHS)
    most = 4 * 8192 * 2048 // (1 if stream == "bf16" else 2)
    T = 1 if path == "norm" and rng.random() < 0.4 else _log_int(rng, 1, min(8192, most // D))
    B = _log_int(rng, 1, max(1, min(256, most // (T * D))))
    pre = rng.random() < 0.85
    return _norm(path, None, B=B, T=T, D=D, stream=stream, branch=branch, out=out,
                 gate=rng.choice(["none", "channel", "channel", "sequence", "token", "full"]),
                 post=rng.random() < 0.7, pre=pre, p=rng.choice([0.0, 0.1]) if path == "train" else 0.0,
                 residual_scale=rng.choice([1.0, 1.0, 0.7]), branch_scale=rng.choice([1.0, 0.25]))


# ------------------------------------------------------------------ inputs

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _drop_inputs(case, seed):
    gen = _gen(seed)
    shape, dt = (case["rows"], case["width"]), DTYPES[case["dtype"]]
    x = torch.randn(shape, generator=gen, device=DEV).to(dt)
    return dict(x=x, dy=torch.randn(shape, generator=gen, device=DEV).to(dt), seed=seed, offset=3)


def _norm_inputs(case, seed):
    """A stream whose channels differ in size, as they do some blocks into a model."""
    gen = _gen(seed)
    B, T, D = (case[k] for k in "BTD")
    xd, rd, yd = (DTYPES[case[k]] for k in ("stream", "branch", "out"))
    r = lambda *s: torch.randn(*s, generator=gen, device=DEV)  # noqa: E731
    s = dict(x=(r(B, T, D) * (0.5 * r(D)).exp()).to(xd), branch=(0.5 * r(B, T, D)).to(rd),
             weight=1 + 0.1 * r(D) if case["pre"] else None,
             post_weight=1 + 0.1 * r(D) if case["post"] else None, gate=None, dh=None, dy=None,
             seed=seed, offset=7)
    g = case["gate"]
    if g == "channel":
        s["gate"] = 0.1 + 0.02 * r(D)
    elif g == "sequence":
        s["gate"] = (0.3 * r(B, 1, D)).to(rd)
    elif g == "token":
        s["gate"] = torch.sigmoid(r(B, T, 1)).to(rd)
    elif g == "full":
        s["gate"] = torch.sigmoid(r(B, T, D)).to(rd)
    if case["path"] == "train":
        s["dh"] = r(B, T, D).to(xd)
        if case["pre"]:
            s["dy"] = r(B, T, D).to(yd)
    return s


LEAVES = ("x", "branch", "weight", "post_weight", "gate")


def _sample_inputs(case, seed):
    """Logits with a long tail and few likely tokens, at random places."""
    gen = _gen(seed)
    B, V = case["B"], case["V"]
    r = lambda *s: torch.rand(*s, generator=gen, device=DEV)  # noqa: E731
    rank = torch.argsort(r(B, V), dim=1) + 1.0
    l = 12 - 1.6 * rank.log() + torch.randn(B, V, generator=gen, device=DEV)
    if case["masked"]:
        l = torch.where(r(B, V) < case["masked"], -math.inf, l)
    width = (V + 127) // 128 * 128 if case["padded"] else V
    logits = torch.full((B, width), 50.0, device=DEV, dtype=DTYPES[case["dtype"]])[:, :V]
    logits.copy_(l)
    s = dict(logits=logits, u=r(B), **{k: case[k] for k in ("temperature", "top_k", "top_p", "min_p")})
    if case["requests"]:
        t = 0.5 + 0.8 * r(B)
        s["temperature"] = torch.where(r(B) < 0.1, 0.0, t)
        k = (1 + 200 * r(B)).to(torch.int32)
        s["top_k"] = torch.where(r(B) < 0.4, torch.zeros_like(k), k)
        s["top_p"] = torch.where(r(B) < 0.3, 1.0, 0.6 + 0.4 * r(B))
        s["min_p"] = torch.where(r(B) < 0.6, 0.0, 0.1 * r(B))
    return s


def _inputs(case, seed):
    p = case["path"]
    return _drop_inputs(case, seed) if p == "drop" else \
        _sample_inputs(case, seed) if p == "sample" else _norm_inputs(case, seed)


def prepare(case, seed):
    s = _inputs(case, seed)
    if case["path"] == "drop":
        s["x"].requires_grad_(True)
    elif case["path"] == "train":
        for n in LEAVES:
            if s[n] is not None:
                s[n].requires_grad_(True)
    return dict(s, case=case)


# ------------------------------------------------------------------ one pass

def run(state):
    path = state["case"]["path"]
    if own:
        return _own_drop(state) if path == "drop" else _own_sample(state) if path == "sample" \
            else _own_norm(state)
    with torch.no_grad():
        return _plain_drop(state) if path == "drop" else _plain_sample(state) if path == "sample" \
            else _plain_norm(state)


def _own_drop(s):
    from nested_recurrent_memory_amd.model_ops import dropout

    y = dropout(s["x"], s["case"]["p"], s["seed"], s["offset"])
    dx, = torch.autograd.grad(y, s["x"], s["dy"])
    return {"y": y.detach(), "dx": dx}


def _own_norm(s):
    from nested_recurrent_memory_amd.model_ops import residual_norm

    c = s["case"]
    out = residual_norm(s["x"], s["branch"], s["weight"], post_weight=s["post_weight"], gate=s["gate"],
                        residual_scale=c["residual_scale"], branch_scale=c["branch_scale"], p=c["p"],
                        seed=s["seed"], offset=s["offset"], eps=EPS, out_dtype=DTYPES[c["out"]])
    h, y = out if c["pre"] else (out, None)
    if c["path"] == "norm":
        return {"h": h, "y": y}
    names = [n for n in LEAVES if s[n] is not None]
    grads = torch.autograd.grad([h] + ([y] if c["pre"] else []), [s[n] for n in names],
                                [s["dh"]] + ([s["dy"]] if c["pre"] else []))
    return {"h": h.detach(), "y": y.detach() if c["pre"] else None,
            **{"d" + n: g for n, g in zip(names, grads)}}


def _own_sample(s):
    from nested_recurrent_memory_amd.model_ops import sample_tokens

    return {"token": sample_tokens(s["logits"], s["u"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])}


M0, M1, W0, W1, LOW = 0xD2511F53, 0xCD9E8D57, 0x9E3779B9, 0xBB67AE85, 0xFFFFFFFF


def _product(m, c):
    """High and low words of m c, both below 2^32, in int64 without overflow."""
    low = m * (c & 0xFFFF)
    top = m * (c >> 16) + (low >> 16)
    return top >> 16, ((top & 0xFFFF) << 16) | (low & 0xFFFF)


def _kept(shape, p, seed, offset):
    n = math.prod(shape)
    block = torch.arange((n + 3) // 4, device=DEV, dtype=torch.int64)
    zero = torch.zeros_like(block)
    c = [block & LOW, block >> 32, zero + (offset & LOW), zero + (offset >> 32)]
    k0, k1 = seed & LOW, seed >> 32
    for _ in range(7):
        h0, l0 = _product(M0, c[0])
        h1, l1 = _product(M1, c[2])
        c = [h1 ^ c[1] ^ k0, l1, h0 ^ c[3] ^ k1, l0]
        k0, k1 = (k0 + W0) & LOW, (k1 + W1) & LOW
    return (torch.stack(c, 1).flatten()[:n] >= round(p * 2 ** 32)).view(shape)


def _plain_drop(s):
    x, p = s["x"], s["case"]["p"]
    keep = _kept(x.shape, p, s["seed"], s["offset"])
    f = lambda t: torch.where(keep, t.float() / (1 - p), 0).to(t.dtype)  # noqa: E731
    return {"y": f(x), "dx": f(s["dy"])}


def _dnorm(dy, n, rstd, w):
    """Gradients of y = n w, n = v rstd(v), for v and w."""
    d = dy * w
    return rstd * (d - n * (d * n).mean(-1, keepdim=True)), (dy * n).sum((0, 1))


def _like(grad, t):
    """Summed over what t was broadcast over, in its type."""
    if t.dim() == 1:
        grad = grad.sum((0, 1))
    else:
        for d in range(3):
            if t.shape[d] == 1 and grad.shape[d] > 1:
                grad = grad.sum(d, keepdim=True)
    return grad.to(t.dtype)


def _plain_norm(s):
    c, x, branch, gate = s["case"], s["x"], s["branch"], s["gate"]
    rstd = lambda v: 1 / ((v * v).mean(-1, keepdim=True) + EPS).sqrt()  # noqa: E731
    b = branch.float()
    if c["post"]:
        sb = rstd(b)
        bn = b * sb
        b = bn * s["post_weight"].float()
    g = gate.float() if gate is not None else None
    u = b * g if gate is not None else b
    keep = _kept(x.shape, c["p"], s["seed"], s["offset"]) if c["p"] else None
    drop = lambda v: torch.where(keep, v / (1 - c["p"]), 0) if c["p"] else v  # noqa: E731
    h = c["residual_scale"] * x.float() + c["branch_scale"] * drop(u)
    out = {"h": h.to(x.dtype), "y": None}
    if c["pre"]:
        sh = rstd(h)
        n, w = h * sh, s["weight"].float()
        out["y"] = (n * w).to(DTYPES[c["out"]])
    if c["path"] == "norm":
        return out
    dh = s["dh"].float()
    if c["pre"]:
        d, dw = _dnorm(s["dy"].float(), n, sh, w)
        dh = dh + d
    out["dx"] = (c["residual_scale"] * dh).to(x.dtype)
    du = c["branch_scale"] * drop(dh)
    db = du * g if gate is not None else du
    if c["post"]:
        db, dpost = _dnorm(db, bn, sb, s["post_weight"].float())
    out["dbranch"] = db.to(branch.dtype)
    if c["pre"]:
        out["dweight"] = dw
    if c["post"]:
        out["dpost_weight"] = dpost
    if gate is not None:
        out["dgate"] = _like(du * b, gate)
    return out


def _plain_sample(s):
    l = s["logits"].double()
    B, V = l.shape
    col = lambda v: torch.as_tensor(v, device=DEV, dtype=torch.float32).double().expand(B).view(B, 1)  # noqa: E731
    t, p, least = col(s["temperature"]), col(s["top_p"]), col(s["min_p"])
    k = torch.as_tensor(s["top_k"], device=DEV).expand(B).view(B, 1)
    v, order = torch.sort(l, dim=1, descending=True, stable=True)
    w = torch.exp((v - v[:, :1]) / torch.where(t > 0, t, 1.0))
    rank = torch.arange(V, device=DEV)
    keep = (k < 1) | (rank < k)
    w = torch.where(keep, w, 0)
    c = w.cumsum(1)
    keep &= (p >= 1) | (rank == 0) | (c - w < p * c[:, -1:])
    keep &= w >= least
    w = torch.zeros_like(w).scatter_(1, order, torch.where(keep, w, 0))
    c = w.cumsum(1)
    token = (c <= s["u"].double().view(B, 1) * c[:, -1:]).sum(1)
    token = torch.where(t[:, 0] > 0, token, order[:, 0])
    return {"token": torch.where(v[:, 0].abs() < math.inf, token, -1)}


# ------------------------------------------------------------------ what a pass cannot do without

_SIZE = {"bf16": 2, "fp32": 4}


def work(case):
    path = case["path"]
    if path == "drop":
        n = case["rows"] * case["width"]
        return {"bytes": 4 * n * _SIZE[case["dtype"]], "flops": 2 * n}
    if path == "sample":
        n = case["B"] * case["V"]
        return {"bytes": n * _SIZE[case["dtype"]] + 12 * case["B"] * (1 + case["requests"]), "flops": 12 * n}
    rows, D = case["B"] * case["T"], case["D"]
    n, e, r, y = rows * D, _SIZE[case["stream"]], _SIZE[case["branch"]], _SIZE[case["out"]]
    gate = {"none": 0, "channel": 4 * D, "sequence": case["B"] * D * r, "token": rows * r, "full": n * r}
    params = 4 * D * (case["post"] + case["pre"]) + gate[case["gate"]]
    moved = n * (2 * e + r + y * case["pre"]) + params
    if path == "norm":
        return {"bytes": moved, "flops": 10 * n}
    return {"bytes": moved + n * (2 * e + r + y * case["pre"]) + params, "flops": 35 * n}


# ------------------------------------------------------------------ the same in float64

def _words(n, seed, offset):
    """The generator's first n words, by numpy's 64-bit products, a run of blocks at a time."""
    out = np.empty(((n + 3) // 4, 4), dtype=np.uint32)
    low, sh = np.uint64(LOW), np.uint64(32)
    for b0 in range(0, out.shape[0], 1 << 15):
        block = np.arange(b0, min(b0 + (1 << 15), out.shape[0]), dtype=np.uint64)
        x0, x1 = block & low, block >> sh
        x2, x3 = np.full_like(block, offset & LOW), np.full_like(block, offset >> 32)
        for r in range(7):
            a, b = x0 * np.uint64(M0), x2 * np.uint64(M1)
            x0 = (b >> sh) ^ x1 ^ np.uint64((seed + r * W0) & LOW)
            x2 = (a >> sh) ^ x3 ^ np.uint64(((seed >> 32) + r * W1) & LOW)
            x1, x3 = b & low, a & low
        for j, x in enumerate((x0, x1, x2, x3)):
            out[b0:b0 + len(block), j] = x
    return out.reshape(-1)[:n]


def _factor(shape, p, seed, offset):
    keep = _words(math.prod(shape), seed, offset) >= np.uint64(round(p * 2 ** 32))
    return torch.from_numpy(keep).to(DEV).view(shape) * (1.0 / (1.0 - p)) if p else 1.0


def exact(case, seed):
    s, path = _inputs(case, seed), case["path"]
    if path == "sample":
        return {"token": _exact_sample(s)}
    if path == "drop":
        f = _factor(s["x"].shape, case["p"], s["seed"], s["offset"])
        return {"y": s["x"].double() * f, "dx": s["dy"].double() * f}
    with torch.enable_grad():
        leaf = {n: s[n].double().requires_grad_(path == "train") for n in LEAVES if s[n] is not None}
        norm = lambda v, w: w * v * torch.rsqrt(v.square().sum(-1, keepdim=True) / case["D"] + EPS)  # noqa: E731
        z = leaf["branch"]
        if case["post"]:
            z = norm(z, leaf["post_weight"])
        if s["gate"] is not None:
            z = z * leaf["gate"]
        if case["p"]:
            z = z * _factor(z.shape, case["p"], s["seed"], s["offset"])
        h = leaf["x"] * case["residual_scale"] + z * case["branch_scale"]
        y = norm(h, leaf["weight"]) if case["pre"] else None
        out = {"h": h.detach(), "y": y.detach() if case["pre"] else None}
        if path == "train":
            grads = torch.autograd.grad([h] + ([y] if case["pre"] else []), list(leaf.values()),
                                        [s["dh"].double()] + ([s["dy"].double()] if case["pre"] else []))
            out.update({"d" + n: g for n, g in zip(leaf, grads)})
    return out


def _exact_sample(s):
    l, u = s["logits"].double().cpu().numpy(), s["u"].double().cpu().numpy()
    B, V = l.shape
    rows = lambda v: np.broadcast_to(  # noqa: E731
        v.cpu().numpy() if torch.is_tensor(v) else np.asarray(v, dtype=np.float32 if isinstance(v, float) else None), (B,))
    T, K, P, least = (rows(s[n]) for n in ("temperature", "top_k", "top_p", "min_p"))
    token = np.empty(B, dtype=np.int64)
    for i in range(B):
        first = int(np.argmax(l[i]))
        token[i] = first if np.isfinite(l[i, first]) else -1
        if T[i] <= 0 or token[i] < 0:
            continue
        w = np.exp((l[i] - l[i, first]) / np.float64(T[i]))
        order = np.argsort(-l[i], kind="stable")[:int(K[i]) if K[i] > 0 else V]
        if P[i] < 1:
            c = np.cumsum(w[order])
            before = np.concatenate(([0.0], c[:-1]))
            order = order[:max(1, int(np.searchsorted(before, np.float64(P[i]) * c[-1], side="left")))]
        order = np.sort(order[w[order] >= np.float64(least[i])])
        c = np.cumsum(w[order])
        token[i] = order[min(int(np.searchsorted(c, u[i] * c[-1], side="right")), len(order) - 1)]
    return torch.from_numpy(token).to(DEV)
