"""Routing by scores, block norm and sampling from their definitions, in 64 bits (numpy), with the rounding bounds of
the kernels' 32-bit parts."""
import numpy as np

U = 2.0 ** -24                                        # half a step of f32
HALF = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}


def first(v, n):
    return np.argsort(-v, kind="stable")[:n]


def route(l, K, score="softmax", bias=None, n_groups=1, top_groups=None, group_best=1, renormalize=True, scale=1.0):
    l = np.asarray(l, np.float64)
    T, E = l.shape
    m = E // n_groups
    ids, w, s_all = np.empty((T, K), np.int32), np.empty((T, K)), np.empty((T, E))
    with np.errstate(all="ignore"):
        for t in range(T):
            on = l[t] > -np.inf
            if score == "sigmoid":
                s = np.where(on, 1.0 / (1.0 + np.exp(-l[t])), 0.0)
            else:
                mx = l[t][on].max() if on.any() else 0.0
                ex = np.where(on, (l[t] == mx) * 1.0 if mx == np.inf else np.exp(l[t] - mx), 0.0)
                s = np.where(on, ex / ex.sum(), 0.0)
            s_all[t] = s
            v = np.where(on, s if bias is None else s + np.asarray(bias, np.float64), -np.inf)
            v = np.where(np.isnan(v), -np.inf, v)
            if n_groups > 1:
                gs = np.full(n_groups, -np.inf)
                for g in range(n_groups):
                    alive = np.sort(v[g * m:(g + 1) * m])[::-1]
                    alive = alive[alive > -np.inf][:group_best]
                    if len(alive):
                        gs[g] = alive.sum()
                keep = first(gs, n_groups if top_groups is None else top_groups)
                for g in set(range(n_groups)) - set(keep.tolist()):
                    v[g * m:(g + 1) * m] = -np.inf
            ids[t] = first(v, K)
            ws = np.where(v[ids[t]] > -np.inf, s[ids[t]], 0.0)
            if renormalize:
                ws = ws / ws.sum() if ws.sum() > 0 else ws * 0.0
            w[t] = float(np.float32(scale)) * ws
    return ids, w, s_all


def _unit(z, e_z, kind, eps, g, c, off, n_red):
    """N(z; g, c) and a bound of its error, given the bound e_z of z's; n_red: roundings of a sum over the row."""
    H = z.shape[1]
    mu, e_mu = 0.0, 0.0
    if kind == "layer":
        mu = z.mean(1, keepdims=True)
        e_mu = e_z.mean(1, keepdims=True) + (n_red + 2) * U * np.abs(z).mean(1, keepdims=True)
    d = z - mu
    e_d = e_z + e_mu + U * np.abs(d)
    ms = np.square(d).mean(1, keepdims=True) + eps
    # the sum of squares: its roundings, and what the terms' errors do to it
    e_ms = (n_red + 4) * U * ms + (2 * np.abs(d) * e_d + e_d * e_d).mean(1, keepdims=True)
    inv = 1.0 / np.sqrt(ms)
    rel_inv = 0.5 * e_ms / np.maximum(ms - e_ms, 1e-300) + 4 * U
    gg = 1.0 if g is None else g + off
    y = d * inv * gg
    e = np.abs(inv * gg) * e_d * (1 + rel_inv) + np.abs(y) * (rel_inv + 4 * U)
    if c is not None:
        y = y + c
        e = e + 2 * U * np.abs(y)
    return y, e


def block_norm(x, branch=None, gate=None, weight=None, bias=None, post_weight=None, post_bias=None, kind="rms",
               eps=1e-6, post_eps=None, post=False, weight_offset=0.0, scale=1.0, gate_act=None):
    """(y, r) before their rounding to the output type, and the bounds of what the f32 arithmetic adds.

    A sum over a row is a chain of at most 64 terms a thread and a tree of at most 20 levels; exp and the divisions
    are taken as 4 half steps each."""
    n_red = 84
    x = np.asarray(x, np.float64)
    r, e_r = x, np.zeros_like(x)
    f = lambda t: None if t is None else np.asarray(t, np.float64)
    weight, bias, post_weight, post_bias, gate = map(f, (weight, bias, post_weight, post_bias, gate))
    eps, off, scale = (float(np.float32(v)) for v in (eps, weight_offset, scale))
    if branch is not None:
        b = f(branch)
        e_b = np.zeros_like(x)
        if b.ndim == 3:
            e_b = b.shape[1] * U * np.abs(b).sum(1)
            b = b.sum(1)
        if post:
            b, e_b = _unit(b, e_b, kind, float(np.float32(eps if post_eps is None else post_eps)), post_weight, post_bias,
                           off, n_red)
        g = np.ones((1, 1)) if gate is None else gate.reshape(-1, 1) if gate.ndim == 1 and len(gate) == len(x) != \
            x.shape[1] else gate.reshape(-1, 1) if gate.ndim == 2 and gate.shape[1] == 1 else gate.reshape(-1, x.shape[1])
        if gate_act == "sigmoid":
            g = 1.0 / (1.0 + np.exp(-g))
        r = x + scale * g * b
        e_r = np.abs(scale * g) * e_b + 12 * U * np.abs(scale * g * b) + U * np.abs(r)
    y, e_y = _unit(r, e_r, kind, eps, weight, bias, off, n_red)
    return y, r, e_y, e_r


def sample(l, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    l = np.asarray(l, np.float64)
    T, V = l.shape
    row = lambda p, t: p[t] if np.ndim(p) else p
    tokens, probs = np.empty(T, np.int32), np.empty(T)
    for t in range(T):
        x = np.where(np.isnan(l[t]), -np.inf, l[t])
        order = np.argsort(-x, kind="stable")
        order = order[x[order] > -np.inf]
        tp, k = float(np.float32(row(temperature, t))), int(row(top_k, t))
        p, mp = float(np.float32(row(top_p, t))), float(np.float32(row(min_p, t)))
        if not len(order):
            tokens[t], probs[t] = -1, 0.0
            continue
        if not tp > 0:
            tokens[t], probs[t] = order[0], 1.0
            continue
        mx = x[order[0]]
        with np.errstate(over="ignore", invalid="ignore"):
            e = (x[order] == mx) * 1.0 if mx == np.inf else np.exp((x[order] - mx) / tp)
        if 0 < k < V:
            e = e[:k]
        if p < 1.0:
            c = np.cumsum(e)
            e = e[:int(np.argmax(c >= max(p, 0.0) * c[-1])) + 1]
        if mp > 0.0:
            e = e[:max(1, int((e >= mp).sum()))]
        c = np.cumsum(e)
        uu = float(np.float32(u[t]))
        uu = min(uu, 1.0 - 2.0 ** -24) if uu > 0 else 0.0
        j = int(np.searchsorted(c, uu * c[-1], side="right"))
        tokens[t], probs[t] = order[j], e[j] / c[-1]
    return tokens, probs
