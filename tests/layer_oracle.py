"""Head norm with rotation, attention and the gated product from their formulas, in numpy and 64 bits."""
import math

import numpy as np
from threadpoolctl import threadpool_limits

EPS = 1e-6


def table(positions, rotary, base=10000.0, factor=1.0, keep_below=0.0, slow_above=0.0):
    half = rotary // 2
    f = base ** (-np.arange(half) / half)
    if factor != 1.0:
        wave = 2 * np.pi / f
        keep = np.zeros(half)
        if slow_above:
            keep = np.clip((slow_above / wave - 1) / (slow_above / keep_below - 1), 0, 1)
        f = f * (keep + (1 - keep) / factor)
    angle = np.arange(positions)[:, None] * f
    return np.stack([np.cos(angle), np.sin(angle)], -1)


def _turn(x, cs, rotary, interleaved, back=False):
    """x (tokens, heads, dim), cs (tokens, rotary / 2, 2)"""
    x = x.copy()
    if not rotary:
        return x
    z = x[..., :rotary]
    a, b = (z[..., 0::2].copy(), z[..., 1::2].copy()) if interleaved else (z[..., : rotary // 2].copy(), z[..., rotary // 2:].copy())
    w = (a + 1j * b) * (cs[:, None, :, 0] + 1j * cs[:, None, :, 1] * (-1 if back else 1))
    if interleaved:
        z[..., 0::2], z[..., 1::2] = w.real, w.imag
    else:
        z[..., : rotary // 2], z[..., rotary // 2:] = w.real, w.imag
    return x


def _angles(t, positions, tokens):
    if t is None:
        return None
    p = np.arange(tokens) if positions is None else np.asarray(positions)
    return np.asarray(t, np.float64)[np.clip(p, 0, len(t) - 1)]


def norm_rotary(x, weight, t, positions, rotary, interleaved, norm):
    x = np.asarray(x, np.float64)
    n = x
    if norm:
        n = x / np.sqrt((x * x).mean(-1, keepdims=True) + EPS) * (1.0 if weight is None else np.asarray(weight, np.float64))
    return _turn(n, _angles(t, positions, len(x)), rotary, interleaved)


def norm_rotary_grad(x, weight, dy, t, positions, rotary, interleaved, norm):
    x, dy = np.asarray(x, np.float64), np.asarray(dy, np.float64)
    g = _turn(dy, _angles(t, positions, len(x)), rotary, interleaved, back=True)
    if not norm:
        return g, None
    w = 1.0 if weight is None else np.asarray(weight, np.float64)
    r = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + EPS)
    u = x * r
    return r * (w * g - u * (w * g * u).mean(-1, keepdims=True)), (g * u).sum((0, 1))


def _seen(nq, nk, causal):
    return (np.arange(nk) <= np.arange(nq)[:, None] + nk - nq) if causal else np.ones((nq, nk), bool)


def _weights(q, k, seen, scale):
    s = np.where(seen, scale * q @ k.T, -np.inf)
    m = s.max(-1, keepdims=True, initial=-np.inf)
    e = np.exp(s - np.where(np.isfinite(m), m, 0))
    total = e.sum(-1, keepdims=True)
    with np.errstate(divide="ignore"):
        lse = np.where(total > 0, np.where(np.isfinite(m), m, 0) + np.log(total), -np.inf)
    return e / np.where(total > 0, total, 1), lse[:, 0]


@threadpool_limits.wrap(limits=1)  # many small products
def attention(q, k, v, q_starts, k_starts, scale, causal, do=None):
    """(o, lse), or with do (dq, dk, dv); NaN in rows of no sequence"""
    q, k, v = (np.asarray(a, np.float64) for a in (q, k, v))
    H, g = q.shape[1], q.shape[1] // k.shape[1]
    o, lse = np.full_like(q, np.nan), np.full((H, len(q)), np.nan)
    dq, dk, dv = np.full_like(q, np.nan), np.full_like(k, np.nan), np.full_like(v, np.nan)
    for i in range(len(q_starts) - 1):
        a, b = slice(q_starts[i], q_starts[i + 1]), slice(k_starts[i], k_starts[i + 1])
        nq, nk = q_starts[i + 1] - q_starts[i], k_starts[i + 1] - k_starts[i]
        dk[b], dv[b] = 0, 0
        for h in range(H):
            e = h // g
            p, lse[h, a] = _weights(q[a, h], k[b, e], _seen(nq, nk, causal), scale)
            o[a, h] = p @ v[b, e]
            if do is not None:
                gr = np.asarray(do, np.float64)[a, h]
                dp = gr @ v[b, e].T
                ds = scale * p * (dp - (p * dp).sum(-1, keepdims=True))
                dq[a, h] = ds @ k[b, e]
                dk[b, e] += ds.T @ q[a, h]
                dv[b, e] += p.T @ gr
    return (o, lse) if do is None else (dq, dk, dv)


_erf = np.vectorize(math.erf, otypes=[np.float64])


def gate(a, act):
    """value and slope"""
    with np.errstate(over="ignore"):
        s = 1 / (1 + np.exp(-a))
    if act == "silu":
        return a * s, s * (1 + a * (1 - s))
    if act == "sigmoid":
        return s, s * (1 - s)
    if act == "relu":
        return np.maximum(a, 0), (a > 0).astype(np.float64)
    p = 0.5 * (1 + _erf(a / math.sqrt(2)))
    return a * p, p + a * np.exp(-0.5 * a * a) / math.sqrt(2 * math.pi)


def gated(x, w, act):
    pre = np.asarray(x, np.float64) @ np.asarray(w, np.float64)
    n = pre.shape[1] // 2
    return gate(pre[:, :n], act)[0] * pre[:, n:], pre


def gated_grad(x, w, pre, dh, act):
    x, w, pre, dh = (np.asarray(a, np.float64) for a in (x, w, pre, dh))
    n = pre.shape[1] // 2
    f, df = gate(pre[:, :n], act)
    dpre = np.concatenate([dh * pre[:, n:] * df, dh * f], 1)
    return dpre @ w.T, x.T @ dpre
