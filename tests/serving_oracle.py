"""The norm of a layer's rows, products in 8-bit integers and attention over a cache in 8 bits from their formulas, in numpy and 64 bits."""
import numpy as np


def layer_norm(x, weight, bias, epsilon):
    """(y, u): the result, and the rows before weight and bias"""
    x = np.asarray(x, np.float64)
    d = x - x.mean(-1, keepdims=True)
    with np.errstate(divide="ignore", invalid="ignore"):
        u = d / np.sqrt((d * d).mean(-1, keepdims=True) + epsilon)
    w = 1.0 if weight is None else np.asarray(weight, np.float64)
    return u * w + (0.0 if bias is None else np.asarray(bias, np.float64)), u


def layer_norm_grad(x, dy, weight, epsilon):
    """(dx, dweight, dbias)"""
    x, g = np.asarray(x, np.float64), np.asarray(dy, np.float64)
    d = x - x.mean(-1, keepdims=True)
    r = 1 / np.sqrt((d * d).mean(-1, keepdims=True) + epsilon)
    u, wg = d * r, g * (1.0 if weight is None else np.asarray(weight, np.float64))
    return r * (wg - wg.mean(-1, keepdims=True) - u * (wg * u).mean(-1, keepdims=True)), (g * u).sum(0), g.sum(0)


def quantize(x):
    """(codes, scales) of rows: the scale is an fp32 number by definition, the codes come from exact quotients (64 bits tell a half of a
    step from what is next to it: x and scale have 24 bits each)"""
    x = np.asarray(x, np.float64)
    good = np.isfinite(x).all(1)
    with np.errstate(invalid="ignore"):
        scales = np.maximum((np.abs(x).max(1, initial=0).astype(np.float32) / np.float32(127)).astype(np.float32), np.float32(2.0 ** -100))
        codes = np.rint(np.where(good[:, None], x, 0) / np.where(good, scales, 1)[:, None].astype(np.float64))
    return codes.astype(np.int8), np.where(good, scales, np.nan).astype(np.float32)


def matmul_int8(x, x_scales, w, w_scales):
    return (x.astype(np.float64) @ w.astype(np.float64).T) * (np.asarray(x_scales, np.float64)[:, None] * np.asarray(w_scales, np.float64))


PAGE = 64


class Cache:
    """pages token by token as the definition has them: codes, scales (powers of two that only grow while a page fills), in float64"""

    def __init__(self, pages, kv_heads, dim):
        self.codes = {n: np.zeros((pages, kv_heads, PAGE, dim)) for n in "kv"}
        self.scales = {n: np.full((pages, kv_heads), np.nan) for n in "kv"}

    @staticmethod
    def _page(table, s, place):
        p = place // PAGE
        return int(table[s][p]) if place >= 0 and p < len(table[s]) else -1

    def _places(self, starts, lengths, table):
        """(row, page, slot) of each row of a call; page -1: none"""
        for s in range(len(lengths)):
            for r in range(starts[s], starts[s + 1]):
                place = int(lengths[s]) - int(starts[s + 1]) + r
                page = self._page(table, s, place)
                yield r, page if 0 <= page < len(self.scales["k"]) else -1, place % PAGE

    def append(self, k, v, starts, lengths, table):
        for name, x in (("k", k), ("v", v)):
            x = np.asarray(x, np.float64)
            runs = {}  # rows of a call that one page gets
            for r, page, slot in self._places(starts, lengths, table):
                if page >= 0:
                    runs.setdefault(page, []).append((r, slot))
            for page, rows in runs.items():
                for h in range(x.shape[1]):
                    new, held = x[[r for r, _ in rows], h], rows[0][1]
                    old = self.scales[name][page, h] if held else 0.0
                    largest = np.abs(new).max()
                    if not np.isfinite(largest):
                        need = np.nan
                    else:
                        need = 2.0 ** -100
                        while 127 * need < largest:
                            need *= 2
                    scale = np.nan if np.isnan(need) or np.isnan(old) else max(need, old)
                    codes = self.codes[name][page, h]
                    if held and not np.isnan(scale):
                        codes[:held] = np.rint(codes[:held] * (old / scale))
                    for (r, slot), row in zip(rows, new):
                        codes[slot] = 0 if np.isnan(scale) else np.rint(row / scale)
                    self.scales[name][page, h] = scale

    def value(self, name, page, h):
        """(token, dim)"""
        return self.codes[name][page, h] * self.scales[name][page, h]

    def read(self, rows, starts, lengths, table, like):
        out = [np.array(a, np.float64) for a in like]
        for r, page, slot in self._places(starts, lengths, table):
            for i, name in enumerate("kv"):
                for h in range(out[i].shape[1]):
                    out[i][r, h] = self.value(name, page, h)[slot] if page >= 0 else 0
        return out


def attention_cache(q, k_values, v_values, starts, lengths, table, pages, scale, causal):
    """(o, lse) over values [page][head][token][dim]; NaN in rows of no sequence"""
    q = np.asarray(q, np.float64)
    H, G = q.shape[1], k_values.shape[1]
    o, lse = np.full_like(q, np.nan), np.full((H, len(q)), np.nan)
    for s in range(len(lengths)):
        n, length = starts[s + 1] - starts[s], int(lengths[s])
        if not n:
            continue
        places = np.arange(min(length, len(table[s]) * PAGE))
        ids = np.asarray(table[s], np.int64)[places // PAGE] if len(places) else np.zeros(0, np.int64)
        there = (ids >= 0) & (ids < pages)
        seen = there & (places <= np.arange(n)[:, None] + length - n) if causal else np.broadcast_to(there, (n, len(places)))
        for h in range(H):
            e = h * G // H
            k, v = (np.where(there[:, None], a[np.where(there, ids, 0), e, places % PAGE], 0) for a in (k_values, v_values))
            t = np.where(seen, scale * (q[starts[s]:starts[s + 1], h] @ k.T), -np.inf)
            m = t.max(1, initial=-np.inf)
            w = np.exp(t - np.where(np.isfinite(m), m, 0)[:, None])
            total = w.sum(1)
            with np.errstate(divide="ignore"):
                lse[h, starts[s]:starts[s + 1]] = np.where(total > 0, np.where(np.isfinite(m), m, 0) + np.log(total), -np.inf)
            o[starts[s]:starts[s + 1], h] = w / np.where(total > 0, total, 1)[:, None] @ v
    return o, lse
