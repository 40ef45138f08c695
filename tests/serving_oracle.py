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
