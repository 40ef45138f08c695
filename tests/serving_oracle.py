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
