"""The layer calls' operators in 64 bits with numpy, from their definitions,
and the error bounds the tests use.

Bounds.  A stored value is off by half a step of its type, HALF[dtype] of the
value (TINY[dtype] where steps no longer shrink).  A sum of n products in f32
is off by at most n * 2^-23 of the sum of the products' magnitudes (2^-24 for
a rounded addition; 2^-23 also covers one that truncates).  The f32
activations and slopes are within (16 + 2 z^2) 2^-24 of the sum of their
parts' magnitudes: a few units in the last place for exp, erfc, expm1, tanh and
the operations around them, and the rounding of the argument of erfc(z / sqrt
2) and exp(-z^2 / 2), which their condition number z^2 magnifies.
"""

import numpy as np
from scipy import special

HALF = {"f64": 2.0 ** -53, "f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}
# Below the smallest normal number a step no longer shrinks with the value.
TINY = {"f64": 2.0 ** -1074, "f32": 2.0 ** -149, "bf16": 2.0 ** -133, "f16": 2.0 ** -24}
U32 = 2.0 ** -24

ACTS = ["none", "relu", "leaky_relu", "elu", "sigmoid", "tanh", "gelu", "swish",
        "mish"]


def sigmoid(z):
    return special.expit(z)


def act(name, z):
    if name == "none":
        return z
    if name == "relu":
        return np.where(z > 0, z, 0.0)
    if name == "leaky_relu":
        return np.where(z > 0, z, 0.01 * z)
    if name == "elu":
        return np.where(z > 0, z, np.expm1(np.minimum(z, 0)))
    if name == "sigmoid":
        return sigmoid(z)
    if name == "tanh":
        return np.tanh(z)
    if name == "gelu":
        return 0.5 * z * special.erfc(-z / np.sqrt(2.0))
    if name == "swish":
        return z * sigmoid(z)
    return z * np.tanh(np.logaddexp(z, 0.0))


def slope(name, z):
    if name == "none":
        return np.ones_like(z)
    if name == "relu":
        return np.where(z > 0, 1.0, 0.0)
    if name == "leaky_relu":
        return np.where(z > 0, 1.0, 0.01)
    if name == "elu":
        return np.where(z > 0, 1.0, np.exp(np.minimum(z, 0)))
    if name == "sigmoid":
        return sigmoid(z) * sigmoid(-z)
    if name == "tanh":
        return 1.0 / np.cosh(np.clip(z, -300, 300)) ** 2
    if name == "gelu":
        return (0.5 * special.erfc(-z / np.sqrt(2.0))
                + z * np.exp(-0.5 * z * z) / np.sqrt(2 * np.pi))
    if name == "swish":
        return sigmoid(z) * (1 + z * sigmoid(-z))
    t = np.tanh(np.logaddexp(z, 0.0))
    return t + z * (1 - t * t) * sigmoid(z)


def slope_parts(name, z):
    """The slope with its terms' magnitudes added instead."""
    if name == "gelu":
        return (0.5 * special.erfc(-z / np.sqrt(2.0))
                + np.abs(z) * np.exp(-0.5 * z * z) / np.sqrt(2 * np.pi))
    if name == "swish":
        return sigmoid(z) * (1 + np.abs(z) * sigmoid(-z))
    if name == "mish":
        t = np.tanh(np.logaddexp(z, 0.0))
        return t + np.abs(z) * (1 - t * t) * sigmoid(z)
    return np.abs(slope(name, z))


def function_err(name, z, parts):
    return 0.0 if name == "none" else (16 + 2 * z * z) * U32 * parts + 2.0 ** -140


def linear(x, w, bias, name, residual, dtype):
    """(y, its bound, z, its bound)."""
    k = x.shape[1]
    z = x @ w
    err = (k + 2) * 2 * U32 * (np.abs(x) @ np.abs(w))
    if bias is not None:
        z = z + bias
        err = err + 2 * U32 * (np.abs(z) + np.abs(bias))
    y = act(name, z)
    # Every activation's slope is within 1.13.
    bound = 1.13 * err + function_err(name, z, np.abs(y))
    if residual is not None:
        y = y + residual
        bound = bound + 2 * U32 * (np.abs(y) + np.abs(residual))
    half = HALF[dtype]
    return (y, bound * (1 + half) + half * np.abs(y) + TINY[dtype],
            z, err * (1 + half) + half * np.abs(z) + TINY[dtype])


def output_grad(dy, z, name, dtype):
    dz = dy * slope(name, z) if name != "none" else dy
    bound = 0 if name == "none" else function_err(
        name, z, np.abs(dy) * slope_parts(name, z))
    return dz, bound * (1 + HALF[dtype]) + HALF[dtype] * np.abs(dz) + TINY[dtype]


def column_sums(dz, dtype):
    s = dz.sum(0)
    err = (dz.shape[0] + 2) * U32 * np.abs(dz).sum(0)
    return s, err * (1 + HALF[dtype]) + HALF[dtype] * np.abs(s) + TINY[dtype]


def product(a, b, dtype, name="none", z=None, residual=None):
    """a . b, times the slope at z, plus the residual, and the bound."""
    p = a @ b
    bound = (a.shape[1] + 2) * 2 * U32 * (np.abs(a) @ np.abs(b))
    if name != "none":
        bound = bound * 1.13 + function_err(name, z, np.abs(p) * slope_parts(name, z))
        p = p * slope(name, z)
    if residual is not None:
        p = p + residual
        bound = bound + 2 * U32 * (np.abs(p) + np.abs(residual))
    half = HALF[dtype]
    return p, bound * (1 + half) + half * np.abs(p) + TINY[dtype]


def unit(dtype):
    return 2.0 ** -53 if dtype == "f64" else 2.0 ** -24


def layer_norm(x, gamma, beta, eps, dtype):
    """((y, bound), (mean, bound), (rstd, bound)).

    A row's sum adds at most cols / 32 + 16 numbers one after another (the
    longest chain of any kernel), so it is off by h * u of the sum of the
    magnitudes.  The differences from a mean that is off by e change the
    variance by e^2 and by the differences' own rounding."""
    cols = x.shape[1]
    u, h = unit(dtype), cols / 32 + 16
    mean = x.mean(1, keepdims=True)
    d = x - mean
    var = (d * d).mean(1, keepdims=True)
    rstd = 1 / np.sqrt(var + eps)
    mean_err = h * u * np.abs(x).mean(1, keepdims=True) + u * np.abs(mean)
    d_err = mean_err + u * (np.abs(d) + np.abs(mean))
    var_err = ((h + 4) * u * var + 2 * (np.abs(d) * d_err).mean(1, keepdims=True)
               + (d_err ** 2).mean(1, keepdims=True))
    rstd_rel = 0.5 * var_err / (var + eps) * 1.1 + 4 * u
    y = d * rstd
    err = rstd * d_err + np.abs(y) * (rstd_rel + 2 * u)
    if gamma is not None:
        y, err = y * gamma, (err + u * np.abs(y)) * np.abs(gamma)
    if beta is not None:
        y = y + beta
        err = err + 2 * u * (np.abs(y) + np.abs(beta))
    half = HALF[dtype]
    return ((y, err * (1 + half) + half * np.abs(y) + 2 * u * np.abs(y) + TINY[dtype]),
            (mean[:, 0], mean_err[:, 0]), (rstd[:, 0], (rstd * rstd_rel)[:, 0]))


def layer_norm_grad(dy, x, mean, rstd, gamma, residual, dtype):
    """((dx, bound), (dgamma, bound), (dbeta, bound)) for the given mean and
    rstd."""
    rows, cols = x.shape
    u, h = unit(dtype), cols / 32 + 20
    m, r = mean[:, None], rstd[:, None]
    xhat = (x - m) * r
    xhat_err = 2 * u * (np.abs(xhat) + np.abs(m * r))
    g = dy if gamma is None else dy * gamma
    a, b = g.mean(1, keepdims=True), (g * xhat).mean(1, keepdims=True)
    a_err = h * u * np.abs(g).mean(1, keepdims=True)
    b_err = (h * u * np.abs(g * xhat).mean(1, keepdims=True)
             + (np.abs(g) * xhat_err).mean(1, keepdims=True))
    dx = r * (g - a - xhat * b)
    err = r * (4 * u * (np.abs(g) + np.abs(a) + np.abs(xhat * b)) + a_err
               + np.abs(xhat) * b_err + xhat_err * np.abs(b))
    if residual is not None:
        dx = dx + residual
        err = err + 2 * u * (np.abs(dx) + np.abs(residual))
    half = HALF[dtype]
    n = rows + 8
    dgamma, dbeta = (dy * xhat).sum(0), dy.sum(0)
    dg_err = n * u * np.abs(dy * xhat).sum(0) + (np.abs(dy) * xhat_err).sum(0)
    db_err = n * u * np.abs(dy).sum(0)
    return ((dx, err * (1 + half) + half * np.abs(dx) + TINY[dtype]),
            (dgamma, dg_err * (1 + half) + half * np.abs(dgamma) + TINY[dtype]),
            (dbeta, db_err * (1 + half) + half * np.abs(dbeta) + TINY[dtype]))
