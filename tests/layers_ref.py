"""Activations of the fused layers in 64 bits, with the error bounds of their
FLOAT32 evaluation (U = 2^-24, half a step)."""
import numpy as np

U = 2.0 ** -24
ACTS = ("none", "relu", "tanh", "sigmoid", "silu", "gelu")


def sigmoid(x):
    e = np.exp(-np.abs(x))
    return np.where(x >= 0, 1 / (1 + e), e / (1 + e))


def act(u, name):
    """act(u), act'(u), and bounds of |act''| and of the evaluation's error of
    either for an exact u.  csrc/jmath.cuh: tanh within 13 and sigmoid within
    3.5 + 1.2 |x| units of 2^-23 (2 U) relative."""
    one = np.ones_like(u)
    if name == "none":
        return u, one, 0.0, 0 * u, 0 * u
    if name == "relu":
        return np.maximum(u, 0), (u > 0) * 1.0, 0.0, 0 * u, 0 * u
    if name == "tanh":
        t = np.tanh(u)
        e = 26 * U * np.abs(t)
        return t, 1 - t * t, 0.77, e, 2 * np.abs(t) * e + 2 * U
    s_of = {"sigmoid": u, "silu": u, "gelu": 2 * np.sqrt(2 / np.pi) * (u + 0.044715 * u ** 3)}[name]
    s = sigmoid(s_of)
    # the argument of gelu's sigmoid is off by at most 6 U of itself: s' |arg| 6 U <= s |arg| 6 U
    es = s * (2 * (3.5 + 1.2 * np.abs(s_of)) + 6 * np.abs(s_of)) * U + 2e-38
    q = s * (1 - s)
    eq = es + 2 * U * q
    if name == "sigmoid":
        return s, q, 0.1, es, eq
    d = one if name == "silu" else 2 * np.sqrt(2 / np.pi) * (1 + 0.134145 * u ** 2)
    slope = s + u * q * d
    return u * s, slope, 0.5 if name == "silu" else 1.2, np.abs(u) * (es + U * s), \
        es + np.abs(u * d) * (eq + 8 * U * q) + 2 * U * (s + np.abs(u * q * d))
