"""The gated feed-forward block and its gradient in float64, and how far fp32 sums may be from them.

u = 2^-24.  A sum of n products in fp32, however it is cut, is off by at most 2 u (n + 16) of the sum of the products' magnitudes: n + 16 additions and multiplications of one step each at most
(a matrix instruction may cut off where it adds).  An activation is evaluated in a few operations: it and its slope are off by at most 16 u of themselves and 8 u in the tails, where the exponential's
argument carries the error, and an error of its argument goes in with at most 1.2 (the largest slope is gelu's, 1.13)."""
import numpy as np
from scipy.special import erfc

from elements import HALF_STEP, SMALLEST, U

ACTS = ["none", "relu", "sigmoid", "tanh", "silu", "gelu", "gelu_tanh"]


def share(v):
    e = np.exp(-np.abs(v))
    return np.where(v >= 0, 1.0, e) / (1.0 + e)


def gate(v, act):
    """-> (the activation, its slope)"""
    if act == "none":
        return v, np.ones_like(v)
    if act == "relu":
        return np.maximum(v, 0.0), (v > 0).astype(np.float64)
    if act == "sigmoid":
        return share(v), share(v) * share(-v)
    if act == "tanh":
        return np.tanh(v), 4.0 * share(2 * v) * share(-2 * v)
    if act == "silu":
        return v * share(v), share(v) * (1.0 + v * share(-v))
    if act == "gelu":
        below = 0.5 * erfc(-v / np.sqrt(2.0))
        return v * below, below + v * np.exp(-0.5 * v * v) / np.sqrt(2.0 * np.pi)
    z = 2.0 * np.sqrt(2.0 / np.pi) * (v + 0.044715 * v ** 3)
    return v * share(z), share(z) + v * share(z) * share(-z) * 2.0 * np.sqrt(2.0 / np.pi) * (1.0 + 3.0 * 0.044715 * v * v)


def sums(W, X, extra=None):
    """-> (W X + extra, the error that fp32 sums may have)"""
    S, off = W @ X, 2 * U * (W.shape[1] + 16) * (np.abs(W) @ np.abs(X))
    if extra is not None:
        S, off = S + extra, off + U * (np.abs(S) + np.abs(extra))
    return S, off


def forward(Wg, Wu, X, act, type_, G0=None, U0=None):
    """-> {name: (value, tolerance)} of H, G and U"""
    G, g_off = sums(Wg, X, G0)
    S, s_off = sums(Wu, X, U0)
    v, _ = gate(G, act)
    H = v * S
    h_off = 1.2 * g_off * (np.abs(S) + s_off) + np.abs(v) * s_off + U * (16 * np.abs(H) + 8 * np.abs(S))
    rounded = lambda want, off: (want, off + HALF_STEP[type_] * (np.abs(want) + off) + SMALLEST[type_])
    return {"H": rounded(H, h_off), "G": rounded(G, g_off), "U": rounded(S, s_off)}


def backward(Wg, Wu, X, act, G, S, dH, type_):
    """-> {name: (value, tolerance)} of dX, dWg, dWu, dG and dU; G and S are the saved sums as they were rounded"""
    v, slope = gate(G, act)
    dG, dU = dH * S * slope, dH * v
    step = lambda want, off: off + HALF_STEP[type_] * (np.abs(want) + off) + SMALLEST[type_]
    dG_off = step(dG, U * (32 * np.abs(dH * S) + 16 * np.abs(dG)))
    dU_off = step(dU, U * (16 * np.abs(dU) + 8 * np.abs(dH)))
    out = {"dG": (dG, dG_off), "dU": (dU, dU_off)}
    m, B = dH.shape

    def product(name, A, A_off, Bs):
        want = sum(a @ b for a, b in zip(A, Bs))
        mag = sum(np.abs(a) @ np.abs(b) for a, b in zip(A, Bs))
        K = sum(a.shape[1] for a in A)
        off = sum(o @ np.abs(b) for o, b in zip(A_off, Bs))
        off = off + 2 * U * (K + 16) * (mag + off)
        out[name] = (want, step(want, off))

    product("dXt", [dG.T, dU.T], [dG_off.T, dU_off.T], [Wg, Wu])
    out["dX"] = tuple(a.T for a in out.pop("dXt"))
    product("dWg", [dG], [dG_off], [X.T])
    product("dWu", [dU], [dU_off], [X.T])
    return out


def check(got, want_and_tolerance, what=""):
    want, tol = want_and_tolerance
    assert got.shape == want.shape
    assert np.all(np.abs(got - want) <= tol), (what, np.nanmax(np.abs(got - want) / tol), int(np.isnan(got).sum()))
