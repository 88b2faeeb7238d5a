"""The gated block's activations and slopes where they are small, in fp32 above all: every value within a few steps of its own, not of the largest one.

u = 2^-24.  W, X and the other projection are ones, so that a sum is the number that its G0 is, exactly.  exp is off by at most a step, 2 u of its value; a sum, a product, a quotient and the fused
multiply-add by u each; an argument of the exponential that is itself rounded costs its size times u.  What is left of 2^-126 and below is held to half a step of the subnormal numbers, times what multiplies it."""
import numpy as np
import pytest

from gated_reference import gate
from elements import HALF_STEP, SMALLEST, U, stored, values
from test_gpu_gated import Arrays

pytestmark = pytest.mark.gpu

V = np.concatenate([np.linspace(-104.0, 104.0, 4001), np.logspace(-6, 0, 200), -np.logspace(-6, 0, 200)]).astype(np.float32).astype(np.float64)
SHARP = ["sigmoid", "silu"]
TINY = 2.0 ** -148            # two steps of the subnormal numbers


def pad_to(v, B):
    return np.concatenate([v, np.zeros(-v.size % B)]).reshape(-1, B)


@pytest.mark.parametrize("B", [1, 7, 64])
@pytest.mark.parametrize("act", SHARP)
def test_values(ctx, act, B):
    """sigmoid: the exponential's step (2 u), a sum and a quotient: 4 u and what they do to one another; silu a product more."""
    G = pad_to(V, B)
    m = G.shape[0]
    a = Arrays(ctx, "f32")
    zero, one = a.put(np.zeros((m, 1)))[0], a.put(np.ones((1, B)))[0]
    H = a.put(np.zeros(G.shape))[0]
    ctx.gated(zero, zero, m, 1, one, B, act, H, dG0=a.put(G)[0], dU0=a.put(np.ones(G.shape))[0])
    want, _ = gate(G, act)
    off = np.abs(H.download().reshape(G.shape).astype(np.float64) - want)
    assert np.all(off <= 6 * U * np.abs(want) + TINY * (1 + np.abs(G))), np.max(off / (U * np.abs(want) + TINY))
    a.free()


@pytest.mark.parametrize("act", SHARP)
def test_slopes(ctx, act):
    """sigmoid: the product of both shares, 3 u and 4 u of their own.  silu: share (1 + v rest); where that is negative its terms cancel, and each is counted."""
    G = pad_to(V, 16)
    m, B = G.shape
    a = Arrays(ctx, "f32")
    ones = a.put(np.ones(G.shape))[0]
    w, x = a.put(np.ones((m, 1)))[0], a.put(np.ones((1, B)))[0]
    dG, dU = (a.put(np.zeros(G.shape))[0] for _ in range(2))
    ctx.gated_grad(w, w, m, 1, x, B, act, a.put(G)[0], ones, ones, None, None, None, dG, dU)
    want, slope = gate(G, act)
    e = np.exp(-np.abs(G))
    share, rest = np.where(G >= 0, 1, e) / (1 + e), np.where(G >= 0, e, 1) / (1 + e)
    terms = share * (1 + np.abs(G) * rest) if act == "silu" else slope
    off = np.abs(dG.download().reshape(G.shape).astype(np.float64) - slope)
    assert np.all(off <= 10 * U * terms + TINY * (1 + np.abs(G))), np.max(off / (U * terms + TINY))
    off = np.abs(dU.download().reshape(G.shape).astype(np.float64) - want)
    assert np.all(off <= 6 * U * np.abs(want) + TINY * (1 + np.abs(G)))
    a.free()


def test_the_normal_distributions_bell(ctx):
    """gelu's slope below -1 is the difference of v times the bell and what is below v; the bell is exp(-v^2 / 2), whose argument's rounding would cost v^2 / 2 steps: with what it leaves put back, 6 u."""
    G = pad_to(V[np.abs(V) < 13], 16)
    m, B = G.shape
    a = Arrays(ctx, "f32")
    ones = a.put(np.ones(G.shape))[0]
    w, x = a.put(np.ones((m, 1)))[0], a.put(np.ones((1, B)))[0]
    dG = a.put(np.zeros(G.shape))[0]
    ctx.gated_grad(w, w, m, 1, x, B, "gelu", a.put(G)[0], ones, ones, None, None, None, dG)
    below, _ = gate(G, "gelu")
    below = np.where(G == 0, 0.5, below / np.where(G == 0, 1, G))
    bell = np.exp(-0.5 * G * G) / np.sqrt(2 * np.pi)
    off = np.abs(dG.download().reshape(G.shape).astype(np.float64) - (below + G * bell))
    # erfc's own error, by its argument's rounding v^2 u of it and 4 steps, is that of the library's function
    assert np.all(off <= U * (10 * np.abs(G) * bell + (12 + 2 * G * G) * below) + TINY * (1 + np.abs(G))), np.max(off / (U * (np.abs(G) * bell + below) + TINY))
    a.free()


@pytest.mark.parametrize("type_", ["f16", "bf16"])
def test_gelu_of_16_bits(ctx, type_):
    """Half a step of the type and 2^-14 of the value: the normal distribution is within 2^-19 of itself, and its exponential's argument, v^2 / 2 < 82, carries 6 u of itself, less than 2^-15."""
    G = pad_to(values(stored(np.concatenate([np.linspace(-12.7, 6.0, 3000), -np.logspace(-3, 1.1, 500)]), type_), type_), 16)
    m, B = G.shape
    a = Arrays(ctx, type_)
    ones = a.put(np.ones(G.shape))[0]
    w, x, zero = a.put(np.ones((m, 1)))[0], a.put(np.ones((1, B)))[0], a.put(np.zeros((m, 1)))[0]
    H, dG, dU = (a.put(np.zeros(G.shape))[0] for _ in range(3))
    at = a.put(G)[0]
    ctx.gated(zero, zero, m, 1, x, B, "gelu", H, dG0=at, dU0=ones, type=type_)
    ctx.gated_grad(w, w, m, 1, x, B, "gelu", at, ones, ones, None, None, None, dG, dU, type=type_)
    want, slope = gate(G, "gelu")
    bell = np.abs(G) * np.exp(-0.5 * G * G) / np.sqrt(2 * np.pi)
    terms = np.where(G == 0, 0.5, np.abs(want / np.where(G == 0, 1, G))) + bell
    for got, value, off in ((H, want, np.abs(want)), (dU, want, np.abs(want)), (dG, slope, terms)):
        off = 2.0 ** -14 * off
        got = values(got.download(), type_).reshape(G.shape)
        assert np.all(np.abs(got - value) <= off + HALF_STEP[type_] * (np.abs(value) + off) + SMALLEST[type_]), np.max(np.abs(got - value) / (np.abs(value) + SMALLEST[type_]))
    a.free()
