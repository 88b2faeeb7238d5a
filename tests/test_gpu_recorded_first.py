"""Kernels whose first launch on a context is inside a recording, with more LDS than a launch has unasked: replayed as often as eager, the same bits."""
import numpy as np
import pytest

import hipabi
from elements import place, stored
from test_gpu_mxfp4 import FORMS, weights

pytestmark = pytest.mark.gpu


def replayed(ctx, calls, outs, inputs, fresh):
    """calls() recorded before any launch of its kernels, then replays and eager calls in turn on new inputs."""
    ctx.graph_begin()
    try:
        calls()
    finally:
        graph = ctx.graph_end()
    for _ in range(3):
        for a in inputs:
            a.upload(fresh(a))
        ctx.graph_launch(graph)
        got = [o.download().copy() for o in outs]
        for o in outs:
            o.upload(np.zeros(o.shape, o.dtype))
        calls()
        for o, g in zip(outs, got):
            assert np.array_equal(o.download().view(np.uint8), g.view(np.uint8)) and g.any()
    ctx.graph_free(graph)


@pytest.mark.parametrize("form", range(1, len(FORMS) + 1))
def test_products(form):
    rng = np.random.default_rng(form)
    ctx = hipabi.Context()
    try:
        m, n, C = 300, 900, 280
        W, _ = weights(ctx, rng, m, n)
        dX, dY, dx, dy = ctx.empty((n, C)), ctx.empty((m, C)), ctx.empty((n,)), ctx.empty((m,))
        with ctx.tuning(SPARSEOPS_MXFP4_MATMUL=form):
            ctx.mxfp4_matmul_reserve(W, C)

            def calls():
                ctx.mxfp4_matmul(W, dX, C, None, dY, "tanh")
                ctx.mxfp4_matvec(W, dx, None, dy)

            replayed(ctx, calls, (dY, dy), (dX, dx), lambda a: rng.standard_normal(a.shape).astype(np.float32))
        W.free()
    finally:
        ctx.close()


def test_a_long_vector():
    rng = np.random.default_rng(0)
    ctx = hipabi.Context()
    try:
        W, _ = weights(ctx, rng, 50, 20000)
        dx, dy = ctx.empty((20000,)), ctx.empty((50,))
        replayed(ctx, lambda: ctx.mxfp4_matvec(W, dx, None, dy), (dy,), (dx,), lambda a: rng.standard_normal(a.shape).astype(np.float32))
        W.free()
    finally:
        ctx.close()


@pytest.mark.parametrize("type_,F,B", [("f32", 8000, 2100), ("bf16", 7001, 4111), ("f16", 9001, 40)])
def test_layer_norm(type_, F, B):
    """All features of a tile in one workgroup, its scales and shifts in LDS, and in parts; the gradient behind it."""
    rng = np.random.default_rng(F)
    ctx = hipabi.Context()
    try:
        dX, dDy, dY, dDx = (place(ctx, np.zeros((F, B)), type_)[0] for _ in range(4))
        dG, dB, dM, dR, dDg, dDb = ctx.array(rng.standard_normal(F).astype(np.float32)), ctx.array(rng.standard_normal(F).astype(np.float32)), ctx.empty((B,)), ctx.empty((B,)), ctx.empty((F,)), ctx.empty((F,))
        ctx.layer_norm_reserve(F, B, type=type_)

        def calls():
            ctx.layer_norm(dX, F, B, dG, dB, 1e-5, dY, dM, dR, type=type_)
            ctx.layer_norm_grad(dX, dDy, F, B, dG, dM, dR, dDx, dDg, dDb, type=type_)

        noise = rng.standard_normal(F * B).astype(np.float32)
        replayed(ctx, calls, (dY, dM, dR, dDx, dDg, dDb), (dX, dDy), lambda a: stored(np.roll(noise, int(rng.integers(F * B))), type_))
    finally:
        ctx.close()
