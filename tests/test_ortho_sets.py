"""Orthogonalised updates and optimiser steps as a network's training loop makes them: ill-conditioned momenta, many layers of
mixed shapes and types in one call."""
import numpy as np
import pytest

from cpmi355 import capi
from lowbits import HALF, TYPES, Mat
from test_ortho import distance, iterate, within

gpu = pytest.mark.gpu


def distance32(U, **more):
    """(the iteration in float64, how far float32 numbers may be off).  X, A and B hold 22 bits or more: four times float32's
    rounding, which `iterate(bits=24)` makes at the same places, and others of that size may cost four times as much."""
    want = iterate(U, **more)
    rms = lambda x: np.sqrt(((x - want) ** 2).mean())
    return want, 16 * rms(iterate(U, bits=24, **more)) + rms(iterate(U, loss=3, **more))


def dominated(rs, rows, cols, top):
    """What a momentum looks like after many steps: a few directions `top` times as strong as the rest."""
    r = min(4, rows, cols)
    return rs.randn(rows, cols) + top * rs.randn(rows, r) @ rs.randn(r, cols)


# ---- precision follows the widest input, not the result ----------------------------------------------------------------------

CONDITIONED = [(40, 300), (300, 40), (64, 500), (130, 260), (260, 130), (256, 576)]


@gpu
@pytest.mark.parametrize("rows,cols", CONDITIONED)
@pytest.mark.parametrize("top", [10.0, 1000.0])
@pytest.mark.parametrize("gk", ["f32", "f16"])
def test_bfloat16_result_of_a_wider_input(ctx, rows, cols, top, gk):
    """The iteration amplifies what is lost of small singular directions by 3.4 a step: 11 bits would cost up to 7 % here."""
    rs = np.random.RandomState(int(top) + rows)
    G, O = Mat(ctx, dominated(rs, rows, cols, top) * 2.0 ** -4, gk), Mat(ctx, np.zeros((rows, cols)), "bf16")
    ctx.orthogonalise(capi.OrthoJobs([(G.ptr, TYPES[gk], rows, cols, O.ptr, TYPES["bf16"])]))
    within(O.get(), *distance32(G.get()), "bf16")


@gpu
@pytest.mark.parametrize("rows,cols", CONDITIONED)
@pytest.mark.parametrize("top", [10.0, 1000.0])
@pytest.mark.parametrize("gk,wk", [("bf16", "bf16"), ("f32", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("nesterov", [True, False])
def test_step_of_an_ill_conditioned_momentum(ctx, rows, cols, top, gk, wk, nesterov):
    rs = np.random.RandomState(int(top) + cols)
    G, M = Mat(ctx, dominated(rs, rows, cols, top / 20), gk), Mat(ctx, dominated(rs, rows, cols, top), "f32")
    W = Mat(ctx, np.zeros((rows, cols)), wk)
    g, m = G.get(), M.get()
    ctx.ortho_step(capi.OrthoStepJobs([(G.ptr, TYPES[gk], rows, cols, M.ptr, W.ptr, TYPES[wk], 1.0)]), 1.0, nesterov=nesterov)
    m2 = 0.95 * m + g
    assert (np.abs(M.get() - m2) <= 2.0 ** -24 * (np.abs(m2) + np.abs(m)) + 1e-30).all()
    # U is a float32 number of the float32 momentum: M's rounding, the factor's, and U's own, half a step each, amplified as any
    # change of U; `moved` is what changes of that size do
    U = g + 0.95 * m2 if nesterov else m2
    want, far = distance32(U)
    moved = iterate(U + 2.0 ** -24 * (np.abs(m2) + np.abs(m) + np.abs(U)) * rs.choice([-1, 1], U.shape)) - want
    within(-W.get(), want, far + 4 * np.sqrt((moved ** 2).mean()), wk)
