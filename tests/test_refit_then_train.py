"""GPU: a layer that the framework has pruned and refitted goes on in the 8-bit products and the orthogonalised step."""
import numpy as np
import pytest

from cpmi355 import capi
from lowbits import Held, Mat, quant
from test_blocks8 import product_bound
from test_ortho import step

pytestmark = pytest.mark.gpu


def real(v, fmt, tile):
    """What a matrix stands for once it is held in 8 bits."""
    q, s = quant(v, fmt, tile)
    return q * s.astype(np.float64).T.repeat(tile, 0)[:v.shape[0]].repeat(128, 1)[:, :v.shape[1]]


@pytest.mark.parametrize("layer,N,c,n,rank", [(2, 600, 64, 48, 32), (3, 400, 96, 130, 55)])
def test_a_refitted_layer_serves_and_trains(ctx, layer, N, c, n, rank):
    import cp_oracle
    import lib.cfgs as cfgs
    import lib.decompose as D
    X, W2, Y, B2 = cp_oracle.synth_layer(layer, N, c, n, 3)
    np.random.seed(1236)
    cfgs.alpha = 1e-3
    kept, newW, newB = D.dictionary(X.astype(np.float64), W2, Y, rank=rank, B2=B2)
    x = np.ascontiguousarray(X[:, kept].reshape(N, -1), dtype=np.float32).astype(np.float64)
    w = np.ascontiguousarray(newW.reshape(n, -1), dtype=np.float32).astype(np.float64)
    b = np.ascontiguousarray(newB, dtype=np.float32)
    k = x.shape[1]
    assert w.shape == (n, k) and k == 9 * int(kept.sum())

    # one training pass in 8 bits: the output with the refit's bias, and the gradients of |y - Y|^2 / 2
    xm, wm = Mat(ctx, x, "f32"), Mat(ctx, w, "f32")
    xq, xt, wq, wt = Held(ctx, N, k, "e4m3", 1), Held(ctx, k, N, "e4m3", 1), Held(ctx, n, k, "e4m3", 128), Held(ctx, k, n, "e4m3", 128)
    gq, gt = Held(ctx, N, n, "e5m2", 1), Held(ctx, n, N, "e5m2", 1)
    y, dx, dw = Mat(ctx, np.zeros((N, n)), "f32"), Mat(ctx, np.zeros((N, k)), "bf16"), Mat(ctx, np.zeros((n, k)), "f32")
    ctx.quant_blocks(xm.ptr, capi.CP_F32, xq.b, xt.b)
    ctx.quant_blocks(wm.ptr, capi.CP_F32, wq.b, wt.b)
    ctx.matmul_blocks(xq.b, wq.b, y.ptr, capi.CP_F32, bias=ctx.to_device(b))
    want, tol = product_bound(real(x, "e4m3", 1), real(w, "e4m3", 128), "f32", b.astype(np.float64))
    assert (np.abs(y.get() - want) <= tol).all()
    # and against the refit in float64: the cast errs by half a step of either operand
    slack = (2.0 ** -3 + 2.0 ** -8) * (np.abs(x) @ np.abs(w).T) + 2.0 ** -9 * np.abs(x).max() * np.abs(w).max() * k
    assert (np.abs(y.get() - (x @ w.T + newB)) <= slack + 1e-6 * np.abs(newB).max()).all()
    g = (y.get() - Y.reshape(N, n)).astype(np.float32).astype(np.float64)
    gm = Mat(ctx, g, "f32")
    ctx.quant_blocks(gm.ptr, capi.CP_F32, gq.b, gt.b)
    ctx.matmul_blocks(gq.b, wt.b, dx.ptr, capi.CP_BF16)
    ctx.matmul_blocks(gt.b, xt.b, dw.ptr, capi.CP_F32)
    for got, l, r, kind in ((dx, real(g, "e5m2", 1), real(w, "e4m3", 128).T, "bf16"), (dw, real(g.T, "e5m2", 1), real(x.T, "e4m3", 1), "f32")):
        want, tol = product_bound(l, r, kind)
        assert (np.abs(got.get() - want) <= tol).all()

    # the refitted weights' step with that gradient
    m = Mat(ctx, np.zeros((n, k)), "f32")
    ctx.ortho_step(capi.OrthoStepJobs([(dw.ptr, capi.CP_F32, n, k, m.ptr, wm.ptr, capi.CP_F32)]), 0.02, weight_decay=0.1)
    m2, w2, far = step(dw.get(), np.zeros((n, k)), w, "f32", 0.02, 0.95, True, 0.1, max(1, n / k) ** 0.5)
    assert (np.abs(m.get() - m2) <= 2.0 ** -24 * np.abs(m2) + 1e-30).all()
    err = np.abs(wm.get() - w2)
    assert (err <= 12 * far + 5 * 2.0 ** -24 * (np.abs(w) + np.abs(w2)) + 2.0 ** -25).all()
