"""8-bit products whose scales lie at the ends of float32's range, and values that are not finite, in every form of the product."""
import numpy as np
import pytest

from cpmi355 import capi
from lowbits import FMT, TYPES, Held, Mat
from test_blocks8 import product_bound, tile_shape  # noqa: F401

gpu = pytest.mark.gpu
SHAPES = [(70, 130), (290, 300)]


def formed(ctx, A, B, out):
    C = Mat(ctx, np.zeros((A.rows, B.rows)), out)
    ctx.matmul_blocks(A.b, B.b, C.ptr, TYPES[out])
    assert C.untouched()
    return C.get()


@gpu
@pytest.mark.parametrize("m,n", SHAPES)
@pytest.mark.parametrize("tb", [1, 128])
@pytest.mark.parametrize("out", ["f32", "bf16"])
def test_scales_whose_product_is_past_float32(ctx, tile_shape, m, n, tb, out):
    """Blocks of 1e30 and of 1e14 that share no column: their product is zero, and the other block's is the result."""
    rs = np.random.RandomState(m)
    a, b = rs.randn(m, 256), rs.randn(n, 256)
    a[:, :64] *= 1e30
    b[:, 64:128] *= 1e14
    a[:, 64:128] = 0
    b[:, :64] = 0
    A, B = Held.of(ctx, a, "e4m3", 1), Held.of(ctx, b, "e4m3", tb)
    want, tol = product_bound(A.real, B.real, out)
    assert np.array_equal(want, A.real[:, 128:] @ B.real[:, 128:].T) and np.abs(want).max() < 1e3
    got = formed(ctx, A, B, out)
    assert (np.abs(got - want) <= tol).all(), np.abs(got - want).max()


@gpu
@pytest.mark.parametrize("m,n", SHAPES)
@pytest.mark.parametrize("tb", [1, 128])
@pytest.mark.parametrize("out", ["f32", "bf16"])
def test_scales_whose_product_is_subnormal(ctx, tile_shape, m, n, tb, out):
    """Operands of 1e-19: the results are ordinary float32 numbers, the product of two scales (2^-144, 2^-151) is not."""
    rs = np.random.RandomState(n)
    A, B = Held.of(ctx, 1e-19 * rs.randn(m, 300), "e5m2" if m < n // 2 + 10 else "e4m3", 1), Held.of(ctx, 1e-19 * rs.randn(n, 300), "e4m3", tb)
    want, tol = product_bound(A.real, B.real, out)
    got = formed(ctx, A, B, out)
    assert (np.abs(got - want) <= tol).all(), float((np.abs(got - want) / tol).max())


@gpu
@pytest.mark.parametrize("tb", [1, 128])
@pytest.mark.parametrize("out", ["f32", "bf16"])
def test_scales_of_every_size(ctx, tile_shape, tb, out):
    """Scales from 2^-110 to 2^50 of A's rows and B's blocks, one size of result: powers of two and others."""
    rs = np.random.RandomState(7)
    m, n, k = 150, 300, 640
    p = rs.randint(-60, 60, size=5).repeat(128)
    A, B = Held.of(ctx, rs.randn(m, k) * 2.0 ** p, "e4m3", 1), Held.of(ctx, rs.randn(n, k) * 2.0 ** -p, "e4m3", tb)
    want, tol = product_bound(A.real, B.real, out)
    got = formed(ctx, A, B, out)
    assert (np.abs(got - want) <= tol).all(), float((np.abs(got - want) / tol).max())


@gpu
@pytest.mark.parametrize("m,n", SHAPES)
@pytest.mark.parametrize("ta,tb", [(1, 1), (128, 128)])
@pytest.mark.parametrize("out,fa", [("f32", "e4m3"), ("bf16", "e5m2"), ("bf16", "e4m3"), ("f16", "e5m2")])
def test_nan_stays_in_its_row_and_column(ctx, tile_shape, m, n, ta, tb, out, fa):
    """An infinity or a NaN in A or B becomes a NaN there: the result's row or column is NaN, everything else is as it was."""
    rs = np.random.RandomState(m + n)
    a, b = rs.randn(m, 300), rs.randn(n, 300)
    a[m // 2, 5], a[m - 1, 299], b[n - 1, 130] = np.nan, -np.inf, np.inf
    mats = []
    for x, f, t in ((a, fa, ta), (b, "e4m3", tb)):
        X, h = Mat(ctx, x, "f32"), Held(ctx, *x.shape, f, t)
        ctx.quant_blocks(X.ptr, capi.CP_F32, h.b)
        mats.append(h)
    got = formed(ctx, *mats, out)
    bad = np.zeros((m, n), dtype=bool)
    bad[[m // 2, m - 1]], bad[:, n - 1] = True, True
    assert np.array_equal(np.isnan(got), bad)
    for x in (a, b):
        x[~np.isfinite(x)] = 0                                   # (a block's scale is that of its finite values)
    want, tol = product_bound(Held.of(ctx, a, fa, ta).real, Held.of(ctx, b, "e4m3", tb).real, out)
    assert (np.abs(got - want)[~bad] <= tol[~bad]).all()


@gpu
@pytest.mark.parametrize("m", [16, 17, 32, 33, 48, 49, 64, 65, 80, 81, 96, 97, 112, 113, 128, 129])
@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("n,k", [(70, 300), (333, 1100)])
def test_every_number_of_row_groups(ctx, m, out, n, k):
    """The few-rows form (asked for) around each number of groups of sixteen rows, and the rule's form, on one shape."""
    from test_blocks8 import check_product
    for knob in (5, 0):
        ctx.lib.cp_debug_knob(3, knob)
        try:
            check_product(ctx, m, n, k, out=out, bias=True, ld=3, lead=1)
        finally:
            ctx.lib.cp_debug_knob(3, 0)
