"""Orthogonalised updates and optimiser steps as a network's training loop makes them: ill-conditioned momenta, many layers of
mixed shapes and types in one call."""
import numpy as np
import pytest

from cpmi355 import capi
from lowbits import HALF, TYPES, Mat
from test_ortho import distance, iterate, tile_shape, within  # noqa: F401

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


# ---- a network's layers in one step --------------------------------------------------------------------------------------------


class Layer:
    """G, M and W of one layer on the device, and what a step has to make of them."""

    def __init__(self, ctx, rs, rows, cols, gk, wk, gamma):
        self.shape, self.gk, self.wk, self.gamma = (rows, cols), gk, wk, gamma
        self.g = Mat(ctx, 1e-3 * dominated(rs, rows, cols, 3.0), gk, ld=cols + rs.randint(3))
        self.m = Mat(ctx, 8e-3 * dominated(rs, rows, cols, 3.0), "f32", ld=cols + rs.randint(3), lead=rs.randint(2))
        self.w = Mat(ctx, 0.05 * rs.randn(rows, cols), wk, ld=cols + rs.randint(3), lead=rs.randint(4))

    def twin(self, ctx):
        """The same layer in memory of its own."""
        t = Layer.__new__(Layer)
        t.__dict__.update(self.__dict__)
        t.m, t.w = Mat(ctx, self.m.get(), "f32"), Mat(ctx, self.w.get(), self.wk)
        return t

    def job(self):
        r, c = self.shape
        return (self.g.ptr, TYPES[self.gk], r, c, self.m.ptr, self.w.ptr, TYPES[self.wk], self.gamma, self.g.ld, self.m.ld, self.w.ld)

    def held(self):
        return self.g.get(), self.m.get(), self.w.get()

    def check(self, before, lr, momentum, nesterov, decay):
        g, m, w = before
        gamma = max(1, self.shape[0] / max(self.shape[1], 1)) ** 0.5 if self.gamma is None else self.gamma
        m2 = momentum * m + g
        U = g + momentum * m2 if nesterov else m2
        O, far = distance32(U)
        # U's float32 roundings (see test_step_of_an_ill_conditioned_momentum)
        signs = np.where((np.arange(U.size).reshape(U.shape) * 2654435761 >> 7) & 1, 1.0, -1.0)
        moved = iterate(U + 2.0 ** -24 * (np.abs(m2) + np.abs(m) + np.abs(U)) * signs) - O
        far = abs(lr * gamma) * (far + 4 * np.sqrt((moved ** 2).mean()))
        want = (1 - lr * decay) * w - lr * gamma * O
        assert (np.abs(self.m.get() - m2) <= 2.0 ** -24 * (np.abs(m2) + np.abs(m)) + 1e-30).all()
        # W: two float32 factors (each off by half a step), a product and a fused multiply-add, and the type's rounding
        slack = 4 * 2.0 ** -24 * (np.abs(w) + np.abs(want)) + HALF[self.wk] * np.abs(want) + 2.0 ** -25
        err = np.abs(self.w.get() - want)
        assert (err <= 12 * far + slack).all() and np.sqrt((err ** 2).mean()) <= far + np.sqrt((slack ** 2).mean()), self.shape
        assert self.m.untouched() and self.w.untouched() and np.array_equal(self.g.raw(), self.g.before)


@gpu
@pytest.mark.parametrize("rows,cols", [(130, 140), (140, 130), (70, 700), (700, 70), (300, 520), (520, 300)])
@pytest.mark.parametrize("gk,wk", [("f32", "f32"), ("bf16", "bf16"), ("f32", "bf16"), ("f16", "f16")])
def test_step_in_every_tile_shape(ctx, tile_shape, rows, cols, gk, wk):
    layer = Layer(ctx, np.random.RandomState(rows + cols), rows, cols, gk, wk, None)
    jobs = capi.OrthoStepJobs([layer.job()])
    for nesterov in (True, False):
        before = layer.held()
        ctx.ortho_step(jobs, 0.02, nesterov=nesterov, weight_decay=0.1)
        layer.check(before, 0.02, 0.95, nesterov, 0.1)


def run_together(ctx, layers, alone):
    """Two steps on all layers in one call, each against float64; `alone(layer)`: and against a call of its own, bit for bit."""
    twins = [(a, a.twin(ctx)) for a in layers if alone(a)]
    jobs = capi.OrthoStepJobs([a.job() for a in layers])
    for _ in range(2):
        before = [a.held() for a in layers]
        ctx.ortho_step(jobs, 0.02, weight_decay=0.1)
        for a, b in zip(layers, before):
            if a.w.rows and a.w.cols:
                a.check(b, 0.02, 0.95, True, 0.1)
    for a, t in twins:
        one = capi.OrthoStepJobs([(a.g.ptr, TYPES[a.gk], *a.shape, t.m.ptr, t.w.ptr, TYPES[a.wk], a.gamma, a.g.ld, t.m.ld, t.w.ld)])
        for _ in range(2):
            ctx.ortho_step(one, 0.02, weight_decay=0.1)
        assert np.array_equal(a.m.get(), t.m.get()) and np.array_equal(a.w.get(), t.w.get()), a.shape


@gpu
@pytest.mark.parametrize("seed", [0, 1])
def test_step_of_a_network(ctx, seed):
    """More layers than a launch's records, tall and wide, large and small, of all types: float32, fp16 and bfloat16 weights
    share the call's counters and pieces."""
    rs = np.random.RandomState(20 + seed)
    kinds = [("f32", "f32"), ("bf16", "bf16"), ("f32", "bf16"), ("bf16", "f32"), ("f16", "f16")]
    shapes = [(int(16 * 24 ** rs.rand()), int(16 * 32 ** rs.rand())) for _ in range(44)]
    shapes += [(70, 5000), (5000, 70), (1, 1), (400, 400), (1, 300), (300, 1)]
    layers = [Layer(ctx, rs, *s, *kinds[i % 5], None if i % 3 else 0.7) for i, s in enumerate(shapes)]
    run_together(ctx, layers, lambda a: min(a.shape) > 64)


@gpu
def test_step_of_many_small_layers(ctx):
    """A call of small matrices alone, more than one kernel's records of a kind."""
    rs = np.random.RandomState(30)
    kinds = [("f32", "f32"), ("bf16", "bf16"), ("f32", "bf16"), ("bf16", "f32"), ("f16", "f16")]
    shapes = [(int(rs.randint(1, 65)), int(rs.randint(1, 513))) for _ in range(60)]
    shapes = [s if i % 2 else s[::-1] for i, s in enumerate(shapes)] + [(64, 512), (512, 64), (64, 64), (1, 1)]
    shapes += [(48, 200)] * 30
    layers = [Layer(ctx, rs, *s, *kinds[i % 5], None if i % 3 else 0.7) for i, s in enumerate(shapes)]
    assert capi.ortho_workspace(capi.OrthoStepJobs([a.job() for a in layers])) == 0
    run_together(ctx, layers, lambda a: True)


# ---- workspaces ------------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("one,many", [((128, 20000), [(4096, 4096)] * 40), ((100, 50000), [(2048, 8192)] * 200), ((70, 9000), [(512, 512)] * 30)])
@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_a_layer_cut_along_k_brings_its_own_pieces_only(one, many, kind):
    """The partial sums of one layer's tiles, not slots for every workgroup of the launch it joins."""
    def need(shapes):
        T, at, jobs = TYPES[kind], 1 << 40, []
        for r, c in shapes:
            jobs.append((at, T, r, c, at + (1 << 34), T))
            at += 1 << 36
        return capi.ortho_workspace(capi.OrthoJobs(jobs))

    # its matrices (what it needs alone), and 16 pieces of each of its 256 x 256 tiles of the first product, of 256 KB
    pieces = 16 * (-(-one[0] // 256)) * (-(-one[0] // 256)) << 18
    assert need(many) < need(many + [one]) <= need(many) + need([one]) + pieces + 65536


@gpu
@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_mixed_call_stays_in_its_workspace(ctx, tile_shape, kind):
    """Layers whose tiles are cut among others whose are not: the same bits as each alone, nothing behind the workspace."""
    rs = np.random.RandomState(40)
    shapes = [(150, 140), (70, 9000), (300, 260), (6000, 130), (200, 70), (129, 4500)]
    T = TYPES[kind]
    Gs, Os = [Mat(ctx, dominated(rs, *s, 2.0), kind) for s in shapes], [Mat(ctx, np.zeros(s), kind) for s in shapes]
    jobs = capi.OrthoJobs([(G.ptr, T, *s, O.ptr, T) for G, O, s in zip(Gs, Os, shapes)])
    need = ctx.ortho_workspace(jobs)
    ws = ctx.to_device(np.full(need + 4096, 0xff, dtype=np.uint8))
    assert ctx.lib.cp_orthogonalise(ctx.h, jobs.n, jobs.c, 5, None, 1e-7, ws.ptr, need) == 0
    assert (ctx.to_host(ws, (need + 4096,), np.uint8)[need:] == 0xff).all()
    for G, O, s in zip(Gs, Os, shapes):
        one = Mat(ctx, np.zeros(s), kind)
        ctx.orthogonalise(capi.OrthoJobs([(G.ptr, T, *s, one.ptr, T)]))
        assert O.untouched() and np.array_equal(one.raw(), O.raw())


# ---- which matrices of a call may lie where ---------------------------------------------------------------------------------------


def cells(at, rows, cols, ld, size):
    return {at + (i * ld + j) * size + b for i in range(rows) for j in range(cols) for b in range(size)}


def test_outputs_are_refused_exactly_where_they_share_memory():
    """Interleaved matrices of any strides and types, against sets of their bytes."""
    rs = np.random.RandomState(50)
    seen = [0, 0]
    for _ in range(4000):
        jobs, bytes_ = [], []
        for i in range(2):
            kind = ("f32", "bf16")[rs.randint(2)]
            size = 4 if kind == "f32" else 2
            rows, cols = rs.randint(1, 7), rs.randint(1, 6)
            ld = cols + (rs.randint(0, 20) if rs.rand() < 0.7 else 0)
            at = 1 << 20 if i == 0 else (1 << 20) + int(rs.randint(-60, 60)) * size
            jobs.append(((1 << 30) + (i << 20), 0, rows, cols, at, TYPES[kind], None, ld))
            bytes_.append(cells(at, rows, cols, ld, size))
        jobs = [j[:6] + (j[3], j[7]) for j in jobs]
        share = bool(bytes_[0] & bytes_[1])
        seen[share] += 1
        if share:
            with pytest.raises(capi.CpError):
                capi.ortho_workspace(capi.OrthoJobs(jobs))
        else:
            capi.ortho_workspace(capi.OrthoJobs(jobs))
    assert min(seen) > 1000


def test_a_tall_matrix_between_the_rows_of_a_wide_one():
    """2^18 rows of three numbers at a stride of their own, beside 2^18 rows of another stride that meet them in one place only."""
    n = 1 << 18
    def call(ld, at):
        return capi.ortho_workspace(capi.OrthoJobs([(1 << 40, 0, n, 3, 1 << 42, 0, 3, 12), (1 << 41, 0, n, 3, (1 << 42) + 4 * at, 0, 3, ld)]))
    call(24, 3)                                                  # every second gap
    call(12, 9)                                                  # the same stride
    call(36, 4)
    call(12 * n - 1, 3)                                          # its second row lies behind the other matrix
    for ld, at in ((25, 3), (36, 10), (24, 1), (6 * n - 1, 3)):
        with pytest.raises(capi.CpError):
            call(ld, at)


# ---- special values in the kernel of small matrices ---------------------------------------------------------------------------------


@gpu
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,cols", [(40, 130), (64, 500), (1, 77), (33, 33)])
def test_special_small_matrices(ctx, kind, rows, cols):
    rs = np.random.RandomState(rows)
    T = TYPES[kind]
    gone = rs.randn(rows, cols)
    gone[1::3], gone[:, 1::5] = 0, 0
    lowrank = rs.randn(rows, 2) @ rs.randn(2, cols)
    spread = rs.randn(rows, cols) * np.logspace(0, -4, rows)[:, None]
    good = [gone, lowrank, spread, np.eye(rows, cols), np.zeros((rows, cols))]
    bad = []
    for v in (np.nan, np.inf, -np.inf):
        b = rs.randn(rows, cols)
        b[rows // 2, cols - 1] = v
        bad.append(b)
    for turn in (lambda x: x, lambda x: x.T):
        mats = [turn(x) for x in good + bad]
        for eps in (1e-7, 0.0):
            Gs, Os = [Mat(ctx, x, kind) for x in mats], [Mat(ctx, np.ones(x.shape), kind) for x in mats]
            jobs = capi.OrthoJobs([(G.ptr, T, *x.shape, O.ptr, T) for G, O, x in zip(Gs, Os, mats)])
            assert ctx.ortho_workspace(jobs) == 0                # the small kernel, all of them in one call
            ctx.orthogonalise(jobs, eps=eps)
            for i, (G, O) in enumerate(zip(Gs, Os)):
                assert O.untouched()
                if i >= len(good):
                    assert np.isnan(O.get()).all()
                elif i == 4:
                    assert (O.get() == 0).all()
                else:
                    want, far = distance(G.get(), kind, eps=eps)
                    within(O.get(), want, far, kind)
                if i == 0:
                    assert (O.get()[(G.get() == 0).all(1)] == 0).all() and (O.get()[:, (G.get() == 0).all(0)] == 0).all()


@gpu
@pytest.mark.parametrize("wk", ["f32", "bf16"])
@pytest.mark.parametrize("rows,cols", [(40, 130), (130, 40), (140, 200), (200, 140)])
def test_a_gradient_that_is_not_finite_spoils_its_own_layer_only(ctx, wk, rows, cols):
    rs = np.random.RandomState(60)
    layers = [Layer(ctx, rs, rows, cols, "f32", wk, None) for _ in range(3)]
    g = layers[1].g.get()
    g[2, 3] = np.inf
    layers[1].g = Mat(ctx, g, "f32")
    before = [a.held() for a in layers]
    ctx.ortho_step(capi.OrthoStepJobs([a.job() for a in layers]), 0.02, weight_decay=0.1)
    for i in (0, 2):
        layers[i].check(before[i], 0.02, 0.95, True, 0.1)
    m = layers[1].m.get()
    assert np.isinf(m[2, 3]) and np.isfinite(np.delete(m.reshape(-1), 2 * cols + 3)).all() and np.isnan(layers[1].w.get()).all()


# ---- coefficients and factors at the ends of their ranges -----------------------------------------------------------------------------


@gpu
@pytest.mark.parametrize("rows,cols", [(40, 130), (140, 200)])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("steps,a", [(3, 1e-6), (5, 2e-5)])
def test_coefficients_that_shrink_every_number(ctx, rows, cols, kind, steps, a):
    """X <- a X, a power of which is what is left of G / |G|_F: numbers as small as float32's and bfloat16's own, at full precision."""
    rs = np.random.RandomState(3)
    G, O = Mat(ctx, rs.randn(rows, cols), kind), Mat(ctx, np.ones((rows, cols)), kind)
    ctx.orthogonalise(capi.OrthoJobs([(G.ptr, TYPES[kind], rows, cols, O.ptr, TYPES[kind])]), steps=steps, coef=(a, 0.0, 0.0), eps=0.0)
    want = iterate(G.get(), steps=steps, coef=[(a, 0.0, 0.0)] * steps, eps=0.0)
    # per step: X and B rounded (11 or 22 bits of the largest number, which is at most eight times the mean), float32 sums
    bits = 11 if kind == "bf16" else 22
    err = np.sqrt(((O.get() - want) ** 2).mean()) / np.sqrt((want ** 2).mean())
    assert err <= (2 * steps + 2) * 2.0 ** -bits + HALF[kind], err


@gpu
def test_factors_past_float32_are_refused(ctx):
    """lr gamma, the momentum and the decay's factor are float32 in the kernels: an infinity there would leave NaN in W."""
    W, M, G = (Mat(ctx, np.ones((3, 4)), "f32") for _ in range(3))
    def call(lr, gamma=1.0, **kw):
        ctx.ortho_step(capi.OrthoStepJobs([(G.ptr, 0, 3, 4, M.ptr, W.ptr, 0, gamma)]), lr, **kw)
    for bad in (dict(lr=1e39), dict(lr=-1e39), dict(lr=1e20, gamma=1e20), dict(lr=1e-3, momentum=1e39), dict(lr=1e20, weight_decay=1e20)):
        with pytest.raises(capi.CpError):
            call(**bad)
    assert np.array_equal(W.raw(), W.before) and np.array_equal(M.raw(), M.before)
    call(1e38, 1e-38)
    assert np.isfinite(W.get()).all()
