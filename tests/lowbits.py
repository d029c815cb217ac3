"""Plain NumPy forms of the low-precision types (bfloat16, float16, the two 8-bit types), and device matrices in them.
Test infrastructure: written from the formats' definitions, shares nothing with the library."""
import contextlib
import ctypes

import numpy as np

from cpmi355 import capi

TYPES = {"f32": capi.CP_F32, "f64": capi.CP_F64, "bf16": capi.CP_BF16, "f16": capi.CP_F16}
HALF = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}      # half a step relative to the value
FMT = {"e4m3": capi.CP_E4M3, "e5m2": capi.CP_E5M2}
FMAX = {"e4m3": 448.0, "e5m2": 57344.0}


def to_bits(a, kind):
    """float array -> the array that holds it on the device (bfloat16 as uint16), rounded to nearest even."""
    a = np.asarray(a)
    if kind == "bf16":
        u = np.ascontiguousarray(a, dtype=np.float32).view(np.uint32)
        r = ((u.astype(np.uint64) + 0x7fff + ((u >> 16) & 1)) >> 16).astype(np.uint16)
        return np.where(np.isnan(a), np.uint16(0x7fc0), r)
    return a.astype({"f32": np.float32, "f64": np.float64, "f16": np.float16}[kind])


def from_bits(b, kind):
    """-> float64"""
    if kind == "bf16":
        return (b.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return b.astype(np.float64)


def size(kind):
    return {"f32": 4, "f64": 8, "bf16": 2, "f16": 2}[kind]


def np_type(kind):
    return {"f32": np.float32, "f64": np.float64, "bf16": np.uint16, "f16": np.float16}[kind]


class Mat:
    """A [rows, cols] device matrix of a type, `ld` elements to a row, `lead` elements behind the buffer's start; what lies
    between and behind the rows holds a pattern that untouched() checks."""

    def __init__(self, ctx, a, kind, ld=None, lead=0):
        a = np.atleast_2d(np.asarray(a, dtype=np.float64))
        self.ctx, self.kind, (self.rows, self.cols) = ctx, kind, a.shape
        self.ld = max(self.cols, 1) if ld is None else ld
        self.lead = lead
        self.n = lead + self.rows * self.ld + 64
        full = np.full(self.n, 0x5a, dtype=np.uint8).repeat(size(kind)).view(np_type(kind))
        self.inside = np.zeros(self.n, dtype=bool)
        for r in range(self.rows):
            o = lead + r * self.ld
            full[o:o + self.cols] = to_bits(a[r], kind)
            self.inside[o:o + self.cols] = True
        self.before = full.copy()
        self.buf = ctx.to_device(full)
        self.ptr = self.buf.ptr + lead * size(kind)

    def raw(self):
        return self.ctx.to_host(self.buf, (self.n,), np_type(self.kind))

    def get(self):
        h = self.raw()
        v = h[self.lead:self.lead + self.rows * self.ld].reshape(self.rows, self.ld)[:, :self.cols]
        return from_bits(np.ascontiguousarray(v), self.kind)

    def untouched(self):
        h = self.raw()
        u = np_type(self.kind)
        return np.array_equal(h.view(np.uint8).reshape(self.n, -1)[~self.inside],
                              self.before.astype(u).view(np.uint8).reshape(self.n, -1)[~self.inside])


def table8(fmt):
    """The 256 values of an 8-bit type."""
    mant, bias = (3, 7) if fmt == "e4m3" else (2, 15)
    out = np.empty(256)
    for c in range(256):
        e, m = (c & 0x7f) >> mant, c & ((1 << mant) - 1)
        v = m * 2.0 ** (1 - bias - mant) if e == 0 else (1 + m * 2.0 ** -mant) * 2.0 ** (e - bias)
        if fmt == "e4m3" and (c & 0x7f) == 0x7f:
            v = np.nan
        if fmt == "e5m2" and e == 31:
            v = np.inf if m == 0 else np.nan
        out[c] = -v if c & 0x80 else v
    return out


def round8(y, fmt):
    """float values -> the nearest 8-bit values (ties to even), |y| <= fmax; NaN stays."""
    y = np.asarray(y, dtype=np.float64)
    mant, low = (3, -6) if fmt == "e4m3" else (2, -14)
    _, e = np.frexp(np.where(np.isfinite(y) & (y != 0), y, 1.0))
    step = np.ldexp(1.0, np.maximum(e - 1, low) - mant)
    return np.rint(y / step) * step


def quant(x, fmt, tile, pow2=False):
    """x -> (values [rows, cols], scales float32 [ceil(cols / 128), rows or ceil(rows / 128)]), by the format's definition."""
    with np.errstate(over="ignore"):
        x = np.asarray(x).astype(np.float32)
    rows, cols = x.shape
    kb, tb = -(-cols // 128), -(-rows // tile)
    q, s = np.empty((rows, cols)), np.empty((kb, tb), dtype=np.float32)
    top = np.float32(FMAX[fmt])
    for k in range(kb):
        for t in range(tb):
            b = x[t * tile:(t + 1) * tile, k * 128:(k + 1) * 128]
            fin = np.abs(b[np.isfinite(b)])
            amax = np.maximum(fin.max() if fin.size else np.float32(0), np.float32(2.0 ** -100))
            sc = amax / top
            if pow2:
                m, e = np.frexp(sc)
                sc = np.ldexp(np.float32(1), e - 1 if m == 0.5 else e)
                inv = np.float32(1) / sc
            else:
                inv = top / amax
            s[k, t] = sc
            y = np.where(np.isfinite(b), np.clip(np.where(np.isfinite(b), b, 0) * inv, -top, top), np.nan)
            q[t * tile:(t + 1) * tile, k * 128:(k + 1) * 128] = round8(y, fmt)
    return q, s


class Held:
    """A Blocks on the device with a pattern around what belongs to it."""

    def __init__(self, ctx, rows, cols, fmt, tile, more_ld=0, more_lds=0):
        self.ctx, self.rows, self.cols, self.fmt, self.tile = ctx, rows, cols, fmt, tile
        self.kb, self.tb = -(-cols // 128), rows if tile == 1 else -(-rows // 128)
        self.ld, self.lds = max(self.kb, 1) * 128 + 128 * more_ld, max(self.tb, 1) + more_lds
        self.qn, self.sn = rows * self.ld + 256, max(self.kb, 1) * self.lds + 64
        self.q = ctx.to_device(np.full(self.qn, 0x33, dtype=np.uint8))
        self.s = ctx.to_device(np.full(self.sn, -7.0, dtype=np.float32))
        self.b = capi.Blocks(self.q, self.s, rows, cols, FMT[fmt], tile, ld=self.ld, lds=self.lds)

    def codes(self):
        return self.ctx.to_host(self.q, (self.qn,), np.uint8)

    def values(self):
        c = self.codes()[:self.rows * self.ld].reshape(self.rows, self.ld)[:, :self.cols]
        return table8(self.fmt)[c]

    def scales(self):
        s = self.ctx.to_host(self.s, (self.sn,), np.float32)
        return s[:max(self.kb, 1) * self.lds].reshape(-1, self.lds)[:self.kb, :self.tb]

    def around(self):
        """The padding is zero, and nothing else outside the matrix was written."""
        c = self.codes()
        body, up = c[:self.rows * self.ld].reshape(self.rows, self.ld), self.kb * 128
        s = self.ctx.to_host(self.s, (self.sn,), np.float32)
        sb = s[:max(self.kb, 1) * self.lds].reshape(-1, self.lds)
        return ((body[:, self.cols:up] == 0).all() and (body[:, up:] == 0x33).all() and (c[self.rows * self.ld:] == 0x33).all()
                and (sb[:, self.tb:] == -7).all() and (s[max(self.kb, 1) * self.lds:] == -7).all())

    @classmethod
    def of(cls, ctx, x, fmt, tile, pow2=False):
        """x held by the definition (no kernel involved), with what it stands for in .real."""
        h = cls(ctx, x.shape[0], x.shape[1], fmt, tile)
        q, s = quant(x, fmt, tile, pow2)
        tab = table8(fmt)
        order = np.argsort(np.where(np.isnan(tab), np.inf, tab), kind="stable")
        order = order[np.isfinite(tab[order])]
        codes = np.zeros((h.rows, h.ld), dtype=np.uint8)
        codes[:, :h.cols] = order[np.searchsorted(tab[order], q)]
        ctx.to_device(np.concatenate([codes.reshape(-1), np.full(256, 0x33, np.uint8)]), h.q)
        sc = np.full((max(h.kb, 1), h.lds), -7, dtype=np.float32)
        sc[:h.kb, :h.tb] = s
        ctx.to_device(np.concatenate([sc.reshape(-1), np.full(64, -7, np.float32)]), h.s)
        ctx.sync()
        h.real = q * s.astype(np.float64).T.repeat(tile, 0)[:h.rows].repeat(128, 1)[:, :h.cols]
        return h


def _hip(ctx, name, *args):
    """A call of the HIP runtime that the library itself is linked to."""
    fn = getattr(ctx.lib, name)
    fn.restype = ctypes.c_int
    rc = fn(*args)
    if rc:
        raise RuntimeError("%s: %d" % (name, rc))


@contextlib.contextmanager
def other_stream(ctx):
    """ctx runs on a stream of the caller's."""
    st = ctypes.c_void_p()
    ctx.sync()
    _hip(ctx, "hipStreamCreateWithFlags", ctypes.byref(st), ctypes.c_uint(1))
    ctx.set_stream(st)
    try:
        yield st
    finally:
        ctx.sync()
        ctx.set_stream(None)
        _hip(ctx, "hipStreamDestroy", st)


class Graph:
    """What `calls` enqueues on ctx's stream (a caller's one), as a graph."""

    def __init__(self, ctx, stream, calls):
        self.ctx, self.stream, self.graph, self.run = ctx, stream, ctypes.c_void_p(), ctypes.c_void_p()
        _hip(ctx, "hipStreamBeginCapture", stream, ctypes.c_int(2))          # relaxed
        try:
            calls()
        finally:
            _hip(ctx, "hipStreamEndCapture", stream, ctypes.byref(self.graph))
        _hip(ctx, "hipGraphInstantiate", ctypes.byref(self.run), self.graph, None, None, ctypes.c_size_t(0))

    def replay(self):
        _hip(self.ctx, "hipGraphLaunch", self.run, self.stream)

    def close(self):
        self.ctx.sync()
        _hip(self.ctx, "hipGraphExecDestroy", self.run)
        _hip(self.ctx, "hipGraphDestroy", self.graph)


class Far:
    """A [rows, cols] matrix of a type whose rows lie `gap` elements apart: bytes past 2^32 from its start.  Only the rows and
    the element before and behind each are filled."""

    def __init__(self, ctx, a, kind, gap):
        self.ctx, self.kind, self.ld, (self.rows, self.cols) = ctx, kind, gap, a.shape
        assert (self.rows - 1) * gap * size(kind) > 1 << 32
        self.buf = ctx.empty(((self.rows - 1) * gap + self.cols + 2) * size(kind))
        self.ptr = self.buf.ptr + size(kind)
        self.edge = np.full(1, 0x5a, dtype=np.uint8).repeat(size(kind)).view(np_type(kind))
        for r in range(self.rows):
            line = np.ascontiguousarray(np.concatenate([self.edge, to_bits(a[r], kind), self.edge]))
            ctx._check(ctx.lib.cp_memcpy_h2d(ctx.h, self.buf.ptr + r * gap * size(kind), line.ctypes.data, line.nbytes), "cp_memcpy_h2d")

    def get(self):
        """The matrix; None if anything beside it was written."""
        out = np.empty((self.rows, self.cols + 2), dtype=np_type(self.kind))
        for r in range(self.rows):
            self.ctx._check(self.ctx.lib.cp_memcpy_d2h(self.ctx.h, out[r].ctypes.data, self.buf.ptr + r * self.ld * size(self.kind),
                                                       out[r].nbytes), "cp_memcpy_d2h")
        ends = np.ascontiguousarray(out[:, [0, -1]]).view(np.uint8)
        return from_bits(np.ascontiguousarray(out[:, 1:-1]), self.kind) if (ends == 0x5a).all() else None
