"""What the binding of the 8-bit and orthogonalised operators refuses before anything reaches the device (no GPU needed: an
argument that came through would end in the library's CP_ERR_ARG for the missing context, a CpError)."""
import numpy as np
import pytest

from cpmi355 import capi


@pytest.fixture
def no_ctx():
    c = capi.Context.__new__(capi.Context)
    c.lib, c.h, c.device, c._given = capi.load(), None, 0, 1
    return c


class Tensor:
    """As much of a device tensor as the binding looks at."""
    is_cuda = True

    def __init__(self, shape, dtype, strides=None, device=0, ptr=4096):
        self.shape, self.dtype, self._strides, self._device, self._ptr = tuple(shape), dtype, strides, device, ptr
        if strides is None:
            self._strides = tuple(int(np.prod(shape[i + 1:])) for i in range(len(shape)))
        self.device = type("Device", (), {"index": device, "type": "cuda"})()

    def dim(self):
        return len(self.shape)

    def stride(self, i=None):
        return self._strides if i is None else self._strides[i]

    def get_device(self):
        return self._device

    def data_ptr(self):
        return self._ptr

    def is_contiguous(self):
        return self._strides == tuple(int(np.prod(self.shape[i + 1:])) for i in range(len(self.shape)))

    @property
    def nbytes(self):
        return int(np.prod(self.shape)) * {"torch.uint8": 1, "torch.float32": 4}.get(str(self.dtype), 1)


class Buf(capi.DevBuf):
    """A DevBuf that allocates nothing."""

    def __init__(self, nbytes, device=0):
        self.nbytes, self.ptr = nbytes, 4096
        self.ctx = type("Ctx", (), {"device": device, "h": None})()


def blocks(rows=5, cols=130, tile=1):
    return capi.Blocks(4096, 4096, rows, cols, capi.CP_E4M3, tile)


# ---- host memory ------------------------------------------------------------------------------------------------------------


def test_host_memory_is_refused(no_ctx):
    import torch
    host = np.zeros((5, 130), dtype=np.float32)
    for bad in (host, torch.from_numpy(host)):
        with pytest.raises(ValueError):
            no_ctx.quant_blocks(bad, capi.CP_F32, blocks())
        with pytest.raises(ValueError):
            no_ctx.matmul_blocks(blocks(), blocks(130), bad, capi.CP_F32)
        for make in (lambda x: capi.OrthoJobs([(x, 0, 5, 130, 4096, 0)]), lambda x: capi.OrthoJobs([(4096, 0, 5, 130, x, 0)]),
                     lambda x: capi.OrthoStepJobs([(x, 0, 5, 130, 4096, 8192, 0)]), lambda x: capi.OrthoStepJobs([(4096, 0, 5, 130, x, 8192, 0)]),
                     lambda x: capi.OrthoStepJobs([(4096, 0, 5, 130, 8192, x, 0)])):
            with pytest.raises(ValueError):
                make(bad)
    q, s = np.zeros((5, 256), dtype=np.uint8), np.ones((2, 5), dtype=np.float32)
    for a, b in ((q, 4096), (4096, s), (torch.from_numpy(q), 4096), (4096, torch.from_numpy(s))):
        with pytest.raises(ValueError):
            capi.Blocks(a, b, 5, 130, capi.CP_E4M3, 1)


def test_bias_and_workspace_are_checked(no_ctx):
    import torch

    def product(**kw):
        no_ctx.matmul_blocks(blocks(), blocks(7), 4096, capi.CP_F32, **kw)

    for bias in (np.zeros(7, dtype=np.float32), torch.zeros(7), Buf(24), Buf(28, device=1)):
        with pytest.raises(ValueError):
            product(bias=bias)
    jobs, steps = capi.OrthoJobs([(4096, 0, 5, 130, 8192, 0)]), capi.OrthoStepJobs([(4096, 0, 5, 130, 8192, 16384, 0)])
    for ws in (np.zeros(512, dtype=np.uint8), torch.zeros(512, dtype=torch.uint8), Buf(512, device=1), 4096,
               Tensor((512,), "torch.uint8", device=1), Tensor((512,), "torch.uint8", strides=(2,))):
        for call in (lambda: product(ws=ws), lambda: no_ctx.orthogonalise(jobs, ws=ws), lambda: no_ctx.ortho_step(steps, 0.1, ws=ws)):
            with pytest.raises(ValueError):
                call()
    for ok in (dict(), dict(bias=Buf(28)), dict(bias=4096), dict(ws=Buf(512)), dict(ws=Tensor((512,), "torch.uint8"))):
        with pytest.raises(capi.CpError):                # through to the library, which misses the context
            product(**ok)


# ---- lists of the other call ---------------------------------------------------------------------------------------------------


def test_a_list_of_the_other_call_is_refused(no_ctx):
    """The records differ: read as the other's, a stride would be taken for an address."""
    jobs, steps = capi.OrthoJobs([(4096, 0, 5, 130, 8192, 0)]), capi.OrthoStepJobs([(4096, 0, 5, 130, 8192, 16384, 0)])
    for bad in (steps, [(4096, 0, 5, 130, 8192, 0)], None):
        with pytest.raises(ValueError):
            no_ctx.orthogonalise(bad)
    for bad in (jobs, [(4096, 0, 5, 130, 8192, 16384, 0)], None):
        with pytest.raises(ValueError):
            no_ctx.ortho_step(bad, 0.1)
    with pytest.raises(ValueError):
        capi.ortho_workspace([(4096, 0, 5, 130, 8192, 0)])


# ---- 8-bit matrices in tensors --------------------------------------------------------------------------------------------------


def held(rows=5, cols=130, fmt=capi.CP_E4M3, tile=1, q=None, scale=None, **kw):
    q = Tensor((rows, 256), "torch.uint8") if q is None else q
    scale = Tensor((2, rows if tile == 1 else -(-rows // 128)), "torch.float32") if scale is None else scale
    return capi.Blocks(q, scale, rows, cols, fmt, tile, **kw)


def test_strides_have_to_be_the_tensors():
    """A stride of the caller's that is not the tensor's reads past its memory."""
    b = held(q=Tensor((5, 256), "torch.uint8", (512, 1)), scale=Tensor((2, 5), "torch.float32", (9, 1)))
    assert (b.ld, b.lds) == (512, 9)
    b = held(q=Tensor((5, 256), "torch.uint8", (512, 1)), scale=Tensor((2, 5), "torch.float32", (9, 1)), ld=512, lds=9)
    assert (b.ld, b.lds) == (512, 9)
    for kw in (dict(ld=512), dict(ld=384), dict(lds=6), dict(lds=1 << 20)):
        with pytest.raises(ValueError):
            held(**kw)
    held(rows=1, q=Tensor((1, 256), "torch.uint8"), ld=1024)                               # one row: its stride leads nowhere
    capi.Blocks(Tensor((5, 128), "torch.uint8"), Tensor((1, 5), "torch.float32"), 5, 100, capi.CP_E4M3, 1, lds=80)   # one block column


def test_types_have_to_be_the_format():
    held(q=Tensor((5, 256), "torch.float8_e4m3fn"))
    held(q=Tensor((5, 256), "torch.float8_e5m2"), fmt=capi.CP_E5M2)
    for t, fmt in (("torch.float8_e4m3fn", capi.CP_E5M2), ("torch.float8_e5m2", capi.CP_E4M3), ("torch.int8", capi.CP_E4M3),
                   ("torch.float8_e4m3fnuz", capi.CP_E4M3)):
        with pytest.raises(ValueError):
            held(q=Tensor((5, 256), t), fmt=fmt)


def test_both_parts_lie_on_one_device():
    two, three = Tensor((2, 5), "torch.float32", device=1), Buf(1 << 16, device=1)
    assert held(q=Tensor((5, 256), "torch.uint8", device=1), scale=three).device == 1
    for kw in (dict(scale=two), dict(scale=three), dict(q=three), dict(q=Buf(1 << 16), scale=three), dict(q=Buf(1 << 16), scale=two)):
        with pytest.raises(ValueError):
            held(**kw)


# ---- sizes that a record does not hold ----------------------------------------------------------------------------------------


def test_sizes_past_the_records_are_refused():
    """2^32 + 64 rows are not 64 of them."""
    for rows, cols in (((1 << 32) + 64, 4), (4, (1 << 32) + 64), (1 << 31, 4)):
        with pytest.raises(ValueError):
            capi.OrthoJobs([(4096, 0, rows, cols, 8192, 0)])
        with pytest.raises(ValueError):
            capi.OrthoStepJobs([(4096, 0, rows, cols, 8192, 16384, 0)])
