"""Run by test_torch_order.py in a process of its own (torch has to come before the first Context): the operators' calls with
torch tensors, among torch's own work on its current stream.  Prints a line per part."""
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path[:0] = [os.path.join(ROOT, "channel-pruning_amd"), ROOT]
from cpmi355 import capi  # noqa: E402

M, N, K = 200, 70, 5000                                       # a product whose tiles are cut along k: it needs scratch
dev = torch.device("cuda", 0)
heavy = torch.randn(8192, 8192, device=dev, dtype=torch.bfloat16)


def delay():
    """About 10 ms of work on the current stream."""
    for _ in range(12):
        torch.mm(heavy, heavy)


def room(rows, cols, tile):
    up = -(-cols // 128) * 128
    return capi.Blocks(torch.zeros(rows, up, dtype=torch.uint8, device=dev),
                       torch.zeros(up // 128, rows if tile == 1 else -(-rows // 128), device=dev), rows, cols, capi.CP_E4M3, tile)


class Layer:
    """A product and a step on torch tensors; the inputs can be overwritten, the results taken."""

    def __init__(self, seed):
        g = torch.Generator(device=dev).manual_seed(seed)
        self.src = {k: torch.randn(s, generator=g, device=dev) for k, s in (("x", (M, K)), ("w", (N, K)), ("g", (N, K)), ("m", (N, K)))}
        self.x, self.w, self.g, self.m = (torch.empty_like(v) for v in self.src.values())
        self.y, self.o = torch.empty(M, N, device=dev), torch.empty(N, K, device=dev)
        self.xq, self.wq = room(M, K, 1), room(N, K, 128)
        self.ortho = capi.OrthoJobs([(self.g, capi.CP_F32, N, K, self.o, capi.CP_F32)])
        self.step = capi.OrthoStepJobs([(self.g, capi.CP_F32, N, K, self.m, self.w, capi.CP_F32)])

    def fill(self):
        for k, v in self.src.items():
            getattr(self, k).copy_(v)

    def spoil(self):
        for t in (self.x, self.w, self.g, self.m, self.y, self.o, self.xq.q, self.wq.q):
            t.fill_(0)

    def calls(self, ctx, ws=None):
        ctx.quant_blocks(self.x, capi.CP_F32, self.xq)
        ctx.quant_blocks(self.w, capi.CP_F32, self.wq)
        ctx.matmul_blocks(self.xq, self.wq, self.y, capi.CP_F32, ws=ws)
        ctx.orthogonalise(self.ortho, ws=ws)
        ctx.ortho_step(self.step, 0.1, ws=ws)

    def pass_(self, ctx, ws=None):
        """Late inputs, the calls, copies of the results, and everything overwritten: all of it enqueued at once."""
        delay()
        self.fill()
        self.calls(ctx, ws)
        out = [t.clone() for t in (self.y, self.o, self.w, self.m)]
        self.spoil()
        return out


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


own, follows = capi.Context(0), capi.Context(0)
layers = [Layer(s) for s in (1, 2, 3)]
want = []
for a in layers:                                              # one thing after the other
    a.fill()
    torch.cuda.synchronize()
    a.calls(own)
    own.sync()
    torch.cuda.synchronize()
    want.append([t.clone() for t in (a.y, a.o, a.w, a.m)])
    assert all(bool(t.isfinite().all()) and bool(t.any()) for t in want[-1])
torch.cuda.synchronize()

side = [torch.cuda.Stream() for _ in range(2)]
for name, ctx in (("own", own), ("follows", follows)):
    for stream in (torch.cuda.default_stream(), side[0], side[1], torch.cuda.default_stream()):
        with torch.cuda.stream(stream):
            for a, w in zip(layers, want):
                if ctx is follows:
                    ctx.use_torch_stream()
                got = a.pass_(ctx)
                torch.cuda.synchronize()
                assert same(got, w), (name, stream)
    print("in order:", name, flush=True)

# two streams at once share the context's scratch: the second's calls have to wait for the first's
for turn in range(3):
    got = []
    for a, stream in zip(layers, (side[0], side[1], torch.cuda.default_stream())):
        with torch.cuda.stream(stream):
            follows.use_torch_stream()
            got.append(a.pass_(follows))
    torch.cuda.synchronize()
    assert all(same(g, w) for g, w in zip(got, want)), turn
print("scratch in order across streams", flush=True)

# captured and replayed, eager work of the same context between the replays
for name, ctx in (("own", own), ("follows", follows)):
    a, b = Layer(5), layers[0]
    a.fill()
    need = max(ctx.matmul_blocks_workspace(a.xq, a.wq, capi.CP_F32), ctx.ortho_workspace(a.ortho), ctx.ortho_workspace(a.step))
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        if ctx is follows:
            ctx.use_torch_stream()
        a.calls(ctx, ws)
    for turn in range(4):
        a.src["x"].mul_(1.25)
        a.fill()
        if ctx is follows:
            ctx.use_torch_stream()
        e = a.pass_(ctx)
        delay()
        a.fill()
        g.replay()
        r = [t.clone() for t in (a.y, a.o, a.w, a.m)]
        if ctx is follows:
            ctx.use_torch_stream()
        assert same(b.pass_(ctx), want[0])
        torch.cuda.synchronize()
        assert same(e, r), turn
    print("captured:", name, flush=True)

# the timed programs, first on the default stream, then on another
from perf import operators as ops  # noqa: E402
ops.own = True
case = dict(op="step", shapes="64x495,300x200", w="f32", g="f32", nesterov=True)
first = {k: v.clone() for k, v in ops.run(ops.prepare(case, 7)).items()}
torch.cuda.synchronize()
with torch.cuda.stream(side[0]):
    st = ops.prepare(case, 7)
    G = [g.clone() for g in st["G"]]
    for g in st["G"]:
        g.zero_()
    delay()
    for g, h in zip(st["G"], G):
        g.copy_(h)
    out = ops.run(st)
    got = {k: v.clone() for k, v in out.items()}
    for v in out.values():
        v.zero_()
    torch.cuda.synchronize()
    assert all(torch.equal(first[k], got[k]) for k in first)
print("perf/operators on another stream", flush=True)
torch.cuda.synchronize()
for c in (own, follows):
    c.close()
print("done", flush=True)
