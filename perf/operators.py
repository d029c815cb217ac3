"""The operators that train and serve a refitted layer, as a user's program calls them, on real sizes.

    quant    a matrix cast to 8-bit floating point with one scale per block of 128 (cp_quant_blocks)
    matmul   the product of two such matrices, C = A B^T (cp_matmul_blocks)
    layer    one training pass of a layer in 8 bits: the output and both gradients (the two above together)
    ortho    the orthogonalised update of a set of layers by Newton-Schulz products (cp_orthogonalise)
    step     a whole optimiser step with it: momentum, orthogonalisation, decay, weights (cp_ortho_step)

`own` chooses between the plain form (elementary torch operations in 32 bits) and the framework's kernels.
"""
import os
import sys

import torch

own = False

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
F8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
FMAX = {"e4m3": 448.0, "e5m2": 57344.0}
TINY = 2.0 ** -100                           # a block's largest magnitude counts as at least this
COEF = (3.4445, -4.7750, 2.0315)             # the quintic of every step
STEPS, EPS = 5, 1e-7
LR, MOMENTUM, DECAY = 0.02, 0.95, 0.1

# weights [n, kept channels * k * k] of the layers that the vgg16 job refits (twelve conv -> conv pairs, int(c / 1.15) kept)
VGG16 = "64x495,128x495,128x999,256x999,256x1998,256x1998,512x1998,512x4005,512x4005,512x4005,512x4005,512x4005"
# and those of the resnet50 job: channel samplers (1 x 1), branch2b (3 x 3) and branch2c (1 x 1) of every stage's blocks
RESNET50 = ("64x35,256x55,64x101,64x459,256x39,64x97,64x450,256x37,128x144,512x106,128x205,128x945,512x72,128x198,128x945,512x72,"
            "128x288,512x110,256x278,1024x225,256x418,256x1881,1024x147,256x407,256x1836,1024x158,256x423,256x1908,1024x155,"
            "256x412,256x1899,1024x148,256x595,1024x213,512x606,2048x433,512x1222,2048x437,512x1147,2048x440")


def listed():
    return [
        # one token's activations before a product
        dict(name="quant one row", op="quant", rows=1, cols=4608, dtype="bf16", fmt="e4m3", tile=1, both=False, pow2=False),
        # the sampled patches of a wide layer at N = 20000, laid out for the product and for the weight gradient
        dict(name="quant patches both ways", op="quant", rows=20000, cols=4608, dtype="f32", fmt="e4m3", tile=1, both=True, pow2=False),
        # a large fully connected layer's weights, once per optimiser step
        dict(name="quant weights", op="quant", rows=4096, cols=25088, dtype="bf16", fmt="e4m3", tile=128, both=True, pow2=True),
        # serving: one token through a square layer
        dict(name="matmul one row", op="matmul", m=1, n=4096, k=4096, out="bf16", a="e4m3", b="e4m3", tile=128, bias=True),
        # a ragged batch at the classifier of the resnet50 network
        dict(name="matmul few rows", op="matmul", m=77, n=1000, k=2048, out="f32", a="e4m3", b="e4m3", tile=128, bias=True),
        # the refitted conv4 layer (445 of 512 channels, 3 x 3) on its N = 5000 sampled patches
        dict(name="matmul conv patches", op="matmul", m=5000, n=512, k=4005, out="bf16", a="e4m3", b="e4m3", tile=128, bias=True),
        # the largest product; both operands scaled row by row, as in a weight gradient
        dict(name="matmul large", op="matmul", m=8192, n=8192, k=8192, out="bf16", a="e4m3", b="e5m2", tile=1, bias=False),
        # one training pass of the 512-channel layer
        dict(name="layer conv", op="layer", m=20000, n=512, k=4005),
        # the smallest update: one early layer
        dict(name="ortho one small layer", op="ortho", shapes="64x576", dtype="bf16"),
        # a large fully connected layer
        dict(name="ortho large", op="ortho", shapes="4096x16384", dtype="bf16"),
        # all refitted layers of the two networks, float32 weights
        dict(name="step vgg16", op="step", shapes=VGG16, w="f32", g="f32", nesterov=True),
        dict(name="step resnet50", op="step", shapes=RESNET50, w="bf16", g="bf16", nesterov=True),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(("quant", "matmul", "layer", "ortho", "step"))
    if op == "quant":
        cols = _log(rng, 16, 25088)
        return dict(op=op, rows=_log(rng, 1, min(20000, 20000 * 4608 // cols)), cols=cols, dtype=rng.choice(("f32", "bf16", "f16")),
                    fmt=rng.choice(("e4m3", "e5m2")), tile=rng.choice((1, 128)), both=rng.random() < 0.5, pow2=rng.random() < 0.5)
    if op == "matmul":
        return dict(op=op, m=_log(rng, 1, 8192), n=_log(rng, 16, 8192), k=_log(rng, 16, 8192), out=rng.choice(("f32", "bf16", "f16")),
                    a="e4m3", b=rng.choice(("e4m3", "e5m2")), tile=rng.choice((1, 128)), bias=rng.random() < 0.5)
    if op == "layer":
        return dict(op=op, m=_log(rng, 64, 20000), n=_log(rng, 16, 1024), k=_log(rng, 64, 4608))
    m = [(_log(rng, 16, 2048), _log(rng, 16, 4608)) for _ in range(1 if rng.random() < 0.4 else _log(rng, 2, 16))]
    shapes = ",".join("%dx%d" % s for s in m)
    if op == "ortho":
        return dict(op=op, shapes=shapes, dtype=rng.choice(("f32", "bf16", "f16")))
    return dict(op=op, shapes=shapes, w=rng.choice(("f32", "bf16")), g=rng.choice(("f32", "bf16")), nesterov=rng.random() < 0.7)


def _shapes(case):
    return [tuple(int(v) for v in s.split("x")) for s in case["shapes"].split(",")]


def _up(v, to=128):
    return (v + to - 1) // to * to


# ---- inputs ---------------------------------------------------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _patches(g, rows, cols, dtype):
    """Activations behind a ReLU: half of them zero, channels of different strength, a few large ones."""
    x = torch.randn(rows, cols, generator=g, device="cuda").clamp_(min=0)
    x *= torch.exp(0.7 * torch.randn(1, cols, generator=g, device="cuda"))
    return x.to(dtype)


def _weights(g, rows, cols, dtype=torch.float32):
    return (0.05 * torch.randn(rows, cols, generator=g, device="cuda")).to(dtype)


def _gradient(g, rows, cols, dtype=torch.float32):
    """A few strong directions over a broad rest, at a gradient's magnitude."""
    r = min(8, rows, cols)
    G = torch.randn(rows, r, generator=g, device="cuda") @ torch.randn(r, cols, generator=g, device="cuda")
    G = G * 0.3 + torch.randn(rows, cols, generator=g, device="cuda")
    return (1e-3 * G).to(dtype)


def _held(x, fmt, tile):
    """(bytes [rows, cols rounded up to 128], scales, what they are): a matrix as it is held in 8 bits, by the plain form."""
    rows, cols = x.shape
    q, s = _quant(x, fmt, tile, False)
    held = torch.zeros(rows, _up(cols), dtype=torch.uint8, device="cuda")
    held[:, :cols] = q.view(torch.uint8)
    return dict(q=held, s=s.contiguous(), rows=rows, cols=cols, fmt=fmt, tile=tile)


def _room(rows, cols, fmt, tile):
    """Memory for a matrix held in 8 bits."""
    return dict(q=torch.zeros(rows, _up(cols), dtype=torch.uint8, device="cuda"), rows=rows, cols=cols, fmt=fmt, tile=tile,
                s=torch.zeros(_up(cols) // 128, rows if tile == 1 else _up(rows) // 128, device="cuda"))


def _together(many):
    """The same values in one buffer, as an optimiser holds its state, each at a multiple of 128 elements: (buffer, views)."""
    at = [0]
    for t in many:
        at.append(at[-1] + _up(t.numel()))
    buf = torch.zeros(at[-1], dtype=many[0].dtype, device=many[0].device)
    views = [buf[o: o + t.numel()].view(t.shape) for o, t in zip(at, many)]
    for v, t in zip(views, many):
        v.copy_(t)
    return buf, views


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    st = dict(case)
    if op == "quant":
        rows, cols = case["rows"], case["cols"]
        st["x"] = _weights(g, rows, cols, DT[case["dtype"]]) if case["tile"] == 128 else _patches(g, rows, cols, DT[case["dtype"]])
        st["out"] = _room(rows, cols, case["fmt"], case["tile"])
        st["out_t"] = _room(cols, rows, case["fmt"], case["tile"]) if case["both"] else None
    elif op == "matmul":
        m, n, k = case["m"], case["n"], case["k"]
        st["A"] = _held(_patches(g, m, k, torch.float32), case["a"], 1)
        st["B"] = _held(_weights(g, n, k), case["b"], case["tile"])
        st["bias_v"] = torch.randn(n, generator=g, device="cuda") if case["bias"] else None
        st["C"] = torch.zeros(m, n, dtype=DT[case["out"]], device="cuda")
    elif op == "layer":
        m, n, k = case["m"], case["n"], case["k"]
        st["x"] = _patches(g, m, k, torch.bfloat16)
        st["w"] = _weights(g, n, k)
        st["dy"] = (1e-4 * torch.randn(m, n, generator=g, device="cuda")).bfloat16()
        st["xq"], st["xt"] = _room(m, k, "e4m3", 1), _room(k, m, "e4m3", 1)
        st["wq"], st["wt"] = _room(n, k, "e4m3", 128), _room(k, n, "e4m3", 128)
        st["gq"], st["gt"] = _room(m, n, "e5m2", 1), _room(n, m, "e5m2", 1)
        st["y"], st["dx"] = (torch.zeros(m, v, dtype=torch.bfloat16, device="cuda") for v in (n, k))
        st["dw"] = torch.zeros(n, k, device="cuda")
    else:
        dt = DT[case["dtype"] if op == "ortho" else case["g"]]
        st["G"] = [_gradient(g, r, c, dt) for r, c in _shapes(case)]
        if op == "ortho":
            st["O"] = [torch.zeros_like(G) for G in st["G"]]
        else:
            st["M_all"], st["M"] = _together([_gradient(g, r, c) * 8 for r, c in _shapes(case)])
            st["W_all"], st["W"] = _together([_weights(g, r, c, DT[case["w"]]) for r, c in _shapes(case)])
    if own:
        _handles(st)
    return st


# ---- the plain form -------------------------------------------------------------------------------------------------------


def _quant(x, fmt, tile, pow2):
    """x [rows, cols] -> its 8-bit values and float32 scales [blocks of columns, rows or blocks of rows]."""
    x = x.float()
    rows, cols = x.shape
    kb, tr = _up(cols) // 128, _up(rows, tile) // tile
    pad = torch.nn.functional.pad(x, (0, kb * 128 - cols, 0, tr * tile - rows)).view(tr, tile, kb, 128)
    amax = pad.abs().amax(dim=(1, 3)).clamp(min=TINY)
    top = torch.full_like(amax, FMAX[fmt])      # a tensor: a division by a number is a product with its inverse
    scale = amax / top
    if pow2:
        frac, e = torch.frexp(scale)
        scale = torch.ldexp(torch.ones_like(scale), e - (frac == 0.5).int())
        inv = 1.0 / scale
    else:
        inv = top / amax
    q = (pad * inv[:, None, :, None]).clamp(-FMAX[fmt], FMAX[fmt]).to(F8[fmt])
    return q.view(tr * tile, kb * 128)[:rows, :cols], scale.t()


def _values(h, dtype=torch.float32):
    """What a matrix held in 8 bits stands for."""
    s = h["s"].t().to(dtype).repeat_interleave(h["tile"], 0)[: h["rows"]].repeat_interleave(128, 1)[:, : h["cols"]]
    return h["q"][:, : h["cols"]].view(F8[h["fmt"]]).to(dtype) * s


def _of(q, s, fmt, tile):
    return _values(dict(q=q.contiguous().view(torch.uint8), s=s, rows=q.shape[0], cols=q.shape[1], fmt=fmt, tile=tile))


def _ortho(G):
    X = G.float()
    tall = X.shape[0] > X.shape[1]
    X = X.t() if tall else X
    X = X / (X.norm() + EPS)
    a, b, c = COEF
    for _ in range(STEPS):
        A = X @ X.t()
        X = a * X + (b * A + c * (A @ A)) @ X
    return X.t() if tall else X


def _plain(st):
    op = st["op"]
    if op == "quant":
        q, s = _quant(st["x"], st["fmt"], st["tile"], st["pow2"])
        if not st["both"]:
            return {"q": q, "scale": s}
        qt, t = _quant(st["x"].t(), st["fmt"], st["tile"], st["pow2"])
        return {"q": q, "scale": s, "qt": qt, "scale_t": t}
    if op == "matmul":
        C = _values(st["A"]) @ _values(st["B"]).t()
        return (C if st["bias_v"] is None else C + st["bias_v"]).to(st["C"].dtype)
    if op == "layer":
        xq, xt = (_of(*_quant(v, "e4m3", 1, False), "e4m3", 1) for v in (st["x"], st["x"].t()))
        wq = _of(*_quant(st["w"], "e4m3", 128, False), "e4m3", 128)
        gq, gt = (_of(*_quant(v, "e5m2", 1, False), "e5m2", 1) for v in (st["dy"], st["dy"].t()))
        return {"y": (xq @ wq.t()).bfloat16(), "dx": (gq @ wq).bfloat16(), "dw": gt @ xt.t()}
    if op == "ortho":
        return [_ortho(G).to(G.dtype) for G in st["G"]]
    for G, M, W in zip(st["G"], st["M"], st["W"]):
        M.mul_(MOMENTUM).add_(G.float())
        U = G.float() + MOMENTUM * M if st["nesterov"] else M
        gamma = max(1.0, W.shape[0] / W.shape[1]) ** 0.5
        W.copy_((1 - LR * DECAY) * W.float() - LR * gamma * _ortho(U))
    return {"M": st["M_all"], "W": st["W_all"]}


# ---- the framework's calls ------------------------------------------------------------------------------------------------

_ctx = None


def _capi():
    global _ctx
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "channel-pruning_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from cpmi355 import capi
    if _ctx is None:
        _ctx = capi.Context(0)
    _ctx.use_torch_stream()                                                # in order with torch's work, whatever stream it is on now
    return capi, _ctx


def _handles(st):
    """What a user's program keeps: the descriptions of its 8-bit matrices, or the list of its layers."""
    capi, ctx = _capi()
    op = st["op"]
    code = {torch.float32: capi.CP_F32, torch.bfloat16: capi.CP_BF16, torch.float16: capi.CP_F16}
    st["code"] = code
    f8 = {"e4m3": capi.CP_E4M3, "e5m2": capi.CP_E5M2}
    for key in ("out", "out_t", "A", "B", "xq", "xt", "wq", "wt", "gq", "gt"):
        h = st.get(key)
        if isinstance(h, dict):
            h["h"] = capi.Blocks(h["q"], h["s"], h["rows"], h["cols"], f8[h["fmt"]], h["tile"])
    if op == "ortho":
        st["jobs"] = capi.OrthoJobs([(G, code[G.dtype], G.shape[0], G.shape[1], O, code[O.dtype]) for G, O in zip(st["G"], st["O"])])
    elif op == "step":
        st["jobs"] = capi.OrthoStepJobs([(G, code[G.dtype], G.shape[0], G.shape[1], M, W, code[W.dtype])
                                         for G, M, W in zip(st["G"], st["M"], st["W"])])


def _calls(st):
    capi, ctx = _capi()
    op = st["op"]
    if op == "quant":
        x, o, t = st["x"], st["out"], st["out_t"]
        ctx.quant_blocks(x, st["code"][x.dtype], o["h"], t["h"] if t else None, flags=capi.CP_QUANT_POW2 if st["pow2"] else 0)
        q = {"q": o["q"][:, : o["cols"]].view(F8[o["fmt"]]), "scale": o["s"]}
        return q | {"qt": t["q"][:, : t["cols"]].view(F8[t["fmt"]]), "scale_t": t["s"]} if t else q
    if op == "matmul":
        ctx.matmul_blocks(st["A"]["h"], st["B"]["h"], st["C"], st["code"][st["C"].dtype], bias=st["bias_v"])
        return st["C"]
    if op == "layer":
        ctx.quant_blocks(st["x"], capi.CP_BF16, st["xq"]["h"], st["xt"]["h"])
        ctx.quant_blocks(st["w"], capi.CP_F32, st["wq"]["h"], st["wt"]["h"])
        ctx.quant_blocks(st["dy"], capi.CP_BF16, st["gq"]["h"], st["gt"]["h"])
        ctx.matmul_blocks(st["xq"]["h"], st["wq"]["h"], st["y"], capi.CP_BF16)
        ctx.matmul_blocks(st["gq"]["h"], st["wt"]["h"], st["dx"], capi.CP_BF16)
        ctx.matmul_blocks(st["gt"]["h"], st["xt"]["h"], st["dw"], capi.CP_F32)
        return {"y": st["y"], "dx": st["dx"], "dw": st["dw"]}
    if op == "ortho":
        ctx.orthogonalise(st["jobs"], steps=STEPS, eps=EPS)
        return st["O"]
    ctx.ortho_step(st["jobs"], LR, momentum=MOMENTUM, nesterov=st["nesterov"], weight_decay=DECAY, steps=STEPS, eps=EPS)
    return {"M": st["M_all"], "W": st["W_all"]}


def run(state):
    return _calls(state) if own else _plain(state)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------------

SIZE = {"f32": 4, "bf16": 2, "f16": 2}


def _blocks_bytes(rows, cols, tile):
    return rows * cols + 4 * (_up(cols) // 128) * (_up(rows, tile) // tile)


def work(case):
    op = case["op"]
    if op == "quant":
        r, c = case["rows"], case["cols"]
        b = r * c * SIZE[case["dtype"]] + _blocks_bytes(r, c, case["tile"]) + (_blocks_bytes(c, r, case["tile"]) if case["both"] else 0)
        return {"bytes": b, "flops": 2 * r * c}
    if op == "matmul":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": _blocks_bytes(m, k, 1) + _blocks_bytes(n, k, case["tile"]) + m * n * SIZE[case["out"]], "flops": 2 * m * n * k}
    if op == "layer":
        m, n, k = case["m"], case["n"], case["k"]
        # inputs once (x, dy 16 bits, w 32), outputs once (y, dx 16 bits, dw 32)
        return {"bytes": 2 * m * k + 2 * m * n + 4 * n * k + 2 * m * n + 2 * m * k + 4 * n * k, "flops": 6 * m * n * k}
    flops = size = 0
    for r, c in _shapes(case):
        m, n = min(r, c), max(r, c)
        flops += STEPS * (m * m * n + m ** 3 + 2 * m * m * n)     # the two symmetric products at half their size
        size += r * c
    if op == "ortho":
        return {"bytes": 2 * SIZE[case["dtype"]] * size, "flops": flops}
    return {"bytes": (SIZE[case["g"]] + 8 + 2 * SIZE[case["w"]]) * size, "flops": flops}


# ---- the definition in 64 bits --------------------------------------------------------------------------------------------


def _round8(v, fmt):
    """v (float64) to the nearest 8-bit value, ties to even."""
    mant, low = (3, -6) if fmt == "e4m3" else (2, -14)
    e = torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -40)))
    e = torch.where(torch.exp2(e) > v.abs(), e - 1, torch.where(torch.exp2(e + 1) <= v.abs(), e + 1, e))
    step = torch.exp2(e.clamp(min=low) - mant)
    return torch.round(v / step) * step


def _exact_quant(x, fmt, tile, pow2):
    """The 8-bit values of x [rows, cols] as float64, and the scales [column blocks, row blocks]. The scale and its inverse are
    float32 numbers by the format's definition, and so is each scaled value before it is cut to 8 bits."""
    rows, cols = x.shape
    top = FMAX[fmt]
    out = torch.empty(rows, cols, dtype=torch.float64, device=x.device)
    n_k = -(-cols // 128)
    scales = torch.empty(n_k, -(-rows // tile), dtype=torch.float64, device=x.device)
    for j in range(n_k):
        part = x[:, 128 * j: 128 * (j + 1)].double()
        peak = part.abs().max(dim=1).values
        if tile > 1:
            peak = torch.stack([p.max() for p in peak.split(tile)])
        peak = torch.maximum(peak, torch.full_like(peak, TINY))
        s = (peak / top).float().double()
        inv = (top / peak).float().double()
        if pow2:
            s = torch.exp2(torch.ceil(torch.log2(s) - 1e-12))
            inv = 1 / s
        scales[j] = s
        if tile > 1:
            inv = inv.repeat_interleave(tile)[:rows]
        out[:, 128 * j: 128 * (j + 1)] = _round8((part * inv[:, None]).float().double().clamp(-top, top), fmt)
    return out, scales


def _exact_product(a, sa, ta, b, sb, tb):
    """sum over the blocks of 128 of a b^T times both scales."""
    va = a * sa.t().repeat_interleave(ta, 0)[: a.shape[0]].repeat_interleave(128, 1)[:, : a.shape[1]]
    vb = b * sb.t().repeat_interleave(tb, 0)[: b.shape[0]].repeat_interleave(128, 1)[:, : b.shape[1]]
    return va @ vb.t()


def _exact_ortho(U):
    """Newton-Schulz on the right singular side: the polynomial of X^T X, whichever way the matrix lies."""
    X = U / (torch.sqrt((U * U).sum()) + EPS)
    if X.shape[0] < X.shape[1]:
        X = X.t()
    a, b, c = COEF
    for _ in range(STEPS):
        S = X.t() @ X
        P = b * S + c * (S @ S)
        P.diagonal().add_(a)
        X = X @ P
    return X.t() if U.shape[0] < U.shape[1] else X


def exact(case, seed):
    global own
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    op = case["op"]
    if op == "quant":
        q, s = _exact_quant(st["x"], case["fmt"], case["tile"], case["pow2"])
        if not case["both"]:
            return {"q": q, "scale": s}
        qt, t = _exact_quant(st["x"].t(), case["fmt"], case["tile"], case["pow2"])
        return {"q": q, "scale": s, "qt": qt, "scale_t": t}
    if op == "matmul":
        A, B = st["A"], st["B"]
        C = _exact_product(A["q"][:, : case["k"]].view(F8[A["fmt"]]).double(), A["s"].double(), 1,
                           B["q"][:, : case["k"]].view(F8[B["fmt"]]).double(), B["s"].double(), B["tile"])
        return C if st["bias_v"] is None else C + st["bias_v"].double()
    if op == "layer":
        x, w, dy = st["x"], st["w"], st["dy"]
        xq, xt = _exact_quant(x, "e4m3", 1, False), _exact_quant(x.t(), "e4m3", 1, False)
        wq, wt = _exact_quant(w, "e4m3", 128, False), _exact_quant(w.t(), "e4m3", 128, False)
        gq, gt = _exact_quant(dy, "e5m2", 1, False), _exact_quant(dy.t(), "e5m2", 1, False)
        return {"y": _exact_product(*xq, 1, *wq, 128), "dx": _exact_product(*gq, 1, *wt, 128), "dw": _exact_product(*gt, 1, *xt, 1)}
    if op == "ortho":
        return [_exact_ortho(G.double()) for G in st["G"]]
    Ms, Ws = [], []
    for G, M, W in zip(st["G"], st["M"], st["W"]):
        M2 = MOMENTUM * M.double() + G.double()
        U = G.double() + MOMENTUM * M2 if case["nesterov"] else M2
        gamma = max(1.0, W.shape[0] / W.shape[1]) ** 0.5
        Ms.append(M2)
        Ws.append((1 - LR * DECAY) * W.double() - LR * gamma * _exact_ortho(U))
    return {"M": _together(Ms)[0], "W": _together(Ws)[0]}
