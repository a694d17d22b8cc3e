"""Layer norm (pyramidkv.norm) against its definition in 64 bits.

Tolerances are bounds, with u = 2^-24 (half a step of fp32) and t = eps/2 of
the result's type.  A sum of C terms, each thread adding at most C / 32 of
them before a tree of 10 levels, is off by at most g = (C / 32 + 16) u times
the sum of magnitudes.  So the mean is off by g max|x|; x - mu by
e = g max|x| + u |x - mu|; the variance by 2 e sigma + g var, so rstd
relatively by r = e / sigma + g + 4 u; and xh by X = e / sigma + |xh| r.
"""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _data(cuda, N, C, G, dt, wt, seed=0, plus=False):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(N, C, generator=g) * torch.exp(0.5 * torch.randn(C, generator=g))
    x = (x + torch.randn(C, generator=g)).to(cuda, dt)
    shape = (G, C) if G > 1 else (C,)
    w = torch.randn(*shape, generator=g).to(cuda, wt)
    b = torch.randn(*shape, generator=g).to(cuda, wt)
    dy = torch.randn(N, C, generator=g).to(cuda, dt)
    return x, w, b, dy


def _exact(x, w, b, dy, eps, plus):
    """Definition and error bounds in 64 bits: {name: (value, bound)}."""
    N, C = x.shape
    xd, dt = x.double(), x.dtype
    G = 1 if w is None or w.dim() == 1 else w.shape[0]
    wd = torch.ones(1, C, dtype=torch.float64, device=x.device) if w is None else \
        w.double().view(G, C) + float(plus)
    bd = torch.zeros_like(wd) if b is None else b.double().view(G, C)
    W = wd.repeat_interleave(N // wd.shape[0], 0)
    B = bd.repeat_interleave(N // bd.shape[0], 0)
    mu = xd.mean(1, keepdim=True)
    d = xd - mu
    sig = ((d * d).mean(1, keepdim=True) + eps).sqrt()
    xh = d / sig
    y = xh * W + B
    g = (C / 32 + 16) * U
    e = g * xd.abs().amax(1, keepdim=True) + U * d.abs()
    e_row = e.amax(1, keepdim=True)
    r = e_row / sig + g + 4 * U
    X = e / sig + xh.abs() * r
    out = {"y": (y, W.abs() * X + 4 * U * ((xh * W).abs() + B.abs()) + _half(dt) * y.abs())}
    if dy is None:
        return out
    dyd = dy.double()
    gr = dyd * W
    c1, c2 = gr.mean(1, keepdim=True), (gr * xh).mean(1, keepdim=True)
    dx = (gr - c1 - xh * c2) / sig
    a1 = gr.abs().mean(1, keepdim=True)
    e1 = (g + 2 * U) * a1
    e2 = (g + 4 * U) * (gr * xh).abs().mean(1, keepdim=True) + X.amax(1, keepdim=True) * a1
    bound = (2 * U * gr.abs() + e1 + X * c2.abs() + xh.abs() * e2
             + 4 * U * (gr.abs() + c1.abs() + (xh * c2).abs())) / sig * (1 + r)
    out["dx"] = (dx, bound + r * dx.abs() + _half(dt) * dx.abs())
    n = N // G
    k = (n + 32) * U
    s = (dyd * xh).view(G, n, C)
    dw = s.sum(1)
    bw = k * s.abs().sum(1) + (dyd.abs() * X).view(G, n, C).sum(1) + _half(FP) * dw.abs()
    db = dyd.view(G, n, C).sum(1)
    bb = k * dyd.abs().view(G, n, C).sum(1)
    if w is not None:
        out["dw"] = (dw.view(w.shape), (bw + _half(w.dtype) * dw.abs()).view(w.shape))
    if b is not None:
        out["db"] = (db.view(b.shape), (bb + _half(b.dtype) * db.abs()).view(b.shape))
    return out


def _within(got, want, name):
    value, bound = want
    tiny = 6e-8 if got.dtype == HF else 1e-37   # half of the smallest fp16 step below its normals
    off = (got.double() - value).abs() - bound - tiny
    assert torch.isfinite(got.float()).all(), name
    assert off.max().item() <= 0, f"{name}: over its bound by {off.max().item():.3e}"


CASES = [
    # rows, cols, groups, type, weight type, one_plus
    (1, 1536, 1, BF, FP, False),        # one row: a block a row
    (3 * 512, 1536, 3, BF, BF, True),   # a warp a row, modulation of each frame
    (700, 1536, 7, BF, FP, True),
    (777, 1111, 1, FP, FP, False),      # odd columns: single elements
    (640, 48, 1, BF, BF, False),        # fewer vectors than a warp
    (601, 1, 1, FP, FP, False),         # one channel: variance 0
    (5, 7, 5, HF, FP, True),            # a group a row
    (600, 520, 1, HF, HF, False),
    (9, 4104, 3, BF, BF, True),         # a block a row, 3 vectors a thread
    (3, 8192, 1, FP, FP, False),
    (2, 8193, 1, BF, BF, False),        # rows too long for registers
    (33, 16392, 3, HF, FP, True),
    (2, 40000, 2, FP, FP, False),
    (1, 1, 1, BF, BF, True),
    # rows enough to fill the GPU: a few lanes a row, ...
    (3000, 24, 1, BF, FP, True),
    (2999, 64, 1, FP, FP, False),
    (2600, 100, 2, HF, HF, True),
    (2400, 250, 3, BF, BF, False),
    (4000, 30, 4000, BF, FP, True),     # ... a group a row
    # ... and fixed columns a thread, of 16, 4 and 2 bytes
    (2400, 777, 8, BF, FP, True),
    (2402, 1534, 2, HF, FP, False),
    (2400, 2050, 1, BF, BF, True),
    (2400, 4100, 3, FP, FP, True),
    (2400, 5001, 2, BF, BF, False),
    (2400, 8192, 1, HF, HF, True),
    (2400, 6000, 240, FP, FP, False),
    (2500, 1536, 2500, BF, FP, True),   # modulation of each row
    (2400, 700, 1200, FP, FP, True),
]


@pytest.mark.parametrize("N,C,G,dt,wt,plus", CASES)
def test_layer_norm_forward_and_gradients(cuda, N, C, G, dt, wt, plus):
    from pyramidkv.norm import layer_norm
    x, w, b, dy = _data(cuda, N, C, G, dt, wt, seed=N + C)
    want = _exact(x, w, b, dy, 1e-6, plus)
    for t in (x, w, b):
        t.requires_grad_(True)
    y = layer_norm(x, w, b, one_plus=plus)
    assert y.dtype == dt and y.shape == x.shape
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    _within(y, want["y"], "y")
    if C > 1:   # of one channel dx is 0 up to rounding noise times 1 / sqrt(eps)
        _within(dx, want["dx"], "dx")
    _within(dw, want["dw"], "dw")
    _within(db, want["db"], "db")
    with torch.no_grad():
        assert torch.equal(layer_norm(x, w, b, one_plus=plus), y)


@pytest.mark.parametrize("have_w,have_b", [(False, False), (True, False), (False, True)])
def test_layer_norm_without_weight_or_bias(cuda, have_w, have_b):
    from pyramidkv.norm import layer_norm
    x, w, b, dy = _data(cuda, 300, 256, 1, BF, FP)
    w, b = w if have_w else None, b if have_b else None
    want = _exact(x, w, b, dy, 1e-5, False)
    leaves = [t for t in (x, w, b) if t is not None]
    for t in leaves:
        t.requires_grad_(True)
    y = layer_norm(x, w, b, eps=1e-5)
    grads = torch.autograd.grad(y, leaves, dy)
    for name, got in zip(["y", "dx"] + ["dw"] * have_w + ["db"] * have_b, (y,) + grads):
        _within(got, want[name], name)


@pytest.mark.parametrize("rows,groups", [(300, 2), (40, 40)])
def test_layer_norm_some_gradients_wanted(cuda, rows, groups):
    """Any subset of x, weight and bias: the bits of the full call."""
    from pyramidkv.norm import layer_norm
    x, w, b, dy = _data(cuda, rows, 256, groups, BF, FP, seed=2)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    want = torch.autograd.grad(layer_norm(*leaves, one_plus=True), leaves, dy)
    for mask in range(1, 8):
        args = [t.clone().requires_grad_(bool(mask >> i & 1)) for i, t in enumerate((x, w, b))]
        picked = [t for t in args if t.requires_grad]
        got = torch.autograd.grad(layer_norm(*args, one_plus=True), picked, dy)
        assert all(torch.equal(p, want[i]) for p, i in
                   zip(got, [i for i in range(3) if mask >> i & 1])), mask


def test_layer_norm_offsets_past_32_bits(cuda):
    """Rows whose element offset passes 2^31 (and byte offset 2^32), forward and
    backward, against the bounds on the last ones."""
    from pyramidkv import _ops
    N, C = 1_400_010, 1536
    ops = _ops.ops()
    x = torch.zeros(N, C, dtype=BF, device=cuda)
    tail, w, b, dy = _data(cuda, 10, C, 1, BF, FP, seed=4)
    x[-10:] = tail
    y, mean, rstd = ops.pkv_layer_norm(x, w, b, 1e-6, False, True)
    want = _exact(tail, w, b, dy, 1e-6, False)
    _within(y[-10:], want["y"], "y")
    del y
    g = torch.zeros(N, C, dtype=BF, device=cuda)
    g[-10:] = dy
    dx, dw, db = ops.pkv_layer_norm_backward(g, x, w, b, mean, rstd, False, True, True, True)
    _within(dx[-10:], want["dx"], "dx")
    _within(dw, want["dw"], "dw")     # the other rows' dy is 0
    _within(db, want["db"], "db")


def test_layer_norm_strided_and_shaped_inputs(cuda):
    """Column slices (row stride three times the width), a transposed view, 4-D
    inputs, expanded gradients, a weight and a bias of different group counts."""
    from pyramidkv.norm import layer_norm
    g = torch.Generator().manual_seed(1)
    big = torch.randn(500, 3 * 128, generator=g).to(cuda, BF)
    x = big[:, 128:256]
    _within(layer_norm(x), _exact(x, None, None, None, 1e-6, False)["y"], "slice")
    xt = torch.randn(96, 200, generator=g).to(cuda, FP).t()
    _within(layer_norm(xt), _exact(xt, None, None, None, 1e-6, False)["y"], "transposed")
    off = torch.randn(64 * 128 + 1, generator=g).to(cuda, BF)[1:].view(64, 128)   # 2-byte aligned
    _within(layer_norm(off), _exact(off, None, None, None, 1e-6, False)["y"], "offset")
    x4 = torch.randn(2, 3, 5, 64, generator=g).to(cuda, FP).requires_grad_(True)
    w = torch.randn(64, generator=g).to(cuda).requires_grad_(True)
    b = torch.randn(2, 64, generator=g).to(cuda).requires_grad_(True)
    y = layer_norm(x4, w, b)
    dy = torch.randn(64, generator=g).to(cuda).expand(2, 3, 5, 64)
    dx, dw, db = torch.autograd.grad(y, (x4, w, b), dy)
    flat, dflat = x4.detach().view(30, 64), dy.reshape(30, 64)
    want = _exact(flat, w.detach().expand(2, 64), b.detach(), dflat, 1e-6, False)
    _within(y.view(30, 64), want["y"], "y")
    _within(dx.view(30, 64), want["dx"], "dx")
    _within(db, want["db"], "db")
    value, bound = want["dw"]
    # the two groups' gradients add up in the shared weight: one more rounding
    _within(dw, (value.sum(0), bound.sum(0) + U * value.abs().sum(0)), "shared dw")


def test_layer_norm_gradient_against_differences(cuda):
    """The kernels' gradient along random directions against central
    differences of the 64-bit definition (h = 1e-5: both errors of the
    differences are below 1e-8 of the terms' size)."""
    from pyramidkv.norm import layer_norm
    x, w, b, dy = _data(cuda, 12, 40, 3, FP, FP, seed=5)
    want = _exact(x, w, b, dy, 1e-6, True)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    grads = torch.autograd.grad(layer_norm(x, w, b, one_plus=True), leaves, dy)

    def f(x, w, b):
        x3 = x.view(3, 4, 40)
        d = x3 - x3.mean(-1, keepdim=True)
        y = d / (d.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * (1 + w)[:, None] + b[:, None]
        return (y.view(12, 40) * dy.double()).sum()

    for i, (t, gr) in enumerate(zip(leaves, grads)):
        v = torch.randn(t.shape, generator=torch.Generator().manual_seed(i)).to(cuda).double()
        args = [s.detach().double() for s in leaves]
        h = 1e-5
        up, down = list(args), list(args)
        up[i], down[i] = args[i] + h * v, args[i] - h * v
        diff = ((f(*up) - f(*down)) / (2 * h)).item()
        bound = (want[("dx", "dw", "db")[i]][1] * v.abs()).sum().item()
        size = (gr.double() * v).abs().sum().item()
        assert abs((gr.double() * v).sum().item() - diff) <= bound + 1e-7 * size


def test_layer_norm_infinities_stay_in_their_row(cuda):
    from pyramidkv.norm import layer_norm
    x, w, b, _ = _data(cuda, 700, 256, 1, BF, BF)
    clean = layer_norm(x, w, b)
    x[3, 5], x[9, 0] = float("inf"), float("nan")
    y = layer_norm(x, w, b)
    assert torch.isnan(y[3]).all() and torch.isnan(y[9]).all()
    rest = [r for r in range(700) if r not in (3, 9)]
    assert torch.equal(y[rest], clean[rest])


def test_layer_norm_no_rows(cuda):
    from pyramidkv.norm import layer_norm
    x = torch.empty(0, 64, device=cuda, requires_grad=True)
    w = torch.ones(64, device=cuda, requires_grad=True)
    y = layer_norm(x, w)
    dx, dw = torch.autograd.grad(y.sum(), (x, w))
    assert y.shape == dx.shape == (0, 64) and (dw == 0).all()


def test_layer_norm_repeats_bit_for_bit(cuda):
    from pyramidkv.norm import layer_norm
    x, w, b, dy = _data(cuda, 5000, 384, 4, BF, FP)
    for t in (x, w, b):
        t.requires_grad_(True)
    first = torch.autograd.grad(layer_norm(x, w, b), (x, w, b), dy)
    for _ in range(3):
        again = torch.autograd.grad(layer_norm(x, w, b), (x, w, b), dy)
        assert all(torch.equal(p, q) for p, q in zip(first, again))


def test_layer_norm_side_stream_and_graph(cuda):
    """Two calls at once on two streams, and one captured step replayed with
    new inputs: the same bits as eager calls."""
    from pyramidkv import _ops
    ops = _ops.ops()
    x, w, b, dy = _data(cuda, 3000, 512, 3, BF, FP)

    def step(x, dy):
        y, m, r = ops.pkv_layer_norm(x, w, b, 1e-6, True, True)
        return (y,) + ops.pkv_layer_norm_backward(dy, x, w, b, m, r, True, True, True, True)

    x2, dy2 = x.flip(0).contiguous(), dy.flip(0).contiguous()
    want, want2 = step(x, dy), step(x2, dy2)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(s1):
        got = step(x, dy)
    with torch.cuda.stream(s2):
        got2 = step(x2, dy2)
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got + got2, want + want2))
    xs, ds = x.clone(), dy.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = step(xs, ds)
    for src, dsrc, ref in ((x2, dy2, want2), (x, dy, want)):
        xs.copy_(src)
        ds.copy_(dsrc)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(res, ref))


def test_layer_norm_captured_backward(cuda):
    """A training step captured through autograd (no eager graph of the same
    leaves alive) and replayed with another gradient: the eager bits."""
    from pyramidkv.norm import layer_norm
    x, w, b, dy = _data(cuda, 640, 256, 2, BF, FP, seed=3)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    static = dy.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = layer_norm(x, w, b, one_plus=True)
        grads = torch.autograd.grad(y, leaves, static)
    other = dy.flip(0).contiguous()
    static.copy_(other)
    graph.replay()
    torch.cuda.synchronize()
    got = [t.clone() for t in grads]
    del y
    want = torch.autograd.grad(layer_norm(x, w, b, one_plus=True), leaves, other)
    assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_layer_norm_refusals(cuda):
    from pyramidkv.norm import layer_norm
    x = torch.randn(6, 8, device=cuda)
    for bad in (dict(weight=torch.ones(7, device=cuda)),            # channels
                dict(weight=torch.ones(4, 8, device=cuda)),         # 4 does not divide 6
                dict(weight=torch.ones(8, device=cuda, dtype=BF)),  # narrower than x
                dict(weight=torch.ones(8)),                         # on the CPU
                dict(weight=torch.ones(1, 1, 8, device=cuda)),
                dict(eps=-1.0)):
        with pytest.raises(RuntimeError, match="pkv_layer_norm"):
            layer_norm(x, **bad)
    with pytest.raises(RuntimeError, match="bf16, fp16 or fp32"):
        layer_norm(x.double())
    leaf = x.clone().requires_grad_(True)
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(layer_norm(leaf).sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="no channels"):
        layer_norm(x[:, :0])
    with pytest.raises(ValueError, match="one type"):
        layer_norm(x.to(BF), torch.ones(8, device=cuda, dtype=BF), torch.ones(8, device=cuda))


@pytest.mark.parametrize("rows,cols,groups", [(37, 1536, 1), (24, 512, 24), (9, 40_000, 3), (40, 9000, 1)])
def test_layer_norm_backward_in_place_through_the_abi(cuda, rows, cols, groups):
    """pkv_layer_norm_backward with dx in dy's memory, rows in registers and
    longer ones: the bits of separate memory."""
    import ctypes
    from pyramidkv import _scatter_ext
    ops = torch.ops.adahead
    _scatter_ext.load_library()
    lib = ctypes.CDLL(_scatter_ext.KERNEL_PATH)
    g = torch.Generator().manual_seed(cols)
    x, dy = (torch.randn(rows, cols, generator=g).to(cuda, torch.bfloat16) for _ in range(2))
    w, b = (torch.randn(groups, cols, generator=g).to(cuda) for _ in range(2))
    _, mean, rstd = ops.pkv_layer_norm(x, w, b, 1e-6, True, True)
    want = ops.pkv_layer_norm_backward(dy, x, w, b, mean, rstd, True, True, True, True)
    ptr, i64, i32 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int
    lib.pkv_layer_norm_workspace_bytes.restype = i64
    need = lib.pkv_layer_norm_workspace_bytes(i64(rows), i64(cols), i64(groups))
    ws = torch.empty(need, dtype=torch.uint8, device=cuda)
    both, dw, db = dy.clone(), torch.empty_like(w), torch.empty_like(b)
    at = lambda t: ptr(t.data_ptr())
    torch.cuda.synchronize()
    rc = lib.pkv_layer_norm_backward(
        at(both), i64(cols), at(x), i64(cols), at(w), at(mean), at(rstd), i32(0), i32(2),
        i64(rows), i64(cols), i64(groups), i32(1), at(both), i64(cols), at(dw), at(db), at(ws),
        i64(need), ptr(torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    assert rc == 0
    for got, ref in zip((both, dw, db), want):
        assert torch.equal(got, ref)
