"""Layer norm on the GPU against its definition in 64 bits.

Tolerances.  e = 2^-24 is half a step of fp32.  A sum of n terms over `d` sequential additions per thread and a tree is off by at
most (d + 16) e times the sum of the magnitudes; that gives the mean, the variance, the two row means of the backward pass and the
column sums.  They enter the results through the formulas as below; the result itself is rounded once to its type (half a step,
finfo.eps / 2, of the value; below the type's smallest normal number the steps stay eps * smallest_normal apart whatever the
value, so that half of that, 2^-25 in fp16, is added: a value of 1e-5 may be off by 3e-8, which is 6 times eps / 2 of it)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


@pytest.fixture(scope="module")
def ops():
    from infinite_texture_gans_amd import ops as o
    return o


def act_of(u, act, slope):
    if act == 1:
        return torch.where(u > 0, u, slope * u), torch.where(u > 0, torch.ones_like(u), torch.full_like(u, slope))
    if act == 2:
        return torch.tanh(u), 1 - torch.tanh(u) ** 2
    return u, torch.ones_like(u)


def oracle(x, w, b, dy, eps, act, slope, t, tw):
    """values and tolerances (y, dx, dw, db) in fp64 for rows x (R, C)"""
    R, C = x.shape
    half = 0 if t == torch.float32 else torch.finfo(t).eps / 2
    halfw = 0 if tw == torch.float32 else torch.finfo(tw).eps / 2
    least, leastw = (torch.finfo(v).eps * torch.finfo(v).smallest_normal / 2 + 1e-30 for v in (t, tw))
    d = C / 64 + 16                                   # sequential additions of a row sum (at least 64 threads share it) + tree
    mean = x.mean(1, keepdim=True)
    var = ((x - mean) ** 2).mean(1, keepdim=True)
    r = 1 / torch.sqrt(var + eps)
    xh = (x - mean) * r
    dmean = (d + 1) * E * x.abs().mean(1, keepdim=True)
    # r: the variance is off by (d + 4) e of itself (+ the square of the mean's error); 1 / sqrt halves that, plus its own rounding
    drel = (d + 8) * E + (dmean * r) ** 2
    exh = dmean * r + xh.abs() * drel + 2 * E * xh.abs()
    ww, bb = (w if w is not None else torch.ones(C, dtype=x.dtype, device=x.device)), (b if b is not None else torch.zeros(C, dtype=x.dtype, device=x.device))
    u = xh * ww + bb
    eu = exh * ww.abs() + 2 * E * ((xh * ww).abs() + bb.abs())
    y, slope_at = act_of(u, act, slope)
    ty = eu * max(1.0, abs(slope)) + (half + 8 * E) * y.abs() + least
    out = [(y, ty)]
    if dy is None:
        return out, u
    # the activation's slope: exact for the linear pieces, |d tanh'| <= 2 |du| for tanh
    esl = 2 * eu + 16 * E if act == 2 else torch.zeros_like(u)
    du = dy * slope_at
    edu = dy.abs() * esl + 2 * E * du.abs()
    g = du * ww
    eg = edu * ww.abs() + 2 * E * g.abs()
    m1, m2 = g.mean(1, keepdim=True), (g * xh).mean(1, keepdim=True)
    em1 = (d + 2) * E * g.abs().mean(1, keepdim=True) + eg.mean(1, keepdim=True)
    em2 = (d + 2) * E * (g * xh).abs().mean(1, keepdim=True) + (eg * xh.abs() + g.abs() * exh).mean(1, keepdim=True)
    inner = g - m1 - xh * m2
    dx = r * inner
    tdx = r * (eg + em1 + xh.abs() * em2 + exh * m2.abs() + 4 * E * (g.abs() + m1.abs() + (xh * m2).abs())) + dx.abs() * (drel + half + 4 * E)
    n = R + 16
    dw, db = (du * xh).sum(0), du.sum(0)
    tdw = n * E * (du * xh).abs().sum(0) + (edu * xh.abs() + du.abs() * exh).sum(0) + (halfw + 4 * E) * dw.abs()
    tdb = n * E * du.abs().sum(0) + edu.sum(0) + (halfw + 4 * E) * db.abs()
    return out + [(dx, tdx + least), (dw, tdw + leastw), (db, tdb + leastw)], u


def near(got, want, what):
    v, tol = want
    got = got.double()
    assert torch.isfinite(got).all(), what
    off = (got - v).abs() / tol
    assert float(off.max()) <= 1.0, "%s: %.3g of the tolerance" % (what, float(off.max()))


def make(rows, c, t, tw, seed=0, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, c, generator=g) * (0.3 + torch.rand(c, generator=g)) + spread * torch.randn(rows, 1, generator=g)).to(t)
    w, b = (1 + 0.3 * torch.randn(c, generator=g)).to(tw), (0.3 * torch.randn(c, generator=g)).to(tw)
    dy = torch.randn(rows, c, generator=g).to(t)
    return [v.cuda() for v in (x, w, b, dy)]


def run(ops, x, w, b, dy, eps=1e-5, act=0, slope=0.0):
    x = x.detach().requires_grad_()
    ps = [p.detach().requires_grad_() if p is not None else None for p in (w, b)]
    y = ops.layer_norm(x, ps[0], ps[1], eps=eps, act=act, slope=slope)
    grads = torch.autograd.grad(y, [x] + [p for p in ps if p is not None], dy)
    return y.detach(), grads


SIZES = [(1, 1), (3, 2), (1, 8), (5, 3), (17, 13), (64, 16), (33, 52), (9, 64), (130, 104), (7, 129), (1, 1021), (70, 416), (257, 1024),
         (3, 2049), (1, 4096), (40, 4096), (2, 8195), (300, 512), (5, 16384), (2, 16389), (3, 40001), (1000, 7), (2049, 26)]


@pytest.mark.parametrize("rows,c", SIZES)
@pytest.mark.parametrize("types", ["f32/f32", "bf16/bf16", "bf16/f32", "f16/f16", "f16/f32"])
def test_forward_and_gradients(ops, rows, c, types):
    t, tw = (TYPES[k] for k in types.split("/"))
    x, w, b, dy = make(rows, c, t, tw, seed=rows + c)
    y, grads = run(ops, x, w, b, dy)
    want, _ = oracle(x.double(), w.double(), b.double(), dy.double(), 1e-5, 0, 0.0, t, tw)
    for got, ref, what in zip((y,) + tuple(grads), want, ("y", "dx", "dw", "db")):
        near(got, ref, what)
    assert y.dtype == t and grads[0].dtype == t and grads[1].dtype == tw and grads[2].dtype == tw


@pytest.mark.parametrize("act,slope", [(1, 0.0), (1, 0.2), (2, 0.0)])
@pytest.mark.parametrize("rows,c", [(50, 13), (31, 416), (6, 5000), (2, 20011)])
@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_activations(ops, rows, c, act, slope, t):
    x, w, b, dy = make(rows, c, TYPES[t], torch.float32, seed=3)
    want, u = oracle(x.double(), w.double(), b.double(), dy.double(), 1e-5, act, slope, TYPES[t], torch.float32)
    if act == 1:      # a value whose sign fp32 cannot tell takes either slope: no gradient passes through it here
        dy = torch.where(u.abs() < 1e-4, torch.zeros_like(dy), dy)
        want, u = oracle(x.double(), w.double(), b.double(), dy.double(), 1e-5, act, slope, TYPES[t], torch.float32)
    y, grads = run(ops, x, w, b, dy, act=act, slope=slope)
    for got, ref, what in zip((y,) + tuple(grads), want, ("y", "dx", "dw", "db")):
        near(got, ref, what)


def test_gradients_against_differences(ops):
    """fp32 central differences of <y, q>: an error of h^2 (third derivatives, O(1) here) and of 1e-6 / h in the quotient."""
    x, w, b, q = make(4, 24, torch.float32, torch.float32, seed=5)
    _, (dx, dw, db) = run(ops, x, w, b, q, act=2)
    h = 1e-2

    def f(x, w, b):
        return float((ops.layer_norm(x, w, b, act=2).double() * q.double()).sum())
    for t, d in ((x, dx), (w, dw), (b, db)):
        for i in range(0, t.numel(), 7):
            e = torch.zeros_like(t).view(-1)
            e[i] = h
            e = e.view(t.shape)
            args = [[a + s * e if a is t else a for a in (x, w, b)] for s in (1, -1)]
            num = (f(*args[0]) - f(*args[1])) / (2 * h)
            assert abs(num - float(d.reshape(-1)[i])) < 5e-3 * max(1.0, abs(num)), (i, num, float(d.reshape(-1)[i]))


@pytest.mark.parametrize("which", ["none", "gamma", "beta"])
def test_without_gain_or_shift(ops, which):
    x, w, b, dy = make(20, 100, torch.float32, torch.float32)
    w, b = (w if which == "gamma" else None), (b if which == "beta" else None)
    y, grads = run(ops, x, w, b, dy)
    want, _ = oracle(x.double(), w.double() if w is not None else None, b.double() if b is not None else None, dy.double(), 1e-5, 0, 0.0,
                     torch.float32, torch.float32)
    near(y, want[0], "y")
    near(grads[0], want[1], "dx")
    if which != "none":
        near(grads[1], want[2 if which == "gamma" else 3], which)


@pytest.mark.parametrize("c", [1, 3, 13, 52, 104, 416, 700])
def test_patch_grid(ops, c):
    """channels 0 .. c of the grid are normalised, the padding channels are written as zeros whatever they held in dy"""
    shape = (2, 3, 1, 4, 5)
    n = 2 * 3 * 4 * 5
    x, w, b, dy = make(n, c, torch.float32, torch.float32, seed=c)
    ld = ops.ld_for(c)
    xt = torch.nn.functional.pad(x, (0, ld - c)).view(*shape, ld).requires_grad_()
    dyt = torch.nn.functional.pad(dy, (0, ld - c), value=7.0).view(*shape, ld)
    w, b = w.requires_grad_(), b.requires_grad_()
    y = ops.layer_norm(ops.GT(xt, c), w, b)
    assert isinstance(y, ops.GT) and y.c == c and y.t.shape == xt.shape
    grads = torch.autograd.grad(y.t, [xt, w, b], dyt)
    want, _ = oracle(x.double(), w.detach().double(), b.detach().double(), dy.double(), 1e-5, 0, 0.0, torch.float32, torch.float32)
    for got, ref, what in zip((y.t.view(n, ld), grads[0].view(n, ld)), want, ("y", "dx")):
        near(got[:, :c].detach(), ref, what)
        assert torch.equal(got[:, c:], torch.zeros_like(got[:, c:]))
    near(grads[1], want[2], "dw")
    near(grads[2], want[3], "db")


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
def test_strides(ops, t):
    """slices of a wider buffer (rows in place, also off any vector alignment), leading dimensions, transposes"""
    t = TYPES[t]
    base = torch.randn(6, 9, 70, device="cuda").to(t)
    w, b = torch.randn(33, device="cuda"), torch.randn(33, device="cuda")
    for x in (base[..., 1:34], base[:, 2:5, 3:36], base[1:4, :, :33], base[:, ::2, 5:38], base.transpose(0, 1)[..., 30:63],
              base.permute(2, 0, 1)[:33].permute(1, 2, 0), base[0, 0, :33], base[:1, :1, 7:40]):
        got = ops.layer_norm(x, w, b)
        same = ops.layer_norm(x.contiguous(), w, b)
        assert torch.equal(got, same) and got.shape == x.shape and got.is_contiguous()
        xs, xc = x.detach().requires_grad_(), x.detach().contiguous().requires_grad_()
        dy = torch.randn(x.shape, device="cuda").to(t)
        dys = torch.empty(x.shape + (2,), device="cuda", dtype=t)[..., 0].copy_(dy)          # no unit stride
        g1, = torch.autograd.grad(ops.layer_norm(xs, w, b), xs, dys)
        g2, = torch.autograd.grad(ops.layer_norm(xc, w, b), xc, dy)
        assert torch.equal(g1, g2)


def test_buffer_behind_the_rows_is_left_alone(ops):
    """the last row's end: neither the padding behind a strided row nor what follows the last one is written"""
    import ctypes as C
    from infinite_texture_gans_amd import _lib
    for t, dt in ((torch.float32, 0), (torch.bfloat16, 1), (torch.float16, 2)):
        for c, ld in ((13, 19), (100, 131), (1021, 1021), (5001, 5003)):
            x = torch.randn(5, ld, device="cuda").to(t)
            y = torch.full((5 * ld + 64,), 3.0, device="cuda", dtype=t)
            _lib.call("itg_layer_norm_fwd", C.c_void_p(x.data_ptr()), ld, None, None, C.c_void_p(y.data_ptr()), ld, None, 5, c, 0, dt, dt,
                      1e-5, 0, 0.0, C.c_void_p(torch.cuda.current_stream().cuda_stream))
            v = y[:5 * ld].view(5, ld)
            assert torch.equal(v[:, :c], ops.layer_norm(x[:, :c]))
            assert torch.equal(v[:, c:], torch.full_like(v[:, c:], 3.0)) and torch.equal(y[5 * ld:], torch.full_like(y[5 * ld:], 3.0))


def test_no_rows_and_one_value(ops):
    w, b = torch.randn(8, device="cuda", requires_grad=True), torch.randn(8, device="cuda", requires_grad=True)
    x = torch.empty(0, 4, 8, device="cuda", requires_grad=True)
    y = ops.layer_norm(x, w, b)
    assert y.shape == x.shape
    g = torch.autograd.grad(y, [x, w, b], torch.empty_like(y))
    assert g[0].shape == x.shape and torch.equal(g[1], torch.zeros(8, device="cuda")) and torch.equal(g[2], torch.zeros(8, device="cuda"))
    one = ops.layer_norm(torch.full((3, 1), 5.0, device="cuda"))          # a single channel: variance 0, y = 0
    assert torch.equal(one, torch.zeros(3, 1, device="cuda"))


@pytest.mark.parametrize("c", [13, 52, 1000, 9000, 40000])
def test_extreme_rows(ops, c):
    """constant rows, rows far from zero, rows with an infinity or a NaN: their neighbours stay as they are"""
    x, w, b, dy = make(9, c, torch.float32, torch.float32, seed=1)
    x[1] = 4.0
    x[3] = x[3] + 1000.0
    clean = ops.layer_norm(x, w, b)
    want, _ = oracle(x.double(), w.double(), b.double(), None, 1e-5, 0, 0.0, torch.float32, torch.float32)
    near(clean, want[0], "y")
    bad = x.clone()
    bad[5, c // 2], bad[7, c - 1] = float("inf"), float("nan")
    got = ops.layer_norm(bad, w, b)
    assert torch.isnan(got[5]).all() and torch.isnan(got[7]).all()
    keep = [0, 1, 2, 3, 4, 6, 8]
    assert torch.equal(got[keep], clean[keep])


def test_same_result_every_time_and_in_a_graph(ops):
    """sums have a fixed order: repeated calls, a call on another stream and every replay of a captured training pass agree bit for bit"""
    x, w, b, dy = make(3000, 52, torch.float32, torch.float32, seed=2)
    xs, ws, bs = x.clone().requires_grad_(), w.clone().requires_grad_(), b.clone().requires_grad_()
    first = torch.autograd.grad(ops.layer_norm(xs, ws, bs), [xs, ws, bs], dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = torch.autograd.grad(ops.layer_norm(xs, ws, bs), [xs, ws, bs], dy)
    torch.cuda.current_stream().wait_stream(side)
    for p, q in zip(first, again):
        assert torch.equal(p, q)
    del first, again, xs, ws, bs
    static = x.clone()
    xg, wg, bg = static.requires_grad_(), w.clone().requires_grad_(), b.clone().requires_grad_()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        y = ops.layer_norm(xg, wg, bg, act=1, slope=0.1)
        grads = torch.autograd.grad(y, [xg, wg, bg], dy)
    for seed in (11, 12, 13):
        new, _, _, _ = make(3000, 52, torch.float32, torch.float32, seed=seed)
        with torch.no_grad():
            static.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        out = [y.detach().clone()] + [t.clone() for t in grads]
        xe, we, be = new.clone().requires_grad_(), w.clone().requires_grad_(), b.clone().requires_grad_()
        ye = ops.layer_norm(xe, we, be, act=1, slope=0.1)
        for p, q in zip(out, (ye.detach(),) + torch.autograd.grad(ye, [xe, we, be], dy)):
            assert torch.equal(p, q)


def test_sinks_accumulate(ops):
    x, w, b, dy = make(200, 26, torch.float32, torch.float32)
    w, b = w.requires_grad_(), b.requires_grad_()
    plain = torch.autograd.grad(ops.layer_norm(x, w, b), [w, b], dy)
    sinks = (torch.full((26,), 2.0, device="cuda"), torch.full((26,), -1.0, device="cuda"))
    xs = x.clone().requires_grad_()
    ops.layer_norm(xs, w, b, sinks=sinks).backward(dy)
    assert w.grad is None and b.grad is None and xs.grad is not None
    assert torch.equal(sinks[0], 2.0 + plain[0]) and torch.equal(sinks[1], -1.0 + plain[1])


def test_only_some_gradients(ops):
    x, w, b, dy = make(64, 48, torch.float32, torch.float32)
    full = run(ops, x, w, b, dy)[1]
    xs = x.clone().requires_grad_()
    assert torch.equal(torch.autograd.grad(ops.layer_norm(xs, w, b), xs, dy)[0], full[0])
    ws = w.clone().requires_grad_()
    assert torch.equal(torch.autograd.grad(ops.layer_norm(x, ws, b), ws, dy)[0], full[1])
    bs = b.clone().requires_grad_()
    assert torch.equal(torch.autograd.grad(ops.layer_norm(x, w, bs), bs, dy)[0], full[2])


def test_refusals(ops):
    from infinite_texture_gans_amd._lib import ItgError
    x, w = torch.randn(4, 8, device="cuda"), torch.randn(8, device="cuda")
    for bad in (lambda: ops.layer_norm(x.double()), lambda: ops.layer_norm(x.cpu()), lambda: ops.layer_norm(x, w[:4]),
                lambda: ops.layer_norm(x, w.cpu()), lambda: ops.layer_norm(x, w.bfloat16()), lambda: ops.layer_norm(x, w.repeat(2)[::2]),
                lambda: ops.layer_norm(x.bfloat16(), w, w.bfloat16()), lambda: ops.layer_norm(x, w, w, eps=-1.0),
                lambda: ops.layer_norm(x, w, w, eps=float("nan")), lambda: ops.layer_norm(x, w, w, act=9),
                lambda: ops.layer_norm(x, w, w, sinks=(w, None)), lambda: ops.layer_norm(x, None, w, sinks=(w, w)),
                lambda: ops.layer_norm(torch.empty(3, 0, device="cuda")), lambda: ops.layer_norm(torch.zeros((), device="cuda")),
                lambda: ops.layer_norm(x.int())):
        with pytest.raises(ItgError):
            bad()


def call(name, *args):
    from infinite_texture_gans_amd import _lib
    return _lib.fn(name)(*[a.data_ptr() if torch.is_tensor(a) else a for a in args], torch.cuda.current_stream().cuda_stream)


@pytest.mark.parametrize("c,pad", [(3, 0), (52, 0), (45, 3), (100, 19), (1021, 0), (4096, 0), (9001, 0), (9001, 5), (20003, 0)])
@pytest.mark.parametrize("t,dt", [(torch.float32, 0), (torch.bfloat16, 1)])
def test_written_over_the_inputs(ops, c, pad, t, dt):
    """y over x, dx over x and dx over dy: the bits that separate buffers give, and in the padding zeros whatever it held"""
    rows, ld = 37, c + pad
    x, w, b, dy = make(rows, ld, t, torch.float32, seed=c)
    w, b = w[:c].contiguous(), b[:c].contiguous()
    if pad:
        x[:, c:], dy[:, c:] = float("nan"), float("inf")
    ws = torch.empty(ops._lib.fn("itg_layer_norm_bwd_workspace")(rows, c), device="cuda")
    for act in (0, 1, 2):
        def fwd(src, out, stat):
            assert call("itg_layer_norm_fwd", src, ld, w, b, out, ld, stat, rows, c, pad, dt, 0, 1e-5, act, 0.1) == 0

        def bwd(src, grad, stat, out, dw, db):
            assert call("itg_layer_norm_bwd", src, ld, grad, ld, stat, w, b, out, ld, dw, db, 0, rows, c, pad, dt, 0, act, 0.1, ws, ws.numel()) == 0

        y, stat, dx = torch.empty_like(x), torch.empty(2 * rows, device="cuda"), torch.empty_like(x)
        dw, db = torch.empty(c, device="cuda"), torch.empty(c, device="cuda")
        fwd(x, y, stat)
        bwd(x, dy, stat, dx, dw, db)
        assert torch.equal(y[:, :c], ops.layer_norm(x[:, :c].contiguous(), w, b, act=act, slope=0.1)) and torch.isfinite(dx).all()
        assert not y[:, c:].any() and not dx[:, c:].any()
        for over in ("x", "dy"):
            a, g = x.clone(), dy.clone()
            ew, eb = torch.empty(c, device="cuda"), torch.empty(c, device="cuda")
            bwd(a, g, stat, a if over == "x" else g, ew, eb)
            assert torch.equal(a if over == "x" else g, dx) and torch.equal(ew, dw) and torch.equal(eb, db), (over, act)
        a, s = x.clone(), torch.empty_like(stat)
        fwd(a, a, s)
        assert torch.equal(a, y) and torch.equal(s, stat)
    # one buffer at two strides is no buffer at all
    assert call("itg_layer_norm_fwd", x, ld, w, b, x, ld + 1, None, rows - 2, c, pad, dt, 0, 1e-5, 0, 0.0) == -1
    assert call("itg_layer_norm_bwd", x, ld, dy, ld, stat, w, b, dy, ld + 1, None, None, 0, rows - 2, c, pad, dt, 0, 0, 0.0, None, 0) == -1


def test_sinks_of_a_frozen_parameter_stay(ops):
    x, w, b, dy = make(200, 26, torch.float32, torch.float32)
    for k in (0, 1):
        ps = [w.clone().requires_grad_(k == 0), b.clone().requires_grad_(k == 1)]
        plain, = torch.autograd.grad(ops.layer_norm(x, *ps), ps[k], dy)
        sinks = (torch.full((26,), 2.0, device="cuda"), torch.full((26,), 2.0, device="cuda"))
        xs = x.clone().requires_grad_()
        ops.layer_norm(xs, *ps, sinks=sinks).backward(dy)
        assert torch.equal(sinks[k], 2.0 + plain) and torch.equal(sinks[1 - k], torch.full((26,), 2.0, device="cuda"))


def test_second_derivatives_are_refused(ops):
    from infinite_texture_gans_amd._lib import ItgError
    x = torch.randn(4, 8, device="cuda", requires_grad=True)
    with pytest.raises(ItgError):
        torch.autograd.grad(ops.layer_norm(x).sum(), x, create_graph=True)


def test_two_captured_graphs_and_rows_far_apart(ops):
    """two captured training passes replayed in turn keep to their own buffers; a row stride that puts rows past 2^31 elements"""
    made, outs = [], []
    for seed, (rows, c) in enumerate(((40, 9001), (300, 416))):
        x, w, b, dy = make(rows, c, torch.float32, torch.float32, seed=seed)
        x, w, b = x.requires_grad_(), w.requires_grad_(), b.requires_grad_()
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            y = ops.layer_norm(x, w, b)
            outs.append([y.detach()] + list(torch.autograd.grad(y, [x, w, b], dy)))
        made.append((graph, x, w, b, dy))
    for turn in range(3):
        for graph, *_ in made if turn % 2 else made[::-1]:
            graph.replay()
        torch.cuda.synchronize()
        for (_, x, w, b, dy), got in zip(made, outs):
            xe, we, be = (v.detach().clone().requires_grad_() for v in (x, w, b))
            y = ops.layer_norm(xe, we, be)
            for p, q in zip(got, [y.detach()] + list(torch.autograd.grad(y, [xe, we, be], dy))):
                assert torch.equal(p, q)
            for p in got:
                p.zero_()
    ld = (1 << 31) + 24
    big = torch.empty(2 * ld + 64, device="cuda", dtype=torch.bfloat16)          # (written only where the three rows lie)
    x = torch.as_strided(big, (3, 52), (ld, 1))
    x.copy_(torch.randn(3, 52))
    xc, dy = x.contiguous().requires_grad_(), torch.randn(3, 52, device="cuda").bfloat16()
    xs = x.detach().requires_grad_()
    ys, yc = ops.layer_norm(xs), ops.layer_norm(xc)
    assert torch.equal(ys, yc) and torch.equal(torch.autograd.grad(ys, xs, dy)[0], torch.autograd.grad(yc, xc, dy)[0])


@pytest.mark.parametrize("rows,c", [(520, 8200), (600, 9001), (1030, 16384), (3, 8200), (511, 8192), (512, 8192)])
@pytest.mark.parametrize("types", ["bf16/bf16", "f16/f32", "f32/f32"])
def test_many_and_few_long_rows(ops, rows, c, types):
    """rows of more than 8192 values: in registers where they are many, swept where they are few"""
    t, tw = (TYPES[k] for k in types.split("/"))
    x, w, b, dy = make(rows, c, t, tw, seed=rows)
    for act, slope in ((0, 0.0), (1, 0.1)):
        want, u = oracle(x.double(), w.double(), b.double(), dy.double(), 1e-5, act, slope, t, tw)
        g = dy if act == 0 else torch.where(u.abs() < 1e-4, torch.zeros_like(dy), dy)
        if act:
            want, _ = oracle(x.double(), w.double(), b.double(), g.double(), 1e-5, act, slope, t, tw)
        y, grads = run(ops, x, w, b, g, act=act, slope=slope)
        for got, ref, what in zip((y,) + tuple(grads), want, ("y", "dx", "dw", "db")):
            near(got, ref, what)


@pytest.mark.parametrize("t,dt", [(torch.bfloat16, 1), (torch.float16, 2)])
def test_many_long_rows_over_the_inputs(ops, t, dt):
    """as test_written_over_the_inputs, for rows that stay in registers in 16 bits, with padding that holds anything"""
    rows, c, pad = 600, 9001, 5
    ld = c + pad
    x, w, b, dy = make(rows, ld, t, torch.float32, seed=5)
    w, b = w[:c].contiguous(), b[:c].contiguous()
    x[:, c:], dy[:, c:] = float("inf"), float("nan")
    ws = torch.empty(ops._lib.fn("itg_layer_norm_bwd_workspace")(rows, c), device="cuda")
    y, stat, dx = torch.empty_like(x), torch.empty(2 * rows, device="cuda"), torch.empty_like(x)
    dw, db = torch.empty(c, device="cuda"), torch.empty(c, device="cuda")
    assert call("itg_layer_norm_fwd", x, ld, w, b, y, ld, stat, rows, c, pad, dt, 0, 1e-5, 1, 0.1) == 0

    def bwd(src, grad, out, gw, gb):
        assert call("itg_layer_norm_bwd", src, ld, grad, ld, stat, w, b, out, ld, gw, gb, 0, rows, c, pad, dt, 0, 1, 0.1, ws, ws.numel()) == 0

    bwd(x, dy, dx, dw, db)
    xs, ps = x[:, :c].contiguous().requires_grad_(), [w.requires_grad_(), b.requires_grad_()]
    want = torch.autograd.grad(ops.layer_norm(xs, *ps, act=1, slope=0.1), [xs] + ps, dy[:, :c].contiguous())
    assert torch.equal(dx[:, :c], want[0]) and not dx[:, c:].any() and torch.equal(dw, want[1]) and torch.equal(db, want[2])
    for over in ("x", "dy"):
        a, g = x.clone(), dy.clone()
        ew, eb = torch.empty(c, device="cuda"), torch.empty(c, device="cuda")
        bwd(a, g, a if over == "x" else g, ew, eb)
        assert torch.equal(a if over == "x" else g, dx) and torch.equal(ew, dw) and torch.equal(eb, db), over


def test_more_than_2_31_values(ops):
    """a contiguous tensor whose later rows lie past 2^31 values: each row as it is alone, the weights' gradients as from its halves"""
    rows, c = (1 << 20) + 5, 2056
    x = torch.empty(rows, c, device="cuda", dtype=torch.bfloat16)
    block = torch.randn(1 << 12, c, device="cuda").bfloat16()
    for k in range(0, rows, 1 << 12):
        x[k:k + (1 << 12)] = block[:min(1 << 12, rows - k)]
    x[-5:] = torch.randn(5, c, device="cuda").bfloat16()
    w, b = torch.randn(c, device="cuda", requires_grad=True), torch.randn(c, device="cuda", requires_grad=True)
    xs = x.requires_grad_()
    y = ops.layer_norm(xs, w, b)
    dx, dw, db = torch.autograd.grad(y, [xs, w, b], x.detach())
    tail = x.detach()[-4101:].clone().requires_grad_()
    yt = ops.layer_norm(tail, w, b)
    dt, = torch.autograd.grad(yt, tail, tail.detach())
    assert torch.equal(y[-4101:], yt) and torch.equal(dx[-4101:], dt)
    first = x.detach()[:1 << 12].clone().requires_grad_()
    yf = ops.layer_norm(first, w, b)
    df, fw, fb = torch.autograd.grad(yf, [first, w, b], first.detach())
    assert torch.equal(y[:1 << 12], yf) and torch.equal(dx[:1 << 12], df)
    last = x.detach()[-5:].clone().requires_grad_()
    _, lw, lb = torch.autograd.grad(ops.layer_norm(last, w, b), [last, w, b], last.detach())
    # 256 blocks of the same rows, and five.  A channel's fp32 sum of 2^20 terms passes through at most 600 additions in a row (4096
    # rows a workgroup's share in four groups, 1024 shares in 64 lanes), the block's through fewer: 600 half steps of the sum of
    # the terms' sizes each, which is below 1.2 a row for normal values over 4096 different rows
    for whole, f, l in ((dw, fw, lw), (db, fb, lb)):
        want = 256 * f.double() + l.double()
        assert float((whole.double() - want).abs().max()) <= 2 * 600 * 2.0 ** -24 * 1.2 * rows


@pytest.mark.parametrize("rows,c", [(40, 7), (40, 52), (70, 1021), (9, 4096), (600, 9001), (5, 20003)])
@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
def test_vectors_at_odd_addresses(ops, rows, c, t):
    """x, dy, gamma and beta one value behind an aligned address: the bits that aligned tensors give"""
    x, w, b, dy = make(rows, c, TYPES[t], TYPES[t], seed=c)
    y, grads = run(ops, x, w, b, dy, act=1, slope=0.1)

    def shift(v):
        return torch.cat([v.new_zeros(1), v.flatten()])[1:].view(v.shape)

    y1, g1 = run(ops, shift(x), shift(w), shift(b), shift(dy), act=1, slope=0.1)
    assert shift(x).data_ptr() % 16 and torch.equal(y, y1)
    for p, q in zip(grads, g1):
        assert torch.equal(p, q)


@pytest.mark.parametrize("t,dt,tw,pdt", [(torch.bfloat16, 1, torch.float32, 0), (torch.bfloat16, 1, torch.bfloat16, 1), (torch.float16, 2, torch.float32, 0)])
@pytest.mark.parametrize("act", [0, 1])
def test_nothing_behind_the_parameters_counts(ops, t, dt, tw, pdt, act):
    """rows of 16-bit values whose padding fills their last vector: NaN behind gamma's and beta's last value changes no bit"""
    rows, c, pad = 600, 9001, 7
    ld = c + pad
    x, w, b, dy = make(rows, ld, t, tw, seed=6)
    x[:, c:], dy[:, c:], w[c:], b[c:] = float("inf"), float("nan"), float("nan"), float("nan")
    ws = torch.empty(ops._lib.fn("itg_layer_norm_bwd_workspace")(rows, c), device="cuda")
    y, stat, dx = torch.empty_like(x), torch.empty(2 * rows, device="cuda"), torch.empty_like(x)
    dw, db = torch.empty(c, device="cuda", dtype=tw), torch.empty(c, device="cuda", dtype=tw)
    assert call("itg_layer_norm_fwd", x, ld, w, b, y, ld, stat, rows, c, pad, dt, pdt, 1e-5, act, 0.1) == 0
    assert call("itg_layer_norm_bwd", x, ld, dy, ld, stat, w, b, dx, ld, dw, db, 0, rows, c, pad, dt, pdt, act, 0.1, ws, ws.numel()) == 0
    xs, ps = x[:, :c].contiguous().requires_grad_(), [w[:c].clone().requires_grad_(), b[:c].clone().requires_grad_()]
    ys = ops.layer_norm(xs, *ps, act=act, slope=0.1)
    want = torch.autograd.grad(ys, [xs] + ps, dy[:, :c].contiguous())
    assert torch.equal(y[:, :c], ys) and not y[:, c:].any()
    assert torch.equal(dx[:, :c], want[0]) and not dx[:, c:].any() and torch.equal(dw, want[1]) and torch.equal(db, want[2])


@pytest.mark.parametrize("rows,c,pad", [(1, 1, 0), (9, 3, 1), (3000, 7, 1), (70, 52, 0), (2000, 1023, 1), (700, 2056, 0), (900, 5000, 0), (600, 9001, 7),
                                        (300, 16384, 0), (40, 9001, 0), (1030, 16392, 0), (96, 40000, 0), (3, 70001, 0)])
@pytest.mark.parametrize("t,dt", [(torch.float32, 0), (torch.bfloat16, 1)])
def test_workspace_is_not_written_past_its_end(ops, rows, c, pad, t, dt):
    """a workspace of the queried size and not a float more, in a buffer whose rest stays as it is; the results do not depend on it"""
    ld = c + pad
    x, w, b, dy = make(rows, ld, t, torch.float32, seed=rows)
    w, b = w[:c].contiguous(), b[:c].contiguous()
    n = ops._lib.fn("itg_layer_norm_bwd_workspace")(rows, c)
    buf = torch.full((n + 4096,), 3.0, device="cuda")
    y, stat, dx = torch.empty_like(x), torch.empty(2 * rows, device="cuda"), torch.empty_like(x)
    dw, db = torch.empty(c, device="cuda"), torch.empty(c, device="cuda")
    assert call("itg_layer_norm_fwd", x, ld, w, b, y, ld, stat, rows, c, pad, dt, 0, 1e-5, 0, 0.0) == 0
    assert call("itg_layer_norm_bwd", x, ld, dy, ld, stat, w, b, dx, ld, dw, db, 0, rows, c, pad, dt, 0, 0, 0.0, buf, n) == 0
    assert call("itg_layer_norm_bwd", x, ld, dy, ld, stat, w, b, dx, ld, dw, db, 0, rows, c, pad, dt, 0, 0, 0.0, buf, n - 1) == -4
    assert torch.equal(buf[n:], torch.full((4096,), 3.0, device="cuda"))
    other, more = [torch.empty_like(v) for v in (dx, dw, db)], torch.empty(4 * n + 4096, device="cuda")
    assert call("itg_layer_norm_bwd", x, ld, dy, ld, stat, w, b, other[0], ld, other[1], other[2], 0, rows, c, pad, dt, 0, 0, 0.0, more, more.numel()) == 0
    for p, q in zip((dx, dw, db), other):
        assert torch.equal(p, q)
    want, _ = oracle(x[:, :c].double(), w.double(), b.double(), dy[:, :c].double(), 1e-5, 0, 0.0, t, torch.float32)
    near(dw, want[2], "dw")
    near(db, want[3], "db")


def test_forward_mode_derivatives_are_refused(ops):
    """a tangent of x, gamma or beta would be lost on the way: with and without a tape, in no_grad, of a GT and through torch.func"""
    import torch.autograd.forward_ad as fwd
    from infinite_texture_gans_amd._lib import ItgError
    x, w, b = torch.randn(4, 8, device="cuda"), torch.randn(8, device="cuda"), torch.randn(8, device="cuda")
    plain = ops.layer_norm(x, w, b)
    with fwd.dual_level():
        for k in range(3):
            args = [fwd.make_dual(v, torch.ones_like(v)) if i == k else v for i, v in enumerate((x, w, b))]
            taped = [a.detach().requires_grad_() if i != k else a for i, a in enumerate(args)]
            for call_args in (args, taped):
                with pytest.raises(ItgError, match="forward"):
                    ops.layer_norm(*call_args)
                with torch.no_grad(), pytest.raises(ItgError, match="forward"):
                    ops.layer_norm(*call_args)
        grid = fwd.make_dual(x.view(1, 1, 1, 1, 4, 8), torch.ones(1, 1, 1, 1, 4, 8, device="cuda"))
        with pytest.raises(ItgError, match="forward"):
            ops.layer_norm(ops.GT(grid, 8), w, b)
        assert torch.equal(ops.layer_norm(x, w, b), plain)                       # no tangent, nothing to lose
        xs = x.clone().requires_grad_()
        assert torch.equal(ops.layer_norm(xs, w, b), plain)
    with pytest.raises(Exception):
        torch.func.jvp(lambda v: ops.layer_norm(v, w, b), (x,), (torch.ones_like(x),))
    assert torch.equal(ops.layer_norm(x, w, b), plain)


@pytest.mark.parametrize("rows,c,t,groups", [((1 << 17) + 5, 2056, "bf16", 512), (1 << 17, 4096, "bf16", 512), (70001, 9001, "bf16", 256), (1 << 18, 416, "f32", 1024),
                                             (100003, 52, "f32", 1024)])
def test_long_column_sums(ops, rows, c, t, groups):
    """Gradients of gamma and beta over many rows against 64-bit sums.  A channel's sum passes through the rows that one thread sees
    (of `groups` workgroups, as the workspace says), the row groups and waves of its workgroup (9 additions at most), 16 shares of
    a lane at most, and 6 steps of the last tree; each addition is off by half a step of a sum that the terms' sizes bound."""
    assert ops._lib.fn("itg_layer_norm_bwd_workspace")(rows, c) == groups * 2 * c
    t, depth = TYPES[t], -(-rows // groups) + 9 + 16 + 6
    x, w, b, dy = make(rows, c, t, torch.float32, seed=c)
    _, (_, dw, db) = run(ops, x, w, b, dy)
    want, size, error = torch.zeros(2, c, device="cuda", dtype=torch.float64), torch.zeros(2, c, device="cuda", dtype=torch.float64), torch.zeros(c, device="cuda", dtype=torch.float64)
    for k in range(0, rows, 1 << 12):
        xs, du = x[k:k + (1 << 12)].double(), dy[k:k + (1 << 12)].double()
        mean = xs.mean(1, keepdim=True)
        r = 1 / torch.sqrt(((xs - mean) ** 2).mean(1, keepdim=True) + 1e-5)
        xh, d = (xs - mean) * r, c / 64 + 16
        dmean = (d + 1) * E * xs.abs().mean(1, keepdim=True)
        exh = dmean * r + xh.abs() * ((d + 10) * E + (dmean * r) ** 2)
        want += torch.stack([(du * xh).sum(0), du.sum(0)])
        size += torch.stack([(du * xh).abs().sum(0), du.abs().sum(0)])
        error += (du.abs() * exh).sum(0)
    for got, k, more in ((dw, 0, error), (db, 1, 0.0)):
        near(got, (want[k], depth * E * size[k] + more + E * want[k].abs() + 1e-30), "dw" if k == 0 else "db")


@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_saved_rows_that_come_back_at_another_stride(ops, t):
    """hooks on saved tensors (offloading, copies) hand the backward pass a contiguous x where rows of a wider buffer were saved: the
    rows are read at the stride that they have then"""
    base = torch.randn(5, 300, 70, device="cuda").to(TYPES[t])
    w, b = torch.randn(33, device="cuda"), torch.randn(33, device="cuda")
    dy = torch.randn(5, 300, 33, device="cuda").to(TYPES[t])

    def grads(x):
        leaves = [x.detach().requires_grad_(), w.clone().requires_grad_(), b.clone().requires_grad_()]
        return torch.autograd.grad(ops.layer_norm(*leaves, act=1, slope=0.1), leaves, dy)

    def widened(v):      # the other way round: contiguous rows that come back inside wider ones
        out = v.new_full(v.shape[:-1] + (v.shape[-1] + 7,), float("nan"))
        out[..., 2:2 + v.shape[-1]] = v
        return out[..., 2:2 + v.shape[-1]]
    hooks = [lambda: torch.autograd.graph.save_on_cpu(), lambda: torch.autograd.graph.saved_tensors_hooks(lambda v: v.clone().contiguous(), lambda v: v),
             lambda: torch.autograd.graph.saved_tensors_hooks(lambda v: v.clone(), lambda v: widened(v) if v.dim() == 3 else v),
             lambda: torch.autograd.graph.saved_tensors_hooks(lambda v: v.clone(), lambda v: v.transpose(0, 1).contiguous().transpose(0, 1) if v.dim() == 3 else v)]
    for x in (base[..., 1:34], base[..., 1:34].contiguous(), base.transpose(0, 1)[:5, :, :33].expand(5, 5, 33)[:, :1].expand(5, 300, 33)):
        want = grads(x)
        for hook in hooks:
            with hook():
                got = grads(x)
            for p, q in zip(got, want):
                assert torch.equal(p, q)


def test_sinks_that_share_values_are_refused(ops):
    """both would be written by different threads; slices side by side of one buffer are two sinks"""
    from infinite_texture_gans_amd._lib import ItgError
    x, w, b, dy = make(40, 26, torch.float32, torch.float32)
    buf = torch.zeros(80, device="cuda")
    for at in ((0, 0), (0, 25), (30, 5)):
        with pytest.raises(ItgError, match="sinks"):
            ops.layer_norm(x, w, b, sinks=tuple(buf[k:k + 26] for k in at))
    w, b = w.requires_grad_(), b.requires_grad_()
    want = torch.autograd.grad(ops.layer_norm(x, w, b), [w, b], dy)
    ops.layer_norm(x.requires_grad_(), w, b, sinks=(buf[26:52], buf[:26])).backward(dy)
    assert torch.equal(buf[26:52], want[0]) and torch.equal(buf[:26], want[1])
