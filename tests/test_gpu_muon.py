"""Newton-Schulz orthogonalisation and the Muon step on the GPU against their definitions in 64 bits.

Tolerances.  fp32 / fp16 matrices: the products are split so that they are as exact as fp32 products.  The oracle runs the same
steps with torch's fp32 products on the CPU too; the kernel may be off by three times what those are off by (its planes carry 22
bits where fp32 carries 24: at most twice the rounding of X, plus the products' own), or by 2e-6 where that is less.  fp16 results
add their rounding, at most 2^-11 of each value; bf16 results: in the 2-norm, 2^-8 in all: rounding takes at most
2^-9 / sqrt(3) * 1.5 of it (values spread over a binade), and the products of planes of 11 bits (2^-12 a value, two factors, 3.4x
amplified once) the rest."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

ABC = (3.4445, -4.7750, 2.0315)
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


@pytest.fixture(scope="module")
def ops():
    from infinite_texture_gans_amd import ops as o
    return o


def steps_of(x, steps=5, abc=ABC):
    """the definition on a (rows, cols) CPU matrix in its own precision"""
    x = x / x.double().norm().to(x.dtype)
    tall = x.shape[0] > x.shape[1]
    x = x.T.contiguous() if tall else x
    for k in range(steps):
        a, b, c = abc if not isinstance(abc[0], tuple) else abc[k]
        s = x @ x.T
        x = a * x + (b * s + c * (s @ s)) @ x
    return x.T if tall else x


def rel(x, y):
    return float((x.double() - y).norm() / y.norm())


def matrix(m, n, seed=0, kind="floor"):
    g = torch.Generator().manual_seed(seed)
    k = min(16, m, n)
    x = torch.randn(m, n, generator=g)
    if kind == "floor":
        x = x + torch.randn(m, k, generator=g) @ torch.randn(k, n, generator=g)
    elif kind == "rank1":
        x = torch.randn(m, 1, generator=g) @ torch.randn(1, n, generator=g) + 1e-3 * x
    elif kind == "powers":
        u, _, v = torch.linalg.svd(x, full_matrices=False)
        x = u @ torch.diag(1.0 / torch.arange(1, min(m, n) + 1)) @ v
    return 1e-3 * x


def check(got, g, t, steps=5, abc=ABC):
    got, g = got.cpu(), g.cpu()
    want = steps_of(g.double(), steps, abc)
    own = rel(steps_of(g.float(), steps, abc), want)
    off = rel(got, want)
    if t == torch.bfloat16:
        assert off <= 2.0 ** -8 + 3 * own, (off, own)
    else:
        assert off <= max(3 * own, 2e-6) + (2.0 ** -11 if t == torch.float16 else 0.0), (off, own)


SIZES = [(1, 1), (1, 9), (7, 1), (2, 3), (3, 117), (13, 26), (64, 48), (48, 64), (64, 64), (65, 64), (63, 65), (128, 128), (13, 1000),
         (1000, 13), (100, 130), (333, 200), (256, 256), (129, 1025), (512, 300), (1, 4099), (520, 700), (200, 4100)]


@pytest.mark.parametrize("m,n", SIZES)
@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
def test_orthogonalize(ops, m, n, t):
    g = matrix(m, n, seed=m * 7 + n).cuda().to(TYPES[t])
    got = ops.orthogonalize(g)
    assert got.shape == g.shape and got.dtype == g.dtype
    check(got, g, TYPES[t])


@pytest.mark.parametrize("m,n", [(1024, 1024), (1100, 2050), (2304, 1153)])
@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_orthogonalize_larger(ops, m, n, t):
    g = matrix(m, n, seed=9).cuda().to(TYPES[t])
    check(ops.orthogonalize(g), g, TYPES[t])


@pytest.mark.parametrize("kind", ["rank1", "powers"])
@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("m,n", [(64, 64), (40, 300), (256, 192)])
def test_spectra(ops, kind, t, m, n):
    """updates of low rank over a faint floor, and spectra that fall off: rounding noise must not be blown up in the empty directions"""
    g = matrix(m, n, seed=4, kind=kind).cuda().to(TYPES[t])
    check(ops.orthogonalize(g), g, TYPES[t])


@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_batches_and_strides(ops, t):
    t = TYPES[t]
    g = torch.stack([matrix(70, 90, seed=s) for s in range(6)]).cuda().to(t).view(2, 3, 70, 90)
    each = torch.stack([ops.orthogonalize(x) for x in g.view(6, 70, 90)]).view(2, 3, 70, 90)
    assert torch.equal(ops.orthogonalize(g), each)
    wide = torch.randn(2, 3, 75, 101, device="cuda").to(t)
    wide[:, :, 2:72, 5:95] = g
    assert torch.equal(ops.orthogonalize(wide[:, :, 2:72, 5:95]), each)                        # rows at a stride
    cols = g.mT.contiguous().mT
    assert torch.equal(ops.orthogonalize(cols), each)                                          # column-major: the transposes' results
    assert torch.equal(ops.orthogonalize(g[0, 0].expand(4, 70, 90)), each[0, 0].expand(4, 70, 90))   # one matrix four times
    inner = g.permute(0, 2, 3, 1).contiguous().permute(0, 3, 1, 2)                             # no unit stride
    assert torch.equal(ops.orthogonalize(inner), each)
    assert torch.equal(ops.orthogonalize(g.transpose(0, 1)), each.transpose(0, 1))
    vec = torch.randn(5, 40, device="cuda").to(t)
    assert torch.equal(ops.orthogonalize(vec.T[:, 2:3]), ops.orthogonalize(vec.T[:, 2:3].contiguous()))
    out = torch.empty_like(g)
    assert ops.orthogonalize(g, out=out) is out and torch.equal(out, each)
    same = g.clone()
    assert ops.orthogonalize(same, out=same) is same and torch.equal(same, each)               # in place


def test_scales_zero_and_not_finite(ops):
    """the result does not depend on the matrix's scale; a zero matrix gives zeros; an infinity or a NaN stays in its own matrix"""
    base = matrix(40, 60, seed=3).cuda()
    want = ops.orthogonalize(base)
    for s in (2.0 ** 70, 2.0 ** -20, 2.0 ** 90):
        assert torch.equal(ops.orthogonalize(base * s), want)
    assert torch.equal(ops.orthogonalize(base * 2.0 ** -100, eps=0.0), want)
    tiny = ops.orthogonalize(base * 2.0 ** -60)                                               # a norm below eps
    assert torch.equal(tiny, torch.zeros_like(tiny))
    for t in (torch.float32, torch.bfloat16, torch.float16):
        g = torch.stack([matrix(40, 60, seed=s) for s in range(5)]).cuda().to(t)
        clean = ops.orthogonalize(g)
        g[1], g[2, 3, 4], g[3, 0, 0] = 0.0, float("inf"), float("nan")
        got = ops.orthogonalize(g, eps=0.0)
        assert torch.equal(got[1], torch.zeros_like(got[1]))
        assert torch.isnan(got[2]).all() and torch.isnan(got[3]).all()
        assert torch.equal(got[0], clean[0]) and torch.equal(got[4], clean[4])
    assert ops.orthogonalize(torch.empty(0, 4, 5, device="cuda")).shape == (0, 4, 5)
    assert ops.orthogonalize(torch.empty(3, 0, 5, device="cuda")).shape == (3, 0, 5)


def test_coefficients_and_steps(ops):
    g = matrix(50, 80, seed=8).cuda()
    check(ops.orthogonalize(g, steps=1), g, torch.float32, 1)
    check(ops.orthogonalize(g, steps=8, coefficients=(1.875, -1.25, 0.375)), g, torch.float32, 8, (1.875, -1.25, 0.375))
    each = ((3.4, -4.7, 2.0), (2.5, -2.5, 1.0), (1.875, -1.25, 0.375))
    check(ops.orthogonalize(g, steps=3, coefficients=each), g, torch.float32, 3, each)


def muon_oracle(p, g, m, ema, shapes, at, lr, mu, nesterov, wd, d, dtype):
    p, g, m = (v.cpu().to(dtype).clone() for v in (p, g, m))
    ema = ema.cpu().to(dtype).clone() if ema is not None else None
    for r, c in shapes:
        s = slice(at, at + r * c)
        m[s] = mu * m[s] + g[s]
        u = g[s] + mu * m[s] if nesterov else m[s]
        p[s] = p[s] * (1 - lr * wd) - lr * math.sqrt(max(1.0, r / c)) * steps_of(u.view(r, c)).reshape(-1)
        if ema is not None:
            ema[s] = d * ema[s] + (1 - d) * p[s]
        at += r * c
    return p, m, ema


SHAPES = [(13, 117), (3, 117), (64, 48), (48, 200), (1, 300), (130, 70), (5, 5)]


@pytest.mark.parametrize("nesterov,wd,with_ema,offset", [(True, 0.0, True, 0), (True, 0.1, False, 7), (False, 0.01, True, 3)])
def test_muon_step(ops, nesterov, wd, with_ema, offset):
    total = offset + sum(r * c for r, c in SHAPES) + 11
    gen = torch.Generator().manual_seed(1)
    p, g, m = (torch.randn(total, generator=gen).cuda() * s for s in (0.05, 1e-3, 1e-3))
    ema = p + 0.01 if with_ema else None
    plan = ops.MuonPlan(SHAPES, "cuda", offset=offset)
    want = muon_oracle(p, g, m, ema, SHAPES, offset, 0.3, 0.9, nesterov, wd, 0.99, torch.float64)
    fp32 = muon_oracle(p, g, m, ema, SHAPES, offset, 0.3, 0.9, nesterov, wd, 0.99, torch.float32)
    before = g.clone()
    ops.muon_step(plan, p, g, m, ema, lr=0.3, momentum=0.9, nesterov=nesterov, weight_decay=wd, ema_decay=0.99)
    assert torch.equal(g, before)
    for got, ref, low, what in zip((p, m, ema), want, fp32, ("p", "m", "ema")):
        if got is None:
            continue
        got = got.cpu()
        assert rel(got, ref) <= max(3 * rel(low, ref), 1e-6), what
        assert torch.equal(got[:offset].double(), ref[:offset]) and torch.equal(got[-11:].double(), ref[-11:])      # outside the matrices


def test_muon_step_of_many_matrices(ops):
    """more matrices than one call of the library takes"""
    shapes = [(4 + i % 5, 6 + i % 7) for i in range(75)]
    total = sum(r * c for r, c in shapes)
    p, g, m = (torch.randn(total, device="cuda") * s for s in (0.05, 1e-3, 1e-3))
    want = muon_oracle(p, g, m, None, shapes, 0, 0.1, 0.95, True, 0.0, 0.0, torch.float64)
    fp32 = muon_oracle(p, g, m, None, shapes, 0, 0.1, 0.95, True, 0.0, 0.0, torch.float32)
    ops.muon_step(ops.MuonPlan(shapes, "cuda"), p, g, m, lr=0.1)
    assert rel(p.cpu(), want[0]) <= max(3 * rel(fp32[0], want[0]), 1e-6) and rel(m.cpu(), want[1]) <= 1e-6


def test_every_replay_of_a_captured_step(ops):
    total = sum(r * c for r, c in SHAPES)
    p, g, m = (torch.randn(total, device="cuda") * s for s in (0.05, 1e-3, 1e-3))
    ema = p.clone()
    plan, other = ops.MuonPlan(SHAPES, "cuda"), ops.MuonPlan(SHAPES, "cuda")
    q, n, f = p.clone(), m.clone(), ema.clone()
    batch = torch.randn(3, 40, 70, device="cuda").bfloat16()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.muon_step(plan, p, g, m, ema)
        o = ops.orthogonalize(batch)
    for k in range(4):
        g.copy_(torch.randn(total, device="cuda") * 1e-3)
        batch.copy_(torch.randn(3, 40, 70, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        ops.muon_step(other, q, g, n, f)
        assert torch.equal(p, q) and torch.equal(m, n) and torch.equal(ema, f), k
        assert torch.equal(o, ops.orthogonalize(batch)), k


def test_two_calls_at_once(ops):
    """calls on two streams have workspaces of their own"""
    a, b = matrix(300, 400, seed=1).cuda(), matrix(120, 700, seed=2).cuda()
    want = ops.orthogonalize(a), ops.orthogonalize(b)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for s in (s1, s2):
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(5):
        with torch.cuda.stream(s1):
            x = ops.orthogonalize(a)
        with torch.cuda.stream(s2):
            y = ops.orthogonalize(b)
        got.append((x, y))
    torch.cuda.synchronize()
    for x, y in got:
        assert torch.equal(x, want[0]) and torch.equal(y, want[1])


def test_refusals(ops):
    from infinite_texture_gans_amd._lib import ItgError
    g = torch.randn(4, 8, device="cuda")
    plan = ops.MuonPlan([(4, 8)], "cuda")
    flat = [torch.zeros(32, device="cuda") for _ in range(3)]
    for bad in (lambda: ops.orthogonalize(g.cpu()), lambda: ops.orthogonalize(g.double()), lambda: ops.orthogonalize(g[0]),
                lambda: ops.orthogonalize(g, steps=0), lambda: ops.orthogonalize(g, steps=17), lambda: ops.orthogonalize(g, eps=-1.0),
                lambda: ops.orthogonalize(g, coefficients=(1.0, 2.0)), lambda: ops.orthogonalize(g, steps=3, coefficients=[(1.5, -0.5, 0.0)] * 2),
                lambda: ops.orthogonalize(g, coefficients=(8.0, 0.0, 0.0)), lambda: ops.orthogonalize(g, coefficients=(float("nan"), 0.0, 0.0)),
                lambda: ops.orthogonalize(g, out=torch.empty(8, 4, device="cuda")), lambda: ops.orthogonalize(g, out=torch.empty(4, 16, device="cuda")[:, ::2]),
                lambda: ops.orthogonalize(g.mT, out=g.mT), lambda: ops.orthogonalize(torch.empty(1, 70000, device="cuda")),
                lambda: ops.MuonPlan([], "cuda"), lambda: ops.MuonPlan([(0, 3)], "cuda"), lambda: ops.MuonPlan([(4, 8)], "cpu"),
                lambda: ops.MuonPlan([(4, 8)], "cuda", offset=-1), lambda: ops.muon_step(plan, flat[0][:31], flat[1], flat[2]),
                lambda: ops.muon_step(plan, flat[0], flat[1].half(), flat[2]), lambda: ops.muon_step(plan, flat[0], flat[1].cpu(), flat[2]),
                lambda: ops.muon_step(plan, flat[0], flat[1], flat[2], steps=0),
                lambda: ops.muon_step(plan, flat[0], torch.zeros(64, device="cuda")[::2], flat[2])):
        with pytest.raises(ItgError):
            bad()


@pytest.mark.parametrize("t,m,n,batch", [("f32", 2048, 2048, 1), ("f32", 1408, 5000, 1), ("f32", 2600, 2500, 1), ("f32", 6000, 900, 2), ("f16", 1030, 8200, 1),
                                         ("bf16", 2560, 2560, 1), ("bf16", 4096, 4100, 1), ("bf16", 9000, 2050, 1), ("bf16", 700, 1100, 9)])
def test_every_tile_size(ops, t, m, n, batch):
    """calls large enough for the larger tiles, alone and mixed between the three products, with whole rounds of tiles and with a
    rest that is split along K; the oracle's products run in 64 bits on the GPU"""
    g = torch.stack([matrix(m, n, seed=s) for s in range(batch)]).cuda().to(TYPES[t])
    got = ops.orthogonalize(g)
    for z in range(batch):
        want, own = steps_of(g[z].double()), steps_of(g[z].float().cpu()).cuda() if m * n < 3e6 else None
        off = rel(got[z], want)
        own = rel(own, want) if own is not None else 4e-6      # fp32 chains of this kind: 2e-6 .. 4e-6 off
        assert off <= (2.0 ** -8 if t == "bf16" else 3 * own + (2.0 ** -11 if t == "f16" else 0.0)), (z, off, own)


def test_overlaps_are_refused(ops):
    """out inside the memory g spans; one buffer in two of a step's places; what lies beside g is fine"""
    from infinite_texture_gans_amd._lib import ItgError
    buf = torch.randn(100 * 80 + 40, device="cuda")
    g, shifted = buf[:8000].view(100, 80), buf[40:].view(100, 80)
    for a, b in ((g, shifted), (shifted, g), (buf[:8000].view(50, 160)[:, :40], buf[4000:6000].view(50, 40))):
        with pytest.raises(ItgError):
            ops.orthogonalize(a, out=b)
    halves = torch.randn(2, 30, 50, device="cuda")
    want = ops.orthogonalize(halves[0])
    assert ops.orthogonalize(halves[0], out=halves[1]) is not None and torch.equal(halves[1], want)
    plan = ops.MuonPlan([(4, 8)], "cuda")
    p, g, m = (torch.randn(32, device="cuda") for _ in range(3))
    for args in ((p, p, m), (p, g, g), (p, g, p), (p, g, m, p), (p, g, m, g), (p, g, m, m)):
        with pytest.raises(ItgError):
            ops.muon_step(plan, *args)


def test_long_batches_of_tiny_matrices(ops):
    """a workgroup per matrix: 200 000 matrices of 1 x 1 (their signs under the iteration's gain) and of 2 x 3"""
    g = torch.randn(200000, 1, 1, device="cuda")
    o = ops.orthogonalize(g)
    want = steps_of(torch.ones(1, 1, dtype=torch.float64)).item()
    assert torch.equal(torch.sign(o), torch.sign(g)) and float((o.abs() - want).abs().max()) < 1e-5
    g = torch.randn(200000, 2, 3, device="cuda")
    o = ops.orthogonalize(g)
    for k in (0, 1, 99999, 199999):
        assert torch.equal(o[k], ops.orthogonalize(g[k]))


@pytest.mark.parametrize("t,m,n,batch", [("f32", 200, 5000, 6), ("f32", 1000, 4100, 1), ("f16", 130, 1400, 33), ("f32", 1900, 450, 5), ("f32", 1930, 1930, 1)])
def test_tall_tiles(ops, t, m, n, batch):
    """calls of 512 and more tiles of 128 columns by 64 rows, with columns behind the last whole tile, alone and split along K"""
    g = torch.stack([matrix(m, n, seed=s) for s in range(batch)]).cuda().to(TYPES[t])
    got = ops.orthogonalize(g)
    for z in range(batch):
        want, own = steps_of(g[z].double()), steps_of(g[z].float().cpu()).cuda()
        off, own = rel(got[z], want), rel(own, want)
        assert off <= 3 * own + (2.0 ** -11 if t == "f16" else 0.0), (z, off, own)


def test_offsets_past_2_31(ops):
    """matrices more than 2^31 values apart, rows more than 2^31 / 64 apart, and filters behind 2^31 values of a flat buffer"""
    big = torch.empty((1 << 32) + (1 << 28), device="cuda", dtype=torch.bfloat16)          # (written only where the matrices lie)
    far = torch.as_strided(big, (2, 70, 130), ((1 << 32) + 7, 130, 1))
    near = torch.randn(2, 70, 130, device="cuda").bfloat16()
    far.copy_(near)
    assert torch.equal(ops.orthogonalize(far), ops.orthogonalize(near))
    wide = torch.as_strided(big, (66, 200), ((1 << 26) + 3, 1))
    flat = torch.randn(66, 200, device="cuda").bfloat16()
    wide.copy_(flat)
    assert torch.equal(ops.orthogonalize(wide), ops.orthogonalize(flat))
    del big, far, wide
    shapes, at = [(64, 48), (130, 300)], (1 << 31) + 5
    total = sum(r * c for r, c in shapes)
    bufs = [torch.empty(at + total, device="cuda") for _ in range(3)]
    small = [torch.randn(total, device="cuda") for _ in range(3)]
    for v, s in zip(bufs, small):
        v[at:].copy_(s)
        v[at - 3:at] = 5.0
    ops.muon_step(ops.MuonPlan(shapes, "cuda", offset=at), *bufs)
    ops.muon_step(ops.MuonPlan(shapes, "cuda"), *small)
    for v, s in zip(bufs, small):
        assert torch.equal(v[at:], s) and torch.equal(v[at - 3:at], torch.full((3,), 5.0, device="cuda"))


@pytest.mark.parametrize("t,m,n,batch", [("f32", 100, 100, 3), ("bf16", 700, 100, 1), ("f32", 128, 128, 1), ("bf16", 4096, 4100, 1), ("f32", 1000, 4100, 1),
                                         ("f16", 60, 5000, 2)])
def test_captured_calls_of_every_path(ops, t, m, n, batch):
    """calls whose kernels ask for more shared memory than the default, split tiles and one-launch matrices, captured and replayed"""
    g = torch.stack([matrix(m, n, seed=s) for s in range(batch)]).cuda().to(TYPES[t])
    static = g.clone()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        o = ops.orthogonalize(static)
    for k in range(3):
        static.copy_(g.roll(k, -1))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, ops.orthogonalize(static)), k
        o.zero_()


@pytest.mark.parametrize("m,n", [(8, 8), (16, 64), (64, 64), (64, 128), (128, 100), (13, 1000), (100, 1000), (333, 1501), (512, 512), (700, 1100), (1030, 2100)])
def test_bf16_results_are_rounded_once(ops, m, n):
    """A bf16 matrix is held in no fewer bits than a float32 one: its result is the float32 path's, rounded at the end.  With y the
    unrounded result and |y - want| <= e (the float32 tests' bound), |bf16(y) - want| <= |bf16(y) - y| + e, and as the distance to
    the nearest bf16 value changes by no more than its argument does, <= |bf16(want) - want| + 2 e."""
    g = matrix(m, n, seed=m + 3 * n).bfloat16()
    want = steps_of(g.double())
    e = max(3 * rel(steps_of(g.float()), want), 2e-6)
    off, once = rel(ops.orthogonalize(g.cuda()).cpu(), want), rel(want.bfloat16(), want)
    assert off <= once + 2 * e, (off, once, e)


def test_steps_on_overlapping_buffers_are_refused(ops):
    """buffers that share values of the plan's matrices, also where the library takes a plan in several calls; slices side by side of
    one allocation, and buffers that overlap outside the matrices, are steps like any other"""
    from infinite_texture_gans_amd._lib import ItgError
    for shapes, offset in (([(4, 8)], 5), ([(3, 5)] * 70, 0)):
        n = sum(r * c for r, c in shapes)
        plan = ops.MuonPlan(shapes, "cuda", offset=offset)
        buf = torch.randn(12 * (n + 16), device="cuda") * 1e-3
        size = offset + n
        before = buf.clone()
        for shift in (1, n - 1):
            for a, b in ((0, 1), (0, 2), (0, 3), (1, 2), (1, 3), (2, 3)):
                at = [k * 2 * (n + 16) for k in range(4)]
                at[b] = at[a] + shift
                with pytest.raises(ItgError):
                    ops.muon_step(plan, *[buf[i:i + size] for i in at])
        assert torch.equal(buf, before)
        at = [0, n, 2 * n, 3 * n]                  # the values in front of a plan's matrices may be another buffer's matrices
        got, alone = [buf[i:i + size] for i in at], [buf[i:i + size].clone() for i in at]
        ops.muon_step(plan, *got, lr=0.1)
        ops.muon_step(ops.MuonPlan(shapes, "cuda", offset=offset), *alone, lr=0.1)
        for x, y in zip(got, alone):
            assert torch.equal(x[offset:], y[offset:])
