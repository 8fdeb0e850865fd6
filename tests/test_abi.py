"""CPU-side checks of the C-ABI boundary: the in-tree library loads, exports every symbol that
include/itg.h declares, the ctypes table mirrors the header, and the host-only helpers (no kernel
launch) behave.  No compute call is made here - there is no GPU in this tier."""
import ctypes
import os
import re

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "itg.h")


def declared():
    src = open(HEADER).read()
    src = re.sub(r"/\*.*?\*/", "", src, flags=re.S)
    return sorted(set(re.findall(r"\b(itg_[a-z0-9_]+)\s*\(", src)))


@pytest.fixture(scope="module")
def lib():
    import __graft_entry__ as ge
    ge.build()
    from infinite_texture_gans_amd import _lib
    return _lib


def test_every_declared_symbol_is_exported(lib):
    names = declared()
    assert len(names) >= 40
    so = ctypes.CDLL(lib.LIB_PATH)
    missing = [n for n in names if not hasattr(so, n)]
    assert not missing, missing


def test_ctypes_table_mirrors_header(lib):
    assert sorted(lib.SIGNATURES) == declared()


def test_argument_counts_match_header(lib):
    src = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    for name, (_, args) in lib.SIGNATURES.items():
        m = re.search(r"\b%s\s*\(([^;]*?)\)\s*;" % name, src, flags=re.S)
        assert m, name
        params = m.group(1).strip()
        n = 0 if params in ("", "void") else len(params.split(","))
        assert n == len(args), (name, n, len(args))


def test_host_only_helpers(lib):
    so = lib.load()
    assert so.itg_version() >= 100
    # packed sizes: rows rounded to 16, K rounded to 16
    assert so.itg_pack_fwd_size(13, 28, 3, 3) == 16 * 256
    assert so.itg_pack_dgrad_size(3, 64, 4, 4, 2) == 4 * 16 * 256
    assert so.itg_pack_dgrad_size(26, 16, 3, 3, 1) == 32 * 144


def test_rejected_calls_return_error_codes_not_crashes(lib):
    so = lib.load()
    # null / inconsistent arguments must come back as ITG_ERR_* (negative), never touch the device
    assert so.itg_bce_logits_fwd(None, 4, ctypes.c_float(1.0), None, None) < 0
    assert so.itg_local_pad_fwd(None, None, 1, 1, 3, 3, 4, 1, 0, None) < 0
    t = lib.Tensor(None, 1, 1, 1, 4, 4, 3, 4)
    assert so.itg_bn_stats(ctypes.byref(t), None, None) < 0
    # the conv family with null tensors / panels / geometry, and a tensor whose pointer is null (the no-gradient-requested
    # shapes a caller can produce: bias None, no weight gradient, no act_out)
    f0 = ctypes.c_float(0.0)
    assert so.itg_conv2d_fwd(None, None, None, None, None, None, None, 0, f0, None, 0, None) < 0
    assert so.itg_conv2d_dgrad(None, None, None, None, None, 0, f0, None, None, 0, None) < 0
    assert so.itg_conv2d_dgrad(ctypes.byref(t), None, None, ctypes.byref(t), None, 0, f0, None, None, 0, None) < 0
    assert so.itg_conv2d_wgrad(None, None, None, None, None, 0, None, 0, None) < 0
    assert so.itg_conv2d_wgrad(ctypes.byref(t), ctypes.byref(t), None, None, None, 0, None, 0, None) < 0
    ok = lib.Tensor(ctypes.c_void_p(64), 1, 1, 1, 4, 4, 3, 4)           # a well-formed descriptor (never dereferenced: the
    assert so.itg_conv2d_dgrad(ctypes.byref(ok), None, None, ctypes.byref(ok), None, 0, f0, None, None, 0, None) < 0   # panel is null)
    assert so.itg_conv2d_wgrad(ctypes.byref(ok), ctypes.byref(ok), None, None, None, 0, None, 0, None) < 0               # geometry is null
    # round 5's entry points: the band halo rows (a band is one 1 x 1-grid image with >= 3 rows; buffer mode needs the buffer),
    # the fused loss head (one-channel logits, a zeroed workspace), the stride-2 Winograd panels
    assert so.itg_band_halo_fill(None, None, None, 1, 1, None) < 0
    assert so.itg_band_halo_fill(ctypes.byref(ok), None, None, 0, 1, None) < 0          # rows from a buffer, no buffer
    assert so.itg_band_halo_fill(ctypes.byref(ok), None, None, 3, 1, None) < 0          # unknown mode
    assert so.itg_band_halo_grad(ctypes.byref(ok), None, None, 1, 0, None) < 0
    assert so.itg_band_rows_get(ctypes.byref(ok), 0, 9, None, None, None) < 0
    assert so.itg_band_interior_copy(ctypes.byref(ok), ctypes.byref(ok), 1, None) < 0   # the band must be two rows shorter
    assert so.itg_logit_loss_grid(None, 0, f0, None, None, None, None) < 0
    assert so.itg_logit_loss_grid(ctypes.byref(ok), 0, f0, ctypes.c_void_p(64), ctypes.byref(ok), ctypes.c_void_p(64), None) < 0   # 3 channels
    one = lib.Tensor(ctypes.c_void_p(64), 1, 1, 1, 4, 4, 1, 4)
    assert so.itg_logit_loss_grid(ctypes.byref(one), 7, f0, ctypes.c_void_p(64), ctypes.byref(one), ctypes.c_void_p(64), None) < 0  # unknown kind
    assert so.itg_logit_loss_grid_workspace() >= 9
    assert so.itg_pack_wino_s2_fwd(None, None, None, 128, 64, 64, None) < 0
    assert so.itg_pack_wino_s2_dgrad(None, None, None, 128, 64, 64, 128, None) < 0
    assert so.itg_pack_wino_s2_size(256, 128) == 25 * 256 * 512 and so.itg_pack_wino_s2_dgrad_size(128, 256) == 25 * 512 * 256
    bad_ld = lib.Tensor(ctypes.c_void_p(64), 1, 1, 1, 4, 4, 3, 3)      # ld not a multiple of 4
    assert so.itg_act_fwd(ctypes.byref(bad_ld), ctypes.byref(bad_ld), 1, ctypes.c_float(0.2), None) == -2


def test_product_has_no_cpu_fallback_and_does_not_import_oracle():
    import subprocess, sys
    code = ("import sys; sys.path.insert(0, %r); import infinite_texture_gans_amd.utils, infinite_texture_gans_amd.engine; "
            "assert not any(m == 'oracle' or m.startswith('oracle.') for m in sys.modules), 'product imported the oracle'; "
            "import torch; from infinite_texture_gans_amd import ops, _lib\n"
            "try:\n    ops.to_grid(torch.zeros(1,3,4,4), 1, 1, True)\n    raise SystemExit('CPU tensor was accepted')\n"
            "except _lib.ItgError: pass") % ROOT
    subprocess.check_call([sys.executable, "-c", code])


def test_struct_layouts_match_the_header(lib, tmp_path):
    """The ctypes mirrors of itg_tensor / itg_conv_geom / itg_bn_bwd_fuse (round 6) have the C structs' sizes and field offsets:
    a C program that includes include/itg.h prints them (gcc is enough - the header is plain C)."""
    import shutil
    import subprocess
    if shutil.which("gcc") is None:
        pytest.skip("gcc not installed")
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "itg.h"\nint main(void) {\n'
                   '  printf("%zu %zu %zu\\n", sizeof(itg_tensor), sizeof(itg_conv_geom), sizeof(itg_bn_bwd_fuse));\n'
                   '  printf("%zu %zu %zu %zu\\n", offsetof(itg_conv_geom, out_stats), offsetof(itg_conv_geom, bn_bwd), '
                   'offsetof(itg_conv_geom, flags), offsetof(itg_conv_geom, wino_v));\n'
                   '  printf("%zu %zu %zu %zu %zu %zu\\n", offsetof(itg_bn_bwd_fuse, x), offsetof(itg_bn_bwd_fuse, ab), '
                   'offsetof(itg_bn_bwd_fuse, mean_rstd), offsetof(itg_bn_bwd_fuse, act), offsetof(itg_bn_bwd_fuse, sums), '
                   'offsetof(itg_bn_bwd_fuse, taken));\n  return 0;\n}\n')
    exe = tmp_path / "layout"
    subprocess.check_call(["gcc", "-std=c99", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)])
    out = subprocess.check_output([str(exe)], text=True).split()
    got = [int(v) for v in out]
    G, F = lib.ConvGeom, lib.BnBwdFuse
    want = [ctypes.sizeof(lib.Tensor), ctypes.sizeof(G), ctypes.sizeof(F),
            G.out_stats.offset, G.bn_bwd.offset, G.flags.offset, G.wino_v.offset,
            F.x.offset, F.ab.offset, F.mean_rstd.offset, F.act.offset, F.sums.offset, F.taken.offset]
    assert got == want, (got, want)


def test_bn_bwd_fuse_is_an_input_gradient_argument_only(lib):
    """itg_conv_geom.bn_bwd (round 6): the forward and the weight gradient reject a geometry that carries it; the input gradient
    validates it (a null BatchNorm input is an argument error, not a crash) and clears `taken` before anything else."""
    so = lib.load()
    f0 = ctypes.c_float(0.0)
    ok = lib.Tensor(ctypes.c_void_p(64), 1, 1, 1, 4, 4, 3, 4)
    fuse = lib.BnBwdFuse(None, None, None, 1, 0.02, None, 7, 0)
    g = lib.ConvGeom(3, 3, 1, 1, 0, bn_bwd=fuse)
    panel = ctypes.c_void_p(64)
    assert so.itg_conv2d_fwd(ctypes.byref(ok), panel, None, None, None, ctypes.byref(ok), ctypes.byref(g), 0, f0, None, 0, None) < 0
    assert so.itg_conv2d_wgrad(ctypes.byref(ok), ctypes.byref(ok), panel, None, ctypes.byref(g), 0, None, 0, None) < 0
    assert so.itg_conv2d_dgrad(ctypes.byref(ok), panel, None, ctypes.byref(ok), None, 0, f0, ctypes.byref(g), None, 0, None) < 0
    assert g.bn_bwd.contents.taken == 0


def test_training_operators_reject_bad_calls_on_the_host(lib):
    """layer norm, Newton-Schulz and Muon entry points: every rejection happens before a launch (there is no GPU in this tier)"""
    so = lib.load()
    f, p = ctypes.c_float, ctypes.c_void_p
    q = p(4096)

    def fwd(x=q, ldx=8, y=q, ldy=8, stat=None, rows=4, c=8, pad=0, dt=0, pdt=0, eps=1e-5, act=0):
        return so.itg_layer_norm_fwd(x, ldx, None, None, y, ldy, stat, rows, c, pad, dt, pdt, f(eps), act, f(0.0), None)

    assert fwd(x=None) == -1 and fwd(y=None) == -1 and fwd(rows=0) == -1 and fwd(c=0) == -1 and fwd(c=(1 << 24) + 1) == -1
    assert fwd(ldx=7) == -1 and fwd(ldy=8, pad=1) == -1 and fwd(pad=-1) == -1 and fwd(dt=3) == -1 and fwd(dt=0, pdt=1) == -1
    assert fwd(dt=1, pdt=2) == -1 and fwd(eps=-1.0) == -1 and fwd(eps=float("nan")) == -1 and fwd(act=3) == -1
    assert fwd(x=p(4098)) == -2 and fwd(dt=1, pdt=1, x=p(4097)) == -2 and fwd(stat=p(4097)) == -2
    assert fwd(rows=1 << 41) == -1 and fwd(rows=1 << 30, ldx=1 << 40) == -1
    assert so.itg_layer_norm_bwd_workspace(0, 4) == -1 and so.itg_layer_norm_bwd_workspace(1000, 10) > 0

    def bwd(stat=q, dx=q, dg=q, ws=q, n=1 << 20, rows=4, c=8, lddx=8):
        return so.itg_layer_norm_bwd(q, 8, q, 8, stat, None, None, dx, lddx, dg, None, 0, rows, c, 0, 0, 0, 0, f(0.0), ws, n, None)

    assert fwd(ldx=9) == -1 and bwd(lddx=9) == -1           # in place at two strides
    assert bwd(stat=None) == -1 and bwd(ws=None) == -4 and bwd(n=7) == -4 and bwd(lddx=4) == -1 and bwd(ws=p(4097)) == -2
    assert bwd(dx=None, dg=None) == 0                       # nothing asked for: nothing launched

    def job(rows=4, cols=8, count=1, reserved=0, io=0, il=8, ist=32, oo=0, ol=8, ost=32):
        return lib.NsJob(rows, cols, count, reserved, io, il, ist, oo, ol, ost)

    def size(j, n=1, dt=0):
        return so.itg_newton_schulz_workspace(ctypes.byref(j) if j is not None else None, n, dt)

    assert size(job()) > 0 and size(job(), dt=1) > 0
    for bad in (job(rows=0), job(cols=0), job(rows=65537), job(count=0), job(reserved=1), job(il=7), job(ol=7), job(io=-1), job(oo=-1),
                job(count=2, ost=31), job(ist=-1), job(il=1 << 62), job(io=(1 << 62)), job(rows=65536, cols=65536, il=65536, ol=65536, count=1 << 30, ost=1 << 40)):
        assert size(bad) == -1
    assert size(None) == -1 and size(job(), n=0) == -1 and size(job(), n=33) == -1 and size(job(), dt=5) == -1
    co = (f * 3)(3.4445, -4.7750, 2.0315)

    def ns(j=job(), n=1, dt=0, g=q, out=q, steps=1, co=co, eps=0.0, ws=q, size=1 << 30):
        return so.itg_newton_schulz(ctypes.byref(j), n, dt, g, out, steps, co, f(eps), ws, size, None)

    assert ns(g=None) == -1 and ns(out=None) == -1 and ns(steps=0) == -1 and ns(steps=17) == -1 and ns(co=None) == -1 and ns(eps=-1.0) == -1
    assert ns(co=(f * 3)(9.0, 0.0, 0.0)) == -1 and ns(co=(f * 3)(float("inf"), 0.0, 0.0)) == -1
    large = job(rows=256, cols=300, il=300, ol=300)
    assert ns(size=size(job()) - 1) == -4 and ns(j=large, size=size(large) - 1) == -4 and size(large) > 4 * 256 * 300
    assert ns(ws=None) == -4 and ns(ws=p(4100)) == -2 and ns(g=p(4098)) == -2

    def muon(j=job(ist=0, ost=0), p_=q, g=q, m=q, e=None, ws=q, size=1 << 30):
        return so.itg_muon_step(ctypes.byref(j), 1, p_, g, m, e, f(0.1), f(0.9), 1, f(0.0), f(0.9), 1, co, f(0.0), ws, size, None)

    assert size(job(rows=1, cols=1, il=1, ist=1, ol=1, ost=1, count=(1 << 24) - 1)) == 16 and size(job(rows=1, cols=1, il=1, ist=1, ol=1, ost=1, count=1 << 24)) == -1
    assert size(job(rows=65, cols=70, il=70, ol=70, ost=4550, count=1 << 23)) == -1 and size(job(rows=65, cols=70, il=70, ol=70, ost=4550, count=(1 << 23) - 1)) == 16
    assert size(job(rows=2, cols=200, il=200, ol=200, ost=400, count=1 << 22)) == -1 and size(job(rows=130, cols=130, il=130, ol=130, ost=16900, count=1 << 21)) == -1

    assert muon(p_=q, g=q) == -1                            # one buffer for two
    q2, q3, q4 = p(1 << 20), p(2 << 20), p(3 << 20)
    assert muon(g=q2, m=q2) == -1 and muon(g=q2, m=q3, e=q3) == -1 and muon(g=q2, m=q3, e=q, ws=q4) == -1
    two = (lib.NsJob * 2)(job(ist=0, ost=0), job(ist=0, ost=0, io=31, oo=31))
    assert so.itg_muon_step(two, 2, q, q2, q3, None, f(0.1), f(0.9), 1, f(0.0), f(0.9), 1, co, f(0.0), q4, 1 << 30, None) == -1      # overlap
    assert muon(p_=None) == -1 and muon(g=None) == -1 and muon(m=None) == -1 and muon(g=q2, m=q3, e=p(4098)) == -2 and muon(g=q2, m=q3, ws=None) == -4
    for bad in (job(count=2), job(il=9), job(io=1, oo=0)):
        assert muon(j=bad, g=q2, m=q3) == -1


def test_training_operators_have_no_cpu_path():
    import torch
    from infinite_texture_gans_amd import ops
    from infinite_texture_gans_amd._lib import ItgError
    x = torch.randn(4, 8)
    for call in (lambda: ops.layer_norm(x), lambda: ops.orthogonalize(x), lambda: ops.MuonPlan([(4, 8)], "cpu"),
                 lambda: ops.layer_norm(ops.GT(x.view(1, 1, 1, 1, 4, 8), 8))):
        with pytest.raises(ItgError):
            call()


ROWS_PROGRAM = r"""
#include "layer_norm_rows.h"
#include <stdio.h>
#include <string.h>
#include <sys/mman.h>
#include <unistd.h>
// gamma ends where readable memory ends: a read behind its c values does not come back
template <typename W> int run(char* end, int c, int pad, int threads, int per) {
  W* gamma = (W*)end - c;
  for (int i = 0; i < c; ++i) { uint32_t b = 0x3f80u + (uint32_t)(i % 97); memcpy(gamma + i, &b, sizeof(W)); }
  const LnV lv = ln_vectors(c, pad, 8);
  int seen = 0;
  for (int i = 0; i < threads * per; ++i) {
    int off, lo, hi;
    ln_place(lv, i, 8, off, lo, hi);
    if (off < 0 || off + 8 > c + pad || lo < 0 || hi > 8) return 1;
    if (hi <= 0) continue;
    Held<W, 8> k;
    memset(&k, 0xff, sizeof(k));
    k.load_first(gamma + off, hi);
    W got[8], want[8];
    memcpy(got, &k, sizeof(got));
    memset(want, 0, sizeof(want));
    memcpy(want, gamma + off, hi * sizeof(W));
    if (memcmp(got, want, sizeof(got))) return 2;
    for (int e = lo; e < hi; ++e) seen += off + e < c;
  }
  return seen == c ? 0 : 3;
}
int main() {
  const size_t page = (size_t)sysconf(_SC_PAGESIZE), room = (16384 * 4 + page - 1) / page * page;
  char* mem = (char*)mmap(0, room + page, PROT_READ | PROT_WRITE, MAP_PRIVATE | MAP_ANONYMOUS, -1, 0);
  if (mem == (char*)MAP_FAILED || mprotect(mem + room, page, PROT_NONE)) return 9;
  for (int c = 8193; c <= 16384; c += c < 8300 || c > 16300 ? 1 : 61)
    for (int pad = 0; pad < 12; ++pad) {
      if (c + pad > 16384 && pad) continue;
      const int a = run<float>(mem + room, c, pad, 1024, 2), b = run<_Float16>(mem + room, c, pad, 1024, 2);
      if (a || b) { printf("%d %d: %d %d\n", c, pad, a, b); return 1; }
    }
  return 0;
}
"""


def test_layer_norm_parameters_are_read_to_their_last_value(tmp_path):
    """long 16-bit rows with padding: the vector of gamma and beta that ends in the padding is read value by value.  The kernel's own
    placement and load, compiled for the host, over a gamma behind whose last value no memory can be read."""
    import shutil
    import subprocess
    import __graft_entry__ as g
    if shutil.which(g.HIPCC) is None:
        pytest.skip("hipcc not installed")
    src, exe = tmp_path / "rows.hip", tmp_path / "rows"
    src.write_text(ROWS_PROGRAM)
    subprocess.check_call([g.HIPCC, "-x", "hip", "--cuda-host-only", "-O1", "-std=c++17", "-I", g.CSRC, "-I", os.path.join(ROOT, "include"), str(src),
                           "-o", str(exe)])
    assert subprocess.run([str(exe)]).returncode == 0
    with open(os.path.join(g.CSRC, "layer_norm.hip")) as f:      # the kernels' only other whole-vector reads of gamma and beta: ln_param's, ln_at's
        kernel = f.read()
    assert kernel.count(".load_first((const W*)p.") == 2 and ".load((const W*)" not in kernel


def test_layer_norm_workspace_is_what_the_backward_pass_writes(lib):
    """a share of dw | db per workgroup that makes one, not per row: with 1024 rows of 40000 / 2^20 / 2^24 channels 312 MiB, 8 GiB and
    128 GiB would be asked for if every row could leave a share, while about 2048 * 256 vectors of channels are swept"""
    size = lib.fn("itg_layer_norm_bwd_workspace")
    for c in (16392, 40000, 1 << 20, 1 << 24):
        for rows in (1, 7, 96, 1024, 5000, 1 << 20):
            # shares: one per 8 rows, and no more than 2048 / ceil(vectors / 256) + 1, with vectors of 4 (fp32) or 8 values
            most = max(min(-(-rows // 8), 2048 // -(-(-(-c // V)) // 256) + 1) for V in (4, 8))
            assert 0 < size(rows, c) <= most * 2 * c, (rows, c)
    assert size(1024, 1 << 24) * 4 <= 256 << 20 and size(1024, 40000) * 4 <= 64 << 20
    for c, groups in ((9001, 256), (16384, 256), (4000, 512), (52, 1024), (3, 256)):      # rows in registers: workgroups of 1024, 512 and 256 threads, the last with 16 or 64 rows a turn and four turns at least
        assert size(1 << 16, c) == groups * 2 * c, c
    assert size(1, 52) == 2 * 52 and size(1 << 40, 1) > 0 and size(0, 8) == -1 and size(8, (1 << 24) + 1) == -1


def test_matrix_sizes_past_32_bits_are_refused():
    """The jobs count rows, columns and matrices in 32 bits: a size that does not fit would be cut to another one (2^32 + 4 rows to 4,
    and the rest of the result left as it was).  The sizes are looked at before the device, so this runs without one: the tensors
    are expanded from one value."""
    import torch
    from infinite_texture_gans_amd import ops
    from infinite_texture_gans_amd._lib import ItgError
    one = torch.zeros(1, 1, 1)
    for shape in ((2 ** 32 + 3, 1, 1), (2 ** 31, 1, 1), (1, 2 ** 32 + 4, 3), (1, 3, 2 ** 32 + 4), (2 ** 20, 2 ** 12 + 1, 1, 1)):
        with pytest.raises(ItgError, match="matrices"):
            ops.orthogonalize(one.expand(*shape))
    for shapes in ([(2 ** 32 + 4, 8)], [(8, 2 ** 32 + 4)], [(4, 8), (65537, 1)], [(-1, 4)]):
        with pytest.raises(ItgError, match="rows and columns"):
            ops.MuonPlan(shapes, "cuda")
    with pytest.raises(ItgError, match="offset"):
        ops.MuonPlan([(4, 8)], "cuda", offset=2 ** 61)


def test_layer_norm_padding_past_32_bits_is_refused():
    """the padding of a pixel is counted in 32 bits too; looked at before the device"""
    import torch
    from infinite_texture_gans_amd import ops
    from infinite_texture_gans_amd._lib import ItgError
    one = torch.zeros(1, 1, 1, 1, 1, 1)
    for ld in (2 ** 32 + 8, 2 ** 24 + 9):
        with pytest.raises(ItgError, match="values a row"):
            ops.layer_norm(ops.GT(one.expand(1, 1, 1, 1, 1, ld), 8))
    with pytest.raises(ItgError, match="channels"):
        ops.layer_norm(ops.GT(one.expand(1, 1, 1, 1, 1, 8), 9))


def test_muon_buffers_that_share_values_are_refused(lib):
    """param, gradient, momentum and EMA of a step are read and written by different workgroups: matrices of two of them that share a
    value have no order.  Buffers that only interleave, their matrices beside each other, are fine (ws None: the check behind)."""
    so = lib.load()
    f, p = ctypes.c_float, ctypes.c_void_p
    co = (f * 3)(3.4445, -4.7750, 2.0315)

    def step(at, jobs=((0, 4, 8),)):
        arr = (lib.NsJob * len(jobs))(*[lib.NsJob(r, c, 1, 0, o, c, 0, o, c, 0) for o, r, c in jobs])
        return so.itg_muon_step(arr, len(jobs), *[p(4096 + 4 * a) if a is not None else None for a in at], f(0.1), f(0.9), 1, f(0.0), f(0.9), 1, co, f(0.0),
                                None, 0, None)

    assert step((0, 32, 64, 96)) == -4 and step((96, 64, 32, 0)) == -4 and step((0, 32, 64, None)) == -4
    for other in range(1, 4):
        for shift in (1, 31, -1, -31):
            at = [1000, 2000, 3000, 4000]
            for k in range(4):
                if k != other:
                    at[other] = at[k] + shift
                    assert step(at) == -1, at
            at[other] = 1000 * (other + 1)
    # two matrices with room between them for the other buffers' matrices
    two = ((0, 4, 8), (200, 4, 8))
    assert step((0, 32, 64, 96), two) == -4 and step((0, 32, 64, 190), two) == -1 and step((0, 231, 400, 800), two) == -1 and step((0, 232, 400, 800), two) == -4
