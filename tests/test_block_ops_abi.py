"""The C ABI of the gated block's operators answers malformed and unhandled calls without touching a GPU, and sizes its workspaces by
the rules its header states (CPU only: no kernel is launched)."""
import array
import ctypes
import os
import re

import pytest
import torch

from conftest import ROOT, sub

native = sub("_native")


def buffer():
    buf = ctypes.create_string_buffer(8192)
    return buf, (ctypes.addressof(buf) + 255) // 256 * 256


def test_block_norm_struct_is_the_headers():
    text = open(os.path.join(ROOT, "include", "weightferry.h")).read()
    body = re.search(r"typedef struct \{([^}]*)\} wf_block_norm;", text).group(1)
    names = [n.strip() for line in body.split(";") for n in re.sub(r"^\s*\w+\s", "", line.strip() + " ", count=1).split(",")]
    assert [f for f, _ in native.BlockNorm._fields_] == [n for n in names if n]
    assert ctypes.sizeof(native.BlockNorm) == 7 * 4 + 2 * 4 + 4 + 3 * 8         # (4 bytes of padding before the 64-bit ones)


def test_block_norm_argument_checks():
    lib = native.lib()
    keep, p = buffer()

    def q(**changed):
        fields = dict(dt=1, post=1, norm=1, plus_one=0, post_weight_dt=1, gate_dt=1, weight_dt=1, scale=1.0, eps=1e-6, groups=2,
                      gate_groups=2, weight_groups=1)
        return native.BlockNorm(**{**fields, **changed})

    def fwd(s=None, x=p, xr=64, h=p, hr=64, y=p, M=4, K=64):
        s = q() if s is None else s
        return lib.wf_block_norm_fwd(ctypes.addressof(s), x, xr, h, hr, None, None, None, None, None, y, None, M, K, None)
    assert fwd(M=0) == native.OK
    for bad in (dict(post=3), dict(norm=0), dict(norm=3), dict(post=-1), dict(groups=0), dict(groups=3), dict(gate_groups=4),
                dict(weight_groups=0)):
        assert fwd(q(**bad)) == native.EINVAL, bad
    for bad in (dict(dt=3), dict(gate_dt=0), dict(weight_dt=0), dict(post_weight_dt=5)):
        assert fwd(q(**bad)) == native.EUNSUPPORTED, bad
    assert fwd(K=16385) == native.EUNSUPPORTED and "32768" in native.last_error()
    assert fwd(q(dt=2, post_weight_dt=2, gate_dt=2, weight_dt=2), K=8193) == native.EUNSUPPORTED
    assert fwd(q(groups=65536, gate_groups=1), M=65536) == native.EUNSUPPORTED
    assert fwd(x=None) == native.EINVAL and fwd(y=None) == native.EINVAL and fwd(xr=-1) == native.EINVAL and fwd(K=0) == native.EINVAL
    assert lib.wf_block_norm_fwd(None, p, 64, p, 64, None, None, None, None, None, p, None, 4, 64, None) == native.EINVAL
    s = q()
    bwd = lambda ws, n, stats=p, dy=p: lib.wf_block_norm_bwd(ctypes.addressof(s), p, 64, p, 64, None, None, None, None, 0, dy, 64,   # noqa: E731
                                                             stats, p, p, None, p, p, None, 4, 64, ws, n, None)
    assert bwd(None, 0) == native.EINVAL and "workspace" in native.last_error()
    assert bwd(p, 8) == native.EINVAL and bwd(p, 8192, stats=None) == native.EINVAL and bwd(p, 8192, dy=None) == native.EINVAL
    need = ctypes.c_int64()
    for M, groups in ((4, 2), (16384, 1), (5152, 2), (65535, 65535)):
        s = q(groups=groups)
        sizes = []
        for sums in range(5):
            assert lib.wf_block_norm_bwd_workspace(ctypes.addressof(s), M, 5120, sums, ctypes.byref(need)) == native.OK
            sizes.append(need.value)
        rows = sizes[1] // (5120 * 4)                              # rows of partial sums: one a group at least, few over all
        assert sizes == [i * sizes[1] for i in range(5)] and groups <= rows <= max(groups, 512)
    assert lib.wf_block_norm_bwd_workspace(ctypes.addressof(s), 4, 64, 5, ctypes.byref(need)) == native.EINVAL


def test_gated_dense_argument_checks():
    lib = native.lib()
    keep, p = buffer()

    def gated(x=p, xr=64, xc=1, w=p, wr=64, wc=1, dt=1, M=4, N=8, K=64, bias=None, bdt=1, act=3, y=p, kept=None, ws=None, n=0):
        return lib.wf_gated_dense(x, xr, xc, w, wr, wc, dt, M, N, K, bias, bdt, act, y, kept, ws, n, None)
    assert gated(dt=2) == native.EUNSUPPORTED and gated(K=(1 << 20) + 1) == native.EUNSUPPORTED
    assert gated(M=(1 << 20) + 1) == native.EUNSUPPORTED and gated(N=(1 << 19) + 1) == native.EUNSUPPORTED
    assert gated(M=-1) == native.EINVAL and gated(K=0) == native.EINVAL and gated(xr=-64) == native.EINVAL
    assert gated(act=5) == native.EINVAL and gated(act=-1) == native.EINVAL and gated(bias=p, bdt=0) == native.EINVAL
    assert gated(x=None) == native.EINVAL and gated(w=None) == native.EINVAL and gated(y=None) == native.EINVAL
    assert gated(x=p + 1) == native.EINVAL and gated(bias=p + 2, bdt=2) == native.EINVAL and gated(kept=p + 1) == native.EINVAL
    assert gated(M=0) == native.OK and gated(N=0) == native.OK
    assert gated(M=256, N=2560, K=5120, xr=5120, wr=5120) == native.EINVAL and "workspace" in native.last_error()

    def bwd(dy=p, kept=p, dt=1, act=3, M=4, N=8, K=64, dx=p, dw=p, db=None, bdt=1, ws=None, n=0):
        return lib.wf_gated_dense_bwd(p, 64, p, 64, 1, dy, 8, kept, dt, act, M, N, K, dx, dw, db, bdt, ws, n, None)
    assert bwd() == native.EINVAL and "workspace" in native.last_error()
    assert bwd(dy=None) == native.EINVAL and bwd(kept=None) == native.EINVAL and bwd(db=p, bdt=0) == native.EINVAL
    assert bwd(M=0) == native.OK and bwd(dt=0, act=9) == native.EINVAL and bwd(dt=2) == native.EUNSUPPORTED
    need = ctypes.c_int64()
    assert lib.wf_gated_dense_bwd_workspace(p, 64, p, 64, 1, 1, 100, 9, 64, 1, 1, 0, ctypes.byref(need)) == native.OK
    assert need.value >= 100 * 24 * 2                              # [dg du]: 18 values up to 24
    assert lib.wf_gated_dense_bwd_workspace(p, 64, p, 64, 1, 1, 100, 9, 64, 0, 0, 0, ctypes.byref(need)) == native.OK
    assert need.value == 0


def test_muon_argument_checks():
    lib = native.lib()
    keep, p = buffer()
    abc = (ctypes.c_double * 3)(3.4445, -4.7750, 2.0315)
    table = array.array("q", [p, p, p])

    def muon(t=table.buffer_info()[0], count=1, rows=8, cols=9, dt=1, mu=0.9, keep_=1.0, rate=0.1, steps=5, c=abc, eps=1e-7, ws=p, n=8192):
        return lib.wf_muon(t, count, rows, cols, dt, mu, 1, keep_, rate, steps, c, eps, ws, n, None)
    assert muon(count=0) == native.OK and muon(rows=0) == native.OK and muon(cols=0) == native.OK
    assert muon(dt=3) == native.EUNSUPPORTED and muon(rows=16385, cols=16385) == native.EUNSUPPORTED
    assert muon(rows=8, cols=(1 << 20) + 1) == native.EUNSUPPORTED and muon(rows=1 << 20, cols=1100) == native.EUNSUPPORTED
    for bad in (dict(count=-1), dict(rows=-1), dict(steps=0), dict(steps=33), dict(c=None), dict(mu=1.0), dict(mu=-0.1), dict(eps=0.0),
                dict(keep_=float("nan")), dict(rate=float("inf")), dict(t=None), dict(ws=None), dict(n=8), dict(ws=p + 8)):
        assert muon(**bad) == native.EINVAL, bad
    assert muon(c=(ctypes.c_double * 3)(4.0, 0.0, 0.0)) == native.EINVAL and "coefficients" in native.last_error()
    assert muon(c=(ctypes.c_double * 3)(float("nan"), 0.0, 0.0)) == native.EINVAL
    for bad in ([0, p, p], [p, 0, p], [p + 1, p, p], [p, p + 1, p], [p, p, p + 2]):
        odd = array.array("q", bad)
        assert muon(t=odd.buffer_info()[0]) == native.EINVAL and "matrix 0" in native.last_error(), bad
    assert lib.wf_orthogonalize(table.buffer_info()[0], 1, 8, 9, 1, 5, abc, 0.0, p, 8192, None) == native.EINVAL
    need = ctypes.c_int64()
    ask = lambda count, rows, cols: (lib.wf_muon_workspace(count, rows, cols, ctypes.byref(need)), need.value)        # noqa: E731
    assert ask(0, 8, 9) == (native.OK, 0) and ask(3, 0, 9) == (native.OK, 0)
    # X twice and its remainder, A and B, in float16; a batch is no larger than fills the chip
    rc, one = ask(1, 13824, 5120)
    assert rc == native.OK and one >= (3 * 13824 * 5120 + 2 * 5120 * 5120) * 2 and ask(9, 13824, 5120)[1] == one
    assert ask(128, 64, 64)[1] == ask(1000, 64, 64)[1] > 0
    assert lib.wf_muon_workspace(1, 8, 9, None) == native.EINVAL


def test_python_refuses_before_the_library(monkeypatch):
    fm, fn, fd = (sub(f"enhancers.{n}") for n in ("fused_muon", "fused_norm", "fused_dense"))
    x, w = torch.zeros(4, 8), torch.zeros(6, 8)
    assert fn.residual_norm(x, x) is None and fn.rms_norm(x) is None and fd.gated_dense(x.bfloat16(), w.bfloat16()) is None
    assert fm.orthogonalize(x) is None
    for bad in (dict(steps=0), dict(coefficients=(1.0, 2.0)), dict(coefficients=(9.0, 0.0, 0.0)), dict(eps=-1.0)):
        with pytest.raises(ValueError):
            fm.orthogonalize(x, **bad)
    with pytest.raises(ValueError):
        fm.muon_step([x], [x], fm.muon_momenta([x]))                # not on a GPU
    with pytest.raises(ValueError):
        fn.residual_norm(x, x, norm="none")
