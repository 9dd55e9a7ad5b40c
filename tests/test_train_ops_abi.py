"""The training-step operators' C ABI answers malformed and unhandled calls without touching a GPU, and sizes its
workspaces by the rules its header states (CPU only: no kernel is launched)."""
import array
import ctypes

import pytest
import torch

from conftest import sub

native = sub("_native")


def buffer():
    buf = ctypes.create_string_buffer(8192)
    return buf, (ctypes.addressof(buf) + 255) // 256 * 256


def test_layer_norm_argument_checks():
    lib = native.lib()
    keep, p = buffer()
    ln = lambda x=p, ldx=64, dt=1, pdt=1, rpg=4, M=4, K=64, y=p: lib.wf_layer_norm(          # noqa: E731
        x, ldx, dt, None, None, pdt, 0, rpg, 1e-5, y, None, M, K, None)
    assert ln(dt=3) == native.EUNSUPPORTED and ln(dt=1, pdt=0) == native.EUNSUPPORTED
    assert ln(K=32769) == native.EUNSUPPORTED and "32768" in native.last_error()
    assert ln(rpg=1, M=65536) == native.EUNSUPPORTED
    assert ln(rpg=3) == native.EINVAL and ln(M=-1) == native.EINVAL and ln(K=0) == native.EINVAL and ln(rpg=0) == native.EINVAL
    assert ln(x=None) == native.EINVAL and ln(y=None) == native.EINVAL and ln(ldx=-1) == native.EINVAL
    assert ln(M=0) == native.OK
    bwd = lambda ws, n: lib.wf_layer_norm_bwd(p, 64, p, 64, 1, None, 1, 0, 4, p, p, p, p, 4, 64, ws, n, None)  # noqa: E731
    assert bwd(None, 0) == native.EINVAL and "workspace" in native.last_error()
    assert bwd(p, 8) == native.EINVAL
    need = ctypes.c_int64()
    for M, rpg in ((4, 4), (100000, 100000), (4096, 2), (65535, 1)):
        assert lib.wf_layer_norm_bwd_workspace(M, 5120, rpg, 1, ctypes.byref(need)) == native.OK
        rows = need.value // (2 * 5120 * 4)                      # rows of partial sums: one a group at least, few over all
        assert M // rpg <= rows <= max(M // rpg, 256) and need.value % (2 * 5120 * 4) == 0
    assert lib.wf_layer_norm_bwd_workspace(5, 64, 2, 1, ctypes.byref(need)) == native.EINVAL


def test_dense_argument_checks():
    lib = native.lib()
    keep, p = buffer()

    def dense(x=p, xr=64, xc=1, w=p, wr=64, wc=1, dt=1, M=4, N=8, K=64, bias=None, bdt=1, act=0, gate=None, gdt=1, rpg=4,
              res=None, rr=8, y=p, h=None, ws=None, n=0):
        return lib.wf_dense(x, xr, xc, w, wr, wc, dt, M, N, K, bias, bdt, act, gate, gdt, rpg, res, rr, y, h, ws, n, None)
    assert dense(dt=2) == native.EUNSUPPORTED and dense(K=(1 << 20) + 1) == native.EUNSUPPORTED
    assert dense(M=(1 << 24) + 1) == native.EUNSUPPORTED
    assert dense(M=-1) == native.EINVAL and dense(K=0) == native.EINVAL and dense(xr=-64) == native.EINVAL
    assert dense(act=5) == native.EINVAL and dense(act=-1) == native.EINVAL
    assert dense(bias=p, bdt=0) == native.EINVAL and dense(gate=p, gdt=0) == native.EINVAL
    assert dense(gate=p, rpg=0) == native.EINVAL and dense(res=p, rr=-1) == native.EINVAL
    assert dense(x=None) == native.EINVAL and dense(w=None) == native.EINVAL and dense(y=None) == native.EINVAL
    assert dense(x=p + 1) == native.EINVAL and dense(bias=p + 2, bdt=2) == native.EINVAL and "aligned" in native.last_error()
    assert dense(M=0) == native.OK and dense(N=0) == native.OK
    # a product that runs in slices asks for its workspace
    need = ctypes.c_int64()
    assert lib.wf_dense_workspace(p, 5120, 1, p, 5120, 1, 1, 256, 5120, 5120, 0, ctypes.byref(need)) == native.OK
    assert need.value > 0 and need.value % (256 * 5120 * 4) == 0
    assert dense(xr=5120, wr=5120, M=256, N=5120, K=5120) == native.EINVAL and "workspace" in native.last_error()
    # whole tiles for the chip: none; an odd row: its operand's copy
    assert lib.wf_dense_workspace(p, 5120, 1, p, 5120, 1, 1, 4096, 5120, 5120, 0, ctypes.byref(need)) == native.OK
    assert need.value == 0
    assert lib.wf_dense_workspace(p, 5121, 1, p, 5120, 1, 1, 4096, 5120, 5120, 0, ctypes.byref(need)) == native.OK
    assert need.value == 4096 * 5120 * 2
    # across K both operands are read as they lie; a fuller epilogue then goes through float32 sums
    across = (p, 1, 4096, p, 1, 5120, 1, 4096, 5120, 5120)
    assert lib.wf_dense_workspace(*across, 0, ctypes.byref(need)) == native.OK and need.value == 0
    assert lib.wf_dense_workspace(*across, 1, ctypes.byref(need)) == native.OK and need.value == 4096 * 5120 * 4
    assert lib.wf_dense_workspace(*across, 8, ctypes.byref(need)) == native.EINVAL

    def bwd(M=4, N=8, K=64, act=0, gate=None, h=None, dy=p, dx=None, dw=None, db=None, dg=None, ws=None, n=0, rpg=4, dt=1):
        return lib.wf_dense_bwd(p, 64, p, 64, 1, dy, 8, h, dt, act, gate, 1, rpg, M, N, K, dx, dw, db, 1, dg, ws, n, None)
    assert bwd(M=(1 << 20) + 4) == native.EUNSUPPORTED and bwd(dt=2) == native.EUNSUPPORTED
    assert bwd(rpg=3) == native.EINVAL and bwd(act=9) == native.EINVAL and bwd(dy=None) == native.EINVAL
    assert bwd(act=1, dx=p) == native.EINVAL                        # a slope without h
    assert bwd(dg=p, h=p) == native.EINVAL                          # a gate's gradient without the gate
    assert bwd(db=p) == native.EINVAL and "workspace" in native.last_error()
    assert bwd(M=0) == native.OK


def test_adamw_argument_checks():
    lib = native.lib()
    keep, p = buffer()

    def step(rows=((p, p, 300),), dt=2, bits=32, m=p, v=p, ms=None, vs=None, blocks=2, t=1, lr=1e-3, b1=0.9, b2=0.99, eps=1e-8):
        table = array.array("q", [x for r in rows for x in r])
        return lib.wf_adamw(table.buffer_info()[0] if rows else None, len(rows), dt, bits, m, v, ms, vs, blocks, t, lr, b1, b2,
                            eps, 0.0, None)
    assert step(dt=3) == native.EUNSUPPORTED and step(bits=16) == native.EUNSUPPORTED
    assert step(t=0) == native.EINVAL and step(b1=1.0) == native.EINVAL and step(eps=-1.0) == native.EINVAL
    assert step(blocks=1) == native.EINVAL and "blocks" in native.last_error()
    assert step(rows=((p, p, -1),), blocks=0) == native.EINVAL
    assert step(rows=((0, p, 300),)) == native.EINVAL and step(rows=((p + 2, p, 300),)) == native.EINVAL
    assert step(m=None) == native.EINVAL and step(m=p + 4) == native.EINVAL
    assert step(bits=8) == native.EINVAL                            # 8-bit moments without scales
    assert step(rows=(), blocks=0) == native.OK and step(rows=((0, 0, 0),), blocks=0) == native.OK
    assert lib.wf_adamw_values(None, None, None, None, 0, None, None, None) == native.OK
    assert lib.wf_adamw_values(None, p, p, p, 1, p, p, None) == native.EINVAL


def test_cpu_tensors_are_not_the_kernels_case():
    x, w = torch.randn(4, 64), torch.randn(8, 64)
    assert sub("enhancers.fused_norm").layer_norm(x, x[0]) is None
    assert sub("enhancers.fused_dense").dense(x.bfloat16(), w.bfloat16()) is None
    fa = sub("enhancers.fused_adamw")
    with pytest.raises(ValueError, match="GPU"):
        fa.adamw_step([x], [x.clone()], fa.adamw_state([x]), 1)


def test_transformed_tensors_are_not_the_kernels_case():
    ops = sub("enhancers.operands")
    x = torch.randn(3, 4)
    seen = []
    torch.func.vmap(lambda t: seen.append(ops.plain(t.device, t)) or t)(x)
    torch.func.grad(lambda t: seen.append(ops.plain(x.device, x)) or t.sum())(x)      # a bystander inside a transform
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        seen += [ops.plain(x.device, dual), not ops.plain(x.device, x)]
    seen += [ops.plain(x.device, torch.nn.Buffer(x) if hasattr(torch.nn, "Buffer") and type(torch.nn.Buffer(x)) is not
                       torch.Tensor else torch._neg_view(x)), ops.plain(torch.device("meta"), x)]
    assert seen == [False] * len(seen) and len(seen) == 6
    assert ops.plain(x.device, x, None, torch.nn.Parameter(x))


def test_gradients_that_are_more_than_memory_are_refused():
    ops = sub("enhancers.operands")
    x = torch.randn(3, 4)
    assert ops.gradient(x) is x and torch.equal(ops.gradient(torch._neg_view(x)), -x)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        assert ops.gradient(x) is x
        with pytest.raises(RuntimeError, match="gradient"):
            ops.gradient(dual)
    with pytest.raises(RuntimeError, match="gradient"):
        torch.func.vmap(lambda t: ops.gradient(t))(x)
    named = x.as_subclass(type("Named", (torch.Tensor,), {}))
    assert type(ops.gradient(named)) is torch.Tensor and ops.gradient(named).data_ptr() == x.data_ptr()

    class Own(torch.Tensor):
        @classmethod
        def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
            return NotImplemented
    with pytest.raises(RuntimeError, match="Own"):
        ops.gradient(torch.Tensor._make_wrapper_subclass(Own, (3, 4)))


def test_traces_are_not_the_kernels_case():
    from torch.fx.experimental.proxy_tensor import make_fx
    ops = sub("enhancers.operands")
    x, seen = torch.randn(3, 4), []

    def ask(t):
        seen.append(ops.plain(x.device, x))
        return t * 2
    torch.jit.trace(ask, (x,), check_trace=False)
    make_fx(ask)(x)
    make_fx(ask, tracing_mode="fake")(x)
    assert seen == [False] * 3 and ops.plain(x.device, x)
    from torch.utils.flop_counter import FlopCounterMode       # a mode that watches, but records no program
    with FlopCounterMode(display=False):
        assert ops.plain(x.device, x)


def test_rows_of_no_values():
    ops = sub("enhancers.operands")
    for shape, rows in (((2, 5, 0), 10), ((0,), 1), ((3, 0), 3), ((0, 4, 0), 0)):
        assert ops.rows_of(torch.empty(shape), 0).shape == (rows, 0)
    assert ops.rows_of(torch.empty(2, 5, 3), 3).shape == (10, 3) and ops.rows_of(torch.empty(0, 5, 3), 3).shape == (0, 3)
