"""Every form in which the 16-bit linear runs a product -- kernel, tiling, whole or in slices of K -- against the formula in
float64: the three products of a plain linear's training pass (its gradient dh is dy itself), and the fuller epilogues.
Tolerances are test_gpu_dense.py's. That these shapes reach every form is checked on the CPU (test_dense_forms.py)."""
import pytest
import torch

from conftest import sub
from test_gpu_dense import check, formula, make

pytestmark = pytest.mark.gpu

fd = sub("enhancers.fused_dense")

# rows, n, k of y = x w^T + b with dx and dw: odd sizes on every side, then widths that need no copies
PLAIN = [(1, 2, 3), (1, 7961, 1), (340, 1, 5684), (8492, 1087, 3), (8627, 1, 4794), (5525, 526, 556), (2030, 274, 7805),
         (278, 3774, 4477), (1451, 6318, 868), (781, 2743, 5481), (5996, 5125, 386), (8757, 395, 904), (8029, 7214, 411),
         (36, 881, 12224), (3124, 1971, 4938), (8685, 271, 12992), (13352, 10875, 266), (5994, 2, 4727), (1247, 45, 10699),
         (55, 13855, 1229), (12562, 145, 12480), (5152, 2048, 2048), (1560, 6912, 1280), (128, 64, 8192), (2000, 320, 320)]

# rows, n, k, groups of y = resid + gate act(x w^T + b): even n runs in the accumulators with one gate row, through float32
# rows in LDS where a tile has rows of two groups; odd n through the same, value by value
FULL = [(13209, 904, 672, 7), (9849, 1158, 827, 7), (9961, 1200, 912, 7), (3075, 3875, 904, 5), (11228, 808, 1496, 7),
        (658, 13690, 1563, 7), (10906, 344, 489, 7), (11081, 333, 466, 7), (10920, 264, 418, 7), (11074, 261, 464, 7),
        (8315, 136, 838, 5), (8491, 129, 776, 7), (258, 16, 96, 3), (264, 18, 51, 3), (8100, 32, 406, 5), (7637, 35, 371, 7)]
TYPES = (torch.bfloat16, torch.float16)


@pytest.mark.parametrize("i", range(len(PLAIN)))
def test_plain_linear_and_gradients(native, i):
    rows, n, k = PLAIN[i]
    print(f"case plain linear rows={rows} n={n} k={k}", flush=True)
    t = make(rows, n, k, TYPES[i % 2], i % 3 == 0, False, 0, i)
    want = formula(t, None)
    names = [s for s in ("x", "w", "b") if t[s] is not None]
    leaf = {s: t[s].detach().clone().requires_grad_() for s in names}
    y = fd.dense(leaf["x"], leaf["w"], leaf.get("b"))
    grads = torch.autograd.grad(y, [leaf[s] for s in names], t["dy"], retain_graph=True)
    check(y.detach(), want["y"], "y")
    for s, g in zip(names, grads):
        check(g, want["d" + s], "d" + s)
    for s in names:                                                # one gradient at a time is the same gradient
        assert torch.equal(torch.autograd.grad(y, leaf[s], t["dy"], retain_graph=True)[0], grads[names.index(s)]), s


@pytest.mark.parametrize("i", range(len(FULL)))
def test_fuller_epilogues(native, i):
    rows, n, k, groups = FULL[i]
    act = ("gelu_tanh", "gelu", "silu", "relu")[i // 2 % 4]
    for g in (1, groups):
        print(f"case epilogue rows={rows} n={n} k={k} groups={g} {act}", flush=True)
        t = make(rows, n, k, TYPES[i // 2 % 2], True, True, g, i)
        y = fd.dense(t["x"], t["w"], t["b"], act, t["r"], t["g"])
        leaf = [t[s].detach().clone().requires_grad_() for s in ("x", "w", "b", "r", "g")]
        z = fd.dense(leaf[0], leaf[1], leaf[2], act, leaf[3], leaf[4])         # keeps the pre-activations besides
        want = formula(t, act)
        check(y, want["y"], "y")
        check(z.detach(), want["y"], "y with h kept")
        for s, got in zip("xwbrg", torch.autograd.grad(z, leaf, t["dy"])):
            check(got, want["d" + s], "d" + s)


@pytest.mark.parametrize("rows,n,k", [(70, 96, 200), (600, 333, 129)])
def test_operands_of_other_strides_in_training(native, rows, n, k):
    # a weight whose columns are two values apart, rows of x and of dy that are all the same memory: each gives the
    # gradients of its copy
    for dtype in TYPES:
        t = make(rows, n, k, dtype, False, False, 0, rows)
        wide = torch.empty(n, 2 * k, device="cuda", dtype=dtype)
        wide[:, ::2] = t["w"]
        forms = {"w": (t["x"], wide[:, ::2], t["dy"]), "x": (t["x"][:1].expand(rows, k), t["w"], t["dy"]),
                 "dy": (t["x"], t["w"], t["dy"][:1].expand(rows, n))}
        for name, (x, w, dy) in forms.items():
            out = []
            for a, b, d in ((x, w, dy), (x.contiguous(), w.contiguous(), dy.contiguous())):
                a, b = a.detach().requires_grad_(), b.detach().requires_grad_()
                y = fd.dense(a, b)
                out.append((y.detach(), *torch.autograd.grad(y, (a, b), d)))
            same = dict(t, x=x, w=w, dy=dy)
            want = formula(same, None)
            for got in out:
                for what, v in zip(("y", "dx", "dw"), got):
                    check(v, want[what], (name, what))


@pytest.mark.parametrize("rows", [1, 37, 500])
def test_one_gate_row_a_row(native, rows):
    t = make(rows, 264, 136, torch.bfloat16, True, True, rows, rows)
    want = formula(t, "gelu")
    leaf = [t[s].detach().clone().requires_grad_() for s in ("x", "w", "b", "r", "g")]
    y = fd.dense(leaf[0], leaf[1], leaf[2], "gelu", leaf[3], leaf[4])
    check(y.detach(), want["y"], "y")
    for s, got in zip("xwbrg", torch.autograd.grad(y, leaf, t["dy"])):
        check(got, want["d" + s], "d" + s)
