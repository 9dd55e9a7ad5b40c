"""The GPU tests' shapes reach every form that the 16-bit linear's plan can give a product (CPU only: wf_dense_plan launches
nothing), so that a change of the plan's time model cannot leave a kernel untested unseen."""
import ctypes
import math
import random

from conftest import sub
from test_gpu_dense_forms import FULL, PLAIN

native = sub("_native")
ROWS, ALONG, FULL_EPILOGUE, W_ACROSS, ACROSS = range(5)
BLOCK_ROWS = (256, 256, 256, 128, 128, 128, 64, 32)                # of the tilings


def plan(M, N, K, x="along", w="along", epilogue=0, x_row=None, w_row=None):
    """(kernel, tiling, in slices), and how the operands get there"""
    at, out = 1 << 20, (ctypes.c_int * 5)()
    xs = (x_row or K, 1) if x == "along" else (1, x_row or M)
    ws = (w_row or K, 1) if w == "along" else (1, w_row or N)
    assert native.lib().wf_dense_plan(at, *xs, at, *ws, 1, M, N, K, epilogue, out) == native.OK, native.last_error()
    return (out[0], out[1], out[2] > 1), tuple(out[3:])


def training(rows, n, k):
    """The products of a plain linear and its gradients."""
    return (plan(rows, n, k), plan(rows, k, n, w="across"), plan(n, k, rows, x="across", w="across"))


def sizes(rng):
    return rng.choice([int(round(math.exp(rng.uniform(0, math.log(14000))))), 8 * rng.randint(1, 1700),
                       64 * rng.randint(1, 216)])


def test_plain_products():
    rng = random.Random(3)
    possible = {p[0] for _ in range(20000) for p in training(sizes(rng), sizes(rng), sizes(rng))}
    reached = {p[0] for s in PLAIN for p in training(*s)}
    assert possible <= reached, sorted(possible - reached)
    assert {f for f, _, _ in reached} == {ROWS, ALONG, W_ACROSS, ACROSS}
    # operands as they lie and copied, in either order
    assert {h for s in PLAIN for p in training(*s) for h in p[1]} >= {0, 1, 2, 3}
    # float16 and bfloat16 (every second shape) each see every kernel
    for first in (0, 1):
        assert {p[0][0] for s in PLAIN[first::2] for p in training(*s)} == {ROWS, ALONG, W_ACROSS, ACROSS}


def test_epilogues():
    reached = {}
    for rows, n, k, groups in FULL:
        (form, tiling, _), _ = plan(rows, n, k, epilogue=5)
        assert form == FULL_EPILOGUE and rows % groups == 0
        spans = (rows // groups) % BLOCK_ROWS[tiling] != 0
        reached.setdefault(tiling, set()).add((n % 8 == 0, spans))
    # each tiling with rows of whole 16-byte runs, a tile that spans two groups among them, and with odd rows
    assert reached.keys() == set(range(8)), reached
    assert all({(True, True), (False, True)} <= v for v in reached.values()), reached


def test_plan_answers():
    out = (ctypes.c_int * 5)()
    ask = lambda *a: native.lib().wf_dense_plan(*a)                                            # noqa: E731
    at = 1 << 20
    assert ask(at, 64, 1, at, 64, 1, 1, 4, 8, 64, 8, out) == native.EINVAL
    assert ask(at, 64, 1, at, 64, 1, 2, 4, 8, 64, 0, out) == native.EUNSUPPORTED
    assert ask(at, 64, 1, at, 64, 1, 1, 0, 8, 64, 0, out) == native.EINVAL
    assert ask(at, 64, 1, at, 64, 1, 1, 4, 8, 64, 0, None) == native.EINVAL
    assert plan(1, 13824, 5120)[0][0] == ROWS and plan(4096, 13824, 5120, epilogue=1)[0][0] == FULL_EPILOGUE
    assert plan(4096, 5120, 13824, w="across", w_row=5121)[1] == (0, 3)
