"""The GPU tests' shapes reach every form that the gated linear's plan can give a product (CPU only: wf_gated_dense_plan launches
nothing), so that a change of the time model cannot leave a kernel untested unseen."""
import ctypes
import math
import random

from conftest import sub
from test_gpu_gated import SHAPES

native = sub("_native")


def plan(M, N, K, keep, w="along"):
    out, need = (ctypes.c_int * 5)(), ctypes.c_int64()
    ws = (K, 1) if w == "along" else (1, 2 * N)
    assert native.lib().wf_gated_dense_plan(1 << 20, K, 1, 1 << 20, *ws, 1, M, N, K, keep, out, ctypes.byref(need)) == native.OK
    return (out[0], out[1], out[2] > 1), tuple(out[3:]), need.value


def sizes(rng):
    return rng.choice([int(round(math.exp(rng.uniform(0, math.log(14000))))), 8 * rng.randint(1, 1700),
                       64 * rng.randint(1, 216)])


def test_every_form_is_reached():
    rng = random.Random(3)
    shapes = [(sizes(rng), sizes(rng), sizes(rng)) for _ in range(20000)]
    for keep in (0, 1):
        possible, reached = ({plan(*s, keep)[0] for s in some} for some in (shapes, SHAPES))
        assert possible <= reached, sorted(possible - reached)
    # float16 and bfloat16 (every second shape) each see the few-rows form, tiles, tiles of rows that start anywhere, and slices
    for first in (0, 1):
        forms = {plan(*s, 1)[0] for s in SHAPES[first::2]}
        assert {f[0] for f in forms} == {0, 1, 2} and {f[2] for f in forms} == {False, True}
    # operands as they lie and copied; a weight that lies across is turned
    assert {plan(*s, 1)[1] for s in SHAPES} >= {(0, 0), (2, 2)}
    assert plan(300, 64, 64, 0, "across")[1][1] == 4


def test_workspace_holds_copies_and_sums():
    (few, tiling, sliced), _, need = plan(256, 2560, 5120, 0)
    assert few == 1 and sliced and need % (256 * 5120 * 4) == 0
    (few, _, _), how, need = plan(300, 300, 2049, 0)
    assert few == 2 and how == (0, 0) and need % (300 * 600 * 4) == 0        # rows that start anywhere are not copied,
    assert plan(300, 300, 7, 0)[1] == (2, 2)                       # but for those shorter than a load
    (few, _, _), how, need = plan(4096, 2560, 333, 0)
    row = 336                                                      # 333 up to whole 16-byte runs
    assert few == 1 and how == (2, 2) and need >= (4096 + 5120) * row * 2
