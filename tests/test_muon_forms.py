"""The GPU tests' shapes reach every form that the orthogonalised updates' plan can give a call (CPU only: wf_muon_plan launches
nothing), so that a change of the time model cannot leave a kernel untested unseen."""
import ctypes
import math
import random

from conftest import sub
from test_gpu_muon import SHAPES
from test_gpu_muon_forms import BATCHES
from test_gpu_muon_forms import SHAPES as MORE

native = sub("_native")


def plan(count, rows, cols):
    out = (ctypes.c_int * 7)()
    assert native.lib().wf_muon_plan(count, rows, cols, out) == native.OK
    return list(out)


def launches(count, rows, cols):
    """How many matrices each launch of a call takes: whole batches, and what is left."""
    n = plan(count, rows, cols)[0]
    return [n] * (count // n) + ([count % n] if count % n else [])


def forms(count, rows, cols):
    found, tall = set(), rows > cols
    for n in set(launches(count, rows, cols)):
        _, narrow, gram, gram_slices, square, square_slices, update = plan(n, rows, cols)
        found |= {("narrow", narrow, tall)} if narrow else {("gram", tall, gram, gram_slices > 1), ("square", square, square_slices > 1),
                                                            ("update", tall, update)}
    return found


def sizes(rng, most):
    return min(most, rng.choice([int(round(math.exp(rng.uniform(0, math.log(most))))), 8 * rng.randint(1, most // 8),
                                 64 * rng.randint(1, most // 64)]))


def random_calls(rng, many):
    for _ in range(many):
        rows, cols = sizes(rng, 1 << 20) if rng.random() < 0.2 else sizes(rng, 16384), sizes(rng, 16384)
        if rng.random() < 0.5:
            rows, cols = cols, rows
        if (rows + 256) * (cols + 8) < 1 << 30:
            yield rng.choice([1, 1, 2, 3, int(round(math.exp(rng.uniform(0, math.log(200)))))]), rows, cols


def test_every_form_is_reached():
    possible = set().union(*(forms(*call) for call in random_calls(random.Random(3), 40000)))
    reached = set().union(*(forms(*s[:3]) for s in SHAPES + MORE))
    assert possible <= reached, sorted(possible - reached, key=str)
    # and by each of the three types, whose last update is code of its own: MORE takes all three
    updates = {f for f in possible if f[0] == "update"}
    assert updates <= set().union(*(forms(*s) for s in MORE))


def test_batches_are_left_over_in_other_forms():
    kinds = set()
    for count, rows, cols in BATCHES:
        whole, *_, left = launches(count, rows, cols)
        a, z = plan(whole, rows, cols), plan(left, rows, cols)
        assert whole > left
        kinds.add((bool(a[1]), a[3] > 1, z[3] > 1))
    assert kinds >= {(True, False, False), (False, False, False), (False, False, True), (False, True, True), (False, True, False)}


def test_the_workspace_holds_the_last_batch_s_sums():
    need = ctypes.c_int64()
    for count, rows, cols in BATCHES:
        whole, *_, left = launches(count, rows, cols)
        sizes = []
        for n in (whole, left, count):
            assert native.lib().wf_muon_workspace(n, rows, cols, ctypes.byref(need)) == native.OK
            sizes.append(need.value)
        a, z = plan(whole, rows, cols), plan(left, rows, cols)
        assert sizes[2] >= max(sizes[:2])
        if z[3] > 1 and a[3] == 1:                                # behind the first launches' matrices, not the last's
            across = -(-min(rows, cols) // (256, 128, 64)[z[2]])
            sums = left * z[3] * (across * (across + 1) // 2) * (256, 128, 64)[z[2]] ** 2 * 4
            assert sizes[2] == sizes[0] + max(0, sums)


def test_the_plan_s_arguments():
    lib, out = native.lib(), (ctypes.c_int * 7)(*[9] * 7)
    assert lib.wf_muon_plan(1, 100, 100, None) == native.EINVAL and lib.wf_muon_plan(-1, 100, 100, out) == native.EINVAL
    assert lib.wf_muon_plan(1, 16385, 16385, out) == native.EUNSUPPORTED
    for empty in ((0, 100, 100), (3, 0, 100), (3, 100, 0)):
        assert lib.wf_muon_plan(*empty, out) == native.OK and not any(out)
    assert plan(1000, 64, 64)[:2] == [128, 4] and plan(1000, 65, 64)[:2] == [128, 4] and plan(5, 65, 66)[:2] == [5, 0]
