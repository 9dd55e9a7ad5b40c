"""A call's kinds, types and groups are handed to the library as a struct's address: the struct lives as long as the call that reads
it, whatever another thread does to the cache it came from (CPU only: no kernel is launched)."""
import ctypes
import gc
import weakref

import pytest

from conftest import sub

fn = sub("enhancers.fused_norm")
HOW = (1, 1, 1, 0, 1, 1, 1, 1.0, 1e-6, 2, 2, 1)


@pytest.fixture(autouse=True)
def empty_caches():
    for cache in (fn._blocks, fn._bytes_block):
        cache._known.clear()
    yield
    for cache in (fn._blocks, fn._bytes_block):
        cache._known.clear()


def test_the_struct_outlives_the_workspace_query(monkeypatch):
    held, real = [], fn._native.call

    def call(name, q, *args):
        # what a forward call on another thread does where it is the 4097th kind: the cache is cleared while the library reads
        fn._blocks._known.clear()
        gc.collect()
        assert held[0]() is not None, "the struct is gone while the library reads it"
        return real(name, q, *args)
    monkeypatch.setattr(fn._native, "call", call)
    monkeypatch.setattr(fn._native, "BlockNorm", type("Seen", (fn._native.BlockNorm,), {
        "__init__": lambda self, *a: (ctypes.Structure.__init__(self, *a), held.append(weakref.ref(self)))[0]}))
    need = fn._bytes_block((HOW, 64, 128, 2))
    assert len(held) == 1 and need > 0


def test_more_kinds_than_the_cache_holds():
    # every scale is a kind of its own
    sizes = {fn._bytes_block((HOW[:7] + (float(i),) + HOW[8:], 64, 128, 2)) for i in range(5000)}
    assert len(sizes) == 1 and len(fn._blocks._known) <= 4097
