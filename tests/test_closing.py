"""A context closes its caches before itself: a cache that outlived it would look for its device and stream in freed memory.  No GPU: the library
is a list of the calls it got."""
import gc

import pytest

from tinytitan_amd import engine


class Library:
    """Hands out handles and writes down what is destroyed, in order."""

    def __init__(self):
        self.destroyed, self.handles = [], 0

    def __getattr__(self, name):
        def call(*args):
            if name.endswith("_destroy"):
                self.destroyed.append((name, args[0]))
            elif "_create" in name:
                self.handles += 1
                return self.handles
            return 0
        return call


@pytest.fixture
def library(monkeypatch):
    library = Library()
    monkeypatch.setattr(engine.capi, "lib", lambda: library)
    monkeypatch.setattr(engine.capi, "calls", lambda: library)
    return library


def test_caches_go_before_their_context(library):
    ctx = engine.HIPContext(0)
    kept = [engine.KVCacheManager(ctx, 1, 2, 64, max_context=64), engine.KVCacheManager(ctx, 1, 2, 64, max_context=64, ring_capacity=64)]
    ctx.close()
    assert sorted(library.destroyed[:2]) == [("tt_hip_kv_destroy", 2), ("tt_hip_kv_destroy", 3)]
    assert library.destroyed[2:] == [("tt_hip_ctx_destroy", 1)]
    assert all(kv.handle is None for kv in kept)
    for kv in kept:
        kv.close()
    ctx.close()
    del kept, kv, ctx
    gc.collect()
    assert len(library.destroyed) == 3


def test_a_closed_cache_is_forgotten(library):
    ctx = engine.HIPContext(0)
    kv = engine.KVCacheManager(ctx, 1, 2, 64, max_context=64)
    kv.close()
    ctx.close()
    assert library.destroyed == [("tt_hip_kv_destroy", 2), ("tt_hip_ctx_destroy", 1)]


def test_a_context_and_a_cache_that_the_collector_takes_together(library):
    # finalised in any order, and the context may be first
    ctx = engine.HIPContext(0)
    kv = engine.KVCacheManager(ctx, 1, 2, 64, max_context=64)
    ctx.cache = kv
    del ctx, kv
    gc.collect()
    names = [name for name, _ in library.destroyed]
    assert names.count("tt_hip_ctx_destroy") == 1 and names[-1] == "tt_hip_ctx_destroy"
