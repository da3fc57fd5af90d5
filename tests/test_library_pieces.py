"""The calls of attention with sinks and of a shared prefix, as far as they go without a device: refusals, argument types, the C++ mirror."""
import ctypes
import os
import shutil
import subprocess
import tempfile

import numpy as np
import pytest

from tinytitan_amd import capi

INC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
BAD = capi.ERR_INVALID_ARGUMENT


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(capi.LIB_PATH):
        pytest.skip("library not built")
    return capi.lib()


def test_null_handles_are_errors_not_crashes(lib):
    one = (ctypes.c_int * 1)(5)
    for table in (None, one):
        assert lib.tt_hip_attn_decode_sinks(None, None, 0, 1, table, table, 8, 4, 8, None, None, 1.0, None) == BAD
        assert lib.tt_hip_attn_verify_sinks(None, None, 0, 1, table, table, 2, 8, 4, 8, None, None, 1.0, None) == BAD
        assert lib.tt_hip_attn_decode_shared(None, None, 0, 1, table, table, 0, 64, 8, None, None, 1.0, None) == BAD
        assert lib.tt_hip_attn_verify_shared(None, None, 0, 1, table, table, 2, 0, 64, 8, None, None, 1.0, None) == BAD
        assert lib.tt_hip_kv_share_prefix(None, 0, 64, 1, table) == BAD
    assert lib.tt_hip_attn_prefill_sinks(None, None, 0, 0, 0, 1, 1, 8, 4, 8, None, 0, None, 0, 1.0, None, 0) == BAD
    assert lib.tt_hip_attn_prefill_shared(None, None, 0, 0, 64, 1, 65, 0, 64, 8, None, 0, None, 0, 1.0, None, 0) == BAD
    for ring, sinks in ((128, 64), (0, 64), (128, -1), (2 ** 31 - 1, 2 ** 31 - 1)):
        err = ctypes.c_int(0)
        assert not lib.tt_hip_kv_create_ring_sinks(None, 1, 2, 64, 1, ring, sinks, 4096, 16, ctypes.byref(err))
        assert err.value == BAD
        assert not lib.tt_hip_kv_create_ring_sinks(None, 1, 2, 64, 1, ring, sinks, 4096, 16, None)


def test_native_calls_take_what_the_c_types_take(lib):
    calls = capi.calls()
    forms = {
        "attn_decode_sinks": lambda n, table=0: calls.attn_decode_sinks(None, None, n, table, table, n, n, n, None, None, 1.0, None),
        "attn_verify_sinks": lambda n, table=(0,): calls.attn_verify_sinks(None, None, n, table, table, n, n, n, n, None, None, 1.0, None),
        "attn_prefill_sinks": lambda n: calls.attn_prefill_sinks(None, None, n, n, n, n, n, n, n, n, None, n, None, n, 1.0, None, n),
        "attn_decode_shared": lambda n, table=0: calls.attn_decode_shared(None, None, n, table, table, n, n, n, None, None, 1.0, None),
        "attn_verify_shared": lambda n, table=(0,): calls.attn_verify_shared(None, None, n, table, table, n, n, n, n, None, None, 1.0, None),
        "attn_prefill_shared": lambda n: calls.attn_prefill_shared(None, None, n, n, n, n, n, n, n, n, None, n, None, n, 1.0, None, n),
    }
    for name, call in forms.items():
        for number in (5, True, np.int64(5), np.array(5)):
            assert call(number) == BAD, name
        for number in (5.0, "5", None):
            with pytest.raises(TypeError):
                call(number)
        if "prefill" not in name:
            assert call(5, [0, 1]) == BAD and call(5, [0] * 100) == BAD, name
            with pytest.raises((TypeError, ValueError)):
                call(5, "five")


@pytest.mark.skipif(shutil.which("g++") is None, reason="no g++")
def test_the_cpp_mirror_has_them(lib):
    src = r'''
#include "TinyTitanHIP.hpp"
#include <cstdio>
using namespace tinytitan;
void use(Context &ctx, KVCacheManager &kv, const tt_half *q, tt_half *out) {
    const SharedPrefix prefix{0, 64};
    kv.sharePrefix(0, 64, {1, 2});
    Attention attention(ctx);
    attention.encodeSWA(kv, 0, q, out, 16, 100, 64, 0.0625f, 1, nullptr, 4);
    attention.encodeBatch(kv, 0, {1, 2}, {65, 70}, prefix, q, out, 16, 0.0625f);
    attention.encodeVerifyRows(kv, 0, {1}, {64}, 3, q, out, 16, 0.0625f, nullptr, 64, 4);
    attention.encodeVerifyRows(kv, 0, {1}, {64}, 3, prefix, q, out, 16, 0.0625f);
    PrefillAttentionParams p;
    p.startPosition = 64;
    p.queryCount = 4;
    p.kvValidCount = 68;
    p.numQHeads = 16;
    p.qStride = p.oStride = 16 * 256;
    PrefillAttention chunk(ctx);
    chunk.encodeCausal(kv, 0, 1, prefix, q, out, p);
    p.slidingWindow = 32;
    p.sinks = 4;
    chunk.encodeCausal(kv, 0, 1, q, out, p);
}
int main(int argc, char **) {
    try {
        Context ctx(0);
        KVCacheManager kv(ctx, 1, 2, 256, 3, 4096);
        if (argc > 1) use(ctx, kv, nullptr, nullptr);
        KVCacheManager::Ring ring;
        ring.capacity = 128;
        ring.sinks = 40;
        KVCacheManager pinned(ctx, 1, 2, 256, 1, 4096, ring);
        if (pinned.capacityTokens() != 128 + 64) return 2;
    } catch (const Error &e) {
        std::printf("status %d\n", e.status());
        return e.status() == TT_HIP_ERR_NO_DEVICE ? 0 : 1;
    }
    return 0;
}
'''
    with tempfile.TemporaryDirectory() as d:
        path, exe, libdir = os.path.join(d, "t.cpp"), os.path.join(d, "t"), os.path.dirname(capi.LIB_PATH)
        open(path, "w").write(src)
        subprocess.run(["g++", "-std=c++17", "-Wall", "-Wextra", "-Werror", "-I", INC, path, "-o", exe, "-L", libdir, "-lctinytitan_hip",
                        f"-Wl,-rpath,{libdir}", "-Wl,-rpath,/opt/rocm/lib", "-L/opt/rocm/lib"], check=True)
        out = subprocess.run([exe], capture_output=True, text=True)
        assert out.returncode == 0, out.stdout + out.stderr
