"""Attention whose keys lie in two pieces at the edges of what its calls allow: the largest windows and sinks, sequences of no keys, more
sequences than a launch takes, other writers and readers of a ring that keeps its first rows, long verify passes behind a prefix."""
import numpy as np
import pytest

from tests.exact_attention import attend, check, dequantise
from tests.test_gpu_attn_shared_prefix import Family
from tests.test_gpu_attn_sinks import Session, _cache, _decode, _dev, _rows

pytestmark = pytest.mark.gpu
MOST = 2 ** 31 - 1


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("ring", [0, 96])
def test_the_largest_windows_and_sinks(gpu_ctx, bits, ring):
    # in a cache that holds every row, and in a ring while nothing has come round
    import torch
    from tinytitan_amd.engine import Attention, PrefillAttention, PrefillAttentionParams
    H, KH, D, length = 8, 2, 128, 150
    kv = _cache(gpu_ctx, KH, D, length, bits, ring=ring, sinks=40 if ring else 0, max_context=10000 if ring else length)
    s = Session(kv, 0, length, 3, bits, ring, 64 if ring else 0)
    q, scale, width = _rows(1, length, H, D), D ** -0.5, H * D
    qd = _dev(q)
    for window, sinks in ((MOST, MOST), (MOST, 0), (MOST, 1), (20, MOST), (1, MOST), (0, MOST), (MOST - 200, 3)):
        got = _decode(gpu_ctx, kv, q[:1], [length], window, sinks, scale)
        check(got, [s.row(q[0], length - 1, window, sinks, scale, None, bits)], f"window {window}, sinks {sinks}")
        out = torch.full((length, H, D), float("nan"), dtype=torch.float16, device="cuda")
        torch.cuda.synchronize()
        Attention(gpu_ctx).encode_verify_rows(kv, 0, qd[:9], out, H, [length - 9], 9, scale, [0], window=window, sinks=sinks)
        gpu_ctx.synchronize()
        check(out.cpu().numpy()[[0, 8]], [s.row(q[i], length - 9 + i, window, sinks, scale, None, bits) for i in (0, 8)], f"verify {window} {sinks}")
        assert out[9:].isnan().all()
        PrefillAttention(gpu_ctx).encode_causal(kv, 0, 0, qd, out, PrefillAttentionParams(0, length, length, H, scale, width, width,
                                                                                          sliding_window=window, sinks=sinks))
        gpu_ctx.synchronize()
        some = [0, 31, 100, length - 1]
        check(out.cpu().numpy()[some], [s.row(q[i], i, window, sinks, scale, None, bits) for i in some], f"chunk {window} {sinks}")
    kv.close()


@pytest.mark.parametrize("H,KH,D,bits", [(16, 2, 256, 16), (32, 8, 128, 8), (4, 4, 64, 4)])
def test_more_sequences_than_a_launch_takes_some_of_them_empty(gpu_ctx, H, KH, D, bits):
    n, window, sinks = 130, 70, 5
    lengths = [(i * 37) % 300 for i in range(n)]
    assert lengths[0] == 0
    kv = _cache(gpu_ctx, KH, D, 300, bits, slots=n)
    some = [0, 1, 63, 64, 65, 127, 128, 129]
    sessions = {i: Session(kv, i, max(lengths[i], 1), i, bits) for i in range(n)}
    q, g = _rows(1, n, H, D), _rows(2, n, H, D)
    got = _decode(gpu_ctx, kv, q, lengths, window, sinks, D ** -0.5, g)
    assert np.isfinite(got).all()
    check(got[some], [sessions[i].row(q[i], lengths[i] - 1, window, sinks, D ** -0.5, g[i], bits) for i in some], "batch")
    kv.close()


def test_the_epilogue_writes_a_ring_with_pinned_rows(gpu_ctx):
    # rows of the epilogue, position by position far past the ring, are those that it writes into a cache that keeps every row
    import torch
    from tinytitan_amd.engine import QKVEpilogue
    H, KH, D, ring, sinks, total = 8, 2, 128, 64, 33, 64 + 3 * 64 + 11
    pinned = 64
    kv, full = _cache(gpu_ctx, KH, D, 0, ring=ring, sinks=sinks, max_context=total), _cache(gpu_ctx, KH, D, total)
    packed, k, v = (_dev(_rows(i, total, w)) for i, w in ((1, H * 2 * D), (2, KH * D), (3, KH * D)))
    weight = torch.full((D,), 0x3f80, dtype=torch.int16, device="cuda")
    q_out, g_out = (torch.empty(total, H, D, dtype=torch.float16, device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    at = 0
    while at < total:
        rows = min(1 + at % 5, pinned - at if at < pinned else ring - (at - pinned) % ring, total - at)
        for cache in (kv, full):
            QKVEpilogue(gpu_ctx).encode(cache, 0, packed[at:], k[at:], v[at:], weight, weight, q_out, g_out, H, [at], rows, 1e-6, 64, 1e7, slots=[0])
        at += rows
    want = full.read(0, 0, 0, total)
    for first, count in ((0, pinned), (pinned + 3 * ring, 11), (pinned + 2 * ring + 11, ring - 11)):
        got = kv.read(0, 0, first, count)
        gpu_ctx.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b[first:first + count]), first
    kv.close()
    full.close()


@pytest.mark.parametrize("bits", [16, 4])
def test_a_snapshot_of_a_ring_with_pinned_rows(gpu_ctx, bits):
    H, KH, D, window, sinks, ring, pinned = 8, 2, 64, 50, 4, 96, 32
    length = pinned + 2 * ring + 21
    a, b = (_cache(gpu_ctx, KH, D, 0, bits, ring=ring, sinks=sinks, max_context=1000) for _ in range(2))
    s = Session(a, 0, length, 9, bits, ring, pinned)
    a.advance(0, length)
    lengths = a.snapshot_segment_lengths(length)
    payload = bytearray()
    a.append_snapshot_payload(payload, lengths)
    b.restore_snapshot(length, lengths, bytes(payload))
    assert b.position(0) == length
    q = _rows(1, 1, H, D)
    got = [_decode(gpu_ctx, kv, q, [length], window, sinks, 0.125) for kv in (a, b)]
    assert np.array_equal(*got)
    check(got[1], [s.row(q[0], length - 1, window, sinks, 0.125, None, bits)], "restored")
    a.close()
    b.close()


@pytest.mark.parametrize("H,KH,D,bits,prefix,rows", [(8, 2, 64, 16, 700, 1100), (4, 1, 128, 8, 2000, 600), (8, 1, 256, 16, 600, 1025)])
def test_long_verify_passes_behind_a_prefix(gpu_ctx, H, KH, D, bits, prefix, rows):
    # more rows than the partial results are kept for at a time, of two sequences and of one
    import torch
    from tinytitan_amd.engine import Attention
    starts = [prefix - 1, prefix + 70]
    f = Family(gpu_ctx, KH, D, prefix, [p + rows for p in starts], bits)
    q = _rows(3, 2, rows, H, D)
    qd = _dev(q)
    for n in (2, 1):
        out = torch.full((2, rows, H, D), float("nan"), dtype=torch.float16, device="cuda")
        torch.cuda.synchronize()
        Attention(gpu_ctx).encode_verify_rows(f.kv, 0, qd, out, H, starts[:n], rows, D ** -0.5, f.slots[:n], prefix=f.prefix)
        gpu_ctx.synchronize()
        got, some = out.cpu().numpy(), sorted({0, 1, 512, min(1023, rows - 1), min(1024, rows - 1), rows - 1})
        for i in range(n):
            check(got[i][some], [f.row(i, q[i, r], starts[i] + r, D ** -0.5) for r in some], f"sequence {i} of {n}")
        assert np.isnan(got[n:]).all()
    f.kv.close()


@pytest.mark.parametrize("bits", [16, 8])
def test_slots_that_lie_past_four_gibibytes(gpu_ctx, bits):
    import torch
    from tinytitan_amd.engine import Attention, KVCacheManager, SharedPrefix
    H, KH, D, prefix, slots = 16, 2, 256, 5005, 9
    capacity = 640_000 if bits == 16 else 1_200_000
    kv = KVCacheManager(gpu_ctx, 1, KH, D, slots=slots, max_context=capacity, initial_capacity=capacity, precision_bits=bits)
    assert kv.token_stride_bytes * capacity * 8 > 2 ** 32
    lengths = {0: prefix + 3, 1: prefix + 40, 6: prefix + 1, 7: prefix + 333}
    home = Session(kv, 8, prefix, 1, bits)
    kv.advance(8, prefix)
    kv.share_prefix(8, prefix, list(lengths))
    own = {}
    for slot, length in lengths.items():
        new = [_dev(part) for part in _rows(slot + 2, 2, length - prefix, KH * D)]
        torch.cuda.synchronize()
        kv.append(0, slot, prefix, *new)
        k, v = kv.export_rows(0, slot, prefix, length - prefix)
        gpu_ctx.synchronize()
        own[slot] = [dequantise(t.cpu().numpy(), KH * D, bits) for t in (k, v)]
    for copies in (1, 16):  # (few rows and many: every way over the shared keys)
        table = list(lengths) * copies
        q = _rows(50 + copies, len(table), H, D)
        qd = _dev(q)
        out = torch.full_like(qd, float("nan"))
        torch.cuda.synchronize()
        Attention(gpu_ctx).encode_full(kv, 0, qd, out, H, [lengths[s] for s in table], 0.0625, slot=table, prefix=SharedPrefix(8, prefix))
        gpu_ctx.synchronize()
        got = out.cpu().numpy()
        for i in range(4):
            k, v = ([np.concatenate(p) for p in zip(front, mine)] for front, mine in zip((home.k64, home.v64), own[table[i]]))
            check(got[i:i + 1], [attend(q[i], k, v, np.arange(len(k[0])) >= 0, 0.0625, None, bits)], f"{copies} copies, sequence {i}")
    q = _rows(60, 1, H, D)
    got = _decode(gpu_ctx, kv, q, [prefix], 300, 7, 0.0625, slots=[8])
    check(got, [home.row(q[0], prefix - 1, 300, 7, 0.0625, None, bits)], "sinks in the last slot")
    kv.close()
