"""A sliding window with sinks through the C ABI, against the definition in 64 bits: the row at position p sees key j <= p where
j > p - window or j < sinks."""
import numpy as np
import pytest

from tests.exact_attention import attend, check, dequantise, stored_rows

pytestmark = pytest.mark.gpu


def _dev(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).to("cuda")


class Session:
    """Rows of one sequence: a slot of the cache, and the same rows here."""

    def __init__(self, kv, slot, length, seed, bits, ring=0, pinned=0):
        import torch
        r = np.random.default_rng(seed)
        width = kv.kv_heads * kv.head_dim
        self.k = stored_rows(r.standard_normal((length, width)), bits)
        self.v = stored_rows(r.standard_normal((length, width)), bits)
        at = 0
        while at < length:
            n = length - at
            if ring:
                n = min(n, pinned - at if at < pinned else ring - (at - pinned) % ring)
            kd, vd = _dev(self.k[at:at + n]), _dev(self.v[at:at + n])
            torch.cuda.synchronize()
            kv.import_rows(0, slot, at, kd, vd)
            kv.ctx.synchronize()
            at += n
        self.k64, self.v64 = dequantise(self.k, width, bits), dequantise(self.v, width, bits)

    def row(self, q, position, window, sinks, scale, gate=None, bits=16):
        keys = np.arange(self.k.shape[0])
        seen = keys <= position
        if window:
            seen &= (keys > position - window) | (keys < sinks)
        return attend(q, self.k64, self.v64, seen, scale, gate, bits)


def _cache(ctx, KH, D, capacity, bits=16, slots=1, ring=0, sinks=0, max_context=None):
    from tinytitan_amd.engine import KVCacheManager
    return KVCacheManager(ctx, 1, KH, D, slots=slots, max_context=max_context or capacity, initial_capacity=capacity, precision_bits=bits,
                          ring_capacity=ring, sink_tokens=sinks)


def _rows(seed, *shape):
    return np.random.default_rng(seed).standard_normal(shape).astype(np.float16)


def _decode(ctx, kv, q, seq_lens, window, sinks, scale, gate=None, slots=None):
    import torch
    from tinytitan_amd.engine import Attention
    n, heads, dim = q.shape
    qd, gd = _dev(q), _dev(gate) if gate is not None else None
    out = torch.full(qd.shape, float("nan"), dtype=torch.float16, device="cuda")
    torch.cuda.synchronize()
    Attention(ctx).encode_swa(kv, 0, qd, out, heads, list(seq_lens), window, scale, slot=slots or list(range(n)), gate=gd, sinks=sinks)
    ctx.synchronize()
    return out.cpu().numpy()


SHAPES = [(16, 2, 256), (8, 2, 256), (24, 2, 256), (32, 8, 128), (4, 1, 128), (16, 4, 64), (6, 3, 64)]


@pytest.mark.parametrize("H,KH,D", SHAPES)
@pytest.mark.parametrize("bits", [16, 8, 4])
def test_decode(gpu_ctx, H, KH, D, bits):
    # windows and sinks that end on blocks and inside them, meet, and leave a gap of less than a block
    length = 1500
    kv = _cache(gpu_ctx, KH, D, length, bits)
    s = Session(kv, 0, length, 7, bits)
    scale = D ** -0.5
    for at, window, sinks in ((1500, 256, 4), (1500, 100, 33), (1499, 31, 1), (1473, 32, 32), (1200, 1, 1), (1200, 1100, 99), (1200, 1100, 100),
                              (1200, 1100, 101), (600, 1000, 4), (65, 64, 1), (66, 33, 32), (2, 1, 1), (1, 5, 3), (1500, 700, 700)):
        q, g = _rows(at, 1, H, D), _rows(at + 1, 1, H, D)
        got = _decode(gpu_ctx, kv, q, [at], window, sinks, scale, g)
        check(got, [s.row(q[0], at - 1, window, sinks, scale, g[0], bits)], f"{at} keys, window {window}, sinks {sinks}")
    kv.close()


@pytest.mark.parametrize("H,KH,D,bits", [(16, 2, 256, 16), (32, 8, 128, 8), (16, 4, 64, 4)])
def test_decode_batch_of_all_ages(gpu_ctx, H, KH, D, bits):
    lengths = [1, 5, 100, 501, 502, 533, 3000, 7001, 900]
    kv = _cache(gpu_ctx, KH, D, max(lengths), bits, slots=len(lengths))
    sessions = [Session(kv, i, n, 30 + i, bits) for i, n in enumerate(lengths)]
    q, g = _rows(1, len(lengths), H, D), _rows(2, len(lengths), H, D)
    for window, sinks in ((500, 2), (3500, 40), (64, 500)):
        for gate in (None, g):
            got = _decode(gpu_ctx, kv, q, lengths, window, sinks, D ** -0.5, gate)
            check(got, [s.row(q[i], n - 1, window, sinks, D ** -0.5, None if gate is None else g[i], bits)
                        for i, (s, n) in enumerate(zip(sessions, lengths))], f"window {window}, sinks {sinks}")
    kv.close()


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("D,window,sinks", [(256, 96, 4), (128, 200, 33), (64, 63, 64)])
def test_a_ring_keeps_its_sinks(gpu_ctx, bits, D, window, sinks):
    # several times round: the window comes out of the ring, the sinks out of the rows in front of it
    H, KH = 8, 2
    ring, pinned = (window + 4 + 30 + 31) // 32 * 32, (sinks + 31) // 32 * 32
    length = pinned + 5 * ring + 17
    kv = _cache(gpu_ctx, KH, D, 0, bits, ring=ring, sinks=sinks, max_context=length)
    assert kv.capacity_tokens == pinned + ring
    s = Session(kv, 0, length, 5, bits, ring, pinned)
    scale = D ** -0.5
    for at in (length, length - 1, length - 40):
        q = _rows(at, 1, H, D)
        first = max(at - window, 0)
        if at != length and length - (first & ~31) > ring:
            continue  # (those rows have been overwritten)
        check(_decode(gpu_ctx, kv, q, [at], window, sinks, scale), [s.row(q[0], at - 1, window, sinks, scale, None, bits)], f"{at} keys")
        # without sinks the window alone, through the same cache
        check(_decode(gpu_ctx, kv, q, [at], window, 0, scale), [s.row(q[0], at - 1, window, 0, scale, None, bits)], f"{at} keys, no sinks")
    kv.close()


def test_ring_rows_are_read_back_from_where_they_lie(gpu_ctx):
    import torch
    KH, D, ring, sinks = 2, 64, 64, 5
    length = 32 + 3 * ring + 9
    for bits in (16, 8):
        kv = _cache(gpu_ctx, KH, D, 0, bits, ring=ring, sinks=sinks, max_context=length)
        s = Session(kv, 0, length, 9, bits, ring, 32)
        positions = [0, 4, 31, length - ring, length - 1, length - 30, length]  # the last is past the context: zeros
        pd = _dev(np.array(positions, np.int32))
        k = torch.full((len(positions), KH * D), float("nan"), dtype=torch.float16, device="cuda")
        v = torch.full_like(k, float("nan"))
        torch.cuda.synchronize()
        kv.gather(0, 0, pd, k, v)
        gpu_ctx.synchronize()
        for i, p in enumerate(positions[:-1]):
            for got, want in ((k, s.k64), (v, s.v64)):
                assert np.abs(got[i].cpu().numpy().astype(np.float64) - (want[0][p] + want[1][p])).max() <= 2.0 ** -9
        limit = kv.max_context
        assert limit >= length and (limit > length or not k[-1].any())
        kv.close()


@pytest.mark.parametrize("H,KH,D,bits,rows", [(16, 2, 256, 16, 4), (24, 2, 256, 4, 3), (32, 8, 128, 8, 5), (16, 4, 64, 16, 8), (16, 2, 256, 8, 2)])
def test_verify_rows(gpu_ctx, H, KH, D, bits, rows):
    import torch
    from tinytitan_amd.engine import Attention
    starts, window, sinks, scale = [0, 20, 318, 320, 333, 2500], 320, 6, D ** -0.5
    kv = _cache(gpu_ctx, KH, D, max(starts) + rows, bits, slots=len(starts))
    sessions = [Session(kv, i, p + rows, 50 + i, bits) for i, p in enumerate(starts)]
    q, g = _rows(3, len(starts), rows, H, D), _rows(4, len(starts), rows, H, D)
    qd, gd = _dev(q), _dev(g)
    out = torch.full(qd.shape, float("nan"), dtype=torch.float16, device="cuda")
    torch.cuda.synchronize()
    Attention(gpu_ctx).encode_verify_rows(kv, 0, qd, out, H, starts, rows, scale, list(range(len(starts))), gate=gd, window=window, sinks=sinks)
    gpu_ctx.synchronize()
    got = out.cpu().numpy()
    for i, p in enumerate(starts):
        check(got[i], [sessions[i].row(q[i, r], p + r, window, sinks, scale, g[i, r], bits) for r in range(rows)], f"sequence {i} at {p}")
    kv.close()


def _prefill(ctx, kv, q, start, rows, valid, window, sinks, scale, gate=None, pad=0, offset=0):
    """Rows inside wider buffers, ``offset`` elements into them; what lies around them has to stay."""
    import torch
    from tinytitan_amd.engine import PrefillAttention, PrefillAttentionParams
    heads, dim = q.shape[1:]
    width, stride = heads * dim, heads * dim + pad

    def wide(a):
        t = torch.full((rows * stride + offset,), 7.0, dtype=torch.float16, device="cuda")
        t[offset:].view(rows, stride)[:, :width] = _dev(a).view(rows, width)
        return t

    qd, gd = wide(q), wide(gate) if gate is not None else None
    out = torch.full((rows * stride + offset + 64,), float("nan"), dtype=torch.float16, device="cuda")
    params = PrefillAttentionParams(start, rows, valid, heads, scale, stride, stride, stride, sliding_window=window, sinks=sinks)
    torch.cuda.synchronize()
    PrefillAttention(ctx).encode_causal(kv, 0, 0, qd[offset:], out[offset:], params, gate=gd[offset:] if gd is not None else None)
    ctx.synchronize()
    res = out.cpu().numpy()
    body = res[offset:offset + rows * stride].reshape(rows, stride)
    assert np.isnan(res[:offset]).all() and np.isnan(body[:, width:]).all() and np.isnan(res[offset + rows * stride:]).all()
    return body[:, :width].reshape(rows, heads, dim)


def _some(rows):
    return sorted({0, 1, 2, rows - 1, rows - 2, *range(0, rows, max(1, rows // 23)), *(r for r in (30, 31, 32, 33, 63, 64, 65) if r < rows)} & set(range(rows)))


@pytest.mark.parametrize("H,KH,D,bits,start,rows,window,sinks,pad,offset", [
    (16, 2, 256, 16, 0, 300, 64, 4, 0, 0), (16, 2, 256, 16, 700, 129, 333, 40, 8, 8), (16, 2, 256, 8, 900, 70, 100, 1, 0, 0),
    (16, 2, 256, 16, 1000, 2100, 512, 64, 0, 0), (24, 2, 256, 16, 2000, 260, 1000, 17, 0, 0), (16, 2, 256, 16, 37, 700, 33, 1, 0, 0),
    (32, 8, 128, 16, 1500, 777, 500, 4, 0, 0), (32, 8, 128, 16, 100, 1500, 90, 95, 0, 0), (32, 8, 128, 8, 3000, 300, 1024, 100, 0, 0),
    (16, 4, 64, 16, 2001, 333, 500, 7, 72, 0), (16, 4, 64, 16, 0, 2500, 31, 31, 0, 0), (16, 4, 64, 4, 200, 500, 150, 32, 5, 3),
    (6, 3, 64, 16, 500, 200, 77, 9, 0, 0), (64, 8, 64, 16, 600, 1100, 320, 65, 0, 0), (40, 8, 128, 16, 40, 600, 256, 3, 0, 1),
    (16, 2, 256, 16, 5, 1, 3, 1, 0, 0), (16, 2, 256, 16, 3000, 40, 2900, 64, 0, 0), (16, 2, 256, 16, 300, 500, 5000, 64, 0, 0),
    (32, 8, 128, 16, 0, 4000, 1, 1, 0, 0)])
def test_chunk(gpu_ctx, H, KH, D, bits, start, rows, window, sinks, pad, offset):
    length, scale = start + rows + 45, D ** -0.5
    kv = _cache(gpu_ctx, KH, D, length, bits)
    s = Session(kv, 0, length, 11, bits)  # (later rows are there, too: not to be seen)
    q, g = _rows(12, rows, H, D), _rows(13, rows, H, D)
    for gate, valid in ((g, start + rows), (None, length)):
        got = _prefill(gpu_ctx, kv, q, start, rows, valid, window, sinks, scale, gate, pad, offset)
        some = _some(rows)
        check(got[some], [s.row(q[r], start + r, window, sinks, scale, None if gate is None else g[r], bits) for r in some], "chunk")
    kv.close()


@pytest.mark.parametrize("H,KH,D,bits,window,sinks,rows", [(16, 2, 256, 16, 200, 5, 130), (32, 8, 128, 16, 300, 33, 700), (16, 4, 64, 8, 100, 2, 90),
                                                           (16, 2, 256, 16, 500, 64, 1500)])
def test_chunk_over_a_ring_that_has_come_round(gpu_ctx, H, KH, D, bits, window, sinks, rows):
    ring, pinned, scale = (window + rows + 30 + 31) // 32 * 32, (sinks + 31) // 32 * 32, D ** -0.5
    start = pinned + 3 * ring
    kv = _cache(gpu_ctx, KH, D, 0, bits, ring=ring, sinks=sinks, max_context=start + rows)
    s = Session(kv, 0, start + rows, 17, bits, ring, pinned)
    q, g = _rows(18, rows, H, D), _rows(19, rows, H, D)
    got = _prefill(gpu_ctx, kv, q, start, rows, start + rows, window, sinks, scale, g)
    some = _some(rows)
    check(got[some], [s.row(q[r], start + r, window, sinks, scale, g[r], bits) for r in some], "ring")
    got = _prefill(gpu_ctx, kv, q, start, rows, start + rows, window, 0, scale, g)
    check(got[some], [s.row(q[r], start + r, window, 0, scale, g[r], bits) for r in some], "ring, no sinks")
    kv.close()


@pytest.mark.parametrize("scale", [0.0, -0.0625, 0.5])
def test_chunk_scales(gpu_ctx, scale):
    H, KH, D, start, rows, window, sinks = 16, 2, 256, 800, 600, 256, 9
    kv = _cache(gpu_ctx, KH, D, start + rows)
    s = Session(kv, 0, start + rows, 21, 16)
    q = _rows(22, rows, H, D)
    got = _prefill(gpu_ctx, kv, q, start, rows, start + rows, window, sinks, scale)
    some = _some(rows)
    check(got[some], [s.row(q[r], start + r, window, sinks, scale) for r in some], f"scale {scale}")
    kv.close()


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("H,KH,D", [(16, 2, 256), (32, 8, 128), (16, 4, 64)])
@pytest.mark.parametrize("rows", [1, 6, 70, 1300])
def test_keys_that_no_row_sees_may_hold_anything(gpu_ctx, bits, H, KH, D, rows):
    # NaN and infinities between the sinks and the window and behind the last row, inside the blocks that are read
    import torch
    start, window, sinks, scale = 1000, 70, 5, D ** -0.5
    length = start + rows + 60
    kv = _cache(gpu_ctx, KH, D, length, bits)
    s = Session(kv, 0, length, 25, bits)
    bad = np.ones(length, bool)
    bad[:sinks] = False
    bad[start + 1 - window:start + rows] = False
    for rows_of, value in ((s.k, np.nan), (s.v, np.inf), (s.v, np.nan)):
        dirty = rows_of.copy()
        halves = dirty if bits == 16 else dirty[:, KH * D * bits // 8:]
        halves[bad] = np.full(halves.shape[1] // 2, value, np.float16).view(np.uint8)
        kd, vd = _dev(dirty if rows_of is s.k else s.k), _dev(dirty if rows_of is s.v else s.v)
        torch.cuda.synchronize()
        kv.import_rows(0, 0, 0, kd, vd)
        gpu_ctx.synchronize()
        q = _rows(26, rows, H, D)
        if rows == 1:
            got = _decode(gpu_ctx, kv, q, [start + 1], window, sinks, scale)
        else:
            got = _prefill(gpu_ctx, kv, q, start, rows, start + rows, window, sinks, scale)
        some = _some(rows)
        check(got[some], [s.row(q[r], start + r, window, sinks, scale, None, bits) for r in some], f"{value} in {'K' if rows_of is s.k else 'V'}")
    kv.close()


def test_without_sinks_it_is_the_window_and_without_a_window_everything(gpu_ctx):
    # bit for bit the calls that were there
    import torch
    from tinytitan_amd.engine import Attention
    H, KH, D, length = 16, 2, 256, 900
    kv = _cache(gpu_ctx, KH, D, length)
    Session(kv, 0, length, 33, 16)
    q = _dev(_rows(34, 1, H, D))
    outs = [torch.zeros(1, H, D, dtype=torch.float16, device="cuda") for _ in range(5)]
    torch.cuda.synchronize()
    a = Attention(gpu_ctx)
    a.encode_swa(kv, 0, q, outs[0], H, length, 200, 0.0625)
    gpu_ctx._check(gpu_ctx._calls.attn_decode_sinks(gpu_ctx.handle, kv.handle, 0, 0, length, 200, 0, H, q, None, 0.0625, outs[1]), "sinks 0")
    a.encode_full(kv, 0, q, outs[2], H, length, 0.0625)
    a.encode_swa(kv, 0, q, outs[3], H, length, 0, 0.0625, sinks=7)
    a.encode_swa(kv, 0, q, outs[4], H, length, length, 0.0625, sinks=7)
    gpu_ctx.synchronize()
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[2], outs[3]) and torch.equal(outs[2], outs[4])
    kv.close()


def test_refusals(gpu_ctx):
    import torch
    from tinytitan_amd import capi
    from tinytitan_amd.engine import Attention, KVCacheManager, PrefillAttention, PrefillAttentionParams, TinyTitanHIPError
    H, KH, D = 8, 2, 64
    q = torch.zeros(4, H, D, dtype=torch.float16, device="cuda")
    out = torch.full_like(q, 3.0)
    a, chunk = Attention(gpu_ctx), PrefillAttention(gpu_ctx)

    def refused(status, call):
        with pytest.raises(TinyTitanHIPError) as e:
            call()
        assert e.value.status == status

    kv = _cache(gpu_ctx, KH, D, 256)
    refused(capi.ERR_INVALID_ARGUMENT, lambda: a.encode_swa(kv, 0, q, out, H, 100, 10, 0.1, sinks=-1))
    refused(capi.ERR_INVALID_ARGUMENT, lambda: a.encode_swa(kv, 0, q, out, H, 100, -10, 0.1, sinks=1))
    refused(capi.ERR_INVALID_ARGUMENT, lambda: a.encode_swa(kv, 0, q, out, H, -1, 10, 0.1, sinks=1))
    refused(capi.ERR_INVALID_ARGUMENT, lambda: a.encode_swa(kv, 0, q, out, H, 100, 10, 0.1, slot=1, sinks=1))
    refused(capi.ERR_INVALID_ARGUMENT, lambda: a.encode_swa(kv, 1, q, out, H, 100, 10, 0.1, sinks=1))
    refused(capi.ERR_SHAPE, lambda: a.encode_swa(kv, 0, q, out, 7, 100, 10, 0.1, sinks=1))
    refused(capi.ERR_CAPACITY, lambda: a.encode_swa(kv, 0, q, out, H, 257, 10, 0.1, sinks=1))
    refused(capi.ERR_INVALID_ARGUMENT, lambda: a.encode_verify_rows(kv, 0, q, out, H, [10], 0, 0.1, [0], window=5, sinks=1))
    refused(capi.ERR_CAPACITY, lambda: a.encode_verify_rows(kv, 0, q, out, H, [254], 4, 0.1, [0], window=5, sinks=1))

    def params(start, rows, valid, stride=H * D, **kw):
        return PrefillAttentionParams(start, rows, valid, H, 0.1, stride, stride, stride, **kw)

    refused(capi.ERR_INVALID_ARGUMENT, lambda: chunk.encode_causal(kv, 0, 0, q, out, params(20, 4, 23, sliding_window=5, sinks=1)))
    refused(capi.ERR_SHAPE, lambda: chunk.encode_causal(kv, 0, 0, q, out, params(20, 4, 24, H * D - 8, sliding_window=5, sinks=1)))
    refused(capi.ERR_CAPACITY, lambda: chunk.encode_causal(kv, 0, 0, q, out, params(254, 4, 258, sliding_window=5, sinks=1)))
    refused(capi.ERR_INVALID_ARGUMENT, lambda: chunk.encode_causal(kv, 0, 0, q, out, params(20, 4, 24, sliding_window=5, sinks=-1)))
    mask = torch.ones(4, 24, dtype=torch.uint8, device="cuda")
    refused(capi.ERR_INVALID_ARGUMENT, lambda: chunk.encode_causal(kv, 0, 0, q, out, params(20, 4, 24, sinks=1), keep_mask=mask))
    kv.close()
    # a ring that has overwritten the first tokens, one that keeps fewer than asked for, and what a ring with sinks serves without a window
    plain = _cache(gpu_ctx, KH, D, 0, ring=128, max_context=1000)
    refused(capi.ERR_CAPACITY, lambda: a.encode_swa(plain, 0, q, out, H, 200, 50, 0.1, sinks=1))
    plain.close()
    kept = _cache(gpu_ctx, KH, D, 0, ring=128, sinks=20, max_context=1000)
    assert kept.capacity_tokens == 160
    refused(capi.ERR_CAPACITY, lambda: a.encode_swa(kept, 0, q, out, H, 200, 50, 0.1, sinks=33))
    refused(capi.ERR_CAPACITY, lambda: a.encode_full(kept, 0, q, out, H, 200, 0.1))
    refused(capi.ERR_CAPACITY, lambda: a.encode_swa(kept, 0, q, out, H, 300, 129, 0.1, sinks=20))
    refused(capi.ERR_CAPACITY, lambda: a.encode_swa(kept, 0, q, out, H, 1025, 50, 0.1, sinks=20))
    k = torch.zeros(20, KH * D, dtype=torch.float16, device="cuda")
    refused(capi.ERR_CAPACITY, lambda: kept.append(0, 0, 150, k, k))  # over the place where the ring comes round
    kept.close()
    for ring, sinks in ((0, 4), (64, -1)):
        refused(capi.ERR_INVALID_ARGUMENT, lambda: KVCacheManager(gpu_ctx, 1, KH, D, max_context=500, ring_capacity=ring, sink_tokens=sinks))
    everything = _cache(gpu_ctx, KH, D, 0, ring=64, sinks=4, max_context=80)  # holds every position: nothing comes round
    assert everything.capacity_tokens == 96
    a.encode_full(everything, 0, q[:1], out[:1], H, 80, 0.1)
    gpu_ctx.synchronize()
    everything.close()
    assert (out[1:] == 3.0).all()


@pytest.mark.parametrize("bits", [16, 8])
def test_a_session_step_by_step_through_its_ring(gpu_ctx, bits):
    # prompt, decode steps and draft rows of one session as a runner makes them: every row written through the epilogue's neighbour, the
    # cache's append, far past the ring; a graph of one step replays it
    import torch
    from tinytitan_amd.engine import Attention, PrefillAttention, PrefillAttentionParams
    H, KH, D, window, sinks, ring = 16, 2, 256, 96, 4, 160
    total, scale = 32 + 3 * ring + 40, D ** -0.5
    r = np.random.default_rng(40)
    k16, v16 = (r.standard_normal((total, KH * D)).astype(np.float16) for _ in range(2))
    kd, vd = _dev(k16), _dev(v16)
    full = _cache(gpu_ctx, KH, D, total, bits)
    full.append(0, 0, 0, kd, vd)
    stored_k, stored_v = full.export_rows(0, 0, 0, total)  # (as the cache rounds them)
    k64, v64 = (dequantise(t.cpu().numpy(), KH * D, bits) for t in (stored_k, stored_v))
    full.close()
    kv = _cache(gpu_ctx, KH, D, 0, bits, ring=ring, sinks=sinks, max_context=total)
    attention, chunks = Attention(gpu_ctx), PrefillAttention(gpu_ctx)

    def expected(q, position):
        keys = np.arange(total)
        return attend(q, k64, v64, (keys <= position) & ((keys > position - window) | (keys < sinks)), scale, None, bits)

    at, graph = 0, None
    while at < total:
        room = 32 - at if at < 32 else ring - (at - 32) % ring
        rows = min(30 if at < 200 else 1 + at % 4, room, total - at)
        q = _rows(at, rows, H, D)
        qd, out = _dev(q), torch.full((rows, H, D), float("nan"), dtype=torch.float16, device="cuda")
        torch.cuda.synchronize()
        kv.append(0, 0, at, kd[at:at + rows], vd[at:at + rows])
        if rows > 8:
            width = H * D
            chunks.encode_causal(kv, 0, 0, qd, out, PrefillAttentionParams(at, rows, at + rows, H, scale, width, width, sliding_window=window, sinks=sinks))
        elif rows > 1:
            attention.encode_verify_rows(kv, 0, qd, out, H, [at], rows, scale, [0], window=window, sinks=sinks)
        else:
            attention.encode_swa(kv, 0, qd, out, H, at + 1, window, scale, sinks=sinks)
        kv.advance(0, rows)
        gpu_ctx.synchronize()
        check(out.cpu().numpy(), [expected(q[i], at + i) for i in range(rows)], f"position {at}, {rows} rows")
        if graph is None and rows == 1 and at > 32 + ring:
            gpu_ctx.graph_begin()
            attention.encode_swa(kv, 0, qd, out, H, at + 1, window, scale, sinks=sinks)
            graph = gpu_ctx.graph_end()
            want = out.clone()
            for _ in range(3):
                out.fill_(float("nan"))
                torch.cuda.synchronize()
                graph.launch()
                gpu_ctx.synchronize()
                assert torch.equal(out, want)
            graph.close()
        at += rows
    assert graph is not None and kv.position(0) == total
    kv.close()
