"""Sequences that share a prefix, through the C ABI, against the definition in 64 bits: key j below the prefix's length is row j of the
prefix's slot, the others are the sequence's own."""
import numpy as np
import pytest

from tests.exact_attention import attend, check, dequantise, stored_rows
from tests.test_gpu_attn_sinks import _dev, _rows, _some

pytestmark = pytest.mark.gpu


def _fill(kv, slot, at, k, v):
    import torch
    if not len(k):
        return
    kd, vd = _dev(k), _dev(v)
    torch.cuda.synchronize()
    kv.import_rows(0, slot, at, kd, vd)
    kv.ctx.synchronize()


class Family:
    """A prefix in slot ``home`` and sequences of ``lengths`` keys in all behind it; what a call must not read holds NaN."""

    def __init__(self, ctx, KH, D, prefix, lengths, bits=16, home=0, spare=40, seed=1):
        from tinytitan_amd.engine import KVCacheManager, SharedPrefix
        n, width, capacity = len(lengths), KH * D, max([prefix, *lengths]) + spare
        self.bits, self.lengths, self.prefix, self.assembled = bits, lengths, SharedPrefix(home, prefix), None
        self.kv = KVCacheManager(ctx, 1, KH, D, slots=n + 1, max_context=capacity, initial_capacity=capacity, precision_bits=bits)
        r = np.random.default_rng(seed)
        junk = stored_rows(np.ones((capacity, width)), bits)
        junk[:, 0 if bits == 16 else width * bits // 8:] = 0xff  # NaN values, or scales and biases
        self.slots = [s for s in range(n + 1) if s != home]
        for slot in self.slots:  # (below the prefix nothing of these is read)
            _fill(self.kv, slot, 0, junk[:prefix // 32 * 32], junk[:prefix // 32 * 32])
        front = [stored_rows(r.standard_normal((prefix, width)), bits) for _ in "kv"]
        _fill(self.kv, home, 0, *front)
        self.kv.advance(home, prefix)
        self.kv.share_prefix(home, prefix, self.slots)
        self.front, self.own = [dequantise(a, width, bits) for a in front], []
        for slot, length in zip(self.slots, lengths):
            assert self.kv.position(slot) == prefix
            own = [stored_rows(r.standard_normal((length - prefix, width)), bits) for _ in "kv"]
            _fill(self.kv, slot, prefix, *own)
            if prefix >= 32:  # (a shorter one is the plain call's, which takes finite values behind the last row for granted)
                _fill(self.kv, slot, length, junk[length:], junk[length:])
            self.own.append(own)

    def row(self, i, q, position, scale, gate=None):
        if self.assembled is None or self.assembled[0] != i:
            self.assembled = i, self.keys(i)
        k, v = self.assembled[1]
        return attend(q, k, v, np.arange(k[0].shape[0]) <= position, scale, gate, self.bits)

    def keys(self, i):
        width = self.front[0][0].shape[1]
        k, v = ([np.concatenate(part) for part in zip(front, dequantise(own, width, self.bits))] for front, own in zip(self.front, self.own[i]))
        return k, v


def _decode(ctx, f, q, scale, gate=None, lengths=None, slots=None):
    import torch
    from tinytitan_amd.engine import Attention
    qd, gd = _dev(q), _dev(gate) if gate is not None else None
    out = torch.full(qd.shape, float("nan"), dtype=torch.float16, device="cuda")
    torch.cuda.synchronize()
    Attention(ctx).encode_full(f.kv, 0, qd, out, q.shape[1], lengths or f.lengths, scale, slot=slots or f.slots, gate=gd, prefix=f.prefix)
    ctx.synchronize()
    return out.cpu().numpy()


@pytest.mark.parametrize("H,KH,D", [(16, 2, 256), (24, 2, 256), (32, 8, 128), (4, 1, 128), (16, 4, 64), (6, 3, 64), (64, 1, 64)])
@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("prefix", [31, 32, 33, 500, 2049])
def test_decode(gpu_ctx, H, KH, D, bits, prefix):
    # sequences that are the prefix alone, one key longer, and longer by unlike lengths
    lengths = [prefix, prefix + 1, prefix + 20, prefix + 33, prefix + 700]
    f = Family(gpu_ctx, KH, D, prefix, lengths, bits, home=2)
    q, g = _rows(3, len(lengths), H, D), _rows(4, len(lengths), H, D)
    for gate in (None, g):
        got = _decode(gpu_ctx, f, q, D ** -0.5, gate)
        check(got, [f.row(i, q[i], n - 1, D ** -0.5, None if gate is None else gate[i]) for i, n in enumerate(lengths)], f"prefix {prefix}")
    f.kv.close()


@pytest.mark.parametrize("H,KH,D,bits,prefix,n", [(16, 2, 256, 16, 9000, 70), (32, 8, 128, 8, 5000, 64), (16, 4, 64, 16, 12321, 66),
                                                  (16, 2, 256, 4, 33000, 40), (8, 2, 256, 8, 6000, 100), (16, 2, 256, 8, 20011, 64)])
def test_a_large_batch(gpu_ctx, H, KH, D, bits, prefix, n):
    # more sequences than one launch takes, and enough rows for the chunk kernel over the shared keys
    lengths = [prefix + 1 + (i * i * 7) % 300 for i in range(n)]
    f = Family(gpu_ctx, KH, D, prefix, lengths, bits)
    q, g = _rows(5, n, H, D), _rows(6, n, H, D)
    got = _decode(gpu_ctx, f, q, D ** -0.5, g)
    some = [0, 31, 32, n - 2, n - 1]
    check(got[some], [f.row(i, q[i], lengths[i] - 1, D ** -0.5, g[i]) for i in some], "batch")
    # a few of them, in another order, one of them twice
    pick = [5, 3, 3, 0]
    got = _decode(gpu_ctx, f, q[pick], D ** -0.5, g[pick], [lengths[i] for i in pick], [f.slots[i] for i in pick])
    check(got, [f.row(i, q[i], lengths[i] - 1, D ** -0.5, g[i]) for i in pick], "picked")
    f.kv.close()


@pytest.mark.parametrize("H,KH,D", [(16, 2, 256), (24, 2, 256), (32, 8, 128), (40, 8, 128), (16, 4, 64), (32, 1, 64)])
@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("prefix,n", [(900, 3), (4500, 7), (10007, 18)])
def test_few_rows_behind_a_long_prefix(gpu_ctx, H, KH, D, bits, prefix, n):
    # tiles that the tokens of several sequences share, whole and ragged, over any number of splits; own keys of one split and of several
    lengths = [prefix + 1 + (i * 37) % 90 + (1500 if i == n - 1 else 0) for i in range(n)]
    f = Family(gpu_ctx, KH, D, prefix, lengths, bits, home=n)
    q, g = _rows(13, n, H, D), _rows(14, n, H, D)
    got = _decode(gpu_ctx, f, q, D ** -0.5, g)
    some = sorted({0, n // 2, n - 1})
    check(got[some], [f.row(i, q[i], lengths[i] - 1, D ** -0.5, g[i]) for i in some], "rows")
    f.kv.close()


@pytest.mark.parametrize("H,KH,D,bits,prefix,rows", [(16, 2, 256, 16, 1000, 4), (24, 2, 256, 4, 2345, 3), (32, 8, 128, 8, 700, 5), (16, 4, 64, 16, 64, 8),
                                                     (16, 2, 256, 16, 5000, 17), (8, 2, 256, 16, 100, 400)])
def test_verify_rows(gpu_ctx, H, KH, D, bits, prefix, rows):
    import torch
    from tinytitan_amd.engine import Attention
    starts = [prefix - 1, prefix, prefix + 45, prefix + 500]
    f = Family(gpu_ctx, KH, D, prefix, [p + rows for p in starts], bits, home=4)
    q, g = _rows(7, len(starts), rows, H, D), _rows(8, len(starts), rows, H, D)
    qd, gd = _dev(q), _dev(g)
    out = torch.full(qd.shape, float("nan"), dtype=torch.float16, device="cuda")
    torch.cuda.synchronize()
    Attention(gpu_ctx).encode_verify_rows(f.kv, 0, qd, out, H, starts, rows, D ** -0.5, f.slots, gate=gd, prefix=f.prefix)
    gpu_ctx.synchronize()
    got, some = out.cpu().numpy(), _some(rows)
    for i, p in enumerate(starts):
        check(got[i][some], [f.row(i, q[i, r], p + r, D ** -0.5, g[i, r]) for r in some], f"sequence {i}")
    f.kv.close()


@pytest.mark.parametrize("H,KH,D,bits,prefix,start,rows,pad,offset", [
    (16, 2, 256, 16, 700, 0, 1, 0, 0), (16, 2, 256, 16, 700, 0, 300, 0, 0), (16, 2, 256, 16, 5000, 10, 130, 8, 8), (16, 2, 256, 8, 5000, 100, 90, 0, 0),
    (16, 2, 256, 16, 4100, 7, 2100, 0, 0), (24, 2, 256, 16, 3333, 40, 600, 0, 0), (32, 8, 128, 16, 2000, 33, 777, 0, 0), (32, 8, 128, 4, 900, 1, 333, 0, 0),
    (32, 8, 128, 16, 321, 0, 3000, 0, 0), (16, 4, 64, 16, 1500, 250, 1234, 72, 0), (16, 4, 64, 8, 8000, 31, 64, 5, 3), (6, 3, 64, 16, 100, 0, 200, 0, 1),
    (40, 8, 128, 16, 40, 3, 700, 0, 0), (16, 2, 256, 8, 3000, 20, 2500, 0, 0), (16, 2, 256, 16, 20, 5, 100, 0, 0), (64, 8, 64, 16, 96, 0, 1500, 0, 0),
    (32, 8, 128, 8, 4100, 500, 1800, 0, 0), (16, 2, 256, 16, 16383, 1, 300, 0, 0)])
def test_chunk(gpu_ctx, H, KH, D, bits, prefix, start, rows, pad, offset):
    import torch
    from tinytitan_amd.engine import PrefillAttention, PrefillAttentionParams
    first = prefix + start
    f = Family(gpu_ctx, KH, D, prefix, [first + rows + 13, first + 5], bits, home=1)
    q, g = _rows(9, rows, H, D), _rows(10, rows, H, D)
    width, stride = H * D, H * D + pad

    def wide(a):
        t = torch.full((rows * stride + offset,), 7.0, dtype=torch.float16, device="cuda")
        t[offset:].view(rows, stride)[:, :width] = _dev(a).view(rows, width)
        return t

    some = _some(rows)
    for gate, valid, scale in ((g, first + rows, D ** -0.5), (None, first + rows + 13, -D ** -0.5)):
        qd, gd = wide(q), wide(gate) if gate is not None else None
        out = torch.full((rows * stride + offset + 64,), float("nan"), dtype=torch.float16, device="cuda")
        params = PrefillAttentionParams(first, rows, valid, H, scale, stride, stride, stride)
        torch.cuda.synchronize()
        PrefillAttention(gpu_ctx).encode_causal(f.kv, 0, f.slots[0], qd[offset:], out[offset:], params,
                                                gate=gd[offset:] if gd is not None else None, prefix=f.prefix)
        gpu_ctx.synchronize()
        res = out.cpu().numpy()
        body = res[offset:offset + rows * stride].reshape(rows, stride)
        assert np.isnan(res[:offset]).all() and np.isnan(body[:, width:]).all() and np.isnan(res[offset + rows * stride:]).all()
        got = body[:, :width].reshape(rows, H, D)
        check(got[some], [f.row(0, q[r], first + r, scale, None if gate is None else gate[r]) for r in some], f"scale {scale}")
    f.kv.close()


def test_the_last_part_block_of_every_layer_is_copied_and_nothing_else(gpu_ctx):
    import torch
    from tinytitan_amd.engine import KVCacheManager
    KH, D, layers, slots = 3, 64, 70, 5
    for bits in (16, 8, 4):
        for prefix in (1, 31, 64, 77):
            kv = KVCacheManager(gpu_ctx, layers, KH, D, slots=slots, max_context=128, initial_capacity=128, precision_bits=bits)
            rows = _dev(_rows(prefix, layers, 128, KH * D))
            marks = torch.full((128, KH * D), 3.0, dtype=torch.float16, device="cuda")
            torch.cuda.synchronize()
            for layer in range(layers):
                kv.append(layer, 2, 0, rows[layer], rows[layer])
                for slot in (0, 1, 3, 4):
                    kv.append(layer, slot, 0, marks, marks)
            kv.advance(2, 100)
            kv.advance(0, 9)
            kv.share_prefix(2, prefix, [0, 4])
            assert [kv.position(s) for s in range(slots)] == [prefix, 0, 100, 0, prefix]
            for layer in (0, 33, 63, 64, 69):
                want, _ = kv.read(layer, 2, 0, 128)
                mark, _ = kv.read(layer, 1, 0, 128)
                for slot in (0, 1, 3, 4):
                    copied = slice(prefix // 32 * 32, prefix // 32 * 32 + (32 if slot in (0, 4) and prefix % 32 else 0))
                    for got in kv.read(layer, slot, 0, 128):
                        expected = mark.clone()
                        expected[copied] = want[copied]
                        assert torch.equal(got, expected), (bits, prefix, layer, slot)
            kv.close()


def test_refusals(gpu_ctx):
    import torch
    from tinytitan_amd import capi
    from tinytitan_amd.engine import (Attention, KVCacheManager, PrefillAttention, PrefillAttentionParams, SharedPrefix, TinyTitanHIPError)
    H, KH, D = 8, 2, 64
    kv = KVCacheManager(gpu_ctx, 1, KH, D, slots=4, max_context=256, initial_capacity=256)
    q = torch.zeros(4, H, D, dtype=torch.float16, device="cuda")
    out = torch.full_like(q, 3.0)
    a, chunk = Attention(gpu_ctx), PrefillAttention(gpu_ctx)

    def refused(status, call):
        with pytest.raises(TinyTitanHIPError) as e:
            call()
        assert e.value.status == status

    bad = capi.ERR_INVALID_ARGUMENT
    refused(capi.ERR_CURSOR, lambda: kv.share_prefix(0, 64, [1]))
    kv.advance(0, 100)
    refused(capi.ERR_CURSOR, lambda: kv.share_prefix(0, 101, [1]))
    for slot, length, slots in ((0, 64, [0, 1]), (0, 64, [4]), (0, 64, [-1]), (0, 64, []), (4, 64, [1]), (-1, 64, [1]), (0, -1, [1])):
        refused(bad, lambda: kv.share_prefix(slot, length, slots))
    refused(capi.ERR_CAPACITY, lambda: kv.share_prefix(0, 257, [1]))
    assert [kv.position(s) for s in range(4)] == [100, 0, 0, 0]
    kv.share_prefix(0, 70, [1, 2])
    p = SharedPrefix(0, 70)
    for lengths, slots in (([69], [1]), ([80, 69], [1, 2]), ([80, 80], [1]), ([80], [9]), ([-1], [1])):
        refused(bad, lambda: a.encode_full(kv, 0, q, out, H, lengths, 0.1, slot=slots, prefix=p))
    for prefix in (SharedPrefix(4, 70), SharedPrefix(-1, 70), SharedPrefix(0, -1)):
        refused(bad, lambda: a.encode_full(kv, 0, q, out, H, [80], 0.1, slot=[1], prefix=prefix))
    refused(bad, lambda: a.encode_full(kv, 0, q, out, H, [10], 0.1, slot=[1], prefix=SharedPrefix(0, 20)))
    refused(capi.ERR_CAPACITY, lambda: a.encode_full(kv, 0, q, out, H, [300], 0.1, slot=[1], prefix=SharedPrefix(0, 260)))
    refused(capi.ERR_CAPACITY, lambda: a.encode_full(kv, 0, q, out, H, [257], 0.1, slot=[1], prefix=p))
    refused(capi.ERR_SHAPE, lambda: a.encode_full(kv, 0, q, out, 7, [80], 0.1, slot=[1], prefix=p))
    refused(bad, lambda: a.encode_full(kv, 1, q, out, H, [80], 0.1, slot=[1], prefix=p))
    refused(bad, lambda: a.encode_verify_rows(kv, 0, q, out, H, [68], 2, 0.1, [1], prefix=p))
    refused(bad, lambda: a.encode_verify_rows(kv, 0, q, out, H, [70], 0, 0.1, [1], prefix=p))
    refused(bad, lambda: a.encode_verify_rows(kv, 0, q, out, H, [70], 2, 0.1, [1], window=9, prefix=p))
    refused(capi.ERR_CAPACITY, lambda: a.encode_verify_rows(kv, 0, q, out, H, [255], 2, 0.1, [1], prefix=p))

    def params(start, rows, valid, stride=H * D, **kw):
        return PrefillAttentionParams(start, rows, valid, H, 0.1, stride, stride, stride, **kw)

    refused(bad, lambda: chunk.encode_causal(kv, 0, 1, q, out, params(68, 4, 72), prefix=p))
    refused(bad, lambda: chunk.encode_causal(kv, 0, 1, q, out, params(70, 4, 73), prefix=p))
    refused(bad, lambda: chunk.encode_causal(kv, 0, 1, q, out, params(70, 4, 74, sliding_window=9), prefix=p))
    refused(capi.ERR_SHAPE, lambda: chunk.encode_causal(kv, 0, 1, q, out, params(70, 4, 74, H * D - 8), prefix=p))
    refused(capi.ERR_CAPACITY, lambda: chunk.encode_causal(kv, 0, 1, q, out, params(254, 4, 258), prefix=p))
    kv.close()
    ring = KVCacheManager(gpu_ctx, 1, KH, D, slots=2, max_context=500, ring_capacity=128)
    refused(capi.ERR_SHAPE, lambda: ring.share_prefix(0, 0, [1]))
    refused(capi.ERR_SHAPE, lambda: a.encode_full(ring, 0, q, out, H, [80], 0.1, slot=[1], prefix=SharedPrefix(0, 64)))
    ring.close()
    gpu_ctx.synchronize()
    assert (out == 3.0).all()


def test_the_prefix_slot_among_the_sequences_and_a_prefix_of_nothing(gpu_ctx):
    import torch
    from tinytitan_amd.engine import Attention, SharedPrefix
    H, KH, D, prefix = 16, 2, 256, 333
    f = Family(gpu_ctx, KH, D, prefix, [400, 350], home=0)
    q = _rows(11, 3, H, D)
    got = _decode(gpu_ctx, f, q, 0.0625, None, [prefix, 400, 350], [0, 1, 2])
    check(got, [f.row(0, q[0], prefix - 1, 0.0625), f.row(0, q[1], 399, 0.0625), f.row(1, q[2], 349, 0.0625)], "the prefix's own slot")
    qd, outs = _dev(q[:1]), [torch.zeros(1, H, D, dtype=torch.float16, device="cuda") for _ in range(2)]
    torch.cuda.synchronize()
    a = Attention(gpu_ctx)
    a.encode_full(f.kv, 0, qd, outs[0], H, [prefix], 0.0625, slot=[0])
    a.encode_full(f.kv, 0, qd, outs[1], H, [prefix], 0.0625, slot=[0], prefix=SharedPrefix(0, 0))
    gpu_ctx.synchronize()
    assert torch.equal(*outs)
    f.kv.close()


@pytest.mark.parametrize("bits", [16, 8])
def test_a_batch_of_sessions_step_by_step(gpu_ctx, bits):
    # a system prompt in one slot; sessions start from it with a chunk of their own each, then decode and verify together; a graph of a
    # step replays it, and a prefix under way grows nothing while it is captured
    import torch
    from tinytitan_amd import capi
    from tinytitan_amd.engine import Attention, HIPContext, KVCacheManager, PrefillAttention, PrefillAttentionParams, SharedPrefix, TinyTitanHIPError
    ctx = HIPContext(0)
    H, KH, D, prefix, n, scale = 16, 2, 256, 2077, 5, 0.0625
    width = H * D
    kv = KVCacheManager(ctx, 2, KH, D, slots=n + 1, max_context=4096, initial_capacity=2112, precision_bits=bits)
    r = np.random.default_rng(3)

    def rows(count):
        return [r.standard_normal((count, KH * D)).astype(np.float16) for _ in range(4)]  # k, v of two layers

    history = [[np.zeros((0, KH * D), np.float16)] * 4 for _ in range(n + 1)]

    def append(slot, at, new):
        dev = [_dev(a) for a in new]
        torch.cuda.synchronize()
        for layer in range(2):
            kv.append(layer, slot, at, dev[2 * layer], dev[2 * layer + 1])
        ctx.synchronize()
        history[slot] = [np.concatenate([a, b]) for a, b in zip(history[slot], new)]

    scratch = KVCacheManager(ctx, 1, KH, D, slots=1, max_context=4096, initial_capacity=4096, precision_bits=bits)

    def stored(a):  # as the cache rounds rows
        d = _dev(a)
        torch.cuda.synchronize()
        scratch.append(0, 0, 0, d, d)
        return dequantise(scratch.export_rows(0, 0, 0, len(a))[0].cpu().numpy(), KH * D, bits)

    def expected(slot, layer, q, position):
        k, v = stored(history[slot][2 * layer]), stored(history[slot][2 * layer + 1])
        return attend(q, k, v, np.arange(len(k[0])) <= position, scale, None, bits)

    append(0, 0, rows(prefix))
    kv.advance(0, prefix)
    kv.share_prefix(0, prefix, list(range(1, n + 1)))
    p = SharedPrefix(0, prefix)
    for slot in range(1, n + 1):
        history[slot] = list(history[0])
    attention, chunks = Attention(ctx), PrefillAttention(ctx)
    positions = [prefix] * n
    kv.reserve(3000)  # (the stores move: the copied part block with them)
    for i in range(n):
        count = [1, 40, 100, 7, 333][i]
        append(i + 1, prefix, rows(count))
        kv.advance(i + 1, count)
        q = _rows(60 + i, count, H, D)
        qd, out = _dev(q), torch.zeros(count, H, D, dtype=torch.float16, device="cuda")
        torch.cuda.synchronize()
        chunks.encode_causal(kv, 1, i + 1, qd, out, PrefillAttentionParams(prefix, count, prefix + count, H, scale, width, width, width), prefix=p)
        ctx.synchronize()
        some = sorted({0, count // 2, count - 1})
        check(out.cpu().numpy()[some], [expected(i + 1, 1, q[t], prefix + t) for t in some], f"first chunk of {i}")
        positions[i] += count
    for step, count in enumerate((1, 3, 1)):
        for i in range(n):
            append(i + 1, positions[i], rows(count))
        q = _rows(80 + step, n, count, H, D)
        qd = _dev(q)
        for layer in range(2):
            out = torch.zeros(n, count, H, D, dtype=torch.float16, device="cuda")
            torch.cuda.synchronize()

            def call():
                if count == 1:
                    attention.encode_full(kv, layer, qd, out, H, [x + 1 for x in positions], scale, slot=list(range(1, n + 1)), prefix=p)
                else:
                    attention.encode_verify_rows(kv, layer, qd, out, H, positions, count, scale, list(range(1, n + 1)), prefix=p)

            call()
            ctx.synchronize()
            got = out.cpu().numpy()
            for i in range(n):
                check(got[i], [expected(i + 1, layer, q[i, t], positions[i] + t) for t in range(count)], f"step {step}, sequence {i}")
            if step == 2:
                want = out.clone()
                ctx.graph_begin()
                call()
                graph = ctx.graph_end()
                for _ in range(3):
                    out.zero_()
                    torch.cuda.synchronize()
                    graph.launch()
                    ctx.synchronize()
                    assert torch.equal(out, want)
                    call()
                    ctx.synchronize()
                graph.close()
        for i in range(n):
            positions[i] += count
            kv.advance(i + 1, count)
    # a capture whose call would have to grow a store is refused and goes on
    big, slots = _dev(_rows(90, n, 200, H, D)), list(range(1, n + 1))
    out = torch.zeros_like(big)
    ctx.graph_begin()
    with pytest.raises(TinyTitanHIPError) as e:
        attention.encode_verify_rows(kv, 0, big, out, H, positions, 200, scale, slots, prefix=p)
    assert e.value.status == capi.ERR_BUSY
    ctx.graph_end().close()
    scratch.close()
    kv.close()
    ctx.close()
