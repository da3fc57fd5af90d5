"""Differential attention through the C ABI against the definition in 64 bits: the difference of two softmax maps over the cache, as a decode
step, as verify rows and as a chunk."""
import numpy as np
import pytest

from tests.exact_attention import stored_rows
from tests.exact_maps import attend_maps, check

pytestmark = pytest.mark.gpu

SHAPES = [(16, 2, 256), (8, 2, 256), (24, 2, 256), (32, 8, 128), (12, 4, 128), (16, 4, 64), (6, 3, 64), (3, 1, 128), (34, 2, 64), (1, 1, 256)]


def _dev(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).to("cuda")


def _randn(seed, *shape):
    return _dev(np.random.default_rng(seed).standard_normal(shape).astype(np.float16))


class Layer:
    """A cache with rows of its sequences, and the heads' factors."""

    def __init__(self, ctx, H, KH, D, lengths, bits=16, window=0, ring=0, extra=0, seed=0, max_context=None):
        from tinytitan_amd.engine import DifferentialAttention, KVCacheManager
        self.ctx, self.H, self.KH, self.D, self.bits, self.window, self.scale = ctx, H, KH, D, bits, window, (D // 2) ** -0.5
        capacity = max(max(lengths) + extra, 32)
        self.kv = KVCacheManager(ctx, 1, KH, D, slots=len(lengths), max_context=max_context or capacity, initial_capacity=capacity, precision_bits=bits,
                                 ring_capacity=ring)
        self.attention = DifferentialAttention(ctx)
        r = np.random.default_rng(seed + 1000)
        self.rows = []
        for slot, n in enumerate(lengths):
            k, v = (stored_rows(r.standard_normal((n, KH * D)), bits) for _ in range(2))
            self.rows.append((k, v))
            self.write(slot, 0, k, v, ring)
        self.norm = (1.0 + 0.2 * r.standard_normal(D)).astype(np.float32)
        self.lambdas = (0.2 + 0.6 * r.random(H)).astype(np.float32)

    def write(self, slot, at, k, v, ring=0):
        import torch
        done = 0
        while done < k.shape[0]:
            n = k.shape[0] - done
            if ring:
                n = min(n, ring - (at + done) % ring)
            kd, vd = _dev(k[done:done + n]), _dev(v[done:done + n])
            torch.cuda.synchronize()
            self.kv.import_rows(0, slot, at + done, kd, vd)
            self.ctx.synchronize()
            done += n

    def heads(self, lambdas=None, normed=True, eps=1e-5, out_scale=0.3):
        import torch
        from tinytitan_amd.engine import DifferentialHeads
        norm = _dev(self.norm).bfloat16() if normed else None
        lambdas = _dev(self.lambdas if lambdas is None else lambdas)
        torch.cuda.synchronize()
        return DifferentialHeads(lambdas, norm_weight=norm, eps=eps, out_scale=out_scale)

    def want(self, q, slot, positions, heads, gate=None, lambdas=None, first=0):
        """q [rows, heads, dim]; the rows from `first` on are in the cache."""
        k, v = self.rows[slot]
        n = max(positions) + 1
        return attend_maps(q, k[first:n], v[first:n], self.KH, positions, np.arange(first, n), self.window, self.scale,
                           heads.lambdas if lambdas is None else lambdas, self.bits, heads.norm_weight, heads.eps, heads.out_scale, gate)

    def decode(self, q, seq_lens, heads, gate=None, slots=None):
        import torch
        out = torch.full(q.shape, float("nan"), dtype=torch.float16, device="cuda")
        torch.cuda.synchronize()
        self.attention.encode_full(self.kv, 0, q, out, self.H, list(seq_lens), self.scale, heads, slot=slots or list(range(len(seq_lens))),
                                   gate=gate, window=self.window)
        self.ctx.synchronize()
        return out

    def verify(self, q, starts, rows, heads, gate=None, slots=None):
        import torch
        out = torch.full(q.shape, float("nan"), dtype=torch.float16, device="cuda")
        torch.cuda.synchronize()
        self.attention.encode_verify_rows(self.kv, 0, q, out, self.H, list(starts), rows, self.scale, heads, slots or list(range(len(starts))),
                                          gate=gate, window=self.window)
        self.ctx.synchronize()
        return out

    def chunk(self, q, start, heads, gate=None, slot=0, pad=0, kv_valid=None, scale=None):
        """q [rows, heads, dim], laid out `pad` elements wider than a row; what lies between the rows has to stay."""
        import torch
        from tinytitan_amd.engine import PrefillAttentionParams
        rows, width = q.shape[0], self.H * self.D
        wide = [None if t is None else torch.full((rows, width + pad), 7.0, dtype=torch.float16, device="cuda") for t in (q, gate, q)]
        wide[0][:, :width] = q.reshape(rows, width)
        if gate is not None:
            wide[1][:, :width] = gate.reshape(rows, width)
        torch.cuda.synchronize()
        params = PrefillAttentionParams(start, rows, kv_valid or start + rows, self.H, scale or self.scale, width + pad, width + pad, width + pad,
                                        sliding_window=self.window)
        self.attention.encode_causal(self.kv, 0, slot, wide[0], wide[2], params, heads, gate=wide[1])
        self.ctx.synchronize()
        assert (wide[2][:, width:] == 7.0).all()
        return wide[2][:, :width].reshape(rows, self.H, self.D).contiguous()

    def close(self):
        self.kv.close()


@pytest.mark.parametrize("H,KH,D", SHAPES)
@pytest.mark.parametrize("bits", [16, 8, 4])
def test_decode(gpu_ctx, H, KH, D, bits):
    layer = Layer(gpu_ctx, H, KH, D, [1500], bits)
    for i, at in enumerate((1, 2, 31, 32, 33, 64, 65, 129, 385, 600, 1500)):
        q, gate = _randn(at, 1, H, D), _randn(at + 1, 1, H, D) if i % 2 else None
        heads = layer.heads(normed=i % 3 != 0)
        check(layer.decode(q, [at], heads, gate), layer.want(q, 0, [at - 1], heads, gate), f"{at} keys")
    layer.close()


@pytest.mark.parametrize("H,KH,D,bits", [(16, 2, 256, 16), (32, 8, 128, 8), (16, 4, 64, 4), (24, 2, 256, 8)])
@pytest.mark.parametrize("window", [0, 500])
def test_decode_batch_of_all_ages(gpu_ctx, H, KH, D, bits, window):
    lengths = [1, 5, 100, 501, 502, 533, 3000, 7001, 900]
    layer = Layer(gpu_ctx, H, KH, D, lengths, bits, window)
    n = len(lengths)
    q, gate = _randn(1, n, H, D), _randn(2, n, H, D)
    by_token = np.random.default_rng(3).random((n, H)).astype(np.float32)
    for lambdas in (None, by_token):
        heads = layer.heads(lambdas)
        got = layer.decode(q, lengths, heads, gate)
        for i, length in enumerate(lengths):
            check(got[i:i + 1], layer.want(q[i:i + 1], i, [length - 1], heads, gate[i:i + 1], None if lambdas is None else _dev(lambdas)[i]), f"{length} keys")
    layer.close()


def test_factors_by_token_in_rows_of_a_wider_buffer(gpu_ctx):
    import torch
    from tinytitan_amd.engine import DifferentialHeads
    H, KH, D, lengths = 16, 2, 256, [40, 700, 90]
    layer = Layer(gpu_ctx, H, KH, D, lengths)
    wide = _dev(np.random.default_rng(1).random((3, H + 5)).astype(np.float32))
    heads = DifferentialHeads(wide[:, 2:2 + H], norm_weight=_dev(layer.norm).bfloat16())
    q = _randn(5, 3, H, D)
    torch.cuda.synchronize()
    got = layer.decode(q, lengths, heads)
    for i, length in enumerate(lengths):
        check(got[i:i + 1], layer.want(q[i:i + 1], i, [length - 1], heads, lambdas=wide[i, 2:2 + H]), f"sequence {i}")
    layer.close()


@pytest.mark.parametrize("D,bits", [(256, 16), (64, 8)])
def test_more_sequences_than_a_launch_takes(gpu_ctx, D, bits):
    # 70 rows: two launches, the factors of the second found behind the first one's; the same slot more than once
    H, KH = 8, 2
    layer = Layer(gpu_ctx, H, KH, D, [300, 77], bits)
    n = 70
    r = np.random.default_rng(9)
    slots, lens = [i % 2 for i in range(n)], [int(r.integers(1, 300 if i % 2 == 0 else 77)) for i in range(n)]
    q, lambdas = _randn(4, n, H, D), r.random((n, H)).astype(np.float32)
    heads = layer.heads(lambdas)
    got = layer.decode(q, lens, heads, slots=slots)
    for i in range(n):
        check(got[i:i + 1], layer.want(q[i:i + 1], slots[i], [lens[i] - 1], heads, lambdas=_dev(lambdas)[i]), f"sequence {i}")
    layer.close()


def test_sequences_without_keys_give_zeros(gpu_ctx):
    H, KH, D = 16, 2, 256
    layer = Layer(gpu_ctx, H, KH, D, [64, 1000, 64])
    q, gate = _randn(1, 3, H, D), _randn(2, 3, H, D)
    for eps in (1e-5, 0.0):
        heads = layer.heads(eps=eps)
        for lens in ([0, 1000, 0], [0, 0, 0], [0, 5, 33]):
            got = layer.decode(q, lens, heads, gate)
            for i, n in enumerate(lens):
                if n == 0:
                    assert (got[i] == 0).all()
                else:
                    check(got[i:i + 1], layer.want(q[i:i + 1], i, [n - 1], heads, gate[i:i + 1]))
    layer.close()


def test_maps_that_cancel_give_zeros_behind_the_norm(gpu_ctx):
    # both maps the same and lambda 1: the difference is exactly zero, whatever eps is
    import torch
    H, KH, D = 4, 2, 128
    layer = Layer(gpu_ctx, H, KH, D, [700])
    k = layer.rows[0][0].view(np.float16).reshape(700, KH, 2, D // 2).copy()
    k[:, :, 1] = k[:, :, 0]
    layer.write(0, 0, k.reshape(700, -1).view(np.uint8), layer.rows[0][1])
    half = _randn(3, 1, H, D // 2)
    q = torch.cat([half, half], -1).contiguous()
    for eps in (1e-5, 0.0):
        got = layer.decode(q, [700], layer.heads(np.ones(H, np.float32), eps=eps))
        assert (got == 0).all()
    layer.close()


@pytest.mark.parametrize("H,KH,D", SHAPES)
@pytest.mark.parametrize("bits", [16, 8, 4])
def test_verify_rows(gpu_ctx, H, KH, D, bits):
    rows, starts = 5, [0, 30, 700]
    layer = Layer(gpu_ctx, H, KH, D, [s + rows for s in starts], bits)
    q, gate = _randn(1, 3, rows, H, D), _randn(2, 3, rows, H, D)
    lambdas = np.random.default_rng(4).random((3 * rows, H)).astype(np.float32)
    heads = layer.heads(lambdas)
    got = layer.verify(q, starts, rows, heads, gate)
    for i, start in enumerate(starts):
        check(got[i], layer.want(q[i], i, [start + r for r in range(rows)], heads, gate[i], _dev(lambdas)[i * rows:(i + 1) * rows]), f"from {start}")
    layer.close()


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("D,window", [(256, 96), (128, 200), (64, 63)])
def test_ring(gpu_ctx, bits, D, window):
    H, KH, rows = 8, 2, 4
    ring = (window + rows + 30 + 31) // 32 * 32
    length = 5 * ring + 17
    layer = Layer(gpu_ctx, H, KH, D, [length], bits, window, ring, max_context=length)
    heads = layer.heads()
    first = max(0, length - ring)
    q = _randn(1, 1, H, D)
    check(layer.decode(q, [length], heads), layer.want(q, 0, [length - 1], heads, first=first), "decode")
    q = _randn(2, 1, rows, H, D)
    start = length - rows
    check(layer.verify(q, [start], rows, heads)[0], layer.want(q[0], 0, list(range(start, length)), heads, first=first), "verify")
    q = _randn(3, rows, H, D)
    check(layer.chunk(q, start, heads), layer.want(q, 0, list(range(start, length)), heads, first=first), "chunk")
    layer.close()


CHUNKS = [  # rows, start, pad
    (1, 0, 0), (2, 0, 5), (31, 1, 0), (32, 0, 8), (33, 40, 0), (65, 31, 3), (96, 500, 72), (130, 0, 0), (257, 900, 0), (300, 3, 8)]


@pytest.mark.parametrize("H,KH,D", SHAPES)
@pytest.mark.parametrize("bits", [16, 8])
def test_chunk(gpu_ctx, H, KH, D, bits):
    layer = Layer(gpu_ctx, H, KH, D, [1200], bits)
    for i, (rows, start, pad) in enumerate(CHUNKS):
        q, gate = _randn(i, rows, H, D), _randn(i + 50, rows, H, D) if i % 2 else None
        lambdas = np.random.default_rng(i).random((rows, H)).astype(np.float32) if i % 3 == 0 else None
        heads = layer.heads(lambdas, normed=i % 4 != 1)
        got = layer.chunk(q, start, heads, gate, pad=pad)
        check(got, layer.want(q, 0, list(range(start, start + rows)), heads, gate), f"{rows} rows behind {start}")
    layer.close()


@pytest.mark.parametrize("H,KH,D,bits,rows,start,window", [
    (16, 2, 256, 16, 1100, 0, 0), (16, 2, 256, 16, 1030, 777, 0), (16, 2, 256, 16, 130, 9000, 0), (24, 2, 256, 8, 520, 3000, 0), (32, 8, 128, 8, 777, 4000, 0),
    (16, 4, 64, 16, 1500, 500, 0), (16, 4, 64, 4, 600, 100, 0), (12, 4, 128, 16, 900, 33, 0), (8, 2, 256, 16, 2050, 0, 0), (16, 2, 256, 16, 1500, 3000, 700),
    (32, 8, 128, 16, 2100, 50, 64), (16, 4, 64, 8, 1999, 4000, 1000), (32, 8, 128, 8, 1100, 900, 256), (6, 3, 64, 16, 1000, 1000, 0)])
def test_long_chunk(gpu_ctx, H, KH, D, bits, rows, start, window):
    layer = Layer(gpu_ctx, H, KH, D, [start + rows], bits, window)
    q, gate = _randn(1, rows, H, D), _randn(2, rows, H, D)
    heads = layer.heads(np.random.default_rng(5).random((rows, H)).astype(np.float32))
    got = layer.chunk(q, start, heads, gate)
    # (some rows of every tile, all of the first and the last ones)
    some = sorted(set(range(0, rows, 7)) | set(range(40)) | set(range(rows - 40, rows)))
    import torch
    at = torch.tensor(some, device="cuda")
    check(got[at], layer.want(q[at], 0, [start + r for r in some], heads, gate[at], heads.lambdas[at]))
    layer.close()


@pytest.mark.parametrize("bits", [16, 8, 4])
def test_what_no_row_sees_does_not_reach_them(gpu_ctx, bits):
    # rows behind the sequence, and in front of its window, that hold infinities and NaN
    H, KH, D, window, length = 16, 2, 256, 200, 900
    layer = Layer(gpu_ctx, H, KH, D, [length], bits, window, extra=100)
    width = KH * D
    bad = np.full((100, width), np.inf, np.float16)
    bad[::2] = np.nan
    if bits == 16:
        stale = bad.view(np.uint8).reshape(100, -1)
    else:
        stale = np.full((100, layer.kv.token_stride_bytes), 255, np.uint8)  # (a scale and a bias of all ones are NaN)
    layer.write(0, length, stale, stale)
    layer.write(0, 0, stale, stale)
    heads = layer.heads()
    for at in (length, length - 1, 400):
        if at == 400:
            layer.write(0, 401, stale[:50], stale[:50])
        q = _randn(at, 1, H, D)
        check(layer.decode(q, [at], heads), layer.want(q, 0, [at - 1], heads, first=at - window), f"{at} keys")
    layer.write(0, 401, *(x[401:451] for x in layer.rows[0]))
    for rows in (7, 64, 500):
        q, start = _randn(rows, rows, H, D), length - rows
        first = start + 1 - window
        check(layer.chunk(q, start, heads), layer.want(q, 0, list(range(start, length)), heads, first=first), f"{rows} rows")
    q = _randn(2, 1, 6, H, D)
    check(layer.verify(q, [length - 6], 6, heads)[0], layer.want(q[0], 0, list(range(length - 6, length)), heads, first=length - 5 - window), "verify")
    layer.close()


@pytest.mark.parametrize("scale", [-0.1, 1e-4, 2.0])
def test_scales(gpu_ctx, scale):
    H, KH, D = 16, 4, 64
    layer = Layer(gpu_ctx, H, KH, D, [700])
    layer.scale = scale
    heads = layer.heads()
    q = _randn(1, 300, H, D)
    check(layer.chunk(q, 400, heads), layer.want(q, 0, list(range(400, 700)), heads))
    check(layer.decode(q[:1], [650], heads), layer.want(q[:1], 0, [649], heads))
    layer.close()


def test_scale_zero_weighs_every_key_the_same(gpu_ctx):
    H, KH, D = 16, 4, 64
    layer = Layer(gpu_ctx, H, KH, D, [600])
    layer.scale = 0.0
    heads = layer.heads(np.full(H, 0.25, np.float32))
    q = _randn(1, 1, H, D)
    check(layer.decode(q, [600], heads), layer.want(q, 0, [599], heads))
    layer.close()


def test_keys_behind_the_chunk_are_valid_but_not_seen(gpu_ctx):
    H, KH, D = 16, 2, 256
    layer = Layer(gpu_ctx, H, KH, D, [2000])
    heads = layer.heads()
    for rows, start in ((50, 100), (1030, 200)):
        q = _randn(rows, rows, H, D)
        check(layer.chunk(q, start, heads, kv_valid=2000), layer.want(q, 0, list(range(start, start + rows)), heads), f"{rows} rows")
    layer.close()


def test_long_contexts(gpu_ctx):
    for H, KH, D, bits in ((16, 2, 256, 16), (32, 8, 128, 8), (16, 4, 64, 4)):
        # (levels' bounds add up over 60,001 keys to as much as the difference: of those the difference itself is looked at, not the norm of it)
        layer = Layer(gpu_ctx, H, KH, D, [60001], bits)
        heads = layer.heads(normed=bits == 16)
        q, gate = _randn(1, 1, H, D), _randn(2, 1, H, D)
        check(layer.decode(q, [60001], heads, gate), layer.want(q, 0, [60000], heads, gate), "decode")
        rows = 40
        q = _randn(3, rows, H, D)
        check(layer.chunk(q, 59961, heads), layer.want(q, 0, list(range(59961, 60001)), heads), "chunk")
        layer.close()


def test_slots_past_four_gibibytes(gpu_ctx):
    from tinytitan_amd.engine import DifferentialAttention, KVCacheManager
    H, KH, D, slots, capacity = 16, 2, 256, 40, 131072
    layer = Layer(gpu_ctx, H, KH, D, [500])
    layer.kv.close()
    layer.kv = KVCacheManager(gpu_ctx, 1, KH, D, slots=slots, max_context=capacity, initial_capacity=capacity)
    layer.write(slots - 1, 0, *layer.rows[0])
    heads = layer.heads()
    q = _randn(1, 1, H, D)
    check(layer.decode(q, [500], heads, slots=[slots - 1]), layer.want(q, 0, [499], heads), "decode")
    q = _randn(2, 400, H, D)
    check(layer.chunk(q, 100, heads, slot=slots - 1), layer.want(q, 0, list(range(100, 500)), heads), "chunk")
    layer.close()


def test_captured_steps_replay_as_they_ran(gpu_ctx):
    # decode, verify and chunk in one graph; between its replays the context's other work, and new queries
    import torch
    H, KH, D = 16, 2, 256
    layer = Layer(gpu_ctx, H, KH, D, [3000, 800])
    from tinytitan_amd.engine import PrefillAttentionParams
    heads, scale, att, kv = layer.heads(), layer.scale, layer.attention, layer.kv
    qs = [_randn(1, 2, H, D), _randn(2, 2, 3, H, D), _randn(3, 1100, H, D)]
    outs = [torch.zeros_like(q) for q in qs]
    params = PrefillAttentionParams(1500, 1100, 2600, H, scale, H * D, H * D)
    torch.cuda.synchronize()

    def step():
        att.encode_full(kv, 0, qs[0], outs[0], H, [3000, 800], scale, heads, slot=[0, 1])
        att.encode_verify_rows(kv, 0, qs[1], outs[1], H, [2990, 700], 3, scale, heads, [0, 1])
        att.encode_causal(kv, 0, 0, qs[2], outs[2], params, heads)

    step()
    gpu_ctx.synchronize()
    gpu_ctx.graph_begin()
    step()
    graph = gpu_ctx.graph_end()
    for turn in range(4):
        for i, q in enumerate(qs):
            q.copy_(_randn(10 * turn + i, *q.shape))
        torch.cuda.synchronize()
        step()
        gpu_ctx.synchronize()
        eager = [o.clone() for o in outs]
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        graph.launch()
        gpu_ctx.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(eager, outs)), f"replay {turn}"
    graph.close()
    layer.close()


def test_on_another_stream(gpu_ctx):
    import torch
    H, KH, D = 32, 8, 128
    layer = Layer(gpu_ctx, H, KH, D, [5000])
    heads = layer.heads()
    q = _randn(1, 1, H, D)
    plain = layer.decode(q, [5000], heads)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        gpu_ctx.use_torch_stream()
        out = torch.zeros_like(q)
        layer.attention.encode_full(layer.kv, 0, q, out, H, 5000, layer.scale, heads)
        copy = out.clone()
    gpu_ctx.set_stream(None)
    stream.synchronize()
    assert torch.equal(copy, plain)
    layer.close()


def test_lambda_from_learned_vectors(gpu_ctx):
    import torch
    from tinytitan_amd.engine import DifferentialAttention
    att = DifferentialAttention(gpu_ctx)
    r = np.random.default_rng(2)
    for heads, dims in ((16, 128), (1, 32), (5, 7), (24, 200)):
        vectors = [0.1 * r.standard_normal((heads, dims)) for _ in range(4)]
        vectors = [v.astype(np.float32) for v in vectors]
        for shared in (False, True):
            mine = [v[0] if shared else v for v in vectors]
            out = torch.zeros(heads, device="cuda")
            tensors = [_dev(v) for v in mine]
            torch.cuda.synchronize()
            att.encode_lambda(*tensors, 0.8, out)
            gpu_ctx.synchronize()
            a, b, c, d = (np.broadcast_to(v, (heads, dims)).astype(np.float64) for v in mine)
            first, second = np.exp((a * b).sum(-1)), np.exp((c * d).sum(-1))
            # a sum of dims products in fp32 (dims + 4 roundings of its magnitudes), exp of it and its own two units, two additions
            room = sum(e * ((dims + 4) * 2.0 ** -24 * m + 2.0 ** -21) for e, m in ((first, (np.abs(a * b)).sum(-1)), (second, (np.abs(c * d)).sum(-1)))) + 2.0 ** -22
            assert (np.abs(out.cpu().numpy() - (first - second + 0.8)) <= room).all()


def test_refusals(gpu_ctx):
    import torch
    from tinytitan_amd import capi
    from tinytitan_amd.engine import DifferentialHeads, KVCacheManager, PrefillAttentionParams, TinyTitanHIPError
    H, KH, D = 8, 2, 128
    layer = Layer(gpu_ctx, H, KH, D, [300, 300])
    att, kv, scale = layer.attention, layer.kv, layer.scale
    heads = layer.heads()
    q = _randn(1, 2, H, D)
    out = torch.full_like(q, 3.0)
    torch.cuda.synchronize()

    def refused(status, call, *args, **kw):
        with pytest.raises(TinyTitanHIPError) as e:
            call(*args, **kw)
        assert e.value.status == status

    bad, shape, capacity, cursor = capi.ERR_INVALID_ARGUMENT, capi.ERR_SHAPE, capi.ERR_CAPACITY, capi.ERR_CURSOR
    refused(shape, att.encode_full, kv, 0, q, out, 7, [5, 5], scale, DifferentialHeads(_dev(np.ones(7, np.float32))), slot=[0, 1])
    refused(shape, att.encode_full, kv, 0, q, out, H, [5, 5], scale, DifferentialHeads(_dev(np.ones(H - 1, np.float32))), slot=[0, 1])
    refused(shape, att.encode_full, kv, 0, q, out, H, [5, 5], scale, DifferentialHeads(_dev(np.ones((3, H), np.float32))), slot=[0, 1])
    refused(shape, att.encode_full, kv, 0, q, out, H, [5, 5], scale, DifferentialHeads(heads.lambdas, norm_weight=torch.ones(D // 2, device="cuda").bfloat16()), slot=[0, 1])
    refused(bad, att.encode_full, kv, 1, q, out, H, [5, 5], scale, heads, slot=[0, 1])
    refused(bad, att.encode_full, kv, 0, q, out, H, [5, 5], scale, heads, slot=[0, 2])
    refused(bad, att.encode_full, kv, 0, q, out, H, [5, -1], scale, heads, slot=[0, 1])
    refused(bad, att.encode_full, kv, 0, q, out, H, [5, 5], scale, heads, slot=[0, 1], window=-1)
    refused(capacity, att.encode_full, kv, 0, q, out, H, [5, kv.capacity_tokens + 1], scale, heads, slot=[0, 1])
    for eps in (-1e-5, float("nan")):
        refused(bad, att.encode_full, kv, 0, q, out, H, [5, 5], scale, DifferentialHeads(heads.lambdas, heads.norm_weight, eps=eps), slot=[0, 1])
    refused(bad, att.encode_verify_rows, kv, 0, q, out, H, [5], 0, scale, DifferentialHeads(heads.lambdas), [0])
    refused(bad, att.encode_verify_rows, kv, 0, q, out, H, [-1], 2, scale, heads, [0])
    refused(bad, att.encode_verify_rows, kv, 0, q, out, H, [5, 6], 1, scale, heads, [0])
    refused(capacity, att.encode_verify_rows, kv, 0, q, out, H, [kv.capacity_tokens - 1], 2, scale, heads, [0])
    width = H * D

    def params(**kw):
        return PrefillAttentionParams(**{**dict(start_position=10, query_count=2, kv_valid_count=12, num_q_heads=H, scale=scale, q_stride=width, o_stride=width), **kw})
    refused(bad, att.encode_causal, kv, 0, 0, q, out, params(sinks=3, sliding_window=5), heads)
    refused(shape, att.encode_causal, kv, 0, 0, q, out, params(q_stride=width - 1), heads)
    refused(shape, att.encode_causal, kv, 0, 0, q, out, params(o_stride=width - 1), heads)
    refused(shape, att.encode_causal, kv, 0, 0, q, out, params(gate_stride=width - 1), heads, gate=q)
    refused(bad, att.encode_causal, kv, 0, 0, q, out, params(kv_valid_count=11), heads)
    refused(bad, att.encode_causal, kv, 0, 2, q, out, params(), heads)
    refused(bad, att.encode_causal, kv, 0, 0, q, out, params(start_position=-1), heads)
    with pytest.raises(TypeError):
        att.encode_full(kv, 0, q, out, H, [5, 5], scale, DifferentialHeads(heads.lambdas.double()), slot=[0, 1])
    # a slot that starts from another's rows, and a ring that keeps sinks behind its first round
    kv.advance(0, 300)
    kv.share_prefix(0, 100, [1])
    refused(cursor, att.encode_full, kv, 0, q, out, H, [200, 200], scale, heads, slot=[0, 1])
    kv.reset(1)
    pinned = KVCacheManager(gpu_ctx, 1, KH, D, slots=1, max_context=1000, initial_capacity=128, ring_capacity=128, sink_tokens=4)
    refused(capacity, att.encode_full, pinned, 0, q[:1].contiguous(), out, H, [500], scale, heads, window=60)
    pinned.close()
    lib = gpu_ctx._lib
    one, five = capi.int_array([0]), capi.int_array([5])
    args = [gpu_ctx.handle, kv.handle, 0, 1, one, five, 0, H, q.data_ptr(), None, scale, heads.lambdas.data_ptr(), 0, None, 0.0, 1.0, out.data_ptr()]
    for at in (0, 1, 4, 5, 8, 11, 16):
        assert lib.tt_hip_attn_decode_diff(*(None if i == at else a for i, a in enumerate(args))) == bad
    args[12] = H - 1
    assert lib.tt_hip_attn_decode_diff(*args) == shape
    gpu_ctx.synchronize()
    assert (out == 3.0).all()
    layer.close()
