"""Differential attention at the edges of what its documentation allows: the largest pages, one slot more than once in a call, a call's smallest and
odd forms."""
import numpy as np
import pytest

from tests.exact_attention import stored_rows
from tests.exact_maps import attend_maps, check
from tests.test_gpu_attn_diff import Layer, _randn

pytestmark = pytest.mark.gpu


def test_a_page_of_two_gibibytes(gpu_ctx):
    # a window at its end: what lies in front is neither written nor read
    from tinytitan_amd.engine import KVCacheManager
    H, KH, D, window, capacity = 4, 1, 256, 600, 4_192_000
    layer = Layer(gpu_ctx, H, KH, D, [32], window=window)
    layer.kv.close()
    layer.kv = KVCacheManager(gpu_ctx, 1, KH, D, slots=1, max_context=capacity, initial_capacity=capacity)
    r, first, end = np.random.default_rng(1), capacity - 2400, capacity
    k, v = (stored_rows(r.standard_normal((end - first, KH * D)), 16) for _ in range(2))
    layer.write(0, first, k, v)
    heads = layer.heads()

    def want(q, positions):
        return attend_maps(q, k, v, KH, positions, np.arange(first, end), window, layer.scale, heads.lambdas, 16, heads.norm_weight, heads.eps, heads.out_scale)

    q = _randn(2, 1, H, D)
    check(layer.decode(q, [end], heads), want(q, [end - 1]), "decode")
    q = _randn(3, 1, 5, H, D)
    check(layer.verify(q, [end - 5], 5, heads)[0], want(q[0], list(range(end - 5, end))), "verify")
    for rows in (33, 300, 1500):
        q = _randn(rows, rows, H, D)
        some = list(range(0, rows, 11)) + [rows - 1]
        check(layer.chunk(q, end - rows, heads)[some], want(q[some], [end - rows + i for i in some]), f"{rows} rows")
    layer.close()


@pytest.mark.parametrize("bits", [16, 8])
def test_one_slot_more_than_once(gpu_ctx, bits):
    H, KH, D = 16, 4, 64
    layer = Layer(gpu_ctx, H, KH, D, [900, 40], bits)
    heads, q = layer.heads(), _randn(1, 5, H, D)
    lengths, slots = [900, 900, 1, 40, 333], [0, 0, 0, 1, 0]
    got = layer.decode(q, lengths, heads, slots=slots)
    for i, (n, slot) in enumerate(zip(lengths, slots)):
        check(got[i:i + 1], layer.want(q[i:i + 1], slot, [n - 1], heads), f"{n} keys of slot {slot}")
    rows, starts = _randn(2, 3, 2, H, D), [898, 100, 38]
    got = layer.verify(rows, starts, 2, heads, slots=[0, 0, 1])
    for i, (start, slot) in enumerate(zip(starts, [0, 0, 1])):
        check(got[i], layer.want(rows[i], slot, [start, start + 1], heads), f"rows {start} of slot {slot}")
    layer.close()


@pytest.mark.parametrize("H,KH,D", [(17, 1, 128), (34, 2, 64), (19, 1, 64), (23, 23, 256), (3, 1, 256)])
def test_heads_whose_maps_part_at_a_tile_s_end(gpu_ctx, H, KH, D):
    # an odd number of rows in a tile: a head's second map may be the next tile's first row
    layer = Layer(gpu_ctx, H, KH, D, [2100])
    heads = layer.heads()
    for n in (1, 65, 300, 2100):
        q, gate = _randn(n, 1, H, D), _randn(n + 1, 1, H, D)
        check(layer.decode(q, [n], heads, gate), layer.want(q, 0, [n - 1], heads, gate), f"{n} keys")
    for start, rows in ((0, 3), (700, 5), (1900, 200)):
        q = _randn(start, rows, H, D)
        check(layer.chunk(q, start, heads), layer.want(q, 0, list(range(start, start + rows)), heads), f"{rows} rows behind {start}")
    layer.close()


def test_a_zero_factor_is_plain_attention_and_one_of_infinity_is_not_hidden(gpu_ctx):
    import torch
    H, KH, D = 8, 2, 128
    layer = Layer(gpu_ctx, H, KH, D, [700])
    q = _randn(1, 1, H, D)
    zero = layer.heads(np.zeros(H, np.float32), normed=False, out_scale=1.0)
    got = layer.decode(q, [700], zero)
    check(got, layer.want(q, 0, [699], zero), "lambda 0")
    lambdas = layer.lambdas.copy()
    lambdas[3] = np.inf
    bad = layer.heads(lambdas)
    got = layer.decode(q, [700], bad)
    others = [h for h in range(H) if h != 3]
    assert not torch.isfinite(got[0, 3]).any() and torch.isfinite(got[0, others]).all()
    want, bound = layer.want(q, 0, [699], layer.heads())
    check(got[:, others].contiguous(), (want[:, others], bound[:, others]), "the other heads")
    layer.close()


@pytest.mark.parametrize("rows", [40, 900])
def test_a_row_that_is_not_finite_stays_alone(gpu_ctx, rows):
    # a query of NaN, in a tile with others
    import torch
    H, KH, D = 16, 4, 128
    layer = Layer(gpu_ctx, H, KH, D, [1000])
    heads = layer.heads()
    start = 1000 - rows
    q = _randn(rows, rows, H, D)
    good = q.clone()
    q[17, 5] = float("nan")
    torch.cuda.synchronize()
    got = layer.chunk(q, start, heads)
    assert torch.isnan(got[17, 5]).all()
    some = [0, 16, 17, 18, 31, 32, rows - 1]
    want, bound = layer.want(good[some], 0, [start + i for i in some], heads)
    got = got[some].clone()
    got[2, 5] = want[2, 5].half()
    check(got, (want, bound + (torch.arange(len(some), device="cuda") == 2)[:, None, None] * 1.0), f"{rows} rows")
    layer.close()


@pytest.mark.parametrize("scale", [-0.05, 0.0])
def test_a_chunk_by_tiles_in_several_passes(gpu_ctx, scale):
    # more rows of both maps than partial results are kept of at a time (131,072 of them), by the way that a scale which is not positive takes
    H, KH, D, rows, start = 64, 8, 64, 1500, 40
    layer = Layer(gpu_ctx, H, KH, D, [start + rows])
    layer.scale = scale
    heads = layer.heads(np.random.default_rng(3).random((rows, H)).astype(np.float32), normed=False)
    q, gate = _randn(1, rows, H, D), _randn(2, rows, H, D)
    from tinytitan_amd.engine import PrefillAttentionParams
    import torch
    out = torch.full_like(q, float("nan"))
    torch.cuda.synchronize()
    layer.attention.encode_causal(layer.kv, 0, 0, q, out, PrefillAttentionParams(start, rows, start + rows, H, scale, H * D, H * D), heads, gate=gate)
    gpu_ctx.synchronize()
    assert torch.isfinite(out).all()
    some = [0, 1, 500, 1022, 1023, 1024, 1025, 1300, 1499]
    check(out[some], layer.want(q[some], 0, [start + i for i in some], heads, gate[some], heads.lambdas[some]), f"scale {scale}")
    layer.close()
