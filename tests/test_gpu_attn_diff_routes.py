"""The ways that a chunk of differential attention is taken -- split-K tiles, the chunk kernel, the chunk kernel over ranges of keys -- over fp16 and
dequantised pages, against the definition in 64 bits, and what is left of them inside a capture."""
import numpy as np
import pytest

from tests.exact_maps import check
from tests.maps_routes import ROUTES
from tests.test_gpu_attn_diff import Layer, _randn

pytestmark = pytest.mark.gpu


def some_rows(rows):
    """The first and the last ones, and some of every tile."""
    return sorted(set(range(0, rows, 13)) | set(range(min(rows, 36))) | set(range(max(rows - 36, 0), rows)))


@pytest.mark.parametrize("H,KH,D,bits,rows,start,window,ring,way", ROUTES)
def test_chunk_by_every_way(gpu_ctx, H, KH, D, bits, rows, start, window, ring, way):
    import torch
    layer = Layer(gpu_ctx, H, KH, D, [start + rows], bits, window, ring=ring, seed=way)
    some = some_rows(rows)
    at = torch.tensor(some, device="cuda")
    for gated, normed, pad in ((False, True, 0), (True, False, 24), (True, True, 5)):
        q, gate = _randn(1 + pad, rows, H, D), _randn(2, rows, H, D) if gated else None
        lambdas = np.random.default_rng(pad).random((rows, H)).astype(np.float32) if pad else None
        heads = layer.heads(lambdas, normed=normed)
        got = layer.chunk(q, start, heads, gate, pad=pad)
        assert torch.isfinite(got).all()
        want = layer.want(q[at], 0, [start + r for r in some], heads, None if gate is None else gate[at], None if lambdas is None else heads.lambdas[at],
                          first=max(0, start + 1 - window) if window else 0)
        check(got[at], want, f"pad {pad}")
    layer.close()


@pytest.mark.parametrize("bits", [16, 8])
def test_the_ways_agree(gpu_ctx, bits):
    # the last rows of a chunk that goes by ranges, of one that goes whole and of one by the tiles are rows of one sequence: a row's result is
    # what the definition says whichever way it takes
    H, KH, D, total = 32, 8, 128, 2600
    layer = Layer(gpu_ctx, H, KH, D, [total], bits)
    heads = layer.heads()
    q = _randn(3, 2600, H, D)
    last = list(range(total - 20, total))
    want = layer.want(q[last], 0, last, heads)
    for rows in (20, 33, 200, 777, 2600):
        got = layer.chunk(q[total - rows:].contiguous(), total - rows, heads)
        check(got[-20:], want, f"{rows} rows")
    layer.close()


@pytest.mark.parametrize("H,KH,D,bits,rows,start", [(16, 2, 256, 16, 333, 2500), (16, 2, 256, 8, 333, 2500), (32, 8, 128, 8, 777, 130)])
def test_capture_before_the_stores_are_there(H, KH, D, bits, rows, start):
    # a context that has run nothing: inside a capture neither partial results nor dequantised pages can be made room for
    import torch
    from tinytitan_amd import capi
    from tinytitan_amd.engine import HIPContext, PrefillAttentionParams, TinyTitanHIPError
    ctx = HIPContext(0)
    layer = Layer(ctx, H, KH, D, [start + rows], bits)
    heads, width = layer.heads(), H * D
    q = _randn(1, rows, H, D)
    out = torch.zeros_like(q)
    params = PrefillAttentionParams(start, rows, start + rows, H, layer.scale, width, width)
    some = some_rows(rows)
    at = torch.tensor(some, device="cuda")
    want = layer.want(q[at], 0, [start + r for r in some], heads)
    torch.cuda.synchronize()

    def captured():
        ctx.graph_begin()
        try:
            layer.attention.encode_causal(layer.kv, 0, 0, q, out, params, heads)
        except TinyTitanHIPError as e:
            ctx.graph_end().close()
            return e.status
        graph = ctx.graph_end()
        for turn in range(3):
            out.fill_(float("nan"))
            torch.cuda.synchronize()
            graph.launch()
            ctx.synchronize()
            check(out[at], want, f"replay {turn}")
            layer.chunk(q, start, heads)
        graph.close()
        return capi.OK

    status = captured()
    assert status in (capi.OK, capi.ERR_BUSY)
    check(layer.chunk(q, start, heads)[at], want, "eager")
    assert captured() == capi.OK
    layer.close()
    ctx.close()


def test_a_row_that_ranges_leave_without_keys_in_most_of_them(gpu_ctx):
    # the first row of a prompt sees one key, of the first range: every other range has nothing for it
    import torch
    H, KH, D, rows = 16, 2, 256, 640
    layer = Layer(gpu_ctx, H, KH, D, [rows + 2000], 16)
    q = _randn(5, rows, H, D)
    heads = layer.heads(normed=False, out_scale=1.0)
    for start in (0, 2000):
        got = layer.chunk(q, start, heads)
        check(got[:3], layer.want(q[:3], 0, [start, start + 1, start + 2], heads), f"behind {start}")
    # (one key: both maps are that key's value, and the difference (1 - lambda) of it)
    got = layer.chunk(q, 0, heads)[0].double()
    v = layer.kv.read(0, 0, 0, 1)[1][0].double()
    torch.cuda.synchronize()
    for h in range(H):
        exact = (1.0 - float(np.float32(layer.lambdas[h]))) * v[h // (H // KH)]
        assert ((got[h] - exact).abs() <= exact.abs() * (2.0 ** -11 + 2.0 ** -20) + v[h // (H // KH)].abs() * 2.0 ** -22 + 2.0 ** -25).all()
    layer.close()
