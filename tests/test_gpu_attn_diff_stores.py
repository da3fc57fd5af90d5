"""What differential attention asks of the stores that a context owns: a call whose launch writes the finished rows keeps no partial results, so that
it can be captured on a context that has run nothing, and leaves captured graphs as they are; a chunk whose partial results find no room takes a way
that keeps none; and of many sequences' rows some are served at a time, so that what is kept of them has a bound."""
import numpy as np
import pytest

from tests.exact_maps import check
from tests.test_gpu_attn_diff import Layer, _randn

pytestmark = pytest.mark.gpu


@pytest.fixture
def new_ctx():
    """A context that has run nothing."""
    from tinytitan_amd.engine import HIPContext
    ctx = HIPContext(0)
    yield ctx
    ctx.close()


def captured(ctx, step):
    """The graph of `step`, or the status that a call of it was refused with."""
    from tinytitan_amd.engine import TinyTitanHIPError
    ctx.graph_begin()
    try:
        step()
    except TinyTitanHIPError as e:
        ctx.graph_end().close()
        return e.status
    return ctx.graph_end()


def replayed(ctx, graph, out, between=None):
    """`out` of three replays, with other work of the context between them; each has to be the first one's."""
    import torch
    first = None
    for _ in range(3):
        out.fill_(float("nan"))
        torch.cuda.synchronize()
        graph.launch()
        ctx.synchronize()
        if first is None:
            first = out.clone()
        assert torch.equal(out, first)
        if between:
            between()
    return first


@pytest.mark.parametrize("H,KH,D,bits", [(16, 2, 256, 16), (32, 8, 128, 16), (16, 4, 64, 8), (24, 2, 256, 4)])
def test_a_launch_that_finishes_its_rows_is_captured_first(new_ctx, H, KH, D, bits):
    import torch
    from tinytitan_amd import capi
    from tinytitan_amd.engine import PrefillAttentionParams
    lengths = [300, 7, 300]
    layer, long = Layer(new_ctx, H, KH, D, lengths, bits), Layer(new_ctx, H, KH, D, [20000], bits)
    heads, att, kv, scale = layer.heads(), layer.attention, layer.kv, layer.scale

    def run(q, step, want, between=None):
        out = torch.zeros_like(q)
        torch.cuda.synchronize()
        graph = captured(new_ctx, lambda: step(out))
        assert not isinstance(graph, int), graph
        got = replayed(new_ctx, graph, out, between)
        want(got)
        graph.close()

    q = _randn(1, 1, H, D)
    run(q, lambda out: att.encode_full(kv, 0, q, out, H, 300, scale, heads), lambda got: check(got, layer.want(q, 0, [299], heads), "one row"))
    qs = _randn(2, 3, H, D)
    run(qs, lambda out: att.encode_full(kv, 0, qs, out, H, lengths, scale, heads, slot=[0, 1, 2]),
        lambda got: [check(got[i:i + 1], layer.want(qs[i:i + 1], i, [n - 1], heads), f"{n} keys") for i, n in enumerate(lengths)])
    rows = _randn(3, 2, 4, H, D)
    run(rows, lambda out: att.encode_verify_rows(kv, 0, rows, out, H, [296, 100], 4, scale, heads, [2, 0]),
        lambda got: [check(got[i], layer.want(rows[i], slot, list(range(at, at + 4)), heads), f"rows {at}") for i, (slot, at) in enumerate(((2, 296), (0, 100)))])
    chunk = _randn(4, 40, H, D)
    params = PrefillAttentionParams(200, 40, 240, H, scale, H * D, H * D)
    run(chunk, lambda out: att.encode_causal(kv, 0, 0, chunk, out, params, heads), lambda got: check(got, layer.want(chunk, 0, list(range(200, 240)), heads), "chunk"))
    # many keys are many splits, whose partial results have to be kept: refused until a call outside has made room
    late, out = _randn(5, 1, H, D), torch.zeros(1, H, D, dtype=torch.float16, device="cuda")
    torch.cuda.synchronize()
    step = lambda: att.encode_full(long.kv, 0, late, out, H, 20000, scale, heads)  # noqa: E731
    assert captured(new_ctx, step) == capi.ERR_BUSY
    # ... which is no harm to a graph from before there was a store
    eager = []
    run(q, lambda out: att.encode_full(kv, 0, q, out, H, 300, scale, heads), lambda got: check(got, layer.want(q, 0, [299], heads), "one row again"),
        lambda: eager.append(long.decode(late, [20000], heads)))
    graph = captured(new_ctx, step)
    # (the definition's bound over so many quantised keys covers a normed difference: the eager result is what a replay has to be)
    assert torch.isfinite(eager[0]).all() and torch.equal(replayed(new_ctx, graph, out), eager[0])
    graph.close()
    layer.close()
    long.close()


def test_a_launch_that_finishes_its_rows_leaves_graphs_as_they_are(new_ctx):
    # a graph over partial results, and then more rows than their store holds, in one split
    import torch
    H, KH, D = 16, 2, 256
    layer = Layer(new_ctx, H, KH, D, [5000] + [300] * 8)
    heads = layer.heads()
    q, out = _randn(1, 1, H, D), torch.zeros(1, H, D, dtype=torch.float16, device="cuda")
    torch.cuda.synchronize()
    step = lambda: layer.attention.encode_full(layer.kv, 0, q, out, H, 5000, layer.scale, heads)  # noqa: E731
    step()
    new_ctx.synchronize()
    graph = captured(new_ctx, step)
    rows = _randn(2, 8, 64, H, D)

    def others():
        got = layer.verify(rows, [236] * 8, 64, heads, slots=list(range(1, 9)))
        check(got[7], layer.want(rows[7], 8, list(range(236, 300)), heads), "many rows")

    check(replayed(new_ctx, graph, out, others), layer.want(q, 0, [4999], heads), "replays")
    graph.close()
    layer.close()


# rows, start, bits: by the tiles in several splits, or by ranges of keys
@pytest.mark.parametrize("H,KH,D,bits,rows,start,staged,status", [
    (16, 2, 256, 16, 24, 3000, False, "OK"), (16, 4, 64, 16, 20, 3000, False, "OK"), (32, 8, 128, 16, 16, 3000, False, "OK"),
    (16, 2, 256, 16, 333, 2500, False, "OK"), (32, 8, 128, 16, 130, 6000, False, "OK"), (16, 2, 256, 16, 100, 17000, False, "OK"),
    (16, 2, 256, 8, 333, 2500, False, "OK"),        # (the tiles: one split)
    (16, 2, 256, 8, 100, 4500, True, "OK"), (16, 2, 256, 4, 20, 3000, True, "OK"),
    (16, 2, 256, 8, 100, 17000, False, "ERR_BUSY"), (16, 2, 256, 4, 20, 3000, False, "ERR_BUSY")])
def test_a_chunk_captured_before_there_is_a_store(new_ctx, H, KH, D, bits, rows, start, staged, status):
    import torch
    from tinytitan_amd import capi
    from tinytitan_amd.engine import PrefillAttentionParams
    layer = Layer(new_ctx, H, KH, D, [max(start + rows, 4500)], bits)
    heads = layer.heads(normed=False)
    if staged:  # by a chunk that leaves dequantised blocks and no partial results: of all keys a workgroup, in the chunk kernel
        layer.chunk(_randn(9, 1500, H, D), 3000, heads)
    q = _randn(1, rows, H, D)
    out = torch.zeros_like(q)
    params = PrefillAttentionParams(start, rows, start + rows, H, layer.scale, H * D, H * D)
    torch.cuda.synchronize()
    step = lambda: layer.attention.encode_causal(layer.kv, 0, 0, q, out, params, heads)  # noqa: E731
    graph = captured(new_ctx, step)
    if status != "OK":
        assert graph == getattr(capi, status)
    else:
        assert not isinstance(graph, int), graph
        some = sorted(set(range(0, rows, 9)) | {rows - 1})
        at = torch.tensor(some, device="cuda")
        # (between the replays the same call makes its stores)
        got = replayed(new_ctx, graph, out, lambda: layer.chunk(q, start, heads))
        check(got[at], layer.want(q[at], 0, [start + r for r in some], heads), "captured")
        graph.close()
    step()
    new_ctx.synchronize()
    graph = captured(new_ctx, step)
    eager = layer.chunk(q, start, heads)
    assert torch.equal(replayed(new_ctx, graph, out), eager)
    graph.close()
    layer.close()


def _several_passes(layer, starts, rows, some):
    """Verify rows with factors by token: `some` of each sequence's against the definition.  Returns what the call has left on the device."""
    import torch

    def used():
        torch.cuda.synchronize()
        free, total = torch.cuda.mem_get_info()
        return total - free - torch.cuda.memory_reserved()

    H, n = layer.H, len(starts)
    q, gate = _randn(1, n, rows, H, layer.D), _randn(2, n, rows, H, layer.D)
    lambdas = np.random.default_rng(3).random((n * rows, H)).astype(np.float32)
    heads = layer.heads(lambdas)
    before = used()
    got = layer.verify(q, starts, rows, heads, gate)
    grown = used() - before
    for i, start in enumerate(starts):
        of = heads.lambdas[i * rows:(i + 1) * rows]
        check(got[i, some], layer.want(q[i, some], i, [start + r for r in some], heads, gate[i, some], of[some]), f"sequence {i}")
    return grown


def test_rows_of_many_sequences_in_several_passes(new_ctx):
    # 17 heads, whose 34 rows of maps are tiles of 17: a head's maps may part, and their partial results are kept whatever the keys are
    H, KH, D, n, rows = 17, 1, 64, 32, 512
    starts = [int(s) for s in np.random.default_rng(1).integers(0, 90, n)]
    layer = Layer(new_ctx, H, KH, D, [s + rows for s in starts])
    at_once = 131072 // (2 * H * n)
    grown = _several_passes(layer, starts, rows, [0, at_once - 1, at_once, at_once + 1, 2 * at_once, rows - 1])
    # 131,072 rows, of 32 a tile 17 in use, 256 values and two statistics each, the store a quarter larger than asked for
    assert grown <= 131072 * 32 / 17 * 1.25 * (256 + 2) * 4 + (32 << 20), grown
    layer.close()


def test_rows_of_unlike_sequences_in_several_passes(new_ctx):
    H, KH, D, n, rows = 16, 2, 256, 20, 300
    starts = [20 * i for i in range(n - 1)] + [20000]
    layer = Layer(new_ctx, H, KH, D, [s + rows for s in starts])
    at_once = 131072 // (2 * H * n)
    assert at_once < rows
    _several_passes(layer, starts, rows, [0, at_once - 1, at_once, rows - 1])
    layer.close()
