"""Chunks behind a shared prefix that the chunk kernel does not take -- groups that are no multiple of four, rows that are not 16-byte
aligned, a scale that is not positive -- go like the plain ones of such shapes: in one launch whatever their rows, by one-head tiles where
packed ones would leave rows empty, and where the store of partial results has no room and a capture forbids to make any."""
import numpy as np
import pytest

from tests.exact_attention import check
from tests.test_gpu_attn_shared_prefix import Family
from tests.test_gpu_attn_sinks import _dev, _rows, _some

pytestmark = pytest.mark.gpu


def _chunk(ctx, kv, slot, q, start, scale, pad, gate, prefix):
    """A call that writes ``out`` when it is made, and what it is made of."""
    import torch
    from tinytitan_amd.engine import PrefillAttention, PrefillAttentionParams
    rows, heads, dim = q.shape
    width, stride = heads * dim, heads * dim + pad

    def wide(a):
        t = torch.zeros(rows, stride, dtype=torch.float16, device="cuda")
        t[:, :width] = _dev(a).view(rows, width)
        return t

    qd, gd = wide(q), wide(gate) if gate is not None else None
    out = torch.full((rows, stride), float("nan"), dtype=torch.float16, device="cuda")
    params = PrefillAttentionParams(start, rows, start + rows, heads, scale, stride, stride, stride)
    torch.cuda.synchronize()
    return out, lambda: PrefillAttention(ctx).encode_causal(kv, 0, slot, qd, out, params, gate=gd, prefix=prefix)


CHUNKS = [(4, 2, 64, 16, 1200, 0, 1000, 0, 0.125), (6, 3, 64, 16, 500, 70, 3000, 0, 0.125), (16, 2, 256, 16, 700, 3, 1100, 5, 0.0625),
          (16, 2, 256, 8, 700, 33, 256, 5, 0.0625), (24, 8, 128, 4, 400, 1, 1300, 0, 0.088), (20, 2, 128, 8, 999, 0, 400, 3, 0.088),
          (16, 2, 256, 16, 320, 0, 1030, 0, -0.0625), (10, 1, 64, 16, 64, 17, 2100, 0, 0.125), (2, 2, 128, 8, 3000, 5, 1700, 0, 0.088)]


@pytest.mark.parametrize("H,KH,D,bits,prefix,start,rows,pad,scale", CHUNKS)
def test_chunks_that_the_chunk_kernel_does_not_take(gpu_ctx, H, KH, D, bits, prefix, start, rows, pad, scale):
    first = prefix + start
    f = Family(gpu_ctx, KH, D, prefix, [first + rows, first + rows], bits, home=1)
    q, g = _rows(9, rows, H, D), _rows(10, rows, H, D)
    some = sorted({*_some(rows), min(1023, rows - 1), min(1024, rows - 1)})
    for gate in (None, g):
        out, call = _chunk(gpu_ctx, f.kv, f.slots[0], q, first, scale, pad, gate, f.prefix)
        call()
        gpu_ctx.synchronize()
        res = out.cpu().numpy()
        assert np.isnan(res[:, H * D:]).all()
        got = res[:, :H * D].reshape(rows, H, D)
        assert np.isfinite(got).all()
        check(got[some], [f.row(0, q[r], first + r, scale, None if gate is None else gate[r]) for r in some], f"gate {gate is not None}")
    f.kv.close()


@pytest.mark.parametrize("H,KH,D,bits,rows,pad", [(4, 2, 64, 16, 1000, 0), (16, 2, 256, 8, 256, 5), (16, 2, 256, 16, 256, 3)])
def test_a_capture_that_finds_no_room_for_partial_results(H, KH, D, bits, rows, pad):
    # in a context that has run nothing before: the plain chunk is captured, and so is the one behind a prefix
    from tinytitan_amd.engine import HIPContext
    ctx = HIPContext(0)
    prefix, scale = 1300, D ** -0.5
    f = Family(ctx, KH, D, prefix, [prefix + rows], bits)
    q = _rows(11, rows, H, D)
    graphs = []
    # (the plain call reads the slot's own pages, which hold NaN below the prefix: what is asked of it is that it is captured)
    for shared in (None, f.prefix):
        out, call = _chunk(ctx, f.kv, f.slots[0], q, prefix, scale, pad, None, shared)
        ctx.graph_begin()
        try:
            call()
        finally:
            graphs.append((ctx.graph_end(), out))
    graph, out = graphs[1]
    some = _some(rows)
    for _ in range(3):
        out.zero_()
        import torch
        torch.cuda.synchronize()
        graph.launch()
        ctx.synchronize()
        got = out.cpu().numpy()[:, :H * D].reshape(rows, H, D)
        check(got[some], [f.row(0, q[r], prefix + r, scale) for r in some], "replayed")
    for graph, _ in graphs:
        graph.close()
    f.kv.close()
    ctx.close()
