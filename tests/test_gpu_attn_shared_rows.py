"""Many rows behind one prefix, whose keys go through tiles of 128 packed rows or through the chunk kernel's ranges: scores that grow along
the keys, tiles whose last rows are few, the same sequence twice, another stream, and graphs of several such calls."""
import numpy as np
import pytest

from tests.exact_attention import check, dequantise, stored_rows
from tests.test_gpu_attn_shared_prefix import Family, _decode, _fill
from tests.test_gpu_attn_sinks import _dev, _rows

pytestmark = pytest.mark.gpu


class Ramp(Family):
    """... whose keys of the prefix grow from a tenth of their size to six times of it, so that rows meet higher scores all along."""

    def __init__(self, ctx, KH, D, prefix, lengths, bits):
        assert prefix % 32 == 0  # (nothing of it is copied)
        super().__init__(ctx, KH, D, prefix, lengths, bits)
        r, width = np.random.default_rng(17), KH * D
        k = r.standard_normal((prefix, width)) * np.linspace(0.1, 6.0, prefix)[:, None]
        front = [stored_rows(k, bits), stored_rows(r.standard_normal((prefix, width)), bits)]
        _fill(self.kv, 0, 0, *front)
        self.front = [dequantise(a, width, bits) for a in front]


@pytest.mark.parametrize("H,KH,D", [(24, 2, 256), (32, 8, 128), (16, 4, 64)])
@pytest.mark.parametrize("bits", [16, 8, 4])
def test_scores_that_grow_along_the_keys(gpu_ctx, H, KH, D, bits):
    prefix, n = 12800, 30
    lengths = [prefix + 1 + (i * 53) % 200 for i in range(n)]
    f = Ramp(gpu_ctx, KH, D, prefix, lengths, bits)
    q, g = _rows(21, n, H, D), _rows(22, n, H, D)
    q[3] *= 4  # (one key takes nearly everything)
    q[4] = 0   # (every key the same)
    got = _decode(gpu_ctx, f, q, D ** -0.5, g)
    some = [0, 3, 4, n - 1]
    check(got[some], [f.row(i, q[i], lengths[i] - 1, D ** -0.5, g[i]) for i in some], "rows")
    f.kv.close()


# rows of a KV head: 128, 129 and 255 of tiles of 128, 10 of the last one, one of 32 in it
@pytest.mark.parametrize("H,KH,D,bits,prefix,n,rows", [(2, 1, 256, 16, 20011, 64, 1), (3, 1, 256, 8, 20011, 43, 1), (5, 1, 128, 16, 30000, 17, 3),
                                                       (24, 2, 256, 4, 12345, 23, 2), (16, 2, 256, 16, 9999, 5, 9), (7, 1, 64, 8, 31111, 23, 1),
                                                       (32, 1, 64, 16, 25000, 9, 4), (40, 8, 128, 4, 8191, 11, 3)])
def test_tiles_whose_last_rows_are_few(gpu_ctx, H, KH, D, bits, prefix, n, rows):
    import torch
    from tinytitan_amd.engine import Attention
    starts = [prefix + (i * 29) % 150 for i in range(n)]
    f = Family(gpu_ctx, KH, D, prefix, [p + rows for p in starts], bits)
    q, g = _rows(31, n, rows, H, D), _rows(32, n, rows, H, D)
    qd, gd = _dev(q), _dev(g)
    room = torch.full((n * rows + 2, H, D), float("nan"), dtype=torch.float16, device="cuda")
    torch.cuda.synchronize()
    Attention(gpu_ctx).encode_verify_rows(f.kv, 0, qd, room[1:-1], H, starts, rows, D ** -0.5, f.slots, gate=gd, prefix=f.prefix)
    gpu_ctx.synchronize()
    assert room[0].isnan().all() and room[-1].isnan().all()
    got = room[1:-1].cpu().numpy().reshape(n, rows, H, D)
    assert np.isfinite(got).all()
    for i in sorted({0, n // 2, n - 1}):
        check(got[i], [f.row(i, q[i, r], starts[i] + r, D ** -0.5, g[i, r]) for r in range(rows)], f"sequence {i}")
    f.kv.close()


@pytest.mark.parametrize("H,KH,D,bits,prefix,n", [(24, 2, 256, 4, 12345, 20), (16, 2, 256, 16, 20011, 64), (32, 8, 128, 16, 30000, 64),
                                                  (16, 2, 256, 8, 3000, 4), (32, 8, 128, 8, 6007, 20)])
def test_graphs_of_several_calls_and_another_stream(gpu_ctx, H, KH, D, bits, prefix, n):
    # two captured steps that share the context's store of partial results, replayed in turn with eager calls between
    import torch
    from tinytitan_amd.engine import Attention, HIPContext
    ctx = HIPContext(0)
    lengths = [prefix + 1 + (i * 41) % 700 for i in range(n)]
    f = Family(ctx, KH, D, prefix, lengths, bits)
    pick = [i for i in range(n) if i % 2] + [1]  # (one of them twice)
    q = _rows(41, n, H, D)
    calls = [(_dev(q), lengths, f.slots), (_dev(q[pick]), [lengths[i] for i in pick], [f.slots[i] for i in pick])]
    outs = [torch.zeros_like(c[0]) for c in calls]
    torch.cuda.synchronize()

    def run(i):
        qd, kv_lens, slots = calls[i]
        Attention(ctx).encode_full(f.kv, 0, qd, outs[i], H, kv_lens, D ** -0.5, slot=slots, prefix=f.prefix)

    for i in range(2):
        run(i)
    ctx.synchronize()
    want = [o.clone() for o in outs]
    some = [0, n // 2, n - 1]
    check(want[0].cpu().numpy()[some], [f.row(i, q[i], lengths[i] - 1, D ** -0.5) for i in some], "eager")
    check(want[1].cpu().numpy()[-1:], [f.row(1, q[1], lengths[1] - 1, D ** -0.5)], "picked")
    graphs = []
    for i in range(2):
        ctx.graph_begin()
        run(i)
        graphs.append(ctx.graph_end())
    for turn in range(3):
        for i in (0, 1, 1, 0):
            outs[i].zero_()
            torch.cuda.synchronize()
            graphs[i].launch()
            ctx.synchronize()
            assert torch.equal(outs[i], want[i]), (turn, i)
            run(1 - i)
            ctx.synchronize()
            assert torch.equal(outs[1 - i], want[1 - i]), (turn, i)
    for graph in graphs:
        graph.close()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for turn in range(4):  # (a call behind another on the other stream, without the program waiting)
        for i in range(2):
            with torch.cuda.stream(streams[(turn + i) % 2]):
                ctx.use_torch_stream()
                run(i)
    torch.cuda.synchronize()
    for i in range(2):
        assert torch.equal(outs[i], want[i])
    f.kv.close()
    ctx.close()
