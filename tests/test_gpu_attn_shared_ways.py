"""Each way of a call of sequences that share a prefix, by calls that the planner sends there (``test_shared_plan`` holds that it does), against
the definition in 64 bits."""
import numpy as np
import pytest

from tests.exact_attention import check
from tests.shared_ways import CASES, RANGES, starts
from tests.test_gpu_attn_shared_prefix import Family
from tests.test_gpu_attn_sinks import _dev, _rows

pytestmark = pytest.mark.gpu


class Call:
    """Verify rows of a family: q and gate from the device's start or, ``off``, half a word behind it, where the chunk kernel does not take them."""

    def __init__(self, ctx, H, KH, D, bits, prefix, n, rows, seed=1, gated=True):
        self.ctx, self.shape, self.starts, self.scale = ctx, (n, rows, H, D), starts(prefix, n), D ** -0.5
        self.f = Family(ctx, KH, D, prefix, [p + rows for p in self.starts], bits, home=n // 2, seed=seed)
        self.q = _rows(seed + 70, n, rows, H, D)
        self.gate = _rows(seed + 71, n, rows, H, D) if gated else None

    def made(self, off=0):
        import torch
        from tinytitan_amd.engine import Attention
        n, rows, H, D = self.shape

        def placed(a):
            room = torch.full((a.size + off + 8,), 7.0, dtype=torch.float16, device="cuda")
            room[off:off + a.size] = _dev(a).view(-1)
            return room[off:off + a.size]

        qd, gd = placed(self.q), placed(self.gate) if self.gate is not None else None
        room = torch.full((self.q.size + 2 * H * D,), float("nan"), dtype=torch.float16, device="cuda")  # a row in front of the output and one behind
        out = room[H * D:-H * D]
        torch.cuda.synchronize()
        return room, lambda: Attention(self.ctx).encode_verify_rows(self.f.kv, 0, qd, out, H, self.starts, rows, self.scale, self.f.slots, gate=gd,
                                                                    prefix=self.f.prefix)

    def check(self, room, what=""):
        n, rows, H, D = self.shape
        res = room.cpu().numpy()
        assert np.isnan(res[:H * D]).all() and np.isnan(res[-H * D:]).all()
        got = res[H * D:-H * D].reshape(self.shape)
        assert np.isfinite(got).all(), what
        for i in sorted({0, 1, n // 2, min(4, n - 1), n - 1}):
            some = sorted({0, 1 % rows, rows // 2, rows - 1})
            want = [self.f.row(i, self.q[i, r], self.starts[i] + r, self.scale, None if self.gate is None else self.gate[i, r]) for r in some]
            check(got[i][some], want, f"{what} sequence {i}")


@pytest.mark.parametrize("H,KH,D,bits,prefix,n,rows,way", CASES)
def test_values(gpu_ctx, H, KH, D, bits, prefix, n, rows, way):
    c = Call(gpu_ctx, H, KH, D, bits, prefix, n, rows, gated=n % 2 == 0)
    room, call = c.made()
    call()
    gpu_ctx.synchronize()
    c.check(room)
    first = room.clone()
    room.fill_(float("nan"))
    call()
    gpu_ctx.synchronize()
    assert np.array_equal(first.cpu().numpy().view(np.uint16), room.cpu().numpy().view(np.uint16))  # (the order of the additions is the call's)
    c.f.kv.close()


@pytest.mark.parametrize("H,KH,D,bits,prefix,n,rows", [c[:-1] for c in CASES if c[-1] == RANGES and c[5:7] in ((5, 200), (32, 32), (64, 4), (16, 32), (40, 8))])
def test_ranges_in_a_graph(H, KH, D, bits, prefix, n, rows):
    # captured behind an eager call of the same shape, and where the store of the ranges' results has not been made and cannot be: then the
    # call goes as rows do that the chunk kernel does not take
    from tinytitan_amd.engine import HIPContext
    for warm in (True, False):
        ctx = HIPContext(0)
        c = Call(ctx, H, KH, D, bits, prefix, n, rows, seed=3)
        other, without = c.made(off=1)
        without()  # (partial results of the two passes have room from here on)
        ctx.synchronize()
        c.check(other, "rows that are not aligned")
        room, call = c.made()
        if warm:
            call()
            ctx.synchronize()
            want = room.clone()
        ctx.graph_begin()
        try:
            call()
        finally:
            graph = ctx.graph_end()
        for turn in range(3):
            room.fill_(float("nan"))
            import torch
            torch.cuda.synchronize()
            graph.launch()
            ctx.synchronize()
            if turn == 0:
                c.check(room, f"replayed, warm {warm}")
                if not warm:
                    want = room.clone()
            assert np.array_equal(want.cpu().numpy().view(np.uint16), room.cpu().numpy().view(np.uint16)), (warm, turn)
            without()
            ctx.synchronize()
        graph.close()
        c.f.kv.close()
        ctx.close()
