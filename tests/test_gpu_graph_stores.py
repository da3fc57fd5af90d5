"""The first allocation of a store that a context owns releases nothing, so that graphs captured before it replay as they did."""
import numpy as np
import pytest

from tests.test_gpu_attn_diff import _randn
from tests.test_gpu_int8_projection import _dev, _tokens, _weights, check, quantised

pytestmark = pytest.mark.gpu


def test_graphs_outlive_the_first_allocation_of_a_store(gpu_ctx):
    import torch
    from tinytitan_amd.engine import Attention, HIPContext, Int8Projection, KVCacheManager, PrefillAttention, PrefillAttentionParams
    ctx = HIPContext(0)
    H, KH, D = 16, 2, 256
    kv = KVCacheManager(ctx, 1, KH, D, slots=1, max_context=1024, initial_capacity=1024)
    kv.append(0, 0, 0, _randn(1, 600, KH * D), _randn(2, 600, KH * D))
    ctx.synchronize()
    attention, q = Attention(ctx), _randn(3, 1, H, D)
    out, rows, chunk = torch.zeros_like(q), _randn(4, 40, H, D), torch.zeros(40, H, D, dtype=torch.float16, device="cuda")
    indices = torch.arange(600, dtype=torch.int32, device="cuda").repeat(40, 1).contiguous()
    counts = torch.full((40,), 600, dtype=torch.int32, device="cuda")
    r = np.random.default_rng(1)
    w, ws = _weights(r, 64, 256)
    x = _tokens(r, 600, 256)
    args = _dev(w), _dev(ws), _dev(x), torch.zeros(600, 64, dtype=torch.float16, device="cuda")
    torch.cuda.synchronize()
    # (300 keys: one split, without a store)
    attention.encode_full(kv, 0, q, out, H, 300, D ** -0.5)
    ctx.synchronize()
    eager = out.clone()
    ctx.graph_begin()
    attention.encode_full(kv, 0, q, out, H, 300, D ** -0.5)
    graph = ctx.graph_end()

    def replay(behind):
        out.zero_()
        torch.cuda.synchronize()
        graph.launch()
        ctx.synchronize()
        assert torch.equal(out, eager), behind

    replay("nothing")
    params = PrefillAttentionParams(560, 40, 600, H, D ** -0.5, H * D, H * D)
    PrefillAttention(ctx).encode_causal(kv, 0, 0, rows, chunk, params, keep_indices=indices, keep_counts=counts)  # the lists' plan
    ctx.synchronize()
    assert torch.isfinite(chunk).all()
    replay("the lists' plan")
    Int8Projection(ctx).encode(*args, 64, 256, 600)  # quantised tokens
    replay("quantised tokens")
    check(args[3].cpu().numpy(), *quantised(x), w, ws)
    graph.close()
    kv.close()
    ctx.close()
