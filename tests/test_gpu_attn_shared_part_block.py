"""The last part block of a prefix that is copied into a slot: the prefix's own slot may go on behind the prefix, and what its rows hold
there, infinities and NaN, is nothing to the sequences that start from it."""
import numpy as np
import pytest

from tests.exact_attention import attend, check, dequantise, stored_rows
from tests.test_gpu_attn_shared_prefix import _fill
from tests.test_gpu_attn_sinks import _dev, _rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("H,KH,D", [(16, 2, 256), (8, 2, 128), (6, 3, 64)])
@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("prefix", [1, 20, 31, 45])
def test_rows_behind_the_prefix_are_not_seen(gpu_ctx, H, KH, D, bits, prefix):
    import torch
    from tinytitan_amd.engine import Attention, KVCacheManager, PrefillAttention, PrefillAttentionParams, SharedPrefix
    width, scale = KH * D, D ** -0.5
    kv = KVCacheManager(gpu_ctx, 1, KH, D, slots=3, max_context=128, initial_capacity=128, precision_bits=bits)
    r = np.random.default_rng(prefix)
    front, own = ([stored_rows(r.standard_normal((n, width)), bits) for _ in "kv"] for n in (prefix, 64))
    _fill(kv, 0, 0, *front)
    for fill in (0x7c, 0xfc, 0xff):  # +inf is 0x7c00
        behind = stored_rows(np.ones((64 - prefix, width)), bits)
        half = behind[:, 0 if bits == 16 else width * bits // 8:].view(np.uint16)
        half[:] = {0x7c: 0x7c00, 0xfc: 0xfc00, 0xff: 0x7e01}[fill]
        _fill(kv, 0, prefix, behind, behind)
        kv.reset(-1)
        kv.advance(0, 64)
        kv.share_prefix(0, prefix, [1, 2])
        for count in (1, 5):
            _fill(kv, 1, prefix, *(part[:count] for part in own))
            q = _rows(count, count, H, D)
            k, v = (dequantise(np.concatenate([a, b[:count]]), width, bits) for a, b in zip(front, own))
            p, starts = SharedPrefix(0, prefix), [prefix]
            qd, outs = _dev(q), [torch.full((count, H, D), float("nan"), dtype=torch.float16, device="cuda") for _ in range(3)]
            torch.cuda.synchronize()
            Attention(gpu_ctx).encode_verify_rows(kv, 0, qd, outs[0], H, starts, count, scale, [1], prefix=p)
            PrefillAttention(gpu_ctx).encode_causal(kv, 0, 1, qd, outs[1], PrefillAttentionParams(prefix, count, prefix + count, H, scale, H * D, H * D,
                                                                                                   H * D), prefix=p)
            Attention(gpu_ctx).encode_full(kv, 0, qd[-1:], outs[2][-1:], H, [prefix + count], scale, slot=[1], prefix=p)
            gpu_ctx.synchronize()
            want = [attend(q[t], k, v, np.arange(prefix + count) <= prefix + t, scale, None, bits) for t in range(count)]
            for out, form in zip(outs, ("verify", "chunk")):
                check(out.cpu().numpy(), want, f"{form}, {count} rows")
            check(outs[2].cpu().numpy()[-1:], want[-1:], "decode")
        # the other slot is the prefix alone
        got = torch.full((1, H, D), float("nan"), dtype=torch.float16, device="cuda")
        Attention(gpu_ctx).encode_full(kv, 0, qd[:1], got, H, [prefix], scale, slot=[2], prefix=p)
        gpu_ctx.synchronize()
        check(got.cpu().numpy(), [attend(q[0], k, v, np.arange(prefix + count) < prefix, scale, None, bits)], "the prefix alone")
    kv.close()


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_finite_rows_behind_the_prefix_are_copied_and_others_are_zeros(gpu_ctx, bits, D):
    # (the rows of the block, as they are stored: only what V holds there that is not finite changes)
    from tinytitan_amd.engine import KVCacheManager
    KH, prefix = 2, 70
    width = KH * D
    kv = KVCacheManager(gpu_ctx, 1, KH, D, slots=2, max_context=128, initial_capacity=128, precision_bits=bits)
    r = np.random.default_rng(D)
    k, v = (stored_rows(r.standard_normal((128, width)), bits) for _ in "kv")
    halves = v[:, 0 if bits == 16 else width * bits // 8:].view(np.uint16)
    bad = np.zeros(halves.shape, bool)
    bad[[3, 69, 70, 75, 80, 95, 96]] = r.random((7, halves.shape[1])) < 0.3
    halves[bad] = r.choice([0x7c00, 0xfc00, 0x7e00, 0xffff], bad.sum())
    _fill(kv, 0, 0, k, v)
    kv.advance(0, 128)
    kv.share_prefix(0, prefix, [1])
    got = [t.cpu().numpy() for t in kv.export_rows(0, 1, 64, 32)]
    gpu_ctx.synchronize()
    bad[:70] = False
    halves[bad] = 0
    assert np.array_equal(got[0], k[64:96]) and np.array_equal(got[1], v[64:96])
    kv.close()
