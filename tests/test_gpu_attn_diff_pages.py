"""Differential attention of a chunk over quantised pages whose dequantised blocks are as long as a page can be, 0x7ff00000 bytes, and longer: the
chunk kernel over the dequantised pages up to there, the split-K tiles over the pages themselves behind it."""
import numpy as np
import pytest

from tests.exact_attention import stored_rows
from tests.exact_maps import attend_maps, check
from tests.test_gpu_attn_diff import Layer, _dev

pytestmark = pytest.mark.gpu

MOST = 0x7ff00000 // 2 // 256  # tokens of a page of heads of 256


@pytest.mark.parametrize("total,bits", [(MOST, 8), (MOST + 1, 8), (MOST + 1, 4)])
def test_dequantised_pages_of_two_gibibytes(gpu_ctx, total, bits):
    # Some keys far apart that every row's two queries point at, with scores of about 31, among rows of zeros: forty keys or more that a row sees, and
    # the zeros' weights together 4.2e6 e^-30 / 40, 1e-8 of the sum; their values are zero.
    import torch
    from tinytitan_amd.engine import KVCacheManager
    H, KH, D, rows = 4, 1, 256, 256
    start, r = total - rows, np.random.default_rng(total + bits)
    layer = Layer(gpu_ctx, H, KH, D, [32], bits)
    layer.kv.close()
    layer.kv = KVCacheManager(gpu_ctx, 1, KH, D, slots=1, max_context=total + 31, initial_capacity=total + 31, precision_bits=bits)
    towards = np.where(r.random(D) < 0.5, -1.0, 1.0)
    at = sorted({0, 31, 32, 5000, 131072, 2 ** 21 - 1, 2 ** 21, 3_000_001, start - 1, start, start + 1, start + 63, start + 64, start + 200, total - 2, total - 1}
                | {int(p) for p in r.integers(0, start, 40)})
    k = stored_rows(towards * 2.8 + 0.1 * r.standard_normal((len(at), D)), bits)
    v = stored_rows(r.standard_normal((len(at), D)), bits)
    zeros = torch.zeros((131072, k.shape[1]), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    for p in range(0, total, len(zeros)):
        some = zeros[:min(len(zeros), total - p)]
        layer.kv.import_rows(0, 0, p, some, some)
    gpu_ctx.synchronize()
    for i, p in enumerate(at):
        layer.write(0, p, k[i:i + 1], v[i:i + 1])
    heads = layer.heads(normed=False, out_scale=0.5)
    q = _dev((towards + 0.05 * r.standard_normal((rows, H, D))).astype(np.float16))
    # (the scores of what is compared, so that the arithmetic above holds: 128 products of about 2.8, over sqrt(128))
    from tests.exact_attention import dequantise
    keys = sum(torch.from_numpy(x) for x in dequantise(k, D, bits)).half().double().cuda()
    scores = torch.stack([(q.double() * half) @ keys.T for half in (torch.arange(D, device="cuda") < D // 2, torch.arange(D, device="cuda") >= D // 2)]) * layer.scale
    assert 30.0 < float(scores.min()) and sum(p <= start for p in at) >= 40
    got = layer.chunk(q, start, heads)
    some = [0, 1, 2, 63, 64, 65, 127, 128, 199, 200, 201, 254, 255]
    out, bound = attend_maps(q[some], k, v, KH, [start + i for i in some], at, 0, layer.scale, heads.lambdas, bits, None, heads.eps, heads.out_scale)
    # (the zeros': 2^-22 of either map's values, which are at most 8)
    check(got[some], (out, bound + 2.0 ** -22 * 8 * 2), f"{total} keys")
    # (what the test notices: zeros in the rows' place, and a third of the keys left out)
    assert ((out.abs() > bound).double().mean(-1) > 0.5).all()
    for j in range(3):
        others = [i for i in range(len(at)) if i * 3 // len(at) != j]
        less, _ = attend_maps(q[some], k[others], v[others], KH, [start + i for i in some], [at[i] for i in others], 0, layer.scale, heads.lambdas, bits, None,
                              heads.eps, heads.out_scale)
        assert ((less - out).abs() > bound).any(-1).all(), j
    layer.close()
