"""A layer's attention half served in 8 bits, as a model runs it: products of 8-bit integers into queries, keys and values, the cache, differential
attention over it -- a prompt in chunks, decode steps, verify rows -- and the output product.  Each call is checked against the
definition from what the call before it left on the device."""
import numpy as np
import pytest

from tests.exact_maps import attend_maps, check
from tests.test_gpu_int8_projection import check as check_product
from tests.test_gpu_int8_projection import quantised

pytestmark = pytest.mark.gpu


class Layer:
    def __init__(self, ctx, width, H, KH, D, bits, window, slots=2, max_context=1024):
        import torch
        from tinytitan_amd.engine import DifferentialAttention, DifferentialHeads, Int8Projection, KVCacheManager
        self.ctx, self.width, self.H, self.KH, self.D, self.bits, self.window, self.scale = ctx, width, H, KH, D, bits, window, (D // 2) ** -0.5
        self.kv = KVCacheManager(ctx, 1, KH, D, slots=slots, max_context=max_context, initial_capacity=max_context, precision_bits=bits)
        self.attention, self.projection = DifferentialAttention(ctx), Int8Projection(ctx)
        r = np.random.default_rng(7)
        self.host, self.weights = {}, {}
        for name, rows, columns in (("q", H * D, width), ("k", KH * D, width), ("v", KH * D, width), ("o", width, H * D)):
            w = r.integers(-127, 128, (rows, columns)).astype(np.int8)
            s = ((0.5 + r.random(rows)) / (64.0 * columns ** 0.5)).astype(np.float32)
            self.host[name] = (w, s)
            self.weights[name] = (torch.from_numpy(w).cuda(), torch.from_numpy(s).cuda())
        self.norm = torch.from_numpy((1.0 + 0.2 * r.standard_normal(D)).astype(np.float32)).cuda().bfloat16()
        vectors = [torch.from_numpy((0.1 * r.standard_normal((H, D // 2))).astype(np.float32)).cuda() for _ in range(4)]
        lambdas = torch.empty(H, device="cuda")
        torch.cuda.synchronize()
        self.attention.encode_lambda(*vectors, 0.8, lambdas)
        ctx.synchronize()
        q1, k1, q2, k2 = (v.double() for v in vectors)
        want = torch.exp((q1 * k1).sum(-1)) - torch.exp((q2 * k2).sum(-1)) + 0.8
        assert ((lambdas.double() - want).abs() <= 2.0 ** -16).all()
        self.heads = DifferentialHeads(lambdas, norm_weight=self.norm, out_scale=0.2)

    def run(self, x, attend):
        """x [tokens][width]; attend(q, out) appends nothing and reads the cache."""
        import torch
        tokens, H, KH, D = x.shape[0], self.H, self.KH, self.D
        levels = torch.empty(tokens, self.width, dtype=torch.int8, device="cuda")
        scales = torch.empty(tokens, device="cuda")
        half = dict(dtype=torch.float16, device="cuda")
        q, k, v = torch.empty(tokens, H * D, **half), torch.empty(tokens, KH * D, **half), torch.empty(tokens, KH * D, **half)
        a, y = torch.full((tokens, H * D), float("nan"), **half), torch.empty(tokens, self.width, **half)
        torch.cuda.synchronize()
        self.projection.quantise(x, levels, scales, self.width, tokens)
        for name, into in (("q", q), ("k", k), ("v", v)):
            self.projection.encode_levels(*self.weights[name], levels, scales, into, into.shape[1], self.width, tokens)
        attend(q, k, v, a)
        self.projection.encode(*self.weights["o"], a, y, self.width, H * D, tokens)
        self.ctx.synchronize()
        got_levels, got_scales = quantised(x.cpu().numpy())
        assert (levels.cpu().numpy() == got_levels).all() and (scales.cpu().numpy() == got_scales).all()
        for name, into in (("q", q), ("k", k), ("v", v)):
            check_product(into.cpu().numpy(), got_levels, got_scales, *self.host[name], what=name)
        check_product(y.cpu().numpy(), *quantised(a.cpu().numpy()), *self.host["o"], what="o")
        return q.reshape(tokens, H, D), k, v, a.reshape(tokens, H, D), y

    def want(self, q, slot, positions):
        first, n = max(0, positions[0] + 1 - self.window) if self.window else 0, max(positions) + 1
        rows = self.kv.export_rows(0, slot, first, n - first)
        self.ctx.synchronize()
        k, v = (r.cpu().numpy() for r in rows)
        return attend_maps(q, k, v, self.KH, positions, np.arange(first, n), self.window, self.scale, self.heads.lambdas, self.bits, self.norm,
                           self.heads.eps, self.heads.out_scale)

    def close(self):
        self.kv.close()


@pytest.mark.parametrize("H,KH,D,bits,window", [(8, 2, 256, 16, 0), (16, 4, 128, 8, 0), (12, 4, 64, 4, 0), (16, 4, 128, 16, 200)])
def test_prompt_decode_and_verify(gpu_ctx, H, KH, D, bits, window):
    from tinytitan_amd.engine import PrefillAttentionParams
    import torch
    width = 640
    layer = Layer(gpu_ctx, width, H, KH, D, bits, window)
    r = np.random.default_rng(11)

    def tokens(n):
        x = r.standard_normal((n, width))
        x[:, ::160] *= 5.0
        return torch.from_numpy(x.astype(np.float16)).cuda()

    lengths = [0, 0]
    for slot, chunks in enumerate(((333, 100), (65,))):  # a prompt in two chunks, a short one
        for n in chunks:
            start = lengths[slot]

            def attend(q, k, v, out):
                layer.kv.append(0, slot, start, k, v)
                params = PrefillAttentionParams(start, n, start + n, H, layer.scale, H * D, H * D, sliding_window=window)
                layer.attention.encode_causal(layer.kv, 0, slot, q, out, params, layer.heads)

            q, _, _, a, _ = layer.run(tokens(n), attend)
            some = list(range(0, n, 9)) + [n - 1]
            at = torch.tensor(some, device="cuda")
            check(a[at], layer.want(q[at], slot, [start + i for i in some]), f"slot {slot}, {n} rows behind {start}")
            lengths[slot] += n
    for _ in range(3):  # both sequences, a token each

        def attend(q, k, v, out):
            for slot in range(2):
                layer.kv.append(0, slot, lengths[slot], k[slot:slot + 1], v[slot:slot + 1])
            layer.attention.encode_full(layer.kv, 0, q, out, H, [n + 1 for n in lengths], layer.scale, layer.heads, slot=[0, 1], window=window)

        q, _, _, a, _ = layer.run(tokens(2), attend)
        for slot in range(2):
            check(a[slot:slot + 1], layer.want(q[slot:slot + 1], slot, [lengths[slot]]), f"slot {slot}, a token behind {lengths[slot]}")
            lengths[slot] += 1
    rows = 4  # both sequences, drafted tokens

    def attend(q, k, v, out):
        for slot in range(2):
            layer.kv.append(0, slot, lengths[slot], k[slot * rows:(slot + 1) * rows], v[slot * rows:(slot + 1) * rows])
        layer.attention.encode_verify_rows(layer.kv, 0, q, out, H, lengths, rows, layer.scale, layer.heads, [0, 1], window=window)

    q, _, _, a, _ = layer.run(tokens(2 * rows), attend)
    for slot in range(2):
        mine = slice(slot * rows, (slot + 1) * rows)
        check(a[mine], layer.want(q[mine], slot, [lengths[slot] + i for i in range(rows)]), f"slot {slot}, {rows} rows behind {lengths[slot]}")
    layer.close()


def test_a_captured_layer_step(gpu_ctx):
    # the whole step as one graph, the output product's workspace and the attention's partial results among what it uses; other work of the
    # context between the replays
    import torch
    H, KH, D, width, context = 16, 2, 256, 512, 900
    layer = Layer(gpu_ctx, width, H, KH, D, 16, 0)
    r = np.random.default_rng(3)
    rows = torch.from_numpy(r.standard_normal((context, KH * D)).astype(np.float16)).cuda()
    torch.cuda.synchronize()
    layer.kv.append(0, 0, 0, rows, rows.flip(0).contiguous())
    half = dict(dtype=torch.float16, device="cuda")
    x, q, k, v = torch.zeros(1, width, **half), torch.empty(1, H * D, **half), torch.empty(1, KH * D, **half), torch.empty(1, KH * D, **half)
    a, y = torch.empty(1, H * D, **half), torch.zeros(1, width, **half)

    def step():
        for name, into in (("q", q), ("k", k), ("v", v)):
            layer.projection.encode(*layer.weights[name], x, into, into.shape[1], width, 1)
        layer.kv.append(0, 0, context, k, v)
        layer.attention.encode_full(layer.kv, 0, q, a, H, context + 1, layer.scale, layer.heads)
        layer.projection.encode(*layer.weights["o"], a, y, width, H * D, 1)

    torch.cuda.synchronize()
    step()
    gpu_ctx.synchronize()
    gpu_ctx.graph_begin()
    step()
    graph = gpu_ctx.graph_end()
    for turn in range(4):
        x.copy_(torch.from_numpy(r.standard_normal((1, width)).astype(np.float16)))
        torch.cuda.synchronize()
        step()
        gpu_ctx.synchronize()
        eager, attended = y.clone(), a.clone()
        y.zero_()
        torch.cuda.synchronize()
        graph.launch()
        gpu_ctx.synchronize()
        assert torch.equal(y, eager) and torch.equal(a, attended) and bool(y.abs().max() > 0)
        check(a.reshape(1, H, D), layer.want(q.reshape(1, H, D), 0, [context]), f"replay {turn}")
    graph.close()
    layer.close()
