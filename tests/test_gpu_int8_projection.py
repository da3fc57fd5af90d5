"""Products of 8-bit integers through the C ABI.  Scales and levels of quantised tokens are exact (fp32 divisions and roundings, which
numpy has too); sums are exact in integers, so that an output is off by three fp32 roundings (the sum as fp32, two products) and one to
fp16: 3 * 2^-24 (and their products, taken as 2^-21) and 2^-11 of it, 2^-25 where it is subnormal."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _dev(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).to("cuda")


def quantised(x):
    """fp16 tokens [n][columns] -> (levels int8, scales fp32)."""
    x = x.astype(np.float32)
    scale = np.abs(x).max(-1) / np.float32(127.0)
    with np.errstate(invalid="ignore", divide="ignore"):
        levels = np.where(scale[:, None] > 0, np.rint(x / scale[:, None]), 0.0)
    return levels.astype(np.int8), scale


def check(got, levels, scales, weights, weight_scales, what=""):
    sums = levels.astype(np.float64) @ weights.astype(np.float64).T
    want = sums * scales.astype(np.float64)[:, None] * weight_scales.astype(np.float64)
    bound = np.abs(want) * (2.0 ** -11 + 2.0 ** -21) + 2.0 ** -25
    g = got.astype(np.float64)
    assert np.isfinite(g).all(), f"{what}: not finite"
    over = np.abs(g - want) - bound
    assert over.max() <= 0, f"{what}: off by {np.abs(g - want).flat[over.argmax()]:.3e} at {np.unravel_index(over.argmax(), over.shape)}, bound {bound.flat[over.argmax()]:.3e}"


def _weights(r, rows, columns):
    w = r.integers(-127, 128, (rows, columns)).astype(np.int8)
    return w, (0.5 + r.random(rows)).astype(np.float32) / np.float32(127.0) / np.float32(columns ** 0.5)


def _tokens(r, tokens, columns):
    x = r.standard_normal((tokens, columns))
    x[:, :: max(columns // 4, 1)] *= 6.0
    return x.astype(np.float16)


class Call:
    def __init__(self, ctx, x, weights, weight_scales, x_pad=0, y_pad=0):
        import torch
        from tinytitan_amd.engine import Int8Projection
        self.ctx, self.projection = ctx, Int8Projection(ctx)
        self.tokens, self.columns = x.shape
        self.rows = weights.shape[0]
        self.x_pad, self.y_pad = x_pad, y_pad
        self.x = torch.full((self.tokens, self.columns + x_pad), float("nan"), dtype=torch.float16, device="cuda")  # (what lies behind a token is not read)
        self.x[:, :self.columns] = _dev(x)
        self.weights, self.weight_scales = _dev(weights), _dev(weight_scales)

    def _y(self):
        import torch
        y = torch.full((self.tokens, self.rows + self.y_pad), 7.0, dtype=torch.float16, device="cuda")
        y[:, :self.rows] = float("nan")
        torch.cuda.synchronize()
        return y

    def _rows(self, y):
        self.ctx.synchronize()
        assert (y[:, self.rows:] == 7.0).all()
        return y[:, :self.rows].cpu().numpy()

    def from_halves(self):
        y = self._y()
        self.projection.encode(self.weights, self.weight_scales, self.x, y, self.rows, self.columns, self.tokens,
                               x_stride=self.columns + self.x_pad, y_stride=self.rows + self.y_pad)
        return self._rows(y)

    def quantise(self, pad=0):
        import torch
        levels = torch.full((self.tokens, self.columns + pad), 99, dtype=torch.int8, device="cuda")
        scales = torch.full((self.tokens,), 5.0, dtype=torch.float32, device="cuda")
        torch.cuda.synchronize()
        self.projection.quantise(self.x, levels, scales, self.columns, self.tokens, x_stride=self.columns + self.x_pad,
                                 levels_stride=self.columns + pad)
        self.ctx.synchronize()
        assert (levels[:, self.columns:] == 99).all()
        return levels, scales

    def from_levels(self, levels, scales):
        y = self._y()
        self.projection.encode_levels(self.weights, self.weight_scales, levels, scales, y, self.rows, self.columns, self.tokens,
                                      levels_stride=levels.shape[1], y_stride=self.rows + self.y_pad)
        return self._rows(y)


TOKENS = [1, 2, 3, 4, 5, 7, 8, 9, 15, 16, 17, 31, 32, 33, 48, 63, 64, 65, 100, 128, 129, 200, 257]


@pytest.mark.parametrize("columns", [16, 32, 48, 64, 80, 112, 128, 144, 256, 272, 1040, 2048, 4112])
@pytest.mark.parametrize("rows", [1, 3, 16, 31, 100, 257])
def test_every_size(gpu_ctx, columns, rows):
    r = np.random.default_rng(columns * 1000 + rows)
    w, ws = _weights(r, rows, columns)
    for i, tokens in enumerate(TOKENS):
        x = _tokens(r, tokens, columns)
        call = Call(gpu_ctx, x, w, ws, x_pad=[0, 8, 40][i % 3], y_pad=[0, 1, 6][i % 3])
        levels, scales = quantised(x)
        check(call.from_halves(), levels, scales, w, ws, f"{tokens} tokens")


@pytest.mark.parametrize("tokens,rows,columns", [(300, 1000, 528), (777, 2311, 1024), (1025, 513, 2064), (513, 5121, 512), (2050, 300, 4096), (4096, 260, 272),
                                                 (1, 9216, 4096), (4, 5121, 6144), (12, 12288, 2048), (40, 4097, 8192), (96, 4608, 5120), (200, 6145, 2048)])
def test_larger_sizes(gpu_ctx, tokens, rows, columns):
    r = np.random.default_rng(tokens + rows)
    w, ws = _weights(r, rows, columns)
    x = _tokens(r, tokens, columns)
    levels, scales = quantised(x)
    call = Call(gpu_ctx, x, w, ws)
    got = call.from_halves()
    check(got, levels, scales, w, ws)
    assert np.array_equal(call.from_levels(*call.quantise()), got)
    assert np.array_equal(call.from_halves(), got)


@pytest.mark.parametrize("columns", [16, 48, 128, 1040, 4096, 20000, 131056])
def test_quantised_tokens_are_exact(gpu_ctx, columns):
    r = np.random.default_rng(columns)
    n = 9
    x = _tokens(r, n, columns)
    x[1] = 0.0                                   # zeros
    x[2] = np.float16(6e-8)                      # the smallest subnormal
    x[3, ::2] = np.float16(65504.0)              # the largest value
    x[4] = np.linspace(-1, 1, columns).astype(np.float16)  # halves of the largest value: ties
    x[5] = np.where(np.arange(columns) % 2, -0.0, 1.0)
    x[6] = (r.integers(-127, 128, columns) / 2.0).astype(np.float16)
    call = Call(gpu_ctx, x, *_weights(r, 3, columns), x_pad=8)
    levels, scales = quantised(x)
    for pad in (0, 16):
        got_levels, got_scales = call.quantise(pad)
        assert np.array_equal(got_scales.cpu().numpy(), scales)
        assert np.array_equal(got_levels[:, :columns].cpu().numpy(), levels)


def test_levels_of_every_half(gpu_ctx):
    # every finite half beside every power of two that bounds it, and some other largest values
    halves = np.arange(0x7c00, dtype=np.uint16).view(np.float16)
    halves = np.concatenate([halves, -halves])
    r = np.random.default_rng(1)
    tops = list(2.0 ** np.arange(-24, 16)) + [float(t) for t in r.choice(halves[1:0x7c00], 60)] + [65504.0]
    columns = 63488 // 16 * 16
    assert columns == len(halves)
    x = np.stack([np.where(np.abs(halves.astype(np.float64)) <= t, halves, np.float16(0.0)) for t in tops])
    x[:, 1] = np.array(tops, np.float16)
    call = Call(gpu_ctx, x, *_weights(r, 1, columns))
    levels, scales = quantised(x)
    got_levels, got_scales = call.quantise()
    assert np.array_equal(got_scales.cpu().numpy(), scales)
    assert np.array_equal(got_levels.cpu().numpy(), levels)


@pytest.mark.parametrize("tokens", [1, 3, 6, 20, 70, 300])
def test_levels_of_all_values_and_the_largest_sums(gpu_ctx, tokens):
    # -128 among levels and weights, and sums next to 2^31, in the given levels' form
    import torch
    r = np.random.default_rng(tokens)
    for columns in (256, 131056):
        w = np.full((5, columns), -128, np.int8)
        w[1] = 127
        w[2] = r.integers(-128, 128, columns)
        ws = np.array([2.0 ** -30, 2.0 ** -28, 1e-7, 0.0, 2.0 ** -40], np.float32)
        levels = r.integers(-128, 128, (tokens, columns)).astype(np.int8)
        levels[0] = -128
        if tokens > 1:
            levels[1] = 127
        scales = r.random(tokens).astype(np.float32)
        call = Call(gpu_ctx, np.zeros((tokens, columns), np.float16), w, ws)
        check(call.from_levels(_dev(levels), _dev(scales)), levels, scales, w, ws, f"{columns} columns")
        torch.cuda.synchronize()


@pytest.mark.parametrize("tokens", [1, 2, 4, 5, 16, 40, 130, 600])
def test_what_is_not_finite_stays_with_its_token(gpu_ctx, tokens):
    r = np.random.default_rng(tokens)
    rows, columns = 37, 272
    w, ws = _weights(r, rows, columns)
    x = _tokens(r, tokens, columns)
    levels, scales = quantised(x)
    bad = sorted({0, tokens // 2, tokens - 1})
    for i, t in enumerate(bad):
        x[t, 5 + 100 * i] = [np.inf, np.nan, -np.inf][i]
    call = Call(gpu_ctx, x, w, ws)
    got = call.from_halves()
    good = [t for t in range(tokens) if t not in bad]
    assert np.isnan(got[bad]).all()
    if good:
        check(got[good], levels[good], scales[good], w, ws)
    got_levels, got_scales = call.quantise()
    assert np.isnan(got_scales.cpu().numpy()[bad]).all() and not got_levels.cpu().numpy()[bad].any()
    assert np.array_equal(call.from_levels(got_levels, got_scales), got, equal_nan=True)


@pytest.mark.parametrize("tokens", [1, 3, 9, 70, 300])
def test_sums_beyond_the_halves_are_infinite(gpu_ctx, tokens):
    columns = 256
    x = np.full((tokens, columns), 60000.0, np.float16)
    w = np.full((4, columns), 127, np.int8)
    w[1] = -127
    w[2] = 0
    w[3, 1:] = 0
    got = Call(gpu_ctx, x, w, np.full(4, 1 / 127.0, np.float32)).from_halves()
    assert np.isposinf(got[:, 0]).all() and np.isneginf(got[:, 1]).all() and (got[:, 2] == 0).all()
    assert (np.abs(got[:, 3].astype(np.float64) - 60000.0) <= 60000.0 * 2.0 ** -10).all()


def test_token_zeros(gpu_ctx):
    r = np.random.default_rng(3)
    w, ws = _weights(r, 40, 128)
    for tokens in (1, 5, 40, 300):
        assert not Call(gpu_ctx, np.zeros((tokens, 128), np.float16), w, ws).from_halves().any()


@pytest.mark.parametrize("tokens", [1, 7, 48, 300])
def test_captured_and_replayed(gpu_ctx, tokens):
    import torch
    r = np.random.default_rng(tokens)
    w, ws = _weights(r, 300, 1040)
    x = _tokens(r, tokens, 1040)
    call = Call(gpu_ctx, x, w, ws)
    call.from_halves()
    y = call._y()
    args = (call.weights, call.weight_scales, call.x, y, 300, 1040, tokens)
    gpu_ctx.graph_begin()
    call.projection.encode(*args)
    graph = gpu_ctx.graph_end()
    for turn in range(4):
        x = _tokens(r, tokens, 1040)
        call.x.copy_(_dev(x))
        torch.cuda.synchronize()
        eager = call.from_halves()
        y.zero_()
        torch.cuda.synchronize()
        graph.launch()
        gpu_ctx.synchronize()
        assert np.array_equal(y.cpu().numpy(), eager), f"replay {turn}"
        check(eager, *quantised(x), w, ws)
    graph.close()


def test_a_capture_does_not_grow_the_store(gpu_ctx):
    import torch
    from tinytitan_amd import capi
    from tinytitan_amd.engine import HIPContext, Int8Projection, TinyTitanHIPError
    ctx = HIPContext(0)
    projection = Int8Projection(ctx)
    r = np.random.default_rng(1)
    w, ws = _weights(r, 64, 256)
    weights, scales = _dev(w), _dev(ws)
    x = _dev(_tokens(r, 600, 256))
    y = torch.zeros(600, 64, dtype=torch.float16, device="cuda")
    torch.cuda.synchronize()
    ctx.graph_begin()
    with pytest.raises(TinyTitanHIPError) as e:
        projection.encode(weights, scales, x, y, 64, 256, 600)
    assert e.value.status == capi.ERR_BUSY
    ctx.graph_end().close()
    projection.encode(weights, scales, x, y, 64, 256, 600)
    ctx.graph_begin()
    projection.encode(weights, scales, x, y, 64, 256, 600)
    graph = ctx.graph_end()
    more = _dev(_tokens(r, 4000, 256))
    many = torch.zeros(4000, 64, dtype=torch.float16, device="cuda")
    torch.cuda.synchronize()
    projection.encode(weights, scales, more, many, 64, 256, 4000)  # the store has moved
    with pytest.raises(TinyTitanHIPError) as e:
        graph.launch()
    assert e.value.status == capi.ERR_STALE
    graph.close()
    ctx.synchronize()
    ctx.close()


def test_on_another_stream(gpu_ctx):
    import torch
    r = np.random.default_rng(2)
    w, ws = _weights(r, 512, 2048)
    call = Call(gpu_ctx, _tokens(r, 40, 2048), w, ws)
    plain = call.from_halves()
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        gpu_ctx.use_torch_stream()
        y = torch.zeros(40, 512, dtype=torch.float16, device="cuda")
        call.projection.encode(call.weights, call.weight_scales, call.x, y, 512, 2048, 40)
        copy = y.clone()
    gpu_ctx.set_stream(None)
    stream.synchronize()
    assert np.array_equal(copy.cpu().numpy(), plain)


def test_weights_past_two_gibibytes(gpu_ctx):
    import torch
    from tinytitan_amd.engine import Int8Projection
    rows, columns = 20000, 131056
    weights = torch.zeros(rows, columns, dtype=torch.int8, device="cuda")
    weights[:, :16] = 3
    weights[rows - 1] = 1
    scales = torch.full((rows,), 2.0 ** -7, device="cuda")
    for tokens in (1, 5, 40, 300):
        x = torch.zeros(tokens, columns, dtype=torch.float16, device="cuda")
        x[:, 0] = 127.0
        x[:, columns - 1] = 127.0
        y = torch.full((tokens, rows), float("nan"), dtype=torch.float16, device="cuda")
        torch.cuda.synchronize()
        Int8Projection(gpu_ctx).encode(weights, scales, x, y, rows, columns, tokens)
        gpu_ctx.synchronize()
        assert (y[:, :rows - 1] == 3 * 127 * 2.0 ** -7).all() and (y[:, rows - 1] == 2 * 127 * 2.0 ** -7).all()


def test_refusals(gpu_ctx):
    import torch
    from tinytitan_amd import capi
    from tinytitan_amd.engine import Int8Projection, TinyTitanHIPError
    p = Int8Projection(gpu_ctx)
    w = torch.ones(10, 64, dtype=torch.int8, device="cuda")
    ws = torch.ones(10, device="cuda")
    x = torch.ones(6, 80, dtype=torch.float16, device="cuda")
    y = torch.full((6, 10), 3.0, dtype=torch.float16, device="cuda")
    levels, scales = torch.zeros(6, 64, dtype=torch.int8, device="cuda"), torch.ones(6, device="cuda")
    torch.cuda.synchronize()

    def refused(status, call, *args, **kw):
        with pytest.raises(TinyTitanHIPError) as e:
            call(*args, **kw)
        assert e.value.status == status

    bad, shape = capi.ERR_INVALID_ARGUMENT, capi.ERR_SHAPE
    for rows, columns, tokens, status in ((0, 64, 4, bad), (10, 0, 4, bad), (10, 64, 0, bad), (-1, 64, 4, bad), (10, 40, 4, shape), (10, 131072, 1, shape)):
        refused(status, p.encode, w, ws, x, y, rows, columns, tokens, x_stride=80 if columns < 100 else columns, y_stride=max(rows, 1))
    refused(shape, p.encode, w, ws, x, y, 10, 64, 4, x_stride=56)
    refused(shape, p.encode, w, ws, x, y, 10, 64, 4, x_stride=68)
    refused(shape, p.encode, w, ws, x, y, 10, 64, 4, x_stride=80, y_stride=9)
    refused(shape, p.encode, w, ws, x.flatten()[1:], y, 10, 64, 4, x_stride=80)
    refused(shape, p.encode, w.flatten()[1:], ws, x, y, 9, 64, 4, x_stride=80)
    refused(bad, p.encode, None, ws, x, y, 10, 64, 4, x_stride=80)
    refused(bad, p.encode, w, None, x, y, 10, 64, 4, x_stride=80)
    refused(bad, p.encode, w, ws, None, y, 10, 64, 4, x_stride=80)
    refused(bad, p.encode, w, ws, x, None, 10, 64, 4, x_stride=80)
    refused(shape, p.quantise, x, levels, scales, 64, 6, x_stride=80, levels_stride=48)
    refused(shape, p.quantise, x, levels, scales, 64, 5, x_stride=80, levels_stride=72)
    refused(shape, p.quantise, x, levels.flatten()[1:], scales, 64, 5, x_stride=80)
    refused(bad, p.quantise, x, levels, None, 64, 5, x_stride=80)
    refused(shape, p.encode_levels, w, ws, levels, scales, y, 10, 64, 4, levels_stride=72)
    refused(shape, p.encode_levels, w, ws, levels, scales, y, 10, 64, 4, levels_stride=48)
    refused(bad, p.encode_levels, w, ws, levels, None, y, 10, 64, 4)
    refused(bad, p.encode_levels, w, ws, None, scales, y, 10, 64, 4)
    for args in ((w.float(), ws, x, y), (w, ws.double(), x, y), (w, ws, x.float(), y), (w, ws, x, y.float()), (w.cpu(), ws, x, y), (w.T, ws, x, y),
                 (torch.ones(10, 80, dtype=torch.int8, device="cuda")[:, :64], ws, x, y)):
        with pytest.raises(TypeError):
            p.encode(*args, 10, 64, 4, x_stride=80)
    gpu_ctx.synchronize()
    assert (y == 3.0).all() and not levels.any()
