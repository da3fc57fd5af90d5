"""What a layer of differential attention needs that is served in 8 bits, as cases that can be timed.

``diff``  attention whose weights are the difference of two softmax maps, over the cache of ``tinytitan_amd.engine``.  A head's query
          row of ``dim`` values is two queries of dim / 2, one behind the other, its KV head's key row two keys of dim / 2, its value
          row one value of ``dim``.  With a factor lambda per head (or per token and head):

              a     = sum_j softmax_j(scale q1.k1_j) v_j - lambda sum_j softmax_j(scale q2.k2_j) v_j
              out   = sigmoid(gate) * out_scale * weight * a / sqrt(mean(a^2) + eps)

          where the norm over the head's values (``normed``) and the gate (``gated``) may be left out.  Row p sees key j <= p, behind
          a ``window`` those with j > p - window.  As a decode step, as a draft's verify rows and as a prefill chunk, over rows of 16,
          8 or 4 bits, linear or in a ring.
``int8``  y[t] = W x[t] over weights of 8-bit integers with a scale for each output channel, and tokens quantised to 8-bit integers with
          a scale for each token:  level = round(x / s), s = max |x| / 127,  y = s * weight_scale * sum(weight_level * level), the
          sum in integers.  From fp16 tokens (the call quantises them), or (``outputs`` 2) from tokens that are quantised once for two
          products, as the projections in front of an attention share their input.

A case's sequences have ``lo`` .. ``hi`` earlier tokens, spread evenly over the logarithm, and ``rows`` new ones each, whose K and V are
already in the cache.
"""
import math

import numpy as np
import torch

own = False

DEVICE = torch.device("cuda", 0)
GROUP = 64  # consecutive values that share a scale and a bias in a cache row of 8 or 4 bits
EPS = 1e-5
LAMBDA_INIT = 0.7

_context = None


def _diff(form, shape, lo, hi=None, seqs=1, rows=1, bits=16, window=0, ring=False, by_token=False, normed=True, gated=True, pad=0, name=None):
    case = {"op": "diff", "form": form, "heads": shape[0], "kv_heads": shape[1], "dim": shape[2], "lo": lo, "hi": hi if hi is not None else lo,
            "seqs": seqs, "rows": rows, "bits": bits, "window": window, "ring": ring, "by_token": by_token, "normed": normed,
            "gated": gated, "pad": pad}
    if name:
        case["name"] = name
    return case


def _int8(tokens, channels, columns, outputs=1, pad=0, name=None):
    case = {"op": "int8", "tokens": tokens, "channels": channels, "columns": columns, "outputs": outputs, "pad": pad}
    if name:
        case["name"] = name
    return case


def listed():
    return [
        # a small model's chat: one token behind a short session, where latency is all
        _diff("decode", (8, 2, 256), 600, name="diff_decode_short"),
        # one user's token late in a long session
        _diff("decode", (16, 2, 256), 100001, name="diff_decode_100k"),
        # a serving batch of all ages over the runtime's default precision, the factor from each token's own projection
        _diff("decode", (32, 8, 128), 300, 30000, seqs=24, bits=8, by_token=True, name="diff_decode_24_8bit"),
        # a draft's four tokens checked for a few sessions on a memory-saving cache that keeps a window
        _diff("verify", (16, 2, 256), 50, 20000, seqs=7, rows=4, bits=4, window=4096, ring=True, name="diff_verify_4bit"),
        # a ragged turn of a small model, its rows inside a wider buffer, without norm and gate
        _diff("prefill", (16, 4, 64), 2001, rows=333, normed=False, gated=False, pad=72, name="diff_chunk_333"),
        # a ragged chunk deep in a session over the default precision
        _diff("prefill", (32, 8, 128), 9000, rows=777, bits=8, by_token=True, name="diff_chunk_777_8bit"),
        # a long document's chunk
        _diff("prefill", (16, 2, 256), 4500, rows=4096, name="diff_chunk_4096"),
        # the output projection of one token
        _int8(1, 2048, 4096, name="int8_token"),
        # the projections in front of an attention for a few drafts' rows: queries and gate, keys and values, from one input
        _int8(7, 9216, 2048, outputs=2, name="int8_rows_7_shared"),
        # a serving batch's step
        _int8(48, 5120, 6144, name="int8_batch_48"),
        # a ragged chunk, an odd number of channels, tokens inside a wider buffer
        _int8(777, 2311, 4096, pad=40, name="int8_chunk_777"),
        # a prompt's chunk at a large model's width
        _int8(4096, 9216, 5120, name="int8_chunk_4096"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    """One more case: both operators, every form, sizes spread over their logarithm."""
    top = [work(c) for c in listed()]
    most_bytes = max(w["bytes"] for w in top)
    while True:
        if rng.random() < 0.4:
            case = _int8(rng.choice([1, _log_int(rng, 1, 64), _log_int(rng, 2, 4096)]), _log_int(rng, 64, 16384),
                         16 * _log_int(rng, 16, 768), outputs=rng.choice([1, 1, 2]), pad=rng.choice([0, 0, 8, 40]))
        else:
            form = rng.choice(["decode", "decode", "verify", "prefill", "prefill"])
            shape = rng.choice([(8, 2, 256), (16, 2, 256), (24, 2, 256), (32, 8, 128), (12, 4, 128), (16, 4, 64)])
            case = _diff(form, shape, _log_int(rng, 1, 131072), bits=rng.choice([16, 16, 8, 8, 4]), by_token=rng.random() < 0.4,
                         normed=rng.random() < 0.75, gated=rng.random() < 0.75)
            case["hi"] = case["lo"]
            if form == "prefill":
                case["rows"] = _log_int(rng, 10, 4096)
                case["pad"] = rng.choice([0, 0, 8, 72, 5])
            else:
                case["seqs"] = rng.choice([1, _log_int(rng, 2, 40)])
                case["rows"] = 1 if form == "decode" else rng.randint(2, 8)
                if case["seqs"] > 1:
                    case["hi"] = _log_int(rng, case["lo"], 131072)
            if rng.random() < 0.35:
                case["window"], case["ring"] = _log_int(rng, 64, 8192), rng.random() < 0.5
        need = work(case)
        # no more than the largest listed case of its operator, and memory for rows padded to the longest sequence
        most_flops = max(w["flops"] for w, c in zip(top, listed()) if c["op"] == case["op"])
        if need["bytes"] > most_bytes or need["flops"] > most_flops:
            continue
        if case["op"] == "int8" or case["seqs"] * _row_count(case) * case["kv_heads"] * case["dim"] * 4 <= 8 << 30:
            return case


# ---- attention ---------------------------------------------------------------------------------------------------------------

def _lengths(case):
    """Earlier tokens of each sequence."""
    n, lo, hi = case["seqs"], case["lo"], case["hi"]
    if n == 1 or lo == hi:
        return [lo] * n
    return [max(lo, min(hi, round(math.exp(math.log(lo) + (math.log(hi) - math.log(lo)) * i / (n - 1))))) for i in range(n)]


def _first_key(case, length):
    """The first key that any of a sequence's new rows sees."""
    return max(0, length + 1 - case["window"]) if case["window"] else 0


def _row_count(case):
    """Rows that the longest sequence's new rows see."""
    return max(n + case["rows"] - _first_key(case, n) for n in _lengths(case))


def _row_bytes(case):
    """Bytes of one token's stored K (or V) row: fp16 values, or levels, then a scale and a bias per group."""
    width = case["kv_heads"] * case["dim"]
    return 2 * width if case["bits"] == 16 else width * case["bits"] // 8 + 4 * (width // GROUP)


def _stored(values, bits):
    """fp16 rows as the cache stores them, in bytes."""
    if bits == 16:
        return values.contiguous().view(torch.uint8)
    rows, width = values.shape
    x = values.float().view(rows, width // GROUP, GROUP)
    bias = x.amin(-1, keepdim=True).half()
    scale = ((x.amax(-1, keepdim=True) - bias.float()) / (2 ** bits - 1)).half()
    levels = ((x - bias.float()) / scale.float().clamp_min(1e-7)).round().clamp(0, 2 ** bits - 1).to(torch.uint8).view(rows, width)
    if bits == 4:
        levels = levels[:, 0::2] | (levels[:, 1::2] << 4)
    params = torch.cat([scale.view(rows, -1), bias.view(rows, -1)], 1).contiguous().view(torch.uint8)
    return torch.cat([levels, params], 1).contiguous()


def _values(stored, case, dtype):
    """Stored rows ``[..., bytes]`` as values ``[..., kv_heads, dim]``."""
    width, bits = case["kv_heads"] * case["dim"], case["bits"]
    shape = stored.shape[:-1] + (case["kv_heads"], case["dim"])
    if bits == 16:
        return stored.contiguous().view(torch.float16).to(dtype).view(shape)
    cut = width * bits // 8
    levels = stored[..., :cut]
    if bits == 4:
        levels = torch.stack([levels & 15, levels >> 4], -1).flatten(-2)
    params = stored[..., cut:].contiguous().view(torch.float16).to(dtype)
    scale, bias = params[..., :width // GROUP, None], params[..., width // GROUP:, None]
    return (levels.to(dtype).unflatten(-1, (width // GROUP, GROUP)) * scale + bias).reshape(shape)


def _diff_inputs(case, seed):
    """What the layers in front leave: queries and gate, the heads' factors, and the cache's rows from each sequence's first seen key on.
    Queries and first tokens' keys lean towards directions of their KV head, a different one for each of the two maps."""
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    heads, kv_heads, dim, rows, seqs = (case[k] for k in ("heads", "kv_heads", "dim", "rows", "seqs"))
    tokens, width, half = seqs * rows, heads * dim, dim // 2

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device=DEVICE, dtype=torch.float16)

    def rand(*shape):
        return torch.rand(*shape, generator=gen, device=DEVICE)

    lean = torch.randn(kv_heads, 2, half, generator=gen, device=DEVICE)
    lean = (lean / (lean * lean).sum(-1, keepdim=True).sqrt() * (3.0 * half ** 0.5) ** 0.5).view(kv_heads, dim)
    x = {"scale": half ** -0.5}
    q = randn(tokens, heads, dim).float() + lean.repeat_interleave(heads // kv_heads, 0)
    x["q"] = torch.zeros(tokens, width + case["pad"], dtype=torch.float16, device=DEVICE)
    x["q"][:, :width] = q.half().view(tokens, width)
    x["gate"] = randn(tokens, width + case["pad"]) if case["gated"] else None
    x["lambdas"] = 0.2 + 0.7 * (rand(tokens, heads) if case["by_token"] else rand(heads))
    x["norm"] = (1.0 + 0.1 * torch.randn(dim, generator=gen, device=DEVICE)).bfloat16() if case["normed"] else None
    x["out_scale"] = 1.0 - LAMBDA_INIT
    x["lengths"] = _lengths(case)
    x["firsts"] = [_first_key(case, n) for n in x["lengths"]]
    longest = _row_count(case)
    x["k"] = torch.zeros(seqs, longest, _row_bytes(case), dtype=torch.uint8, device=DEVICE)
    x["v"] = torch.zeros_like(x["k"])
    for i, (first, length) in enumerate(zip(x["firsts"], x["lengths"])):
        n = length + rows - first
        k = randn(n, kv_heads, dim)
        if first < 4:
            k[:4 - first] = (k[:4 - first].float() + lean).half()
        x["k"][i, :n], x["v"][i, :n] = _stored(k.view(n, -1), case["bits"]), _stored(randn(n, kv_heads * dim), case["bits"])
    return x


class State:
    """What a program has in hand between calls."""


def _fill(kv, slot, first, k, v, ring):
    """Stored rows into their places of a slot, on a ring a run that does not wrap at a time."""
    at = 0
    while at < k.shape[0]:
        n = k.shape[0] - at
        if ring:
            n = min(n, ring - (first + at) % ring)
        kv.import_rows(0, slot, first + at, k[at:at + n].contiguous(), v[at:at + n].contiguous())
        at += n


def _own_context():
    from tinytitan_amd.engine import HIPContext
    global _context
    if _context is None:
        _context = HIPContext(0)
    _context.use_torch_stream()
    return _context


def _prepare_diff(s, case, seed):
    x = s.x = _diff_inputs(case, seed)
    s.out = torch.zeros(case["seqs"] * case["rows"], case["heads"] * case["dim"] + case["pad"], dtype=torch.float16, device=DEVICE)
    if not own:
        return s
    from tinytitan_amd.engine import DifferentialAttention, DifferentialHeads, KVCacheManager
    context = _own_context()
    total = max(x["lengths"]) + case["rows"]
    ring = -(-(case["window"] + case["rows"] + 32) // 32) * 32 if case["ring"] else 0
    s.kv = KVCacheManager(context, 1, case["kv_heads"], case["dim"], slots=case["seqs"], max_context=total, initial_capacity=total,
                          precision_bits=case["bits"], ring_capacity=ring)
    for i, (first, length) in enumerate(zip(x["firsts"], x["lengths"])):
        n = length + case["rows"] - first
        _fill(s.kv, i, first, x["k"][i, :n], x["v"][i, :n], ring)
    s.slots = list(range(case["seqs"]))
    s.heads = DifferentialHeads(x["lambdas"], norm_weight=x["norm"], eps=EPS, out_scale=x["out_scale"])
    s.attention = DifferentialAttention(context)
    return s


def _run_own_diff(s):
    from tinytitan_amd.engine import PrefillAttentionParams
    case, x = s.case, s.x
    heads, rows, width = case["heads"], case["rows"], case["heads"] * case["dim"]
    if case["form"] == "prefill":
        start, stride = x["lengths"][0], width + case["pad"]
        params = PrefillAttentionParams(start, rows, start + rows, heads, x["scale"], stride, stride, stride, sliding_window=case["window"])
        s.attention.encode_causal(s.kv, 0, 0, x["q"], s.out, params, s.heads, gate=x["gate"])
    elif case["form"] == "verify":
        s.attention.encode_verify_rows(s.kv, 0, x["q"], s.out, heads, x["lengths"], rows, x["scale"], s.heads, s.slots, gate=x["gate"],
                                       window=case["window"])
    else:
        s.attention.encode_full(s.kv, 0, x["q"], s.out, heads, [n + 1 for n in x["lengths"]], x["scale"], s.heads, slot=s.slots,
                                gate=x["gate"], window=case["window"])
    return s.out[:, :width]


def _run_plain_diff(s):
    case, x = s.case, s.x
    heads, kv_heads, dim, rows, seqs = (case[k] for k in ("heads", "kv_heads", "dim", "rows", "seqs"))
    group, width, half = heads // kv_heads, heads * dim, dim // 2
    q = x["q"][:, :width].float().view(seqs, rows, kv_heads, group, 2, half) * x["scale"]
    q = q.permute(0, 2, 4, 1, 3, 5).reshape(seqs, kv_heads, 2, rows * group, half)
    # keys [seqs, kv_heads, 2, half, keys], values [seqs, kv_heads, keys, dim]
    k = _values(x["k"], case, torch.float32).unflatten(-1, (2, half)).permute(0, 2, 3, 4, 1).contiguous()
    v = _values(x["v"], case, torch.float32).permute(0, 2, 1, 3).contiguous()
    at = (torch.tensor(x["lengths"], device=DEVICE)[:, None] + torch.arange(rows, device=DEVICE))[:, :, None]
    keys = (torch.tensor(x["firsts"], device=DEVICE)[:, None] + torch.arange(k.shape[-1], device=DEVICE))[:, None]
    seen = keys <= at
    if case["window"]:
        seen = seen & (keys > at - case["window"])
    hidden = ~seen[:, None].repeat_interleave(group, 2)
    maps = []
    for m in range(2):
        scores = torch.matmul(q[:, :, m], k[:, :, m].contiguous()).masked_fill(hidden, float("-inf"))
        weights = torch.exp(scores - scores.amax(-1, keepdim=True))
        maps.append(torch.matmul(weights, v) / weights.sum(-1, keepdim=True))
    first, second = (m.view(seqs, kv_heads, rows, group, dim).permute(0, 2, 1, 3, 4).reshape(seqs * rows, heads, dim) for m in maps)
    out = first - x["lambdas"][..., None] * second
    if x["norm"] is not None:
        out = out / (out * out).mean(-1, keepdim=True).add(EPS).sqrt() * x["norm"].float()
    out = (out * x["out_scale"]).view(seqs * rows, width)
    if x["gate"] is not None:
        out = out / (1.0 + torch.exp(-x["gate"][:, :width].float()))
    s.out[:, :width] = out.half()
    return s.out[:, :width]


def _exact_diff(case, seed):
    """The definition in 64 bits: sequence by sequence and head by head, some rows at a time."""
    x = _diff_inputs(case, seed)
    heads, kv_heads, dim, rows = (case[k] for k in ("heads", "kv_heads", "dim", "rows"))
    group, half = heads // kv_heads, dim // 2
    result = torch.zeros(case["seqs"] * rows, heads, dim, dtype=torch.float64, device=DEVICE)
    lambdas = x["lambdas"].double().expand(case["seqs"] * rows, heads)
    for i, (first, length) in enumerate(zip(x["firsts"], x["lengths"])):
        n = length + rows - first
        k, v = _values(x["k"][i, :n], case, torch.float64), _values(x["v"][i, :n], case, torch.float64)
        position = torch.arange(first, first + n, device=DEVICE)
        for r0 in range(0, rows, 512):
            r1 = min(r0 + 512, rows)
            distance = torch.arange(length + r0, length + r1, device=DEVICE)[:, None] - position[None]
            hidden = distance < 0
            if case["window"]:
                hidden |= distance >= case["window"]
            lines = slice(i * rows + r0, i * rows + r1)
            for h in range(heads):
                row = x["q"][lines, h * dim:(h + 1) * dim].double()
                both = 0.0
                for part, sign in ((slice(0, half), 1.0), (slice(half, dim), -lambdas[lines, h, None])):
                    logits = (row[:, part] @ k[:, h // group, part].T.contiguous()) * x["scale"]
                    logits[hidden] = -np.inf
                    both = both + sign * torch.softmax(logits, -1)
                result[lines, h] = both @ v[:, h // group].contiguous()
    if x["norm"] is not None:
        result *= torch.rsqrt(result.square().mean(-1, keepdim=True) + EPS) * x["norm"].double()
    result = result.flatten(1) * x["out_scale"]
    if x["gate"] is not None:
        result *= torch.sigmoid(x["gate"][:, :heads * dim].double())
    return result


# ---- products of 8-bit integers --------------------------------------------------------------------------------------------------

def _channels(case):
    """Output channels of each product: of two, the second is an eighth of the first, as keys and values beside queries."""
    return [case["channels"], max(1, case["channels"] // 8)][:case["outputs"]]


def _int8_inputs(case, seed):
    """Tokens as a norm leaves them, a few of their columns much larger than the rest, and weights quantised channel by channel."""
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    tokens, columns = case["tokens"], case["columns"]
    x = torch.randn(tokens, columns + case["pad"], generator=gen, device=DEVICE)
    loud = torch.randint(0, columns, (max(1, columns // 256),), generator=gen, device=DEVICE)
    x[:, loud] *= 6.0
    inputs = {"x": x.half(), "weights": [], "scales": []}
    for channels in _channels(case):
        w = torch.randn(channels, columns, generator=gen, device=DEVICE) * columns ** -0.5
        scale = w.abs().amax(-1) / 127.0
        inputs["weights"].append((w / scale[:, None]).round().to(torch.int8))
        inputs["scales"].append(scale)
    return inputs


def _prepare_int8(s, case, seed):
    s.x = _int8_inputs(case, seed)
    tokens, columns = case["tokens"], case["columns"]
    s.outs = [torch.zeros(tokens, n, dtype=torch.float16, device=DEVICE) for n in _channels(case)]
    if not own:
        return s
    from tinytitan_amd.engine import Int8Projection
    s.projection = Int8Projection(_own_context())
    s.levels = torch.empty(tokens, columns, dtype=torch.int8, device=DEVICE)
    s.token_scales = torch.empty(tokens, dtype=torch.float32, device=DEVICE)
    return s


def _run_own_int8(s):
    case, x = s.case, s.x
    tokens, columns, stride = case["tokens"], case["columns"], case["columns"] + case["pad"]
    if case["outputs"] == 1:
        s.projection.encode(x["weights"][0], x["scales"][0], x["x"], s.outs[0], case["channels"], columns, tokens, x_stride=stride)
    else:
        s.projection.quantise(x["x"], s.levels, s.token_scales, columns, tokens, x_stride=stride)
        for w, scale, y in zip(x["weights"], x["scales"], s.outs):
            s.projection.encode_levels(w, scale, s.levels, s.token_scales, y, w.shape[0], columns, tokens)
    return s.outs


def _run_plain_int8(s):
    x, columns = s.x, s.case["columns"]
    tokens = x["x"][:, :columns].float()
    token_scale = tokens.abs().amax(-1, keepdim=True) / 127.0
    levels = torch.where(token_scale > 0, tokens / token_scale, torch.zeros_like(tokens)).round()
    for w, scale, y in zip(x["weights"], x["scales"], s.outs):
        y.copy_((torch.matmul(levels, w.float().T.contiguous()) * scale * token_scale).half())
    return s.outs


def _exact_int8(case, seed):
    """The definition in 64 bits; the scales are the 32-bit numbers that the operator hands on."""
    inputs = _int8_inputs(case, seed)
    x = inputs["x"][:, :case["columns"]].double()
    s = (x.abs().max(dim=1).values.float() / np.float32(127.0)).double()[:, None]
    levels = torch.round(x / s.clamp_min(1e-300))
    return [(levels @ w.double().T.contiguous()) * (s * scale.double()[None]) for w, scale in zip(inputs["weights"], inputs["scales"])]


# ---- the cases' interface -------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    s = State()
    s.case = case
    return (_prepare_diff if case["op"] == "diff" else _prepare_int8)(s, case, seed)


def run(s):
    if s.case["op"] == "diff":
        return _run_own_diff(s) if own else _run_plain_diff(s)
    return _run_own_int8(s) if own else _run_plain_int8(s)


def exact(case, seed):
    return _exact_diff(case, seed) if case["op"] == "diff" else _exact_int8(case, seed)


def work(case):
    if case["op"] == "int8":
        tokens, columns, channels = case["tokens"], case["columns"], sum(_channels(case))
        return {"bytes": channels * (columns + 4) + tokens * columns * 2 + tokens * channels * 2, "flops": 2 * tokens * columns * channels}
    heads, dim, rows, seqs = (case[k] for k in ("heads", "dim", "rows", "seqs"))
    keys = pairs = 0
    for length in _lengths(case):
        keys += length + rows - _first_key(case, length)
        for p in range(length, length + rows):
            pairs += min(p + 1, case["window"]) if case["window"] else p + 1
    moved = keys * 2 * _row_bytes(case) + seqs * rows * heads * dim * 2 * (3 if case["gated"] else 2)
    return {"bytes": moved + 4 * heads * (seqs * rows if case["by_token"] else 1), "flops": 6 * dim * heads * pairs}
