"""Attention whose keys lie in two pieces of the cache, as cases that can be timed.

Two operators over the cache of ``tinytitan_amd.engine``, each as a decode step (one token a sequence), as verify rows (a draft's
few tokens a sequence) and as a prefill chunk (many tokens of one sequence), over rows of 16, 8 or 4 bits:

``sinks``   a sliding window and a few first tokens that stay visible.  The row at position p sees key j <= p where
            j > p - window or j < sinks.
``shared``  sequences that start from one prefix.  Key j < prefix of any of them is row j of the prefix's slot, which is stored and
            read once for all of them; key j >= prefix is row j of the sequence's own slot.

Both end in the softmax-weighted sum of the values and, with ``gated``, the output gate: out = sigmoid(gate) * sum_j softmax_j(scale q.k_j) v_j.

A case's sequences have ``lo`` .. ``hi`` earlier tokens (of ``shared``: behind the prefix), spread evenly over the logarithm, and
``rows`` new ones each, whose K and V are already in the cache.
"""
import math

import numpy as np
import torch

own = False

DEVICE = torch.device("cuda", 0)
GROUP = 64  # consecutive values that share a scale and a bias in a row of 8 or 4 bits

_context = None


def _case(op, form, shape, lo, hi=None, seqs=1, rows=1, bits=16, window=0, sinks=0, ring=False, prefix=0, gated=True, pad=0, name=None):
    case = {"op": op, "form": form, "heads": shape[0], "kv_heads": shape[1], "dim": shape[2], "lo": lo, "hi": hi if hi is not None else lo,
            "seqs": seqs, "rows": rows, "bits": bits, "window": window, "sinks": sinks, "ring": ring, "prefix": prefix, "gated": gated,
            "pad": pad}
    if name:
        case["name"] = name
    return case


def listed():
    return [
        # a small model's chat that has just outgrown its window: one token, where latency is all
        _case("sinks", "decode", (8, 2, 256), 600, window=256, sinks=4, name="sinks_decode_short"),
        # one user's token late in a long session of a model with a wide window
        _case("sinks", "decode", (16, 2, 256), 100001, window=32000, sinks=128, name="sinks_decode_100k"),
        # a serving batch of endless sessions over the runtime's default precision, each in a ring of bounded memory
        _case("sinks", "decode", (32, 8, 128), 2999, 120000, seqs=24, bits=8, window=4096, sinks=4, ring=True, name="sinks_decode_ring_8bit"),
        # a draft's four tokens checked for a few sessions of all ages, some younger than the window, on a memory-saving cache
        _case("sinks", "verify", (16, 2, 256), 20, 50000, seqs=7, rows=4, bits=4, window=1024, sinks=33, ring=True, name="sinks_verify_4bit"),
        # a ragged turn of a small model, its rows inside a wider buffer
        _case("sinks", "prefill", (16, 4, 64), 2001, rows=333, window=500, sinks=7, gated=False, pad=72, name="sinks_chunk_333"),
        # a ragged chunk deep in a session over the default precision and a ring
        _case("sinks", "prefill", (32, 8, 128), 30000, rows=777, bits=8, window=2048, sinks=4, ring=True, name="sinks_chunk_777_8bit"),
        # a long document's chunk
        _case("sinks", "prefill", (16, 2, 256), 9000, rows=4096, window=4096, sinks=64, name="sinks_chunk_4096"),
        # two samples of one short prompt on a small model: latency again
        _case("shared", "decode", (16, 4, 64), 20, 90, seqs=2, prefix=300, name="shared_decode_2"),
        # a serving batch behind one system prompt over the default precision
        _case("shared", "decode", (32, 8, 128), 1, 500, seqs=20, bits=8, prefix=6007, name="shared_decode_20_8bit"),
        # many samples, or many users' questions, about one long document
        _case("shared", "decode", (16, 2, 256), 50, 2000, seqs=64, prefix=30011, name="shared_decode_64"),
        # a draft's three tokens for a few of them on a memory-saving cache, at a head count that fills no tile
        _case("shared", "verify", (24, 2, 256), 10, 300, seqs=6, rows=3, bits=4, prefix=12345, name="shared_verify_4bit"),
        # a session's own first chunk behind a system prompt that another slot holds
        _case("shared", "prefill", (16, 2, 256), 0, rows=2048, prefix=8200, name="shared_chunk_2048"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    """One more case: both operators and every form, sizes spread over their logarithm."""
    top = [work(c) for c in listed()]
    most_bytes, most_flops = max(w["bytes"] for w in top), max(w["flops"] for w in top)
    while True:
        op, form = rng.choice(["sinks", "shared"]), rng.choice(["decode", "decode", "verify", "prefill"])
        shape = rng.choice([(8, 2, 256), (16, 2, 256), (24, 2, 256), (32, 8, 128), (16, 4, 64)])
        case = _case(op, form, shape, 1, bits=rng.choice([16, 16, 8, 8, 4]), gated=rng.random() < 0.75)
        if form == "prefill":
            case["rows"] = _log_int(rng, 10, 4096)
            case["pad"] = rng.choice([0, 0, 8, 72, 5])
        else:
            case["seqs"] = rng.choice([1, _log_int(rng, 2, 40)]) if op == "sinks" else _log_int(rng, 2, 64)
            case["rows"] = 1 if form == "decode" else rng.randint(2, 8)
        if op == "sinks":
            case["window"], case["sinks"], case["ring"] = _log_int(rng, 64, 8192), _log_int(rng, 1, 300), rng.random() < 0.5
            case["lo"] = _log_int(rng, 1, 131072)
            case["hi"] = _log_int(rng, case["lo"], 131072) if case["seqs"] > 1 else case["lo"]
        else:
            case["prefix"] = _log_int(rng, 17, 65536)
            case["lo"] = _log_int(rng, 1, 2000)
            case["hi"] = _log_int(rng, case["lo"], 4000) if case["seqs"] > 1 else case["lo"]
        need = work(case)
        # no more than the largest listed cases, and memory for the slots' pages and for rows padded to the longest sequence
        slots, tokens = case["seqs"] + (op == "shared"), case["prefix"] + case["hi"] + case["rows"]
        if case["ring"]:
            tokens = case["window"] + case["rows"] + 400
        if need["bytes"] <= most_bytes and need["flops"] <= most_flops and slots * tokens * shape[1] * shape[2] * 4 <= 8 << 30:
            return case


def _lengths(case):
    """Earlier tokens of each sequence (of ``shared``: behind the prefix)."""
    n, lo, hi = case["seqs"], case["lo"], case["hi"]
    if n == 1 or lo == hi:
        return [lo] * n
    return [max(lo, min(hi, round(math.exp(math.log(lo) + (math.log(hi) - math.log(lo)) * i / (n - 1))))) for i in range(n)]


def _key_positions(case, length):
    """Positions of the rows of a sequence's own slot that its new rows see."""
    if case["op"] == "shared":
        return list(range(case["prefix"], case["prefix"] + length + case["rows"]))
    first = max(0, length + 1 - case["window"])
    return list(range(min(case["sinks"], first))) + list(range(first, length + case["rows"]))


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


def _inputs(case, seed):
    """What the layers in front leave: queries and gate, and the cache's rows with their positions.  The queries lean towards a
    direction of their KV head, and the first tokens' keys do too, as first tokens do that a model keeps returning to."""
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    heads, kv_heads, dim, rows, seqs = (case[k] for k in ("heads", "kv_heads", "dim", "rows", "seqs"))
    tokens, width = seqs * rows, heads * dim

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device=DEVICE, dtype=torch.float16)

    lean = torch.nn.functional.normalize(torch.randn(kv_heads, dim, generator=gen, device=DEVICE), dim=-1) * (3.0 * dim ** 0.5) ** 0.5
    x = {"scale": dim ** -0.5}
    q = randn(tokens, heads, dim).float() + lean.repeat_interleave(heads // kv_heads, 0)
    x["q"] = torch.zeros(tokens, width + case["pad"], dtype=torch.float16, device=DEVICE)
    x["q"][:, :width] = q.half().view(tokens, width)
    x["gate"] = randn(tokens, width + case["pad"]) if case["gated"] else None

    def stored(n, first_tokens=0):
        k = randn(n, kv_heads, dim)
        if first_tokens:
            k[:first_tokens] = (k[:first_tokens].float() + lean).half()
        return _stored(k.view(n, -1), case["bits"]), _stored(randn(n, kv_heads * dim), case["bits"])

    if case["op"] == "shared":
        x["prefix_k"], x["prefix_v"] = stored(case["prefix"], min(4, case["prefix"]))
    x["lengths"] = _lengths(case)
    positions = [_key_positions(case, n) for n in x["lengths"]]
    longest = max(len(p) for p in positions)
    x["positions"] = torch.tensor([p + [1 << 40] * (longest - len(p)) for p in positions], device=DEVICE)  # (padding: behind every row)
    x["k"] = torch.zeros(seqs, longest, _row_bytes(case), dtype=torch.uint8, device=DEVICE)
    x["v"] = torch.zeros_like(x["k"])
    for i, p in enumerate(positions):
        first_tokens = sum(1 for j in p[:case["sinks"]] if j < case["sinks"])
        x["k"][i, :len(p)], x["v"][i, :len(p)] = stored(len(p), first_tokens)
    x["own_counts"] = [len(p) for p in positions]
    return x


class State:
    """What a program has in hand between calls."""


def _fill(kv, slot, positions, k, v, ring, pinned):
    """Stored rows into their places of a slot, a run of consecutive positions (on a ring: that does not wrap) at a time."""
    at = 0
    while at < len(positions):
        n = 1
        while at + n < len(positions) and positions[at + n] == positions[at] + n:
            n += 1
        p = positions[at]
        if ring:
            n = min(n, pinned - p if p < pinned else ring - (p - pinned) % ring)
        kv.import_rows(0, slot, p, k[at:at + n].contiguous(), v[at:at + n].contiguous())
        at += n


def prepare(case, seed):
    s = State()
    s.case, s.x = case, _inputs(case, seed)
    tokens, width, pad = case["seqs"] * case["rows"], case["heads"] * case["dim"], case["pad"]
    s.out = torch.zeros(tokens, width + pad, dtype=torch.float16, device=DEVICE)
    if not own:
        return s
    from tinytitan_amd.engine import Attention, HIPContext, KVCacheManager, PrefillAttention, SharedPrefix
    global _context
    if _context is None:
        _context = HIPContext(0)
    _context.use_torch_stream()
    x, prefix = s.x, case["prefix"]
    total = prefix + max(x["lengths"]) + case["rows"]
    if case["op"] == "shared":
        s.kv = KVCacheManager(_context, 1, case["kv_heads"], case["dim"], slots=case["seqs"] + 1, max_context=total, initial_capacity=total,
                              precision_bits=case["bits"])
        s.kv.import_rows(0, 0, 0, x["prefix_k"], x["prefix_v"])
        s.kv.advance(0, prefix)
        s.slots = list(range(1, case["seqs"] + 1))
        s.kv.share_prefix(0, prefix, s.slots)
        s.prefix = SharedPrefix(0, prefix)
    else:
        ring = -(-(case["window"] + case["rows"] + 32) // 32) * 32 if case["ring"] else 0
        s.kv = KVCacheManager(_context, 1, case["kv_heads"], case["dim"], slots=case["seqs"], max_context=total, initial_capacity=total,
                              precision_bits=case["bits"], ring_capacity=ring, sink_tokens=case["sinks"] if ring else 0)
        s.slots, s.prefix = list(range(case["seqs"])), None
    pinned = -(-case["sinks"] // 32) * 32
    for i, slot in enumerate(s.slots):
        n = x["own_counts"][i]
        ring = -(-(case["window"] + case["rows"] + 32) // 32) * 32 if case["ring"] else 0
        _fill(s.kv, slot, x["positions"][i, :n].tolist(), x["k"][i, :n], x["v"][i, :n], ring, pinned)
    s.starts = [prefix + n for n in x["lengths"]]
    s.attention, s.chunks = Attention(_context), PrefillAttention(_context)
    return s


def _run_own(s):
    from tinytitan_amd.engine import PrefillAttentionParams
    case, x = s.case, s.x
    heads, rows, width, stride = case["heads"], case["rows"], case["heads"] * case["dim"], case["heads"] * case["dim"] + case["pad"]
    if case["form"] == "prefill":
        start = s.starts[0]
        params = PrefillAttentionParams(start, rows, start + rows, heads, x["scale"], stride, stride, stride, sliding_window=case["window"],
                                        sinks=case["sinks"])
        s.chunks.encode_causal(s.kv, 0, s.slots[0], x["q"], s.out, params, gate=x["gate"], prefix=s.prefix)
    elif case["form"] == "verify" and case["op"] == "sinks":
        s.attention.encode_verify_rows(s.kv, 0, x["q"], s.out, heads, s.starts, rows, x["scale"], s.slots, gate=x["gate"],
                                       window=case["window"], sinks=case["sinks"])
    elif case["form"] == "verify":
        s.attention.encode_verify_rows(s.kv, 0, x["q"], s.out, heads, s.starts, rows, x["scale"], s.slots, gate=x["gate"], prefix=s.prefix)
    elif case["op"] == "sinks":
        s.attention.encode_swa(s.kv, 0, x["q"], s.out, heads, [p + 1 for p in s.starts], case["window"], x["scale"], slot=s.slots,
                               gate=x["gate"], sinks=case["sinks"])
    else:
        s.attention.encode_full(s.kv, 0, x["q"], s.out, heads, [p + 1 for p in s.starts], x["scale"], slot=s.slots, gate=x["gate"],
                                prefix=s.prefix)
    return s.out[:, :width]


def run(s):
    if own:
        return _run_own(s)
    case, x = s.case, s.x
    heads, kv_heads, dim, rows, seqs = (case[k] for k in ("heads", "kv_heads", "dim", "rows", "seqs"))
    group, width = heads // kv_heads, heads * dim
    q = x["q"][:, :width].float().view(seqs, rows, kv_heads, group, dim) * x["scale"]
    # own keys: [seqs, kv_heads, rows * group, keys]
    k = _values(x["k"], case, torch.float32).permute(0, 2, 3, 1).contiguous()
    v = _values(x["v"], case, torch.float32).permute(0, 2, 1, 3).contiguous()
    scores = torch.matmul(q.permute(0, 2, 1, 3, 4).reshape(seqs, kv_heads, rows * group, dim), k)
    start = torch.tensor([case["prefix"] + n for n in x["lengths"]], device=DEVICE)
    at = (start[:, None] + torch.arange(rows, device=DEVICE))[:, :, None]
    keys = x["positions"][:, None, :]
    seen = keys <= at
    if case["op"] == "sinks":
        seen = seen & ((keys > at - case["window"]) | (keys < case["sinks"]))
    scores = scores.masked_fill(~seen[:, None].repeat_interleave(group, 2), float("-inf"))
    top = scores.amax(-1, keepdim=True)
    if case["op"] == "shared":
        # the prefix's keys for all sequences at once: [kv_heads, seqs * rows * group, keys]
        pk = _values(x["prefix_k"], case, torch.float32).permute(1, 2, 0).contiguous()
        pv = _values(x["prefix_v"], case, torch.float32).permute(1, 0, 2).contiguous()
        first = torch.matmul(q.permute(2, 0, 1, 3, 4).reshape(kv_heads, seqs * rows * group, dim), pk)
        by_seq = (kv_heads, seqs, rows * group, 1)
        top = torch.maximum(top, first.amax(-1).view(by_seq).transpose(0, 1))
        first = torch.exp(first - top.transpose(0, 1).reshape(kv_heads, -1, 1))
    weights = torch.exp(scores - top)
    total, out = weights.sum(-1, keepdim=True), torch.matmul(weights, v)
    if case["op"] == "shared":
        total = total + first.sum(-1).view(by_seq).transpose(0, 1)
        out = out + torch.matmul(first, pv).view(kv_heads, seqs, rows * group, dim).transpose(0, 1)
    out = (out / total).view(seqs, kv_heads, rows, group, dim).permute(0, 2, 1, 3, 4).reshape(seqs * rows, width)
    if x["gate"] is not None:
        out = out / (1.0 + torch.exp(-x["gate"][:, :width].float()))
    s.out[:, :width] = out.half()
    return s.out[:, :width]


def exact(case, seed):
    """The definition in 64 bits: sequence by sequence, KV head by KV head, each over the keys in the order of their positions."""
    x = _inputs(case, seed)
    heads, kv_heads, dim, rows = (case[k] for k in ("heads", "kv_heads", "dim", "rows"))
    group, width = heads // kv_heads, heads * dim
    result = torch.zeros(case["seqs"] * rows, width, dtype=torch.float64, device=DEVICE)
    if case["op"] == "shared":
        front = [_values(x[name], case, torch.float64) for name in ("prefix_k", "prefix_v")]
    for i, length in enumerate(x["lengths"]):
        n = x["own_counts"][i]
        k, v = _values(x["k"][i, :n], case, torch.float64), _values(x["v"][i, :n], case, torch.float64)
        position = x["positions"][i, :n].double()
        if case["op"] == "shared":
            k, v = torch.cat([front[0], k]), torch.cat([front[1], v])
            position = torch.cat([torch.arange(case["prefix"], device=DEVICE, dtype=torch.float64), position])
        for first in range(0, rows, 512):
            some = range(first, min(first + 512, rows))
            at = torch.tensor([case["prefix"] + length + r for r in some], device=DEVICE, dtype=torch.float64)
            distance = at[:, None] - position[None]
            hidden = distance < 0
            if case["op"] == "sinks":
                hidden |= (distance >= case["window"]) & (position[None] >= case["sinks"])
            lines = slice(i * rows + some[0], i * rows + some[-1] + 1)
            for h in range(heads):
                columns = slice(h * dim, (h + 1) * dim)
                logits = (x["q"][lines, columns].double() @ k[:, h // group].T.contiguous()) * x["scale"]
                logits[hidden] = -np.inf
                result[lines, columns] = torch.softmax(logits, -1) @ v[:, h // group].contiguous()
    if x["gate"] is not None:
        result *= torch.sigmoid(x["gate"][:, :width].double())
    return result


def work(case):
    heads, kv_heads, dim, rows, seqs = (case[k] for k in ("heads", "kv_heads", "dim", "rows", "seqs"))
    keys = case["prefix"]  # (of ``shared``: once for all)
    pairs = 0
    for length in _lengths(case):
        if case["op"] == "shared":
            keys += length + rows
            pairs += rows * (case["prefix"] + length) + rows * (rows + 1) // 2
            continue
        keys += len(_key_positions(case, length))
        for r in range(rows):
            p, w, s = length + r, case["window"], case["sinks"]
            pairs += p + 1 if p < w else w + min(s, p + 1 - w)
    moved = keys * 2 * _row_bytes(case) + seqs * rows * heads * dim * 2 * (3 if case["gated"] else 2)
    return {"bytes": moved, "flops": 4 * dim * heads * pairs}
