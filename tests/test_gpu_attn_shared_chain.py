"""A slot that starts from another's prefix holds none of it but the last part block: what needs rows that are not there is refused --
such a slot as a prefix of its own, a shorter prefix than the one it started from -- and what has them is served again."""
import numpy as np
import pytest

from tests.exact_attention import attend, check, dequantise, stored_rows
from tests.test_gpu_attn_shared_prefix import _fill
from tests.test_gpu_attn_sinks import _dev, _rows

pytestmark = pytest.mark.gpu

H, KH, D, SCALE = 8, 2, 64, 0.125


class Slots:
    """A cache whose rows are known: what each slot was written with, position by position."""

    def __init__(self, ctx, slots, capacity, bits=16):
        from tinytitan_amd.engine import KVCacheManager
        self.ctx, self.bits = ctx, bits
        self.kv = KVCacheManager(ctx, 1, KH, D, slots=slots, max_context=capacity, initial_capacity=capacity, precision_bits=bits)
        r = np.random.default_rng(5)
        self.rows = [[stored_rows(r.standard_normal((capacity, KH * D)), bits) for _ in "kv"] for _ in range(slots)]

    def write(self, slot, first, last):
        _fill(self.kv, slot, first, *(part[first:last] for part in self.rows[slot]))

    def call(self, form, slot, length, prefix):
        """The last row of ``length`` keys of ``slot``; its queries and what came out."""
        import torch
        from tinytitan_amd.engine import Attention, PrefillAttention, PrefillAttentionParams, SharedPrefix
        q = _rows(length, 1, H, D)
        qd, out, p = _dev(q), torch.full((1, H, D), 3.0, dtype=torch.float16, device="cuda"), SharedPrefix(*prefix)
        torch.cuda.synchronize()
        try:
            if form == "decode":
                Attention(self.ctx).encode_full(self.kv, 0, qd, out, H, [length], SCALE, slot=[slot], prefix=p)
            elif form == "verify":
                Attention(self.ctx).encode_verify_rows(self.kv, 0, qd, out, H, [length - 1], 1, SCALE, [slot], prefix=p)
            else:
                PrefillAttention(self.ctx).encode_causal(self.kv, 0, slot, qd, out,
                                                         PrefillAttentionParams(length - 1, 1, length, H, SCALE, H * D, H * D, H * D), prefix=p)
        finally:
            self.ctx.synchronize()
            self.out = out.cpu().numpy()
        return q[0], self.out

    def served(self, slot, length, prefix):
        home, front = prefix
        for form in ("decode", "verify", "prefill"):
            q, out = self.call(form, slot, length, prefix)
            k, v = (dequantise(np.concatenate([a[:front], b[front:length]]), KH * D, self.bits) for a, b in zip(self.rows[home], self.rows[slot]))
            check(out, [attend(q, k, v, np.ones(length, bool), SCALE, None, self.bits)], f"{form}, slot {slot} behind {prefix}")

    def refused(self, slot, length, prefix):
        from tinytitan_amd import capi
        from tinytitan_amd.engine import TinyTitanHIPError
        for form in ("decode", "verify", "prefill"):
            with pytest.raises(TinyTitanHIPError) as e:
                self.call(form, slot, length, prefix)
            assert e.value.status == capi.ERR_CURSOR, form
            assert (self.out == 3.0).all(), form

    def not_shared(self, home, length, slots):
        from tinytitan_amd import capi
        from tinytitan_amd.engine import TinyTitanHIPError
        before = [self.kv.position(s) for s in range(len(self.rows))]
        with pytest.raises(TinyTitanHIPError) as e:
            self.kv.share_prefix(home, length, slots)
        assert e.value.status == capi.ERR_CURSOR
        assert [self.kv.position(s) for s in range(len(self.rows))] == before


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("prefix", [33, 96, 500])
def test_a_slot_that_starts_from_a_prefix_is_none_itself(gpu_ctx, bits, prefix):
    s = Slots(gpu_ctx, 4, prefix + 140, bits)
    s.write(0, 0, prefix)
    s.kv.advance(0, prefix)
    s.kv.share_prefix(0, prefix, [1])
    s.write(1, prefix, prefix + 100)
    s.kv.advance(1, 100)
    s.served(1, prefix + 100, (0, prefix))
    # a conversation forked from slot 1, whose pages do not hold the prompt
    for length in (1, 31, prefix, prefix + 100):
        s.not_shared(1, length, [2])
    s.refused(2, prefix + 1, (1, prefix))
    s.refused(1, prefix + 100, (1, prefix))
    # ... and a call that says less of the prompt is another slot's than is
    if prefix >= 64:
        s.refused(1, prefix + 100, (0, 33))
    s.refused(1, prefix + 100, (0, 31))
    # the prompt, not its first user, is what the fork starts from
    s.kv.share_prefix(0, prefix, [2])
    s.write(2, prefix, prefix + 7)
    s.served(2, prefix + 7, (0, prefix))
    s.served(1, prefix + 100, (0, prefix))
    s.kv.close()


def test_rows_of_its_own_make_it_one_again(gpu_ctx):
    s = Slots(gpu_ctx, 3, 700)
    s.write(0, 0, 500)
    s.kv.advance(0, 500)
    for again in (lambda: s.kv.reset(1), lambda: s.kv.reset(-1), lambda: s.kv.rewind(1, 0), lambda: s.kv.share_prefix(0, 0, [1])):
        s.kv.share_prefix(0, 500, [1])
        s.not_shared(1, 400, [2])
        again()
        assert s.kv.position(1) == 0
        s.write(1, 0, 600)
        s.kv.advance(1, 600)
        s.kv.share_prefix(1, 600, [2])
        s.write(2, 600, 640)
        s.served(2, 640, (1, 600))
        s.kv.reset(-1)
        s.kv.advance(0, 500)
    s.kv.close()


def test_a_slot_taken_back_into_its_prefix(gpu_ctx):
    s = Slots(gpu_ctx, 2, 700)
    s.write(0, 0, 500)
    s.kv.advance(0, 500)
    s.kv.share_prefix(0, 500, [1])
    s.kv.rewind(1, 96)  # (whole blocks: the rows from there on are all its own)
    s.write(1, 96, 300)
    s.kv.advance(1, 204)
    s.served(1, 300, (0, 96))
    s.kv.reset(1)
    s.kv.share_prefix(0, 500, [1])
    s.kv.rewind(1, 100)  # (of this block it has the rows from 100 on only, until it is shared at that length)
    s.write(1, 100, 300)
    s.refused(1, 300, (0, 100))
    s.kv.share_prefix(0, 100, [1])
    s.write(1, 100, 300)
    s.served(1, 300, (0, 100))
    s.kv.close()


def test_a_prefix_of_less_than_a_block_goes_on_from_slot_to_slot(gpu_ctx):
    # (it is copied whole, so every slot has it)
    s = Slots(gpu_ctx, 3, 128)
    s.write(0, 0, 20)
    s.kv.advance(0, 20)
    s.kv.share_prefix(0, 20, [1])
    s.kv.share_prefix(1, 20, [2])
    s.write(2, 20, 41)
    s.served(2, 41, (0, 20))
    s.kv.close()


def test_a_restored_snapshot_is_rows_of_its_own(gpu_ctx):
    s, other = Slots(gpu_ctx, 2, 256), Slots(gpu_ctx, 2, 256)
    other.write(0, 0, 200)
    other.kv.advance(0, 200)
    lengths, payload = other.kv.snapshot_segment_lengths(200), bytearray()
    other.kv.append_snapshot_payload(payload, lengths)
    s.write(1, 0, 100)
    s.kv.advance(1, 100)
    s.kv.share_prefix(1, 100, [0])
    s.not_shared(0, 64, [1])
    s.kv.restore_snapshot(200, lengths, bytes(payload))
    s.rows[0] = other.rows[0]
    s.kv.share_prefix(0, 200, [1])
    s.write(1, 200, 230)
    s.served(1, 230, (0, 200))
    s.kv.close()
    other.kv.close()
