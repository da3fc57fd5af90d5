"""Calls of sequences that share a prefix, by the way that the planner sends them on a device of 256 CUs: ``test_shared_plan`` holds the ways,
``test_gpu_attn_shared_ways`` the values that come out of each."""

ONE_PASS, TILES, PACKED_ROWS, RANGES = range(4)  # tt::SharedWay

# q heads, kv heads, dim, bits, prefix, sequences, rows of each, way
CASES = [
    (16, 2, 256, 16, 500, 5, 1, ONE_PASS), (32, 8, 128, 8, 700, 3, 4, ONE_PASS), (16, 4, 64, 4, 900, 8, 2, ONE_PASS),
    (16, 2, 256, 16, 2047, 20, 1, TILES), (32, 8, 128, 16, 6007, 9, 4, TILES), (16, 4, 64, 16, 8191, 9, 1, TILES), (32, 8, 128, 8, 4100, 9, 1, TILES),
    (32, 8, 128, 4, 20011, 3, 2, TILES), (8, 2, 256, 4, 16384, 9, 1, TILES),
    (24, 2, 256, 16, 8200, 32, 1, PACKED_ROWS), (16, 2, 256, 8, 8192, 32, 4, PACKED_ROWS), (32, 4, 128, 4, 8193, 16, 8, PACKED_ROWS),
    (16, 4, 64, 16, 8200, 64, 4, PACKED_ROWS),
    # over fp16 pages, over staged ones; groups of 4, 8, 12 and 16; tiles whose last rows are few; a prefix that ends on a block and not;
    # rows one by one, some without keys of their own
    (16, 2, 256, 16, 4096, 64, 16, RANGES), (16, 2, 256, 16, 4111, 5, 200, RANGES), (8, 2, 256, 16, 8223, 32, 32, RANGES),
    (24, 2, 256, 16, 2080, 5, 200, RANGES), (24, 2, 256, 16, 4100, 3, 100, RANGES), (32, 8, 128, 16, 4096, 64, 4, RANGES),
    (128, 8, 128, 16, 4096, 64, 1, RANGES), (32, 4, 128, 16, 4096, 32, 32, RANGES),
    (16, 2, 256, 8, 4096, 16, 32, RANGES), (16, 2, 256, 8, 20011, 64, 4, RANGES), (8, 2, 256, 8, 16384, 32, 16, RANGES),
    (24, 2, 256, 8, 1055, 8, 100, RANGES), (24, 2, 256, 8, 2064, 2, 200, RANGES), (32, 8, 128, 8, 4096, 64, 16, RANGES),
    (16, 2, 256, 4, 4096, 40, 8, RANGES), (24, 2, 256, 4, 32768, 64, 2, RANGES), (16, 2, 256, 4, 2049, 5, 199, RANGES),
    (64, 4, 256, 4, 8192, 48, 2, RANGES),
]


def starts(prefix, sequences):
    """Positions of the sequences' first rows: one that sees the prefix alone, one behind it, others at unlike distances."""
    return [prefix - 1 + (i * i * 37) % 301 + (900 if i == 4 else 0) for i in range(sequences)]
