// Workgroups of the few tokens' 8-bit products.  Host arithmetic without a device, so that it can be run over any shape anywhere.
#pragma once

namespace tt {

// Channels of a workgroup, in tiles of 16: the fewest of one, two and four with which every CU has one workgroup at most, since a second round
// of them waits for the first.  us by one tile / two / four, weights out of memory, 256 CUs:
//   2,048 columns, one token: 4,096 channels 5.1 / 4.7 / 6.4, 4,352 5.9 / 4.8 / 6.5, 8,192 6.6 / 5.7 / 6.9, 8,224 8.3 / 8.4 / 6.9, 9,152 8.9 / 8.9 / 7.0, 16,384 11.8 /
//   10.2 / 8.5; 32 tokens that are quantised already: 4,096 5.1 / 5.8 / 8.1, 4,352 8.4 / 5.9 / 8.3, 8,192 9.0 / 6.9 / 9.1, 8,224 11.9 / 10.3 / 8.9, 16,384 16.9 / 11.9 / 10.7
//   4,096 columns, one token: 4,096 6.4 / 7.3 / 9.3, 4,352 8.1 / 7.3 / 9.3, 8,192 9.6 / 9.5 / 10.8, 8,224 11.2 / 13.5 / 10.6; 32 tokens: 4,096 7.6 / 8.5 / 11.8, 4,352 11.9 /
//   8.5 / 12.0, 8,192 13.7 / 10.3 / 13.4, 8,224 17.2 / 15.3 / 13.3
inline int int8_ring_tiles(int n_cus, int rows) {
    for (int tiles = 1; tiles < 4; tiles *= 2)
        if (((long long)rows + 16 * tiles - 1) / (16 * tiles) <= n_cus) return tiles;
    return 4;
}

}  // namespace tt
