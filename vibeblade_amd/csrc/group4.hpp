// 4-bit weights with one scale (and zero point) per group of a row, as they
// lie in HBM.
//
// Rows are taken 16 at a time and k 256 at a time: such a block is one run of
// memory, codes, scales and zero points together, and the blocks of a row tile
// follow each other along k, so that a wave reads one linear stream.  (As three
// planes the small pieces cost more than their bytes: 14336 x 4096 with groups
// of 128 took 11.3 us to read, its codes alone 8.9.)  A block holds
//
//   codes   2 steps of 128 k, 1 KB each, in the order in which the lanes of a
//           wave feed them to the matrix cores.  Lane l holds row l % 16 and,
//           in its dword t (t = 0..3, one per 32 of k), the codes of k = 32 t
//           + 8 (l / 16) + 0..7, code i at bit 4 i, with its top bit flipped
//           (q - 8 in two's complement).
//   scales  4 x 2 G x 4 fp16, G = 4, 2, 1 groups per 128 for groups of 32, 64
//           and 128 or more (a longer group repeats its scale): [c][step and
//           group][row 4 c + 0..3], the scales that the lanes of c = l / 16
//           multiply their four outputs by
//   zeros   in the order of the scales, 4 bits each, as the codes (z - 8);
//           none for symmetric weights (zero point 8)
//
// Rows and k past the tensor have scale 0 and the code of 0.
#pragma once

#include <cstdint>

namespace vb {

constexpr int GROUP4_K = 256;  // of a block

struct Group4Layout {
    int64_t tiles, blocks;  // row tiles, blocks per tile
    int32_t per;            // groups per 128 of k
    int32_t scales, zeros;  // byte offsets in a block (codes at 0)
    int32_t bytes;          // of a block
    int64_t total;
};

// false for shapes and groups that there is no layout for
inline bool group4_layout(int64_t rows, int64_t k, int32_t group, bool has_zeros, Group4Layout* out) {
    if (rows <= 0 || k <= 0 || rows > 0x7fffffff || k > 1 << 28 || group <= 0) return false;  // a row tile below 4 GB
    if (group != 32 && group != 64 && group % 128 != 0) return false;
    out->tiles = (rows + 15) / 16;
    out->blocks = (k + GROUP4_K - 1) / GROUP4_K;
    out->per = group >= 128 ? 1 : 128 / group;
    out->scales = 16 * GROUP4_K / 2;
    out->zeros = out->scales + 64 * out->per;
    out->bytes = out->zeros + (has_zeros ? 16 * out->per : 0);  // a multiple of 16
    out->total = out->tiles * out->blocks * out->bytes;
    return true;
}

}  // namespace vb
