// 4-bit weights with one scale (and zero point) per group of a row, as they
// lie in HBM.
//
// Rows are taken 16 at a time and k 128 at a time: a block of 16 x 128 codes
// is 1 KB, in the order in which the lanes of a wave feed them to the matrix
// cores.  Lane l holds row l % 16 and, in its dword t (t = 0..3, one per 32 of
// k), the codes of k = 32 t + 8 (l / 16) + 0..7, code i at bit 4 i, with its
// top bit flipped (q - 8 in two's complement).  A wave reads a block with one
// 16-byte load per lane, and block after block along k as one linear stream.
//
// Planes, each [row tile][128-step][...]:
//   codes   1024 bytes
//   scales  4 x G x 4 fp16 (G = 4, 2, 1 groups per 128 for groups of 32, 64
//           and 128 or more; a longer group repeats its scale): the scales
//           that lane l multiplies its four outputs (rows 4 (l / 16) + 0..3)
//           by lie together
//   zeros   in the order of the scales, 4 bits each, as the codes (z - 8); no
//           plane for symmetric weights (zero point 8)
// Rows and k past the tensor have scale 0 and the code of 0.
#pragma once

#include <cstdint>

namespace vb {

struct Group4Layout {
    int64_t tiles, steps, per;  // row tiles, 128-steps, groups per step
    int64_t scales, zeros, total;  // byte offsets of the planes (codes at 0), bytes in all
};

// false for shapes and groups that there is no layout for
inline bool group4_layout(int64_t rows, int64_t k, int32_t group, bool has_zeros, Group4Layout* out) {
    if (rows <= 0 || k <= 0 || rows > 0x7fffffff || k > 1 << 28 || group <= 0) return false;  // a row tile below 4 GB
    if (group != 32 && group != 64 && group % 128 != 0) return false;
    out->tiles = (rows + 15) / 16;
    out->steps = (k + 127) / 128;
    out->per = group >= 128 ? 1 : 128 / group;
    const int64_t blocks = out->tiles * out->steps;
    out->scales = blocks * 1024;
    out->zeros = out->scales + blocks * out->per * 32;
    out->total = out->zeros + (has_zeros ? blocks * out->per * 8 : 0);
    return true;
}

}  // namespace vb
