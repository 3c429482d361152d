// Matrices of 8-bit integers with one scale per row, as they lie in HBM: the
// weights (a scale per output channel) and the activations (one per token) of
// an integer product, alike.
//
// Rows are taken 16 at a time and k 64 at a time: such a block is 1 KB of
// memory, in the order in which the lanes of a wave feed it to
// v_mfma_i32_16x16x64_i8.  Lane l holds row l % 16 and k = 16 (l / 16) + 0..15,
// so one 16-byte load per lane is an operand, and a wave reads whole KB.  The
// blocks of a row tile follow each other along k; then come the tiles, then the
// scales (fp32, a row each).  Rows and k past the matrix are 0.
#pragma once

#include <cstdint>

namespace vb {

constexpr int INT8_ROWS = 16;      // of a block
constexpr int INT8_K = 64;
constexpr int INT8_BLOCK = INT8_ROWS * INT8_K;
// sums of products of two codes (-128..127) stay within 32 bits
constexpr int64_t INT8_MAX_K = 131071;

struct Int8Layout {
    int64_t tiles, blocks;  // row tiles, blocks of a tile
    int64_t scales, total;  // byte offset of the scales, bytes
};

// rows that a workgroup of 512 threads a tile can be launched for
constexpr int64_t INT8_MAX_ROWS = 1 << 26;

// false for shapes that there is no layout for
inline bool int8_layout(int64_t rows, int64_t k, Int8Layout* out) {
    if (rows <= 0 || k <= 0 || rows > INT8_MAX_ROWS || k > INT8_MAX_K) return false;
    out->tiles = (rows + INT8_ROWS - 1) / INT8_ROWS;
    out->blocks = (k + INT8_K - 1) / INT8_K;
    out->scales = out->tiles * out->blocks * INT8_BLOCK;
    out->total = out->scales + out->tiles * INT8_ROWS * 4;
    return true;
}

}  // namespace vb
