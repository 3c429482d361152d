// Products of a few tokens with 4-bit weights of one scale and zero point per
// group (layout in group4.hpp), and the packing, quantizing and decoding of
// such weights:
//
//   W[n, k] = (q[n, k] - z[n, g]) * s[n, g],   g = k / group,  z = 8 without zeros
//   y[t, n] = sum_k W[n, k] x[t, k]
//
// One wave per row.
#include "elem_types.hpp"
#include "group4.hpp"
#include "../../include/vbhip.h"

namespace vb {
namespace {

struct G4Weights {
    const uint8_t* w;
    Group4Layout l;
    int64_t rows, k;
    bool has_zeros;
};

__device__ __forceinline__ int64_t block_of(const G4Weights& g, int64_t row, int64_t k) {
    return (row >> 4) * g.l.steps + (k >> 7);
}

__device__ __forceinline__ float g4_value(const G4Weights& g, int64_t row, int64_t k) {
    const int64_t b = block_of(g, row, k);
    const int r = static_cast<int>(row & 15), kk = static_cast<int>(k & 127), j = kk & 7;
    const uint32_t word = reinterpret_cast<const uint32_t*>(g.w)[b * 256 + (((kk >> 3) & 3) * 16 + r) * 4 + (kk >> 5)];
    const int q = (word >> ((j >> 1) * 4 + (j & 1) * 16)) & 15;
    const int64_t gi = b * g.l.per + (kk * g.l.per >> 7);
    const float s = static_cast<float>(reinterpret_cast<const _Float16*>(g.w + g.l.scales)[gi * 16 + r]);
    const int z = g.has_zeros ? (g.w[g.l.zeros + gi * 8 + (r >> 1)] >> ((r & 1) * 4)) & 15 : 8;
    return static_cast<float>(q - z) * s;
}

// Work items of 256-thread workgroups, as many per thread as it takes: a
// launch has fewer than 2^32 threads.
__device__ __forceinline__ int64_t first_item() { return static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; }
__device__ __forceinline__ int64_t item_stride() { return static_cast<int64_t>(gridDim.x) * 256; }
uint32_t item_blocks(int64_t n) { return static_cast<uint32_t>(n > (1 << 28) ? 1 << 20 : (n + 255) / 256); }

// One thread per dword of codes, then per group of 16 scales (and zeros).
__global__ void __launch_bounds__(256) g4_pack_codes_kernel(const uint8_t* packed, uint32_t* out, Group4Layout l,
                                                            int64_t rows, int64_t k) {
    for (int64_t i = first_item(); i < l.tiles * l.steps * 256; i += item_stride()) {
        const int64_t b = i >> 8;
        const int lane = static_cast<int>(i >> 2) & 63, t = static_cast<int>(i) & 3;
        const int64_t row = b / l.steps * 16 + (lane & 15), k0 = b % l.steps * 128 + t * 32 + (lane >> 4) * 8;
        uint32_t word = 0;
        if (row < rows)
            for (int j = 0; j < 8 && k0 + j < k; j++) {
                const uint32_t byte = packed[row * ((k + 1) >> 1) + ((k0 + j) >> 1)];
                word |= ((j & 1 ? byte >> 4 : byte) & 15u) << ((j >> 1) * 4 + (j & 1) * 16);
            }
        out[i] = word;
    }
}

__global__ void __launch_bounds__(256) g4_pack_groups_kernel(const _Float16* scales, const uint8_t* zeros, uint8_t* out,
                                                             Group4Layout l, int64_t rows, int64_t k, int32_t group,
                                                             int64_t groups) {
    for (int64_t i = first_item(); i < l.tiles * l.steps * l.per; i += item_stride()) {
        const int64_t b = i / l.per, tile = b / l.steps;
        const int64_t gi = (b % l.steps * 128 + i % l.per * (128 / l.per)) / group;
        uint64_t zs = 0;
        for (int r = 0; r < 16; r++) {
            const int64_t row = tile * 16 + r;
            const bool in = row < rows && gi < groups;
            reinterpret_cast<_Float16*>(out + l.scales)[i * 16 + r] =
                in ? scales[row * groups + gi] : static_cast<_Float16>(0.f);
            if (zeros && in) zs |= static_cast<uint64_t>(zeros[row * groups + gi] & 15) << (4 * r);
        }
        if (zeros) reinterpret_cast<uint64_t*>(out + l.zeros)[i] = zs;
    }
}

__global__ void __launch_bounds__(256) g4_dequant_kernel(G4Weights g, float* out) {
    for (int64_t i = first_item(); i < g.rows * g.k; i += item_stride()) out[i] = g4_value(g, i / g.k, i % g.k);
}

// One thread per group of a row.  Symmetric: s = absmax / 7, codes 1..15
// around 8.  With zeros: the range is stretched to hold 0, s = (hi - lo) / 15,
// z = round(-lo / s).  s is rounded to fp16 first and the codes go by that.
__global__ void __launch_bounds__(256) g4_quantize_kernel(const void* src, int32_t type, int64_t ld, int64_t rows,
                                                          int64_t k, int32_t group, int64_t groups, uint8_t* codes,
                                                          _Float16* scales, uint8_t* zeros) {
    for (int64_t i = first_item(); i < rows * groups; i += item_stride()) {
        const int64_t row = i / groups, k0 = i % groups * group, end = k0 + group < k ? k0 + group : k;
        float lo = 0.f, hi = 0.f;
        for (int64_t j = k0; j < end; j++) {
            const float v = elem_ld(src, row * ld + j, type);
            lo = fminf(lo, v);
            hi = fmaxf(hi, v);
        }
        const float want = zeros ? (hi - lo) / 15.f : fmaxf(hi, -lo) / 7.f;
        const _Float16 sh = static_cast<_Float16>(fminf(want, 65504.f));
        const float s = static_cast<float>(sh);
        const float z = !zeros ? 8.f : s > 0.f ? fminf(fmaxf(rintf(-lo / s), 0.f), 15.f) : 0.f;
        scales[i] = sh;
        if (zeros) zeros[i] = static_cast<uint8_t>(z);
        for (int64_t j = k0; j < end; j += 2) {
            uint32_t byte = 0;
            for (int h = 0; h < 2 && j + h < end; h++) {
                const float v = elem_ld(src, row * ld + j + h, type);
                const float q = s > 0.f ? fminf(fmaxf(rintf(v / s) + z, 0.f), 15.f) : z;
                byte |= static_cast<uint32_t>(q) << (4 * h);
            }
            codes[row * ((k + 1) >> 1) + (j >> 1)] = static_cast<uint8_t>(byte);
        }
    }
}

__global__ void __launch_bounds__(256) g4_gemv_kernel(G4Weights g, const void* x, int32_t type, int64_t ld, int m,
                                                      float* y) {
    for (int64_t row = first_item() >> 6; row < g.rows; row += item_stride() >> 6)
        for (int t = 0; t < m; t++) {
            float s = 0.f;
            for (int64_t i = threadIdx.x & 63; i < g.k; i += 64) s += g4_value(g, row, i) * elem_ld(x, t * ld + i, type);
            s = wave_sum_dpp(s);
            if ((threadIdx.x & 63) == 0) y[t * g.rows + row] = s;
        }
}

// The layout of a call's weights, or an error.
int layout_of(const char* what, int64_t rows, int64_t k, int32_t group, int32_t has_zeros, Group4Layout* l) {
    if (!group4_layout(rows, k, group, has_zeros != 0, l)) {
        set_error("%s: no layout for %lld x %lld in groups of %d (32, 64 or a multiple of 128)", what,
                  static_cast<long long>(rows), static_cast<long long>(k), group);
        return E_INVAL;
    }
    return OK;
}

}  // namespace
}  // namespace vb

using namespace vb;

extern "C" {

int64_t vb_group4_bytes(int64_t rows, int64_t k, int32_t group, int32_t has_zeros) {
    Group4Layout l;
    return group4_layout(rows, k, group, has_zeros != 0, &l) ? l.total : -1;
}

int vb_group4_pack(const uint8_t* packed, const void* scales, const uint8_t* zeros, void* w, int64_t rows, int64_t k,
                   int32_t group, void* stream) {
    Group4Layout l;
    if (const int rc = layout_of("vb_group4_pack", rows, k, group, zeros != nullptr, &l); rc != OK) return rc;
    if (!packed || !scales || !w || reinterpret_cast<uintptr_t>(w) % 16 != 0) {
        set_error("vb_group4_pack: null pointer, or w not 16-byte aligned");
        return E_INVAL;
    }
    hipStream_t st = as_stream(stream);
    g4_pack_codes_kernel<<<item_blocks(l.tiles * l.steps * 256), 256, 0, st>>>(packed, static_cast<uint32_t*>(w), l,
                                                                                  rows, k);
    if (const int rc = check_launch("vb_group4_pack"); rc != OK) return rc;
    g4_pack_groups_kernel<<<item_blocks(l.tiles * l.steps * l.per), 256, 0, st>>>(
        static_cast<const _Float16*>(scales), zeros, static_cast<uint8_t*>(w), l, rows, k, group, (k + group - 1) / group);
    return check_launch("vb_group4_pack");
}

int vb_group4_quantize(const void* src, int32_t type, int64_t ld, int64_t rows, int64_t k, int32_t group,
                       uint8_t* packed, void* scales, uint8_t* zeros, void* stream) {
    Group4Layout l;
    if (const int rc = layout_of("vb_group4_quantize", rows, k, group, zeros != nullptr, &l); rc != OK) return rc;
    if (!elem_type(type) || !src || !packed || !scales || (rows > 1 && ld < 0)) {
        set_error("vb_group4_quantize: null pointer, element type %d or row stride %lld", type,
                  static_cast<long long>(ld));
        return E_INVAL;
    }
    const int64_t groups = (k + group - 1) / group;
    g4_quantize_kernel<<<item_blocks(rows * groups), 256, 0, as_stream(stream)>>>(
        src, type, ld, rows, k, group, groups, packed, static_cast<_Float16*>(scales), zeros);
    return check_launch("vb_group4_quantize");
}

int vb_group4_dequant_rows(const void* w, float* out, int64_t rows, int64_t k, int32_t group, int32_t has_zeros,
                           void* stream) {
    G4Weights g{static_cast<const uint8_t*>(w), {}, rows, k, has_zeros != 0};
    if (const int rc = layout_of("vb_group4_dequant_rows", rows, k, group, has_zeros, &g.l); rc != OK) return rc;
    if (!w || !out || reinterpret_cast<uintptr_t>(w) % 16 != 0) {
        set_error("vb_group4_dequant_rows: null pointer, or w not 16-byte aligned");
        return E_INVAL;
    }
    g4_dequant_kernel<<<item_blocks(rows * k), 256, 0, as_stream(stream)>>>(g, out);
    return check_launch("vb_group4_dequant_rows");
}

int vb_group4_gemv(const void* w, int64_t rows, int64_t k, int32_t group, int32_t has_zeros, const void* x,
                   int32_t x_type, int64_t x_ld, int64_t m, float* y, void* stream) {
    G4Weights g{static_cast<const uint8_t*>(w), {}, rows, k, has_zeros != 0};
    if (const int rc = layout_of("vb_group4_gemv", rows, k, group, has_zeros, &g.l); rc != OK) return rc;
    if (!elem_type(x_type) || m < 0 || m > 0x7fffffff || (m > 1 && x_ld < 0)) {
        set_error("vb_group4_gemv: bad arguments (x type %d, m=%lld, row stride %lld)", x_type,
                  static_cast<long long>(m), static_cast<long long>(x_ld));
        return E_INVAL;
    }
    if (m == 0) return OK;
    if (!w || !x || !y || reinterpret_cast<uintptr_t>(w) % 16 != 0) {
        set_error("vb_group4_gemv: null pointer, or w not 16-byte aligned");
        return E_INVAL;
    }
    g4_gemv_kernel<<<item_blocks(rows * 64), 256, 0, as_stream(stream)>>>(g, x, x_type, x_ld, static_cast<int>(m), y);
    return check_launch("vb_group4_gemv");
}

}  // extern "C"
