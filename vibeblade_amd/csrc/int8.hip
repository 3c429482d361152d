// Products in 8-bit integers with a scale per token and one per output channel
// (layout of both operands in int8.hpp), and the quantizing, packing and
// decoding of such matrices:
//
//   s[r] = max(max_k |x[r, k]| / 127, 2^-126)  (fp32; 0 values: 0)
//   q[r, k] = x[r, k] / s[r], to the nearest integer, ties to even
//   y[t, n] = s_x[t] s_w[n] sum_k q_x[t, k] q_w[n, k]  (+ bias[n])
//
// Sums of products are exact 32-bit integers, so no order of them shows in a
// result.  A row that holds a NaN or an infinity has the scale NaN and codes 0.
#include <type_traits>

#include "elem_types.hpp"
#include "int8.hpp"
#include "vb_internal.hpp"
#include "../../include/vbhip.h"

namespace vb {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));

constexpr int I8_PACKED = 3;  // x_type of an operand that is packed already

__device__ __forceinline__ i32x4 mfma_i8(i32x4 a, i32x4 b, i32x4 c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
}

// ---- quantizing, packing, decoding ---------------------------------------------

// The scale of a row whose largest magnitude is `big`.
__device__ __forceinline__ float scale_of(float big) {
    return big > 0.f ? fmaxf(big / 127.f, 0x1p-126f) : 0.f;
}

// v / s to the nearest integer, ties to even: the quotient of fp32's division may
// have been rounded onto a tie, which the remainder tells.
__device__ __forceinline__ int code_of(float v, float s, float inv) {
    float q = rintf(v * inv);
    // v - q s is exact in the fma; a code that is not the nearest is off by one
    const float r = __builtin_fmaf(-q, s, v), half = 0.5f * s;
    if (r > half || (r == half && (static_cast<int>(q) & 1))) q += 1.f;
    else if (r < -half || (r == -half && (static_cast<int>(q) & 1))) q -= 1.f;
    return static_cast<int>(q);
}

// Byte k of row r in the codes.
__device__ __forceinline__ int64_t code_at(int64_t blocks, int64_t r, int64_t k) {
    return ((r >> 4) * blocks + (k >> 6)) * INT8_BLOCK + (((k >> 4) & 3) * 16 + (r & 15)) * 16 + (k & 15);
}

struct I8Rows {
    const void* src;
    uint8_t* w;
    Int8Layout l;
    int64_t ld, rows, k;
};

// One workgroup a row (rows to the end of the last tile: zeros).
template <int TYPE>
__global__ void __launch_bounds__(256) i8_quantize_kernel(I8Rows a) {
    __shared__ float bigs[4];
    const int wave = static_cast<int>(threadIdx.x) >> 6;
    for (int64_t row = blockIdx.x; row < a.l.tiles * INT8_ROWS; row += gridDim.x) {
        float big = 0.f;
        bool bad = false;
        if (row < a.rows)
            for (int64_t i = threadIdx.x; i < a.k; i += 256) {
                const float v = fabsf(elem_ld(a.src, row * a.ld + i, TYPE));
                bad = bad || !(v < INFINITY);
                big = fmaxf(big, v);
            }
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) big = fmaxf(big, __shfl_xor(big, o, 64));
        if ((threadIdx.x & 63) == 0) bigs[wave] = big;
        bad = __syncthreads_or(bad);
        big = fmaxf(fmaxf(bigs[0], bigs[1]), fmaxf(bigs[2], bigs[3]));
        const float s = bad ? 0.f : scale_of(big), inv = s > 0.f ? 1.f / s : 0.f;
        for (int64_t i = threadIdx.x; i < a.l.blocks * INT8_K; i += 256) {
            const float v = s > 0.f && i < a.k ? elem_ld(a.src, row * a.ld + i, TYPE) : 0.f;
            a.w[code_at(a.l.blocks, row, i)] = static_cast<uint8_t>(code_of(v, s, inv));
        }
        if (threadIdx.x == 0) reinterpret_cast<float*>(a.w + a.l.scales)[row] = bad ? NAN : s;
        __syncthreads();
    }
}

uint32_t i8_grid(int64_t n) { return static_cast<uint32_t>(n < (1 << 20) ? n : 1 << 20); }

// One thread per 16 codes, then a scale a row.
__global__ void __launch_bounds__(256) i8_pack_kernel(const int8_t* q, int64_t ld, const float* scales, uint8_t* w, Int8Layout l,
                                                      int64_t rows, int64_t k) {
    const int64_t pieces = l.tiles * l.blocks * 64, stride = static_cast<int64_t>(gridDim.x) * 256;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < pieces; i += stride) {
        const int64_t block = i >> 6, row = block / l.blocks * 16 + (i & 15), k0 = block % l.blocks * 64 + ((i >> 4) & 3) * 16;
        uint32_t word[4] = {0, 0, 0, 0};
        if (row < rows)
            for (int j = 0; j < 16 && k0 + j < k; j++)
                word[j >> 2] |= static_cast<uint32_t>(static_cast<uint8_t>(q[row * ld + k0 + j])) << 8 * (j & 3);
        reinterpret_cast<uint4*>(w)[i] = make_uint4(word[0], word[1], word[2], word[3]);
    }
    for (int64_t r = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; r < l.tiles * INT8_ROWS; r += stride)
        reinterpret_cast<float*>(w + l.scales)[r] = r < rows ? scales[r] : 0.f;
}

__global__ void __launch_bounds__(256) i8_dequant_kernel(const uint8_t* w, Int8Layout l, int64_t rows, int64_t k, float* out) {
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < rows * k;
         i += static_cast<int64_t>(gridDim.x) * 256) {
        const int64_t row = i / k;
        const float q = static_cast<float>(static_cast<int8_t>(w[code_at(l.blocks, row, i % k)]));
        out[i] = q * reinterpret_cast<const float*>(w + l.scales)[row];
    }
}

// ---- products ---------------------------------------------------------------

struct I8Args {
    const uint8_t* w;
    const uint8_t* x;  // packed
    const float* bias;
    void* y;
    Int8Layout wl, xl;
    int64_t n, m;
    int32_t out_type;
};

__device__ __forceinline__ void i8_store(const I8Args& a, int64_t t, int64_t n, int sum) {
    const float sx = reinterpret_cast<const float*>(a.x + a.xl.scales)[t], sw = reinterpret_cast<const float*>(a.w + a.wl.scales)[n];
    float v = static_cast<float>(sum) * sx * sw;
    if (a.bias) v += a.bias[n];
    elem_st(a.y, t * a.n + n, a.out_type, v);
}

// 16 rows of the weights by 16 tokens a workgroup, k over its four waves.
__global__ void __launch_bounds__(256) i8_gemm_kernel(I8Args a) {
    __shared__ i32x4 part[4][64];
    const int lane = static_cast<int>(threadIdx.x) & 63, wave = static_cast<int>(threadIdx.x) >> 6;
    for (int64_t item = blockIdx.x; item < a.wl.tiles * a.xl.tiles; item += gridDim.x) {
        const int64_t tile = item % a.wl.tiles, cols = item / a.wl.tiles;
        const i32x4* pw = reinterpret_cast<const i32x4*>(a.w) + tile * a.wl.blocks * 64 + lane;
        const i32x4* px = reinterpret_cast<const i32x4*>(a.x) + cols * a.wl.blocks * 64 + lane;
        i32x4 acc = {0, 0, 0, 0};
        for (int64_t b = wave; b < a.wl.blocks; b += 4) acc = mfma_i8(pw[b * 64], px[b * 64], acc);
        part[wave][lane] = acc;
        __syncthreads();
        if (wave == 0) {
            const i32x4 sum = (part[0][lane] + part[1][lane]) + (part[2][lane] + part[3][lane]);
            const int64_t t = cols * 16 + (lane & 15);
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int64_t n = tile * 16 + 4 * (lane >> 4) + r;
                if (t < a.m && n < a.n) i8_store(a, t, n, sum[r]);
            }
        }
        __syncthreads();
    }
}

int i8_quantize(const I8Rows& a, int32_t type, hipStream_t st) {
    const uint32_t grid = i8_grid(a.l.tiles * INT8_ROWS);
    if (type == ELEM_F32) i8_quantize_kernel<ELEM_F32><<<grid, 256, 0, st>>>(a);
    else if (type == ELEM_F16) i8_quantize_kernel<ELEM_F16><<<grid, 256, 0, st>>>(a);
    else i8_quantize_kernel<ELEM_BF16><<<grid, 256, 0, st>>>(a);
    return check_launch("vb_int8_quantize");
}

int i8_layout_of(const char* what, int64_t rows, int64_t k, Int8Layout* l) {
    if (!int8_layout(rows, k, l)) {
        set_error("%s: no layout for %lld x %lld (k at most %lld)", what, static_cast<long long>(rows),
                  static_cast<long long>(k), static_cast<long long>(INT8_MAX_K));
        return E_INVAL;
    }
    return OK;
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

}  // namespace
}  // namespace vb

using namespace vb;

extern "C" {

int64_t vb_int8_bytes(int64_t rows, int64_t k) {
    Int8Layout l;
    return int8_layout(rows, k, &l) ? l.total : -1;
}

int vb_int8_pack(const int8_t* codes, int64_t ld, const float* scales, void* w, int64_t rows, int64_t k, void* stream) {
    Int8Layout l;
    if (const int rc = i8_layout_of("vb_int8_pack", rows, k, &l); rc != OK) return rc;
    if (!codes || !scales || !w || !aligned16(w) || (rows > 1 && ld < 0)) {
        set_error("vb_int8_pack: null pointer, w not 16-byte aligned, or row stride %lld", static_cast<long long>(ld));
        return E_INVAL;
    }
    const int64_t groups = (l.tiles * l.blocks * 64 + 255) / 256;
    i8_pack_kernel<<<i8_grid(groups), 256, 0, as_stream(stream)>>>(codes, ld, scales, static_cast<uint8_t*>(w), l, rows, k);
    return check_launch("vb_int8_pack");
}

int vb_int8_quantize(const void* src, int32_t type, int64_t ld, int64_t rows, int64_t k, void* w, void* stream) {
    Int8Layout l;
    if (const int rc = i8_layout_of("vb_int8_quantize", rows, k, &l); rc != OK) return rc;
    if (!elem_type(type) || !src || !w || !aligned16(w) || (rows > 1 && ld < 0)) {
        set_error("vb_int8_quantize: null pointer, w not 16-byte aligned, element type %d or row stride %lld", type,
                  static_cast<long long>(ld));
        return E_INVAL;
    }
    return i8_quantize(I8Rows{src, static_cast<uint8_t*>(w), l, ld, rows, k}, type, as_stream(stream));
}

int vb_int8_dequant_rows(const void* w, float* out, int64_t rows, int64_t k, void* stream) {
    Int8Layout l;
    if (const int rc = i8_layout_of("vb_int8_dequant_rows", rows, k, &l); rc != OK) return rc;
    if (!w || !out || !aligned16(w)) {
        set_error("vb_int8_dequant_rows: null pointer, or w not 16-byte aligned");
        return E_INVAL;
    }
    i8_dequant_kernel<<<i8_grid((rows * k + 255) / 256), 256, 0, as_stream(stream)>>>(static_cast<const uint8_t*>(w), l, rows, k, out);
    return check_launch("vb_int8_dequant_rows");
}

int64_t vb_int8_workspace(int64_t m, int64_t rows, int64_t k, int32_t x_type) {
    Int8Layout wl, xl;
    if (m < 0 || m > 0x7fffffff - 255 || (x_type != I8_PACKED && !elem_type(x_type)) || !int8_layout(rows, k, &wl)) return -1;
    if (m == 0 || x_type == I8_PACKED) return 0;
    return int8_layout(m, k, &xl) ? xl.total : -1;
}

int vb_int8_gemm(const void* w, int64_t rows, int64_t k, const void* x, int32_t x_type, int64_t x_ld, int64_t m,
                 const float* bias, void* y, int32_t y_type, void* workspace, size_t workspace_bytes, void* stream) {
    Int8Layout l;
    if (const int rc = i8_layout_of("vb_int8_gemm", rows, k, &l); rc != OK) return rc;
    const int64_t need = vb_int8_workspace(m, rows, k, x_type);
    if (need < 0 || !elem_type(y_type) || (m > 1 && x_type != I8_PACKED && x_ld < 0)) {
        set_error("vb_int8_gemm: bad arguments (x type %d, y type %d, m=%lld, row stride %lld)", x_type, y_type,
                  static_cast<long long>(m), static_cast<long long>(x_ld));
        return E_INVAL;
    }
    if (m == 0) return OK;
    if (!w || !x || !y || !aligned16(w) || (x_type == I8_PACKED && !aligned16(x))) {
        set_error("vb_int8_gemm: null pointer, or packed operands not 16-byte aligned");
        return E_INVAL;
    }
    if (static_cast<int64_t>(workspace_bytes) < need || (need > 0 && (!workspace || !aligned16(workspace)))) {
        set_error("vb_int8_gemm: workspace of %zu bytes (16-byte aligned) is below the %lld needed", workspace_bytes,
                  static_cast<long long>(need));
        return E_INVAL;
    }
    I8Args a{};
    a.w = static_cast<const uint8_t*>(w);
    a.wl = l;
    int8_layout(m, k, &a.xl);
    a.x = static_cast<const uint8_t*>(x);
    if (x_type != I8_PACKED) {
        a.x = static_cast<const uint8_t*>(workspace);
        if (const int rc = i8_quantize(I8Rows{x, static_cast<uint8_t*>(workspace), a.xl, x_ld, m, k}, x_type, as_stream(stream));
            rc != OK)
            return rc;
    }
    a.bias = bias;
    a.y = y;
    a.n = rows;
    a.m = m;
    a.out_type = y_type;
    i8_gemm_kernel<<<i8_grid(a.wl.tiles * a.xl.tiles), 256, 0, as_stream(stream)>>>(a);
    return check_launch("vb_int8_gemm");
}

}  // extern "C"
