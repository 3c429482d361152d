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
//
// Few tokens are memory's: 128256 x 4096, one token 82 us, 6.4 TB/s; 14336 x 4096
// 12.3 and 4.8, of which 1.9 is the launch and 1 to 2 the first loads; 1024 x 4096
// 4.4.  Many are the matrix cores': 4096 tokens of 14336 x 4096 214 us (2.25 POP/s),
// of 4096 x 14336 175 (2.75), 8192 x 8192 x 8192 402 to 435 (2.5 to 2.7; the
// library's product of that size reaches 2.02, of 16384 2.36).  There the clock is
// at 2.0 GHz of 2.4 under the load and the cores are busy for 53 to 64 % of it.
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

// v / s to the nearest integer, ties to even, with inv = 1 / s rounded: the
// remainder v - q s, exact in the fma, tells a q that is not the nearest.
__device__ __forceinline__ int code_of(float v, float s, float inv) {
    const float q = rintf(v * inv), r = __builtin_fmaf(-q, s, v), twice = r + r;
    const int c = static_cast<int>(q);
    // one further where more than half a step is left, or half of one behind an odd code
    const bool off = fabsf(twice) > s || (fabsf(twice) == s && (c & 1));
    return off ? c + (r > 0.f ? 1 : -1) : c;
}

// 16 consecutive values of a row, from k0 on (0 past the row's end), as they lie
// in memory: a thread holds several such pieces.
template <int TYPE>
struct Values {
    static constexpr int WORDS = TYPE == ELEM_F32 ? 16 : 8;
    uint32_t raw[WORDS];
    __device__ __forceinline__ void load(const void* row, int64_t k0, int64_t k) {
        if (k0 + 16 <= k) {  // (rows begin at any element; a load of 16 bytes does not mind)
            typedef uint32_t v4 __attribute__((ext_vector_type(4), aligned(2)));
            const v4* p = reinterpret_cast<const v4*>(static_cast<const uint8_t*>(row) + k0 * (TYPE == ELEM_F32 ? 4 : 2));
#pragma unroll
            for (int i = 0; i < WORDS / 4; i++) {
                const v4 q = p[i];
#pragma unroll
                for (int j = 0; j < 4; j++) raw[4 * i + j] = q[j];
            }
        } else if constexpr (TYPE == ELEM_F32) {
#pragma unroll
            for (int i = 0; i < 16; i++) raw[i] = k0 + i < k ? static_cast<const uint32_t*>(row)[k0 + i] : 0u;
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const uint32_t lo = k0 + 2 * i < k ? static_cast<const uint16_t*>(row)[k0 + 2 * i] : 0u;
                const uint32_t hi = k0 + 2 * i + 1 < k ? static_cast<const uint16_t*>(row)[k0 + 2 * i + 1] : 0u;
                raw[i] = lo | hi << 16;
            }
        }
    }
    __device__ __forceinline__ float value(int i) const {
        if constexpr (TYPE == ELEM_F32) return __uint_as_float(raw[i]);
        else if constexpr (TYPE == ELEM_BF16) return __uint_as_float(i & 1 ? raw[i >> 1] & 0xffff0000u : raw[i >> 1] << 16);
        else return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(raw[i >> 1] >> 16 * (i & 1))));
    }
    // the largest magnitude as bits: infinities and NaN from 0x7f800000 on
    __device__ __forceinline__ uint32_t largest() const {
        uint32_t b = 0;
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const uint32_t m = __float_as_uint(value(i)) & 0x7fffffffu;
            b = m > b ? m : b;
        }
        return b;
    }
    // The low byte of v / s + 3 * 2^22, rounded by one fma, is the code, unless the
    // remainder of one of the sixteen says that its quotient is not the nearest
    // (or a tie): then all by code_of.
    __device__ __forceinline__ uint4 codes(float s, float inv) const {
        if (!(s > 0.f)) return make_uint4(0, 0, 0, 0);
        uint32_t t[16], w[4];
        float most = 0.f;
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const float v = value(i), q = __builtin_fmaf(v, inv, 12582912.f);
            t[i] = __float_as_uint(q);
            most = fmaxf(most, fabsf(__builtin_fmaf(12582912.f - q, s, v)));
        }
        if (!(most + most < s)) {
#pragma unroll
            for (int i = 0; i < 16; i++) t[i] = static_cast<uint32_t>(code_of(value(i), s, inv));
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            // bytes 0 of two values, twice
            const uint32_t lo = __builtin_amdgcn_perm(t[4 * i + 1], t[4 * i], 0x0c0c0400u);
            w[i] = __builtin_amdgcn_perm(t[4 * i + 3], t[4 * i + 2], 0x04000c0cu) | lo;
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
};

__device__ __forceinline__ uint32_t wave_max_bits(uint32_t v) {
    const auto take = [&](uint32_t u) { v = u > v ? u : v; };
    take(__builtin_amdgcn_update_dpp(v, v, 0xB1, 0xF, 0xF, false));   // quad_perm [1,0,3,2]
    take(__builtin_amdgcn_update_dpp(v, v, 0x4E, 0xF, 0xF, false));   // quad_perm [2,3,0,1]
    take(__builtin_amdgcn_update_dpp(v, v, 0x141, 0xF, 0xF, false));  // row_half_mirror
    take(__builtin_amdgcn_update_dpp(v, v, 0x140, 0xF, 0xF, false));  // row_mirror
    take(__builtin_amdgcn_update_dpp(v, v, 0x142, 0xA, 0xF, false));  // row_bcast:15 into rows 1, 3
    take(__builtin_amdgcn_update_dpp(v, v, 0x143, 0xC, 0xF, false));  // row_bcast:31 into rows 2, 3
    return __builtin_amdgcn_readlane(v, 63);
}

// The scale of a row by the bits of its largest magnitude: codes by s (0: all
// 0), and what is stored.
struct RowScale {
    float s, inv, stored;
    __device__ __forceinline__ explicit RowScale(uint32_t bits) {
        const bool bad = bits >= 0x7f800000u;
        s = bad ? 0.f : scale_of(__uint_as_float(bits));
        inv = s > 0.f ? 1.f / s : 0.f;
        stored = bad ? NAN : s;
    }
};

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

// A row by a workgroup, which few rows need; a thread's first HELD pieces of 16
// values are read once, longer rows again for their codes.  Rows to the end of the
// last tile are zeros.
template <int TYPE, int WAVES>
__global__ void __launch_bounds__(64 * WAVES) i8_quantize_rows_kernel(I8Rows a) {
    __shared__ uint32_t bigs[16];
    const int lane = static_cast<int>(threadIdx.x) & 63, wave = static_cast<int>(threadIdx.x) >> 6;
    const int at = static_cast<int>(threadIdx.x);
    constexpr int SPAN = 64 * WAVES, HELD = WAVES == 16 ? 1 : 2;
    const int64_t pieces = a.l.blocks * 4, all = a.l.tiles * INT8_ROWS;
    for (int64_t row = blockIdx.x; row < all; row += gridDim.x) {
        const bool in = row < a.rows;
        const uint8_t* src = static_cast<const uint8_t*>(a.src) + (in ? row * a.ld * (TYPE == ELEM_F32 ? 4 : 2) : 0);
        Values<TYPE> held[HELD];
        uint32_t big = 0;
#pragma unroll
        for (int h = 0; h < HELD; h++) {
            const int64_t p = at + h * SPAN;
            if (in && p < pieces) {
                held[h].load(src, p * 16, a.k);
                const uint32_t b = held[h].largest();
                big = b > big ? b : big;
            }
        }
        for (int64_t p = at + HELD * SPAN; in && p < pieces; p += SPAN) {
            Values<TYPE> v;
            v.load(src, p * 16, a.k);
            const uint32_t b = v.largest();
            big = b > big ? b : big;
        }
        big = wave_max_bits(big);
        if (lane == 0) bigs[wave] = big;
        __syncthreads();
        big = wave_max_bits(lane < WAVES ? bigs[lane] : 0);
        __syncthreads();
        const RowScale s(big);
        uint8_t* to = a.w + code_at(a.l.blocks, row, 0);
#pragma unroll
        for (int h = 0; h < HELD; h++) {
            const int64_t p = at + h * SPAN;
            if (p < pieces) *reinterpret_cast<uint4*>(to + (p >> 2) * INT8_BLOCK + (p & 3) * 256) =
                in ? held[h].codes(s.s, s.inv) : make_uint4(0, 0, 0, 0);
        }
        for (int64_t p = at + HELD * SPAN; p < pieces; p += SPAN) {
            uint4 c = make_uint4(0, 0, 0, 0);
            if (in) {
                Values<TYPE> v;
                v.load(src, p * 16, a.k);
                c = v.codes(s.s, s.inv);
            }
            *reinterpret_cast<uint4*>(to + (p >> 2) * INT8_BLOCK + (p & 3) * 256) = c;
        }
        if (at == 0) reinterpret_cast<float*>(a.w + a.l.scales)[row] = in ? s.stored : 0.f;
    }
}

// A tile of 16 rows by a workgroup: a wave's lanes are the pieces of one block, so
// that it is written as one run (by rows they are 16 bytes every 256: 4096 x 4096
// bf16 17.5 us).
template <int TYPE>
__global__ void __launch_bounds__(1024) i8_quantize_tiles_kernel(I8Rows a) {
    __shared__ uint32_t bigs[16][16];
    constexpr int WAVES = 16, HELD = TYPE == ELEM_F32 ? 3 : 4;  // (four of fp32 spill)
    const int lane = static_cast<int>(threadIdx.x) & 63, wave = static_cast<int>(threadIdx.x) >> 6;
    const int j = lane & 15, k16 = 16 * (lane >> 4);
    for (int64_t tile = blockIdx.x; tile < a.l.tiles; tile += gridDim.x) {
        const int64_t row = tile * INT8_ROWS + j;
        const bool in = row < a.rows;
        const uint8_t* src = static_cast<const uint8_t*>(a.src) + (in ? row * a.ld * (TYPE == ELEM_F32 ? 4 : 2) : 0);
        Values<TYPE> held[HELD];
        uint32_t big = 0;
#pragma unroll
        for (int h = 0; h < HELD; h++) {
            const int64_t b = wave + h * WAVES;
            if (in && b < a.l.blocks) held[h].load(src, b * INT8_K + k16, a.k);
        }
#pragma unroll
        for (int h = 0; h < HELD; h++) {
            if (in && wave + h * WAVES < a.l.blocks) {
                const uint32_t b = held[h].largest();
                big = b > big ? b : big;
            }
        }
        for (int64_t b = wave + HELD * WAVES; in && b < a.l.blocks; b += WAVES) {
            Values<TYPE> v;
            v.load(src, b * INT8_K + k16, a.k);
            const uint32_t most = v.largest();
            big = most > big ? most : big;
        }
#pragma unroll
        for (int o = 16; o <= 32; o <<= 1) {
            const uint32_t u = __shfl_xor(big, o, 64);
            big = u > big ? u : big;
        }
        if (lane < 16) bigs[wave][lane] = big;
        __syncthreads();
#pragma unroll
        for (int v = 0; v < WAVES; v++) big = bigs[v][j] > big ? bigs[v][j] : big;
        __syncthreads();
        const RowScale s(big);
        uint4* to = reinterpret_cast<uint4*>(a.w) + tile * a.l.blocks * 64 + lane;
#pragma unroll
        for (int h = 0; h < HELD; h++) {
            const int64_t b = wave + h * WAVES;
            if (b < a.l.blocks) to[b * 64] = in ? held[h].codes(s.s, s.inv) : make_uint4(0, 0, 0, 0);
        }
        for (int64_t b = wave + HELD * WAVES; b < a.l.blocks; b += WAVES) {
            uint4 c = make_uint4(0, 0, 0, 0);
            if (in) {
                Values<TYPE> v;
                v.load(src, b * INT8_K + k16, a.k);
                c = v.codes(s.s, s.inv);
            }
            to[b * 64] = c;
        }
        if (threadIdx.x < 16) reinterpret_cast<float*>(a.w + a.l.scales)[row] = in ? s.stored : 0.f;
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
//
// A workgroup makes a tile of weight rows by tokens from stages of one block of
// k (64): its blocks of both operands go by DMA into one of four images in LDS,
// each wave bringing its share of whole 1 KB blocks, and every wave reads the
// blocks of its own rows and tokens, a conflict-free 16 bytes a lane each.  A
// block is an operand as it lies in memory, so nothing is shuffled anywhere.
//
// (Blocks through registers and ds_write, or by DMA of 4 bytes a lane, or each
// wave's DMA together behind another wave's products: 8192 x 8192 x 8192 430 us to
// 468, 472 and 462.)
//
// While a wave multiplies a stage's operands it reads the next stage's from
// their image and requests the blocks of the fourth stage on, into the image that
// all have read: one barrier a stage says that an image has landed and that
// another is free.
//
// A operands are the weights, B the tokens: a lane's four results are then four
// neighbouring outputs of one token.

struct I8Args {
    const uint8_t* w;
    const uint8_t* x;  // packed
    const float* bias;
    void* y;
    int32_t* partial;  // [chunk of k][token][row of the last tile too], or null: y
    Int8Layout wl, xl;
    int64_t n, m;
    int32_t out_type;
    int32_t chunk;     // blocks of k of a chunk
};

// The wave's LDS reads and all but its last N loads have landed, then everyone's.
template <int N>
__device__ __forceinline__ void landed_barrier() {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(0x0070 | (N & 15) | ((N >> 4) << 14));
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// The wave's LDS accesses are done, then everyone's; its loads stay in flight.
__device__ __forceinline__ void lds_barrier() {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(0xC07F);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// 16 bytes a lane from a buffer's at + 16 * lane into the 1 KB of LDS at `lds`.  In
// asm, as the compiler would wait for other images' DMA before it reads one; the
// waits are landed_barrier's.  (Writing M0 takes a wait state before its use.)
__device__ __forceinline__ void dma_block(u32x4 rsrc, uint32_t lds, uint32_t lane16, uint32_t at) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
                 :: "s"(lds), "v"(lane16), "s"(rsrc), "s"(at) : "memory");
}

__device__ __forceinline__ u32x4 buffer_of(const void* base, uint32_t bytes) {
    const uint64_t p = reinterpret_cast<uintptr_t>(base);
    return u32x4{static_cast<uint32_t>(p), static_cast<uint32_t>(p >> 32) & 0xffffu, bytes, 0x00020000u};
}

// The results of four neighbouring rows n ... n + 3 and a token.
__device__ __forceinline__ float4 i8_results(const I8Args& a, int64_t n, i32x4 sum, float sx, float4 sw) {
    float4 v = make_float4(static_cast<float>(sum[0]) * sx * sw.x, static_cast<float>(sum[1]) * sx * sw.y,
                           static_cast<float>(sum[2]) * sx * sw.z, static_cast<float>(sum[3]) * sx * sw.w);
    if (a.bias) {
        v.x += n < a.n ? a.bias[n] : 0.f;
        v.y += n + 1 < a.n ? a.bias[n + 1] : 0.f;
        v.z += n + 2 < a.n ? a.bias[n + 2] : 0.f;
        v.w += n + 3 < a.n ? a.bias[n + 3] : 0.f;
    }
    return v;
}

// Four results as bf16 or fp16.
__device__ __forceinline__ uint2 i8_halves(const I8Args& a, float4 v) {
    if (a.out_type == ELEM_BF16) return make_uint2(f32_bf16x2(v.x, v.y), f32_bf16x2(v.z, v.w));
    typedef _Float16 h4 __attribute__((ext_vector_type(4)));
    const h4 h = {static_cast<_Float16>(v.x), static_cast<_Float16>(v.y), static_cast<_Float16>(v.z), static_cast<_Float16>(v.w)};
    return __builtin_bit_cast(uint2, h);
}

__device__ __forceinline__ void i8_store4(const I8Args& a, int64_t t, int64_t n, i32x4 sum, float sx, float4 sw, bool vec) {
    const float4 v = i8_results(a, n, sum, sx, sw);
    const int64_t at = t * a.n + n;
    if (vec && n + 4 <= a.n) {
        if (a.out_type == ELEM_F32) *reinterpret_cast<float4*>(static_cast<float*>(a.y) + at) = v;
        else *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.y) + at) = i8_halves(a, v);
        return;
    }
    const float u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int r = 0; r < 4; r++)
        if (n + r < a.n) elem_st(a.y, at + r, a.out_type, u[r]);
}

// Whether rows of y take whole stores of four values.
__device__ __forceinline__ bool i8_vec(const I8Args& a) {
    return (a.n & 3) == 0 && (reinterpret_cast<uintptr_t>(a.y) & (a.out_type == ELEM_F32 ? 15 : 7)) == 0;
}

// The tile of this workgroup, or x < 0: none.  Workgroups go to the eight dies in
// turn, and each die has an L2 of its own: a die takes one run of the tiles, in
// panels of PANEL column tiles, so that the 32 that it has at once share both
// their rows and their columns.
constexpr int I8_DIES = 8, I8_PANEL = 4;
__device__ __forceinline__ int2 tile_of(int rows, int cols) {
    const int all = rows * cols, each = (all + I8_DIES - 1) / I8_DIES;
    const int b = static_cast<int>(blockIdx.x), at = b % I8_DIES * each + b / I8_DIES;
    if (b / I8_DIES >= each || at >= all) return make_int2(-1, 0);
    const int panel = at / (rows * I8_PANEL), in = at % (rows * I8_PANEL);
    const int wide = cols - panel * I8_PANEL < I8_PANEL ? cols - panel * I8_PANEL : I8_PANEL;
    return make_int2(in / wide, panel * I8_PANEL + in % wide);
}

// Tile of (16 FR WR) weight rows by (16 FT WT) tokens by WR x WT waves, FR x FT
// operands each.
template <int FR, int FT, int WR, int WT>
__global__ void __launch_bounds__(64 * WR * WT) i8_tile_kernel(I8Args a, int32_t row_tiles, int32_t col_tiles) {
    constexpr int AR = FR * WR, AT = FT * WT, WAVES = WR * WT, SHARE = (AR + AT + WAVES - 1) / WAVES;
    constexpr int IMAGE = (AR + AT) * INT8_BLOCK;
    __shared__ i32x4 images[4 * IMAGE / 16];
    const int lane = static_cast<int>(threadIdx.x) & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wr = wave / WT, wt = wave % WT;
    const int64_t blocks = a.wl.blocks;
    const int2 at = tile_of(row_tiles, col_tiles);
    if (at.x < 0) return;
    const int64_t row0 = static_cast<int64_t>(at.x) * AR, col0 = static_cast<int64_t>(at.y) * AT;
    const int64_t first = static_cast<int64_t>(blockIdx.y) * a.chunk;
    const int count = static_cast<int>(blocks - first < a.chunk ? blocks - first : a.chunk);
    // past the matrix, the last rows of blocks again: their results are dropped
    const int64_t rows_here = a.wl.tiles - row0 < AR ? a.wl.tiles - row0 : AR, cols_here = a.xl.tiles - col0 < AT ? a.xl.tiles - col0 : AT;
    const u32x4 ws = buffer_of(a.w + row0 * blocks * INT8_BLOCK, static_cast<uint32_t>(rows_here * blocks * INT8_BLOCK));
    const u32x4 xs = buffer_of(a.x + col0 * blocks * INT8_BLOCK, static_cast<uint32_t>(cols_here * blocks * INT8_BLOCK));
    typedef __attribute__((address_space(3))) i32x4* lds_ptr;
    const uint32_t lds = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_ptr)images)), lane16 = 16u * lane;
    // the wave's blocks of an image (where they do not come out even, the last one
    // twice: the waits count the same loads in every wave), from the first stage on
    u32x4 source[SHARE];
    uint32_t from[SHARE], to[SHARE];
#pragma unroll
    for (int i = 0; i < SHARE; i++) {
        const int b = wave + i * WAVES < AR + AT ? wave + i * WAVES : AR + AT - 1;
        const int last = static_cast<int>(b < AR ? rows_here : cols_here) - 1, tile = b < AR ? b : b - AR;
        source[i] = b < AR ? ws : xs;
        from[i] = static_cast<uint32_t>(((tile < last ? tile : last) * blocks + first) * INT8_BLOCK);
        to[i] = lds + b * INT8_BLOCK;
    }
    // block i of stage s (the last one again past the end) into image q
    const auto request = [&](int s, int q, int i) __attribute__((always_inline)) {
        dma_block(source[i], to[i] + q * IMAGE, lane16, from[i] + static_cast<uint32_t>(s < count ? s : count - 1) * INT8_BLOCK);
    };
    i32x4 acc[FR][FT], fr[2][FR], ft[2][FT];
#pragma unroll
    for (int r = 0; r < FR; r++)
#pragma unroll
        for (int t = 0; t < FT; t++) acc[r][t] = i32x4{0, 0, 0, 0};
    const i32x4* mine_r = images + wr * FR * 64 + lane;
    const i32x4* mine_t = images + (AR + wt * FT) * 64 + lane;
    // operand i (tokens, then rows) from image q
    const auto read = [&](int q, int p, int i) __attribute__((always_inline)) {
        if (i < FT) ft[p][i] = mine_t[q * (IMAGE / 16) + i * 64];
        else fr[p][i - FT] = mine_r[q * (IMAGE / 16) + (i - FT) * 64];
    };
    // stage s, whose image was q, with the operands of parity p
    const auto step = [&](int s, int q, int p) __attribute__((always_inline)) {
        landed_barrier<2 * SHARE>();
#pragma unroll
        for (int r = 0; r < FR; r++) {
#pragma unroll
            for (int i = r * (FR + FT) / FR; i < (r + 1) * (FR + FT) / FR; i++) read((q + 1) & 3, p ^ 1, i);
#pragma unroll
            for (int i = r * SHARE / FR; i < (r + 1) * SHARE / FR; i++) request(s + 4, q, i);
#pragma unroll
            for (int t = 0; t < FT; t++) acc[r][t] = mfma_i8(fr[p][r], ft[p][t], acc[r][t]);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
#pragma unroll
    for (int q = 0; q < 4; q++)
#pragma unroll
        for (int i = 0; i < SHARE; i++) request(q, q, i);
    landed_barrier<3 * SHARE>();
#pragma unroll
    for (int i = 0; i < FR + FT; i++) read(0, 0, i);
    for (int s = 0;; s += 4) {
        step(s, 0, 0);
        if (s + 1 >= count) break;
        step(s + 1, 1, 1);
        if (s + 2 >= count) break;
        step(s + 2, 2, 0);
        if (s + 3 >= count) break;
        step(s + 3, 3, 1);
        if (s + 4 >= count) break;
    }
    // No DMA is in flight, and all have read their last operands: the images are
    // free.  A lane's results are four rows of a token, and 16 rows of 16 tokens
    // would be pieces of 32 bytes: the wave's go through its share of LDS, 16
    // tokens at a time, and out as whole runs of its rows.
    landed_barrier<0>();
    const int size = a.partial || a.out_type == ELEM_F32 ? 4 : 2, pitch = 16 * FR * size + 16;
    uint8_t* mine = reinterpret_cast<uint8_t*>(images) + wave * (16 * (64 * FR + 16));
    static_assert(WAVES * 16 * (64 * FR + 16) <= 4 * IMAGE, "the waves' shares");
    const int64_t n0 = (row0 + wr * FR) * 16, width = a.partial ? a.wl.tiles * 16 : a.n;
    uint8_t* const y = a.partial ? reinterpret_cast<uint8_t*>(a.partial) + static_cast<int64_t>(blockIdx.y) * a.m * width * 4
                                 : static_cast<uint8_t*>(a.y);
    // the bytes that every run of a token's results begins at a multiple of
    const uint32_t apart = static_cast<uint32_t>(width * size) | static_cast<uint32_t>(reinterpret_cast<uintptr_t>(y)) | 16u;
    const int unit = static_cast<int>(apart & (0u - apart));
#pragma unroll
    for (int t = 0; t < FT; t++) {
        const int64_t t0 = (col0 + wt * FT + t) * 16;
        if (t0 >= a.m) break;
        const int64_t token = t0 + (lane & 15) < a.m ? t0 + (lane & 15) : a.m - 1;
        const float sx = reinterpret_cast<const float*>(a.x + a.xl.scales)[token];
#pragma unroll
        for (int r = 0; r < FR; r++) {
            const int64_t n = n0 + r * 16 + 4 * (lane >> 4);
            uint8_t* to = mine + (lane & 15) * pitch + (r * 16 + 4 * (lane >> 4)) * size;
            if (a.partial) {
                *reinterpret_cast<i32x4*>(to) = acc[r][t];
            } else {
                const bool in = n < a.wl.tiles * 16;
                const float4 v = i8_results(a, n, acc[r][t], sx,
                                            in ? *reinterpret_cast<const float4*>(a.w + a.wl.scales + 4 * n) : make_float4(0.f, 0.f, 0.f, 0.f));
                if (size == 4) *reinterpret_cast<float4*>(to) = v;
                else *reinterpret_cast<uint2*>(to) = i8_halves(a, v);
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        const auto out = [&](auto piece) __attribute__((always_inline)) {
            using P = decltype(piece);
            const int each = static_cast<int>(sizeof(P)) / size, pieces = 16 * FR / each;  // values of a piece, pieces of a token
            for (int i = lane; i < 16 * pieces; i += 64) {
                const int row = i / pieces, n = i % pieces * each;
                if (t0 + row >= a.m || n0 + n >= width) continue;
                *reinterpret_cast<P*>(y + ((t0 + row) * width + n0 + n) * size) = *reinterpret_cast<const P*>(mine + row * pitch + n * size);
            }
        };
        if (unit == 16) out(uint4{});
        else if (unit == 8) out(uint2{});
        else if (unit == 4) out(uint32_t{});
        else out(uint16_t{});
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
}

// The chunks' sums of four neighbouring rows and a token a thread; where rows of y
// do not take whole stores, of one row, so that a wave's are a run (203 tokens of
// 5121 rows in two chunks: 6.2 us by fours).
__global__ void __launch_bounds__(256) i8_join_kernel(I8Args a, int32_t chunks) {
    const int64_t fours = a.wl.tiles * 4, all = a.m * fours, stride = static_cast<int64_t>(gridDim.x) * 256;
    if (i8_vec(a)) {
        for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < all; i += stride) {
            const int64_t t = i / fours, n = i % fours * 4;
            if (n >= a.n) continue;
            const i32x4* p = reinterpret_cast<const i32x4*>(a.partial) + i;
            i32x4 sum = p[0];
            for (int c = 1; c < chunks; c++) sum += p[c * all];
            i8_store4(a, t, n, sum, reinterpret_cast<const float*>(a.x + a.xl.scales)[t],
                      *reinterpret_cast<const float4*>(a.w + a.wl.scales + 4 * n), true);
        }
    } else {
        for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < 4 * all; i += stride) {
            const int64_t t = i / (4 * fours), n = i % (4 * fours);
            if (n >= a.n) continue;
            int sum = a.partial[i];
            for (int c = 1; c < chunks; c++) sum += a.partial[i + c * 4 * all];
            float v = static_cast<float>(sum) * reinterpret_cast<const float*>(a.x + a.xl.scales)[t] *
                      reinterpret_cast<const float*>(a.w + a.wl.scales)[n];
            if (a.bias) v += a.bias[n];
            elem_st(a.y, t * a.n + n, a.out_type, v);
        }
    }
}

// ---- a few tokens -------------------------------------------------------------
//
// Up to 16 tokens are one operand's columns, and the weights one stream: a wave
// takes every KS-th block of a row tile, KB by KB, sixteen of them under way, and
// the KS waves of a workgroup add their sums through LDS.
//
// One token's values (x_type 0 to 2) every workgroup quantizes for itself while
// its first weights are under way, a piece of 16 a thread at a time, into the
// operand's order in LDS: a launch less.  Otherwise the tokens are packed, and a
// wave loads its operands beside the weights.
constexpr int I8_BATCH = 8;  // blocks; two batches are under way

struct I8Few {
    I8Args g;
    const void* raw;  // one token's values
    int64_t k;
};

template <int XT, int KS>
__global__ void __launch_bounds__(64 * KS) i8_few_kernel(I8Few a) {
    constexpr bool SELF = XT != I8_PACKED;
    extern __shared__ i32x4 few_lds[];  // the waves' sums, then the tokens' codes
    __shared__ uint32_t bigs[16];
    const int lane = static_cast<int>(threadIdx.x) & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int m = static_cast<int>(a.g.m), blocks = static_cast<int>(a.g.wl.blocks);
    const int mine = (blocks - wave + KS - 1) / KS;  // blocks of a tile
    const int j = lane & 15, token = j < m ? j : m - 1;
    const int64_t tile = blockIdx.x;
    const i32x4* pw = reinterpret_cast<const i32x4*>(a.g.w) + tile * blocks * 64 + lane;
    // block i of the wave's (past them the last one again)
    const auto block = [&](int i) __attribute__((always_inline)) { return wave + (i < mine ? i : mine - 1) * KS; };
    i32x4 w[2][I8_BATCH];
    const auto load_w = [&](int q, int i0) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < I8_BATCH; i++) w[q][i] = __builtin_nontemporal_load(pw + block(i0 + i) * 64);
    };
    if (mine > 0) {
        load_w(0, 0);
        if (mine > I8_BATCH) load_w(1, I8_BATCH);
    }
    i32x4* codes = few_lds + KS * 64;
    float sx = 0.f;
    if constexpr (SELF) {
        const int pieces = blocks * 4, at = static_cast<int>(threadIdx.x);
        Values<XT> first;
        uint32_t big = 0;
        if (at < pieces) {
            first.load(a.raw, at * 16, a.k);
            big = first.largest();
        }
        for (int p = at + 64 * KS; p < pieces; p += 64 * KS) {
            Values<XT> v;
            v.load(a.raw, p * 16, a.k);
            const uint32_t b = v.largest();
            big = b > big ? b : big;
        }
        big = wave_max_bits(big);
        if (lane == 0) bigs[wave] = big;
        lds_barrier();
        big = wave_max_bits(lane < KS ? bigs[lane] : 0);
        const RowScale s(big);
        sx = s.stored;
        if (at < pieces) reinterpret_cast<uint4*>(codes)[at] = first.codes(s.s, s.inv);
        for (int p = at + 64 * KS; p < pieces; p += 64 * KS) {
            Values<XT> v;
            v.load(a.raw, p * 16, a.k);
            reinterpret_cast<uint4*>(codes)[p] = v.codes(s.s, s.inv);
        }
        lds_barrier();
    } else {
        sx = reinterpret_cast<const float*>(a.g.x + a.g.xl.scales)[token];
    }
    const i32x4* px = SELF ? codes + (lane >> 4) : reinterpret_cast<const i32x4*>(a.g.x) + (lane >> 4) * 16 + token;
    i32x4 acc = {0, 0, 0, 0}, x[SELF ? 1 : 2][I8_BATCH];
    const auto load_x = [&](int q, int i0) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < I8_BATCH; i++) x[q][i] = px[block(i0 + i) * (SELF ? 4 : 64)];
    };
    const auto batch = [&](auto parity, int i0) __attribute__((always_inline)) {
        constexpr int q = decltype(parity)::value, qx = SELF ? 0 : q;
        if constexpr (SELF) load_x(0, i0);
        if (i0 + I8_BATCH <= mine) {
#pragma unroll
            for (int i = 0; i < I8_BATCH; i++) acc = mfma_i8(w[q][i], x[qx][i], acc);
        } else {
#pragma unroll
            for (int i = 0; i < I8_BATCH; i++)
                if (i0 + i < mine) acc = mfma_i8(w[q][i], x[qx][i], acc);
        }
        if (i0 + 2 * I8_BATCH < mine) {
            load_w(q, i0 + 2 * I8_BATCH);
            if constexpr (!SELF) load_x(qx, i0 + 2 * I8_BATCH);
        }
    };
    if (mine > 0) {
        if constexpr (!SELF) {
            load_x(0, 0);
            if (mine > I8_BATCH) load_x(SELF ? 0 : 1, I8_BATCH);
        }
        for (int i0 = 0; i0 < mine; i0 += 2 * I8_BATCH) {
            batch(std::integral_constant<int, 0>{}, i0);
            if (i0 + I8_BATCH < mine) batch(std::integral_constant<int, 1>{}, i0 + I8_BATCH);
        }
    }
    few_lds[wave * 64 + lane] = acc;
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int v = 1; v < KS; v++) acc += few_lds[v * 64 + lane];
    const int64_t n = tile * 16 + 4 * (lane >> 4);
    if (j < m && n < a.g.n)
        i8_store4(a.g, j, n, acc, sx, *reinterpret_cast<const float4*>(a.g.w + a.g.wl.scales + 4 * n), i8_vec(a.g));
}

struct I8Plan {
    bool few, self;  // i8_few_kernel, which quantizes the token itself
    int ks;          // its waves a tile
    int shape;       // of the tiles
    int64_t chunks;  // of k
    int64_t chunk;   // blocks of k
    int64_t packed, workspace;
};

// The tiles: rows, tokens, and of what a workgroup takes, in us: a stage, where
// it has its CU to itself and where it shares it, and everything before and behind
// the stages.  (4096 rows of k = 4096, us: 256 tokens in tiles of 128 x 64 15.7,
// of 128 x 128 19.3; 1024 25.6 and 25.9; 4096 62.8 by 256 x 256, 79 by 128 x 128,
// 93 by 128 x 64.  128 tokens by 128 x 32 12.6, by 128 x 64 14.2.)
struct I8Shape {
    int rows, cols;
    float alone, shared, ends;
};
constexpr I8Shape I8_SHAPES[] = {{256, 256, 0.87f, 0.87f, 4.f}, {224, 256, 0.77f, 0.77f, 4.f}, {128, 128, 0.31f, 0.27f, 3.f},
                                 {128, 64, 0.21f, 0.165f, 2.f}, {128, 32, 0.16f, 0.12f, 1.5f}};
constexpr int I8_MAX_CHUNKS = 8;

// The shape and the chunks of k that the above makes shortest: workgroups a CU
// times what each takes, and with chunks the launch that adds them and its bytes.
// (17 tokens of 4096 x 14336: whole 28 us, in eight chunks 18.8; 4096 tokens of
// 14336 x 4096: four rounds of 256 rows 224 us, of 224 rows 217.)  It ranks shapes
// and is no forecast: there is no term for the memory, which bounds tens to hundreds
// of tokens.  Modelled, measured: 4096 tokens of 14336 x 4096 213, 214; of 4096 x
// 14336 199, 175; 203 of 5121 x 4100 9.8 and 5.6 to add the chunks, 15.1 and 5.5; 64
// of 14336 x 4096 12, 20.5 of which quantizing is about 3.
void i8_best_tiles(const Int8Layout& wl, int64_t m, int64_t cus, int* shape, int64_t* chunks) {
    float best = INFINITY;
    for (int s = 0; s < 5; s++) {
        const I8Shape& t = I8_SHAPES[s];
        const int64_t tiles = ((wl.tiles * 16 + t.rows - 1) / t.rows) * ((m + t.cols - 1) / t.cols);
        for (int c = 1; c <= I8_MAX_CHUNKS && c <= wl.blocks; c++) {
            const int64_t each = (tiles * c + cus - 1) / cus, stages = (wl.blocks + c - 1) / c;
            float us = static_cast<float>(each) * (static_cast<float>(stages) * (each == 1 ? t.alone : t.shared) + t.ends);
            if (c > 1) us += 2.5f + static_cast<float>(c) * static_cast<float>(m) * static_cast<float>(wl.tiles) * 16e-6f;
            if (us < best) {
                best = us;
                *shape = s;
                *chunks = c;
            }
        }
    }
}

I8Plan i8_plan(const Int8Layout& wl, const Int8Layout& xl, int64_t m, bool packed) {
    I8Plan p{};
    if (m <= 16) {
        p.few = true;
        // one token of 14336 x 4096: 13.4 us, so quantized first 16.1; two 16.9 and 16.6
        p.self = !packed && m == 1;
        // (us by two, four and eight waves a tile: 14336 x 4096 13.1, 13.4, 19.1; 4096 x 14336 19.9, 15.2, 14.2;
        // 16384 x 1024 5.8, 8.1, 12.5; 1024 x 16384 18.3, 11.8, 10.5)
        p.ks = wl.blocks < 32 ? 2 : wl.tiles < 2 * num_cus() && wl.blocks >= 64 ? 8 : 4;
        p.packed = p.workspace = packed || p.self ? 0 : xl.total;
        p.chunks = 1;
        return p;
    }
    i8_best_tiles(wl, m, num_cus(), &p.shape, &p.chunks);
    p.chunk = (wl.blocks + p.chunks - 1) / p.chunks;
    p.chunks = (wl.blocks + p.chunk - 1) / p.chunk;
    p.packed = packed ? 0 : xl.total;
    p.workspace = p.packed + (p.chunks > 1 ? p.chunks * m * wl.tiles * 64 : 0);
    return p;
}

template <int FR, int FT, int WR, int WT>
int i8_tile(const I8Args& a, const I8Plan& p, hipStream_t st) {
    const int64_t rows = (a.wl.tiles + FR * WR - 1) / (FR * WR), cols = (a.xl.tiles + FT * WT - 1) / (FT * WT);
    if (rows * cols * p.chunks * 64 * WR * WT >= int64_t(1) << 32) {  // threads of a launch
        set_error("vb_int8_gemm: %lld x %lld outputs are too many for a launch", static_cast<long long>(a.m),
                  static_cast<long long>(a.n));
        return E_INVAL;
    }
    const dim3 grid(static_cast<uint32_t>((rows * cols + I8_DIES - 1) / I8_DIES * I8_DIES), static_cast<uint32_t>(p.chunks));
    i8_tile_kernel<FR, FT, WR, WT><<<grid, 64 * WR * WT, 0, st>>>(a, static_cast<int32_t>(rows), static_cast<int32_t>(cols));
    return check_launch("vb_int8_gemm");
}

template <int XT>
int i8_few(const I8Few& a, const I8Plan& p, hipStream_t st) {
    const uint32_t grid = static_cast<uint32_t>(a.g.wl.tiles);
    const uint32_t lds = static_cast<uint32_t>(p.ks * 1024 + (p.self ? a.g.wl.blocks * INT8_K : 0));
    if (p.ks == 2) i8_few_kernel<XT, 2><<<grid, 128, lds, st>>>(a);
    else if (p.ks == 4) i8_few_kernel<XT, 4><<<grid, 256, lds, st>>>(a);
    else i8_few_kernel<XT, 8><<<grid, 512, lds, st>>>(a);
    return check_launch("vb_int8_gemm");
}

int i8_run(I8Args a, const I8Plan& p, hipStream_t st) {
    a.chunk = static_cast<int32_t>(p.chunk);
    if (p.chunks == 1) a.partial = nullptr;
    int rc = OK;
    switch (p.shape) {
        case 0: rc = i8_tile<8, 4, 2, 4>(a, p, st); break;
        case 1: rc = i8_tile<7, 4, 2, 4>(a, p, st); break;
        case 2: rc = i8_tile<4, 4, 2, 2>(a, p, st); break;
        case 3: rc = i8_tile<4, 2, 2, 2>(a, p, st); break;
        default: rc = i8_tile<2, 2, 4, 1>(a, p, st); break;
    }
    if (rc != OK || p.chunks == 1) return rc;
    i8_join_kernel<<<i8_grid((a.m * a.wl.tiles * ((a.n & 3) == 0 ? 4 : 16) + 255) / 256), 256, 0, st>>>(a, static_cast<int32_t>(p.chunks));
    return check_launch("vb_int8_gemm");
}

template <int TYPE>
int i8_quantize_type(const I8Rows& a, hipStream_t st) {
    // a workgroup a row, of four waves where those hold it, until tiles alone give half of the CUs one
    if (a.l.tiles * 2 >= num_cus()) i8_quantize_tiles_kernel<TYPE><<<i8_grid(a.l.tiles), 1024, 0, st>>>(a);
    else if (a.l.blocks <= 128) i8_quantize_rows_kernel<TYPE, 4><<<i8_grid(a.l.tiles * INT8_ROWS), 256, 0, st>>>(a);
    else i8_quantize_rows_kernel<TYPE, 16><<<i8_grid(a.l.tiles * INT8_ROWS), 1024, 0, st>>>(a);
    return check_launch("vb_int8_quantize");
}

int i8_quantize(const void* src, int32_t type, int64_t ld, int64_t rows, int64_t k, uint8_t* w, const Int8Layout& l,
                hipStream_t st) {
    const I8Rows a{src, w, l, ld, rows, k};
    if (type == ELEM_F32) return i8_quantize_type<ELEM_F32>(a, st);
    if (type == ELEM_F16) return i8_quantize_type<ELEM_F16>(a, st);
    return i8_quantize_type<ELEM_BF16>(a, st);
}

int i8_layout_of(const char* what, int64_t rows, int64_t k, Int8Layout* l) {
    if (!int8_layout(rows, k, l)) {
        set_error("%s: no layout for %lld x %lld (at most %lld rows, k at most %lld)", what, static_cast<long long>(rows),
                  static_cast<long long>(k), static_cast<long long>(INT8_MAX_ROWS), static_cast<long long>(INT8_MAX_K));
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
    return i8_quantize(src, type, ld, rows, k, static_cast<uint8_t*>(w), l, as_stream(stream));
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
    if (m < 0 || m > INT8_MAX_ROWS || (x_type != I8_PACKED && !elem_type(x_type)) || !int8_layout(rows, k, &wl)) return -1;
    if (m == 0) return 0;
    return int8_layout(m, k, &xl) ? i8_plan(wl, xl, m, x_type == I8_PACKED).workspace : -1;
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
    const I8Plan p = i8_plan(l, a.xl, m, x_type == I8_PACKED);
    a.x = static_cast<const uint8_t*>(x);
    if (x_type != I8_PACKED && !p.self) {
        a.x = static_cast<const uint8_t*>(workspace);
        if (const int rc = i8_quantize(x, x_type, x_ld, m, k, static_cast<uint8_t*>(workspace), a.xl, as_stream(stream)); rc != OK)
            return rc;
    }
    a.partial = reinterpret_cast<int32_t*>(static_cast<uint8_t*>(workspace) + p.packed);
    a.bias = bias;
    a.y = y;
    a.n = rows;
    a.m = m;
    a.out_type = y_type;
    if (!p.few) return i8_run(a, p, as_stream(stream));
    const I8Few f{a, x, k};
    if (!p.self) return i8_few<I8_PACKED>(f, p, as_stream(stream));
    if (x_type == ELEM_F32) return i8_few<ELEM_F32>(f, p, as_stream(stream));
    if (x_type == ELEM_F16) return i8_few<ELEM_F16>(f, p, as_stream(stream));
    return i8_few<ELEM_BF16>(f, p, as_stream(stream));
}

}  // extern "C"
