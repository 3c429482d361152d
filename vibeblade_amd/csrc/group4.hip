// Products of a few tokens with 4-bit weights of one scale and zero point per
// group (layout in group4.hpp), and the packing, quantizing and decoding of
// such weights:
//
//   W[n, k] = (q[n, k] - z[n, g]) * s[n, g],   g = k / group,  z = 8 without zeros
//   y[t, n] = sum_k W[n, k] x[t, k]
#include "elem_types.hpp"
#include "group4.hpp"
#include "vb_internal.hpp"
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

// Row r's scale of group g among the 16 x per of a block.
__device__ __forceinline__ int scale_at(int r, int g, int per) { return ((r >> 2) * per + g) * 4 + (r & 3); }

__device__ __forceinline__ float g4_value(const G4Weights& g, int64_t row, int64_t k) {
    const int64_t b = block_of(g, row, k);
    const int r = static_cast<int>(row & 15), kk = static_cast<int>(k & 127), j = kk & 7;
    const uint32_t word = reinterpret_cast<const uint32_t*>(g.w)[b * 256 + (((kk >> 3) & 3) * 16 + r) * 4 + (kk >> 5)];
    const int q = (word >> ((j >> 1) * 4 + (j & 1) * 16)) & 15;
    const int per = static_cast<int>(g.l.per), gi = kk * per >> 7, zi = r * per + gi;
    const float s = static_cast<float>(reinterpret_cast<const _Float16*>(g.w + g.l.scales)[b * per * 16 + scale_at(r, gi, per)]);
    const int z = g.has_zeros ? (g.w[g.l.zeros + b * per * 8 + (zi >> 1)] >> ((zi & 1) * 4)) & 15 : 8;
    return static_cast<float>(q - z) * s;
}

// Work items of 256-thread workgroups, as many per thread as it takes: a
// launch has fewer than 2^32 threads.
__device__ __forceinline__ int64_t first_item() { return static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; }
__device__ __forceinline__ int64_t item_stride() { return static_cast<int64_t>(gridDim.x) * 256; }
uint32_t item_blocks(int64_t n) { return static_cast<uint32_t>(n > (1 << 28) ? 1 << 20 : (n + 255) / 256); }

// One thread per dword of codes, then per block's scales and zero points.
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
                                                             Group4Layout l, int64_t rows, int32_t group, int64_t groups) {
    const int per = static_cast<int>(l.per);
    for (int64_t b = first_item(); b < l.tiles * l.steps; b += item_stride()) {
        const int64_t tile = b / l.steps, k0 = b % l.steps * 128;
        _Float16* so = reinterpret_cast<_Float16*>(out + l.scales) + b * per * 16;
        uint8_t* zo = out + l.zeros + b * per * 8;
        for (int i = 0; i < 16 * per; i += 2) {  // a byte of zero points: rows or groups next to each other
            uint32_t zs = 0;
            for (int h = 0; h < 2; h++) {
                const int r = (i + h) / per, g = (i + h) % per;
                const int64_t row = tile * 16 + r, gi = (k0 + g * (128 / per)) / group;
                const bool in = row < rows && gi < groups;
                so[scale_at(r, g, per)] = in ? scales[row * groups + gi] : static_cast<_Float16>(0.f);
                if (zeros && in) zs |= (zeros[row * groups + gi] & 15u) << (4 * h);
            }
            if (zeros) zo[i >> 1] = static_cast<uint8_t>(zs);
        }
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

// ---- products ---------------------------------------------------------------
//
// A wave takes a row tile (16 rows) and every KS-th of its 128-steps: one
// 16-byte load per lane brings a step's codes in the order of the A operand of
// v_mfma_f32_16x16x32_f16 (group4.hpp).  Two codes become two halves by one
// mask: in the low bits of the mantissa of 1024 (codes at bits 0-3) or at bit 4
// of that of 64 (codes at bits 4-7) they are 1024 + q and 64 + q, and a packed
// subtraction leaves q - z exactly.  The scale stays out of the operand: a
// group's products are summed in fp32 and then scaled, so nothing is rounded
// but the sums.
//
// The B operand's 16 columns are the tokens.  fp16 activations are taken as
// they are; fp32 ones as two halves hi + lo in two columns (22 bits), bf16 ones
// as one (all 8 bits), each block of 128 brought to [2^14, 2^15) by a power of
// two that the group's sum is multiplied back by.  Columns past the tokens
// repeat the last one and are dropped.
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef float float4_t __attribute__((ext_vector_type(4)));

constexpr int G4_WAVES = 8;
constexpr int G4_THREADS = 64 * G4_WAVES;

struct G4Args {
    const uint8_t* w;
    Group4Layout l;
    const void* x;
    float* y;
    int64_t x_ld, rows, k;
    int32_t m;          // tokens of this launch
    int32_t ks;         // waves that share a row tile
    int32_t groups;     // sets of G4_WAVES / ks row tiles
    int32_t chunk;      // 128-steps of x in LDS at a time
    bool whole;         // all of x fits: staged once
};

template <int XT>
struct XUnit {
    uint32_t u[XT == ELEM_F32 ? 8 : 4];
};

template <int XT>
__device__ __forceinline__ XUnit<XT> x_load(const G4Args& a, int token, int64_t k0) {
    XUnit<XT> r;
    if constexpr (XT == ELEM_F32) {
        typedef uint32_t v4 __attribute__((ext_vector_type(4), aligned(4)));
        const float* p = static_cast<const float*>(a.x) + token * a.x_ld + k0;
        if (k0 + 8 <= a.k) {
            const v4 lo = *reinterpret_cast<const v4*>(p), hi = *reinterpret_cast<const v4*>(p + 4);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                r.u[i] = lo[i];
                r.u[4 + i] = hi[i];
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) r.u[i] = k0 + i < a.k ? __float_as_uint(p[i]) : 0u;
        }
    } else {
        typedef uint32_t v4 __attribute__((ext_vector_type(4), aligned(2)));
        const uint16_t* p = static_cast<const uint16_t*>(a.x) + token * a.x_ld + k0;
        if (k0 + 8 <= a.k) {
            const v4 v = *reinterpret_cast<const v4*>(p);
#pragma unroll
            for (int i = 0; i < 4; i++) r.u[i] = v[i];
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint32_t lo = k0 + 2 * i < a.k ? p[2 * i] : 0u, hi = k0 + 2 * i + 1 < a.k ? p[2 * i + 1] : 0u;
                r.u[i] = lo | hi << 16;
            }
        }
    }
    return r;
}

// The same without a branch around a load: a piece that reaches past k (k >= 8)
// takes the row's last eight values and moves its own to the front.
template <int XT>
__device__ __forceinline__ XUnit<XT> x_load_whole(const G4Args& a, int token, int64_t k0) {
    XUnit<XT> r;
    k0 = k0 + 8 <= a.k ? k0 : a.k - 8;
    if constexpr (XT == ELEM_F32) {
        typedef uint32_t v4 __attribute__((ext_vector_type(4), aligned(4)));
        const v4* p = reinterpret_cast<const v4*>(static_cast<const float*>(a.x) + token * a.x_ld + k0);
        const v4 lo = p[0], hi = p[1];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            r.u[i] = lo[i];
            r.u[4 + i] = hi[i];
        }
    } else {
        typedef uint32_t v4 __attribute__((ext_vector_type(4), aligned(2)));
        const v4 v = *reinterpret_cast<const v4*>(static_cast<const uint16_t*>(a.x) + token * a.x_ld + k0);
#pragma unroll
        for (int i = 0; i < 4; i++) r.u[i] = v[i];
    }
    return r;
}

template <int XT>
__device__ __forceinline__ void x_shift(XUnit<XT>& r, int by) {  // values `by`.. of the eight to the front, zeros behind
    if constexpr (XT == ELEM_F32) {
#pragma unroll
        for (int b = 4; b >= 1; b >>= 1) {
            if (!(by & b)) continue;
#pragma unroll
            for (int i = 0; i < 8; i++) r.u[i] = i + b < 8 ? r.u[i + b] : 0u;
        }
        if (by & 8) {
#pragma unroll
            for (int i = 0; i < 8; i++) r.u[i] = 0u;
        }
    } else {
#pragma unroll
        for (int b = 4; b >= 1; b >>= 1) {
            if (!(by & (2 * b))) continue;
#pragma unroll
            for (int i = 0; i < 4; i++) r.u[i] = i + b < 4 ? r.u[i + b] : 0u;
        }
        if (by & 1) {
#pragma unroll
            for (int i = 0; i < 4; i++) r.u[i] = r.u[i] >> 16 | (i < 3 ? r.u[i + 1] << 16 : 0u);
        }
    }
}

// The largest of 16 lanes' values (a DPP row), in each of them.
__device__ __forceinline__ float row_max(float v) {
    v = fmaxf(v, dpp_f<0xB1>(v));
    v = fmaxf(v, dpp_f<0x4E>(v));
    v = fmaxf(v, dpp_f<0x141>(v));
    return fmaxf(v, dpp_f<0x140>(v));
}

__device__ __forceinline__ uint32_t pack_half2(float a, float b) {
    const half2_t h = {static_cast<_Float16>(a), static_cast<_Float16>(b)};
    return __builtin_bit_cast(uint32_t, h);
}

// A unit's columns into LDS.  xs: [step][t][c][col] of 8 halves; inv: [step][token].
template <int XT>
__device__ __forceinline__ void x_store(const XUnit<XT>& r, uint4* xs, float* inv, int cols, int m, int token, int kc) {
    uint4* at = xs + static_cast<int64_t>(kc) * cols + (XT == ELEM_F32 ? 2 * token : token);
    if constexpr (XT == ELEM_F16) {
        *at = make_uint4(r.u[0], r.u[1], r.u[2], r.u[3]);
    } else {
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            if constexpr (XT == ELEM_F32) v[i] = __uint_as_float(r.u[i]);
            else v[i] = __uint_as_float(i & 1 ? r.u[i >> 1] & 0xffff0000u : r.u[i >> 1] << 16);
        }
        // the largest magnitude of the 128 by its bits (NaN and infinity are the largest)
        uint32_t big = 0;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const uint32_t b = __float_as_uint(v[i]) & 0x7fffffffu;
            big = b > big ? b : big;
        }
        const uint32_t top = static_cast<uint32_t>(row_max(static_cast<float>(big >> 23)));  // its exponent
        // 2^(14 - exponent), within the normal numbers with its reciprocal; 1 for a block without bounds
        uint32_t f = top == 255 ? 127 : 268 - top;
        f = f > 253 ? 253 : f;
        const float scale = __uint_as_float(f << 23);
        float hi[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            v[i] *= scale;
            hi[i] = static_cast<float>(static_cast<_Float16>(v[i]));
        }
        *at = make_uint4(pack_half2(hi[0], hi[1]), pack_half2(hi[2], hi[3]), pack_half2(hi[4], hi[5]),
                         pack_half2(hi[6], hi[7]));
        if constexpr (XT == ELEM_F32) {
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = top == 255 ? 0.f : v[i] - hi[i];
            at[1] = make_uint4(pack_half2(v[0], v[1]), pack_half2(v[2], v[3]), pack_half2(v[4], v[5]),
                               pack_half2(v[6], v[7]));
        }
        if ((kc & 15) == 0) inv[(kc >> 4) * m + token] = __uint_as_float((254 - f) << 23);
    }
}

// The wave's LDS accesses are done, then everyone's; its loads from memory stay in flight.
__device__ __forceinline__ void lds_barrier() {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(0xC07F);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

typedef _Float16 half4_t __attribute__((ext_vector_type(4)));

// What a wave loads of one block.
template <int PER, bool ZEROS>
struct WStep {
    u32x4 q;
    half4_t s[PER];
    uint32_t z;  // zero points of 8 / PER rows, the lane's among them
};

template <int PER>
constexpr int g4_depth() { return PER == 1 ? 8 : 4; }  // blocks in flight per wave

template <int PER, bool ZEROS, int XT, int NT>
__global__ void __launch_bounds__(G4_THREADS, NT == 4 ? 2 : 4) g4_gemv_kernel(G4Args a) {
    constexpr int DEPTH = g4_depth<PER>();
    constexpr int PARTS = XT == ELEM_F32 ? 2 : 1;
    extern __shared__ uint4 lds[];
    const int tid = static_cast<int>(threadIdx.x), lane = tid & 63, n = lane & 15, c = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int cols = PARTS * a.m, ks = a.ks, sub = wave % ks, local = wave / ks, per_group = G4_WAVES / ks;
    const int steps = static_cast<int>(a.l.steps), tiles = static_cast<int>(a.l.tiles);
    float4_t* red = reinterpret_cast<float4_t*>(lds);  // [wave][nt][lane]
    float* inv = reinterpret_cast<float*>(lds + (ks > 1 ? G4_WAVES * NT * 64 : 0));
    uint4* xs = reinterpret_cast<uint4*>(inv) + (XT == ELEM_F16 ? 0 : (a.chunk * a.m + 3) / 4);

    int col[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) col[t] = t * 16 + n < cols ? t * 16 + n : cols - 1;

    const int pieces = a.chunk * 16, units = pieces * a.m;  // of a token, of all tokens in a chunk
    auto stage = [&](int first, int from) {                 // pieces from .. of steps first .. first + chunk of x
#pragma unroll 1
        for (int u = from + tid; u < units; u += G4_THREADS) {
            const int token = u / pieces, kc = u % pieces;
            x_store<XT>(x_load<XT>(a, token, (static_cast<int64_t>(first) * 16 + kc) * 8), xs, inv, cols, a.m, token, kc);
        }
    };
    // Loads of the ring: a step or tile past the last is outside of its
    // buffer and reads nothing.  (A branch around a load would make the
    // compiler wait for all loads in flight.)
    auto load = [&](int tile, int step, WStep<PER, ZEROS>& r) __attribute__((always_inline)) {
        const bool in = tile < tiles;
        const int64_t b = in ? static_cast<int64_t>(tile) * steps : 0;
        const uint32_t size = in ? static_cast<uint32_t>(steps) : 0u;
        const __amdgpu_buffer_rsrc_t rq = make_rsrc(a.w + b * 1024, size * 1024);
        const __amdgpu_buffer_rsrc_t rs = make_rsrc(a.w + a.l.scales + b * (32 * PER), size * (32 * PER));
        r.q = buf_ld128(rq, static_cast<uint32_t>(step) * 1024 + lane * 16, 0);
        const uint32_t so = (static_cast<uint32_t>(step) * 4 + c) * (8 * PER);
        if constexpr (PER == 1) {
            typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
            r.s[0] = __builtin_bit_cast(half4_t, __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(rs, static_cast<int>(so), 0, 0)));
        } else {
#pragma unroll
            for (int g = 0; g < PER; g += 2) {
                const half8_t v = __builtin_bit_cast(half8_t, buf_ld128(rs, so + 8 * g, 0));
                r.s[g] = half4_t{v[0], v[1], v[2], v[3]};
                r.s[g + 1] = half4_t{v[4], v[5], v[6], v[7]};
            }
        }
        if constexpr (ZEROS) {
            const __amdgpu_buffer_rsrc_t rz = make_rsrc(a.w + a.l.zeros + b * (8 * PER), size * (8 * PER));
            r.z = __builtin_amdgcn_raw_buffer_load_b32(rz, static_cast<int>(step * (8 * PER) + n * PER / 8 * 4), 0, 0);
        }
        __builtin_amdgcn_sched_barrier(0);  // slot after slot, as they are waited for
    };
    float4_t acc[NT];
    auto multiply = [&](const WStep<PER, ZEROS>& r, int at) __attribute__((always_inline)) {  // step `at` of the chunk
        const uint4* xb = xs + (at * 16 + c) * cols;
        float4_t p[NT], sum[NT];
        half8_t xv[4][NT];
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int u = 0; u < NT; u++) xv[t][u] = __builtin_bit_cast(half8_t, xb[t * 4 * cols + col[u]]);
#pragma unroll
        for (int t = 0; t < 4; t++) {
            const int g = t * PER / 4;
            uint32_t z = 8;
            if (ZEROS) z = (r.z >> (n * PER % 8 * 4 + 4 * g)) & 15;
            const half2_t z0 = __builtin_bit_cast(half2_t, z * 0x00010001u + 0xE400E400u);  // -(1024 + z)
            const half2_t z1 = __builtin_bit_cast(half2_t, z * 0x00100010u + 0xD400D400u);  // -(64 + z)
            const uint32_t q = r.q[t], qh = q >> 8;
            const half2_t h0 = __builtin_bit_cast(half2_t, (q & 0x000f000fu) | 0x64006400u) + z0;
            const half2_t h1 = __builtin_bit_cast(half2_t, (q & 0x00f000f0u) | 0x54005400u) + z1;
            const half2_t h2 = __builtin_bit_cast(half2_t, (qh & 0x000f000fu) | 0x64006400u) + z0;
            const half2_t h3 = __builtin_bit_cast(half2_t, (qh & 0x00f000f0u) | 0x54005400u) + z1;
            const half8_t wv = {h0[0], h0[1], h1[0], h1[1], h2[0], h2[1], h3[0], h3[1]};
#pragma unroll
            for (int u = 0; u < NT; u++) {
                const float4_t zero = {0.f, 0.f, 0.f, 0.f};
                p[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wv, xv[t][u], t % (4 / PER) == 0 ? zero : p[u], 0, 0, 0);
                if ((t + 1) % (4 / PER) == 0) {
                    // fp16 x adds to acc; the others to the block's sum, which then takes the block's power of two
                    float4_t& to = XT == ELEM_F16 ? acc[u] : sum[u];
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float s = static_cast<float>(r.s[g][i]);
                        to[i] = XT != ELEM_F16 && g == 0 ? s * p[u][i] : __builtin_fmaf(s, p[u][i], to[i]);
                    }
                }
            }
        }
        if (XT != ELEM_F16) {
#pragma unroll
            for (int u = 0; u < NT; u++) {
                const float f = inv[at * a.m + col[u] / PARTS];
#pragma unroll
                for (int i = 0; i < 4; i++) acc[u][i] = __builtin_fmaf(f, sum[u][i], acc[u][i]);
            }
        }
    };

    // The wave's steps of a tile: sub, sub + ks, ..., in rounds of DEPTH; the
    // last rounds load the next tile's first ones.
    const int rounds = (steps + ks * DEPTH - 1) / (ks * DEPTH);
    const int hop = static_cast<int>(gridDim.x) * per_group;
    int tile = static_cast<int>(blockIdx.x) * per_group + local;
    WStep<PER, ZEROS> ring[DEPTH];
    // x first, as loads come back in order: pieces past HELD per thread, then
    // HELD of them on the way together with the ring's first round.
    constexpr int HELD = 4;
    XUnit<XT> held[HELD];
    const bool hold = a.k >= 8;
    stage(0, hold ? HELD * G4_THREADS : 0);
    if (hold) {
#pragma unroll
        for (int i = 0; i < HELD; i++) {
            const int u = i * G4_THREADS + tid, v = u < units ? u : units - 1;
            held[i] = x_load_whole<XT>(a, v / pieces, static_cast<int64_t>(v % pieces) * 8);
        }
    }
#pragma unroll
    for (int d = 0; d < DEPTH; d++) load(tile, sub + d * ks, ring[d]);
    if (hold) {
#pragma unroll
        for (int i = 0; i < HELD; i++) {
            const int u = i * G4_THREADS + tid;
            if (u >= units) continue;
            const int token = u / pieces, kc = u % pieces;
            if (kc * 8 + 8 > a.k) x_shift<XT>(held[i], static_cast<int>(kc * 8 >= a.k ? 8 : kc * 8 + 8 - a.k));
            x_store<XT>(held[i], xs, inv, cols, a.m, token, kc);
        }
    }
    lds_barrier();
    bool staged = true;  // the chunk in LDS is the next one to be used
    for (int grp = static_cast<int>(blockIdx.x); grp < a.groups; grp += static_cast<int>(gridDim.x), tile += hop) {
#pragma unroll
        for (int t = 0; t < NT; t++) acc[t] = float4_t{0.f, 0.f, 0.f, 0.f};
        int first = 0;  // of the chunk (whose length is whole rounds)
        for (int i = 0; i < rounds; i++) {
            const int s = i * ks * DEPTH + sub;
            if (s - sub == first + a.chunk) first += a.chunk;
            if (!a.whole && s - sub == first) {
                if (!staged) {
                    lds_barrier();  // the chunk before is read
                    stage(first, 0);
                    lds_barrier();
                }
                staged = false;
            }
            const bool last = i + 1 == rounds;
            const int next = last ? tile + hop : tile, from = last ? sub : s + DEPTH * ks;
#pragma unroll
            for (int d = 0; d < DEPTH; d++) {
                if (tile < tiles && s + d * ks < steps) multiply(ring[d], s + d * ks - first);
                load(next, from + d * ks, ring[d]);
            }
        }
        if (ks == 1) {
            // the wave's tile is done: its lanes hold rows 4 c + 0..3 of column n
#pragma unroll
            for (int t = 0; t < NT; t++) {
                if (PARTS == 2) {
#pragma unroll
                    for (int i = 0; i < 4; i++) acc[t][i] += dpp_f<0xB1>(acc[t][i]);
                }
                const int cc = t * 16 + n;
                const int64_t row = static_cast<int64_t>(tile) * 16 + 4 * c;
                if (tile < tiles && cc < cols && cc % PARTS == 0) {
                    float* y = a.y + static_cast<int64_t>(cc / PARTS) * a.rows + row;
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if (row + i < a.rows) y[i] = acc[t][i];
                }
            }
            continue;
        }
        // y: the waves of a tile, and the two halves of fp32 activations, added in order
#pragma unroll
        for (int t = 0; t < NT; t++) red[(wave * NT + t) * 64 + lane] = acc[t];
        lds_barrier();
        const float* rf = reinterpret_cast<const float*>(red);
        for (int o = tid; o < per_group * 16 * a.m; o += G4_THREADS) {
            const int r = o & 15, tt = (o >> 4) % per_group, token = (o >> 4) / per_group;
            const int64_t row = (static_cast<int64_t>(grp) * per_group + tt) * 16 + r;
            float sum = 0.f;
#pragma unroll
            for (int h = 0; h < PARTS; h++) {
                const int cc = PARTS * token + h;
                for (int v = 0; v < ks; v++)
                    sum += rf[(((tt * ks + v) * NT + (cc >> 4)) * 64 + (r >> 2) * 16 + (cc & 15)) * 4 + (r & 3)];
            }
            if (row < a.rows) a.y[static_cast<int64_t>(token) * a.rows + row] = sum;
        }
        lds_barrier();  // red is free
    }
}

template <int PER, bool ZEROS, int XT>
void g4_launch(const G4Args& a, int nt, uint32_t grid, uint32_t lds, hipStream_t st) {
    if (nt == 1) g4_gemv_kernel<PER, ZEROS, XT, 1><<<grid, G4_THREADS, lds, st>>>(a);
    else if (nt == 2) g4_gemv_kernel<PER, ZEROS, XT, 2><<<grid, G4_THREADS, lds, st>>>(a);
    else if constexpr (XT == ELEM_F16) g4_gemv_kernel<PER, ZEROS, XT, 4><<<grid, G4_THREADS, lds, st>>>(a);
}

template <int PER, bool ZEROS>
void g4_launch_x(const G4Args& a, int xt, int nt, uint32_t grid, uint32_t lds, hipStream_t st) {
    if (xt == ELEM_F32) g4_launch<PER, ZEROS, ELEM_F32>(a, nt, grid, lds, st);
    else if (xt == ELEM_F16) g4_launch<PER, ZEROS, ELEM_F16>(a, nt, grid, lds, st);
    else g4_launch<PER, ZEROS, ELEM_BF16>(a, nt, grid, lds, st);
}

constexpr int64_t G4_LDS = 120 << 10;  // of x in LDS, at most

int g4_run(G4Args a, int x_type, bool has_zeros, hipStream_t st) {
    const int parts = x_type == ELEM_F32 ? 2 : 1, cols = parts * a.m, nt = cols <= 16 ? 1 : cols <= 32 ? 2 : 4;
    const int depth = a.l.per == 1 ? g4_depth<1>() : g4_depth<4>();
    const int64_t slots = 16 * num_cus();  // waves that are resident at once
    a.ks = 1;
    while (a.ks < G4_WAVES && a.l.tiles * a.ks * 2 <= slots && a.ks < a.l.steps) a.ks *= 2;
    // the 128-steps of x that LDS takes, whole rounds of the ring (64 columns are 16 KB a step)
    const int64_t step_bytes = 256 * cols + (x_type == ELEM_F16 ? 0 : 4 * a.m);
    int64_t chunk = G4_LDS / step_bytes;
    a.whole = chunk >= a.l.steps;
    while (!a.whole && a.ks > 1 && chunk < depth * a.ks) a.ks /= 2;
    chunk = a.whole ? a.l.steps : chunk / (depth * a.ks) * (depth * a.ks);
    if (chunk == 0) chunk = depth;
    a.chunk = static_cast<int32_t>(chunk);
    const int per_group = G4_WAVES / a.ks;
    a.groups = static_cast<int32_t>((a.l.tiles + per_group - 1) / per_group);
    const uint32_t lds = static_cast<uint32_t>((a.ks > 1 ? G4_WAVES * nt * 1024 : 0) +
                                               (x_type == ELEM_F16 ? 0 : (chunk * a.m + 3) / 4 * 16) + chunk * 256 * cols);
    const int64_t most = (lds > (80 << 10) ? 1 : 2) * num_cus();
    const uint32_t grid = static_cast<uint32_t>(a.groups < most ? a.groups : most);
    const int per = static_cast<int>(a.l.per);
    if (has_zeros) {
        if (per == 1) g4_launch_x<1, true>(a, x_type, nt, grid, lds, st);
        else if (per == 2) g4_launch_x<2, true>(a, x_type, nt, grid, lds, st);
        else g4_launch_x<4, true>(a, x_type, nt, grid, lds, st);
    } else {
        if (per == 1) g4_launch_x<1, false>(a, x_type, nt, grid, lds, st);
        else if (per == 2) g4_launch_x<2, false>(a, x_type, nt, grid, lds, st);
        else g4_launch_x<4, false>(a, x_type, nt, grid, lds, st);
    }
    return check_launch("vb_group4_gemv");
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
    g4_pack_groups_kernel<<<item_blocks(l.tiles * l.steps), 256, 0, st>>>(
        static_cast<const _Float16*>(scales), zeros, static_cast<uint8_t*>(w), l, rows, group, (k + group - 1) / group);
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
    // tokens a launch takes: 32 columns of scaled activations, 64 of fp16 ones (the registers of four column tiles)
    const int64_t slab = x_type == ELEM_F32 ? 16 : x_type == ELEM_F16 ? 64 : 32;
    for (int64_t t = 0; t < m; t += slab) {
        const void* xt = static_cast<const uint8_t*>(x) + t * x_ld * elem_bytes(x_type);
        const G4Args a{g.w, g.l, xt, y + t * rows, x_ld, rows, k, static_cast<int32_t>(m - t < slab ? m - t : slab),
                       0, 0, 0, false};
        if (const int rc = g4_run(a, x_type, g.has_zeros, as_stream(stream)); rc != OK) return rc;
    }
    return OK;
}

}  // extern "C"
