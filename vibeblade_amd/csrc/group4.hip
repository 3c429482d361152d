// Products of a few tokens with 4-bit weights of one scale and zero point per
// group (layout in group4.hpp), and the packing, quantizing and decoding of
// such weights:
//
//   W[n, k] = (q[n, k] - z[n, g]) * s[n, g],   g = k / group,  z = 8 without zeros
//   y[t, n] = sum_k W[n, k] x[t, k]
#include <type_traits>

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

// Row r's scale of group g (of 2 per) among the 32 x per of a block.
__device__ __forceinline__ int scale_at(int r, int g, int per) { return ((r >> 2) * 2 * per + g) * 4 + (r & 3); }

__device__ __forceinline__ float g4_value(const G4Weights& g, int64_t row, int64_t k) {
    const uint8_t* b = g.w + ((row >> 4) * g.l.blocks + k / GROUP4_K) * g.l.bytes;
    const int r = static_cast<int>(row & 15), kk = static_cast<int>(k & (GROUP4_K - 1));
    const uint32_t word = reinterpret_cast<const uint32_t*>(b)[(kk >> 7) * 256 + (((kk >> 3) & 3) * 16 + r) * 4 + ((kk >> 5) & 3)];
    const int q = (word >> (kk & 7) * 4) & 15, at = scale_at(r, kk * g.l.per >> 7, g.l.per);
    const float s = static_cast<float>(reinterpret_cast<const _Float16*>(b + g.l.scales)[at]);
    const int z = g.has_zeros ? (b[g.l.zeros + (at >> 1)] >> ((at & 1) * 4)) & 15 : 0;
    return static_cast<float>((q ^ 8) - (z ^ 8)) * s;
}

// Work items of 256-thread workgroups, as many per thread as it takes: a
// launch has fewer than 2^32 threads.
__device__ __forceinline__ int64_t first_item() { return static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; }
__device__ __forceinline__ int64_t item_stride() { return static_cast<int64_t>(gridDim.x) * 256; }
uint32_t item_blocks(int64_t n) { return static_cast<uint32_t>(n > (1 << 28) ? 1 << 20 : (n + 255) / 256); }

// One thread per dword of codes, then per block's scales and zero points.
__global__ void __launch_bounds__(256) g4_pack_codes_kernel(const uint8_t* packed, uint8_t* out, Group4Layout l,
                                                            int64_t rows, int64_t k) {
    for (int64_t i = first_item(); i < l.tiles * l.blocks * 512; i += item_stride()) {
        const int64_t b = i >> 9;
        const int step = static_cast<int>(i >> 8) & 1, lane = static_cast<int>(i >> 2) & 63, t = static_cast<int>(i) & 3;
        const int64_t row = b / l.blocks * 16 + (lane & 15);
        const int64_t k0 = b % l.blocks * GROUP4_K + step * 128 + t * 32 + (lane >> 4) * 8;
        uint32_t word = 0;
        if (row < rows)
            for (int j = 0; j < 8 && k0 + j < k; j++) {
                const uint32_t byte = packed[row * ((k + 1) >> 1) + ((k0 + j) >> 1)];
                word |= (((j & 1 ? byte >> 4 : byte) & 15u) ^ 8u) << (4 * j);
            }
        reinterpret_cast<uint32_t*>(out + b * l.bytes)[i & 511] = word;
    }
}

__global__ void __launch_bounds__(256) g4_pack_groups_kernel(const _Float16* scales, const uint8_t* zeros, uint8_t* out,
                                                             Group4Layout l, int64_t rows, int32_t group, int64_t groups) {
    const int per = l.per;
    for (int64_t b = first_item(); b < l.tiles * l.blocks; b += item_stride()) {
        const int64_t tile = b / l.blocks, k0 = b % l.blocks * GROUP4_K;
        _Float16* so = reinterpret_cast<_Float16*>(out + b * l.bytes + l.scales);
        uint8_t* zo = out + b * l.bytes + l.zeros;
        for (int i = 0; i < 32 * per; i += 2) {  // two rows of a group: a byte of zero points
            uint32_t zs = 0;
            for (int h = 0; h < 2; h++) {
                const int r = i / (8 * per) * 4 + (i & 3) + h, g = i / 4 % (2 * per);
                const int64_t row = tile * 16 + r, gi = (k0 + g * (128 / per)) / group;
                const bool in = row < rows && gi < groups;
                so[i + h] = in ? scales[row * groups + gi] : static_cast<_Float16>(0.f);
                if (zeros && in) zs |= ((zeros[row * groups + gi] & 15u) ^ 8u) << (4 * h);
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
// z = round(-lo / s).  s is rounded to fp16 first (at most 65504, and weights
// past its codes take the last one) and the codes go by that.  A NaN or an
// infinity has no code: its group's scale is NaN.
__global__ void __launch_bounds__(256) g4_quantize_kernel(const void* src, int32_t type, int64_t ld, int64_t rows,
                                                          int64_t k, int32_t group, int64_t groups, uint8_t* codes,
                                                          _Float16* scales, uint8_t* zeros) {
    for (int64_t i = first_item(); i < rows * groups; i += item_stride()) {
        const int64_t row = i / groups, k0 = i % groups * group, end = k0 + group < k ? k0 + group : k;
        float lo = 0.f, hi = 0.f;
        bool finite = true;
        for (int64_t j = k0; j < end; j++) {
            const float v = elem_ld(src, row * ld + j, type);
            finite = finite && fabsf(v) < INFINITY;
            lo = fminf(lo, v);
            hi = fmaxf(hi, v);
        }
        const float want = zeros ? (hi - lo) / 15.f : fmaxf(hi, -lo) / 7.f;
        const _Float16 sh = static_cast<_Float16>(finite ? fminf(want, 65504.f) : NAN);
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
// A wave takes a row tile (16 rows) and every ks-th of its blocks of 256 k: one
// 16-byte load per lane brings half a block's codes in the order of the A operand of
// v_mfma_i32_16x16x64_i8 (group4.hpp).  The operand needs no more than a shift
// and two masks per eight codes: a nibble in the high half of a byte, as int8,
// is 16 (q - 8).  Fp16 operands take five times the instructions, and
// instructions are what bounds a wave here: at the memory's rate a CU has about
// 100 issue slots for a step's 1 KB.
//
// Bound by memory where the weights are large (one token, us and TB/s of weights:
// 128256 x 4096 44 and 6.2, 128256 x 14336 147 and 6.5); below that by what comes
// before and behind the stream (14336 x 4096 9.0 and 3.4, 4096 x 4096 5.9, of
// which a launch is 1.9, the first loads, digits and barrier about 2 and the
// sums over waves 0.5); with more tokens by staging them and, in groups of 32,
// by the multiplications and sums of each group (128256 x 4096, five tokens 54).
//
// The B operand's 16 columns are the activations as integers: each block of 128
// of a token, brought by a power of two to |X| < 2^30 (fp32 x) or 2^22 (16-bit
// x) and rounded, is split into 4 or 3 signed digits to the base 256, one
// column each.  fp32 values keep all their bits down to 2^-6 of the block's
// largest, bf16 and fp16 ones down to 2^-14 and 2^-11; what is lost below is at
// most 2^-30 (2^-22) of the largest.  Sums over a group are exact:
//
//   sum (q - z) X = sum (q - 8) X - (z - 8) sum X
//
// with sum X found once as x is staged.  Then, in fp32, a group's sum is
// multiplied by its scale and the block's power of two and added up; the digits
// of a token meet at the end.  Until then each digit counts as the top one, so a
// sum may be up to 4 sum |W| max |x| (over each block) and has to stay below
// 2^128.  A block with a NaN or an infinity has the power
// NaN, which stays in its token.  Columns past the tokens repeat the last one
// and are dropped.
//
// More than a few 16-bit tokens would take two or three such sets of columns, so
// they go to v_mfma_f32_16x16x32_f16 as they are, a column each: fp16 values
// unchanged, bf16 ones brought to |x| < 2^15 by a power of two for each block of
// 128 (exact down to 2^-31 of its largest, below that cut to multiples of fp16's
// 2^-24, at most 2^-38 of it).  The weights' codes become fp16 integers q - z, exactly; a group's
// products are summed in fp32.
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef float float4_t __attribute__((ext_vector_type(4)));
typedef int int4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr int G4_WAVES = 8;  // of a workgroup, at most

struct G4Args {
    const uint8_t* w;
    Group4Layout l;
    const void* x;
    uint8_t* image;  // x as digits, chunk after chunk, laid out for LDS (null: the workgroups make it)
    float* partial;  // [chunk][token][row]: sums of a chunk, where there are several
    float* y;
    int64_t x_ld, rows, k;
    int32_t x_type, parts;  // digits of a value (1: fp16 operands)
    int32_t m;              // tokens of this launch
    int32_t ks;             // waves of a workgroup that share a row tile
    int32_t kz, chunk;      // chunks of k, each a workgroup's of its own, and their blocks
    int32_t groups;         // sets of waves / ks row tiles, one a workgroup's turn
};

// Eight activations as loaded: fp32 (8 dwords) or 16-bit (4).
template <int PARTS>
struct XUnit {
    uint32_t u[PARTS == 4 ? 8 : 4];
};

// Values k0 .. k0 + 7 of a token, zeros past k.  WHOLE: without a branch around
// a load (k >= 8): a piece that reaches past k takes the row's last eight values,
// and x_shift moves its own to the front.
template <int PARTS, bool WHOLE>
__device__ __forceinline__ XUnit<PARTS> x_load(const G4Args& a, int token, int64_t k0) {
    constexpr int N = PARTS == 4 ? 8 : 4, SIZE = PARTS == 4 ? 4 : 2;
    typedef uint32_t v4 __attribute__((ext_vector_type(4), aligned(2)));
    XUnit<PARTS> r;
    if (WHOLE || k0 + 8 <= a.k) {
        const int64_t from = k0 + 8 <= a.k ? k0 : a.k - 8;
        const v4* p = reinterpret_cast<const v4*>(static_cast<const uint8_t*>(a.x) + (token * a.x_ld + from) * SIZE);
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const v4 v = p[i / 4];
#pragma unroll
            for (int j = 0; j < 4; j++) r.u[i + j] = v[j];
        }
    } else if constexpr (PARTS == 4) {
        const uint32_t* p = static_cast<const uint32_t*>(a.x) + token * a.x_ld + k0;
#pragma unroll
        for (int i = 0; i < 8; i++) r.u[i] = k0 + i < a.k ? p[i] : 0u;
    } else {
        const uint16_t* p = static_cast<const uint16_t*>(a.x) + token * a.x_ld + k0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t lo = k0 + 2 * i < a.k ? p[2 * i] : 0u, hi = k0 + 2 * i + 1 < a.k ? p[2 * i + 1] : 0u;
            r.u[i] = lo | hi << 16;
        }
    }
    return r;
}

template <int PARTS>
__device__ __forceinline__ void x_shift(XUnit<PARTS>& r, int by) {  // values `by`.. (0 to 8) to the front, zeros behind
    constexpr int N = PARTS == 4 ? 8 : 4;
    const int words = PARTS == 4 ? by : by >> 1;
#pragma unroll
    for (int b = N; b >= 1; b >>= 1) {
        if (!(words & b)) continue;
#pragma unroll
        for (int i = 0; i < N; i++) r.u[i] = i + b < N ? r.u[i + b] : 0u;
    }
    if (PARTS != 4 && (by & 1)) {
#pragma unroll
        for (int i = 0; i < N; i++) r.u[i] = r.u[i] >> 16 | (i + 1 < N ? r.u[i + 1] << 16 : 0u);
    }
}

template <int CTRL>
__device__ __forceinline__ int dpp_i(int v) {
    return __builtin_amdgcn_update_dpp(0, v, CTRL, 0xF, 0xF, false);
}

// x of a chunk as a workgroup reads it.
//   digits  [step][half][c][col] of 16 bytes: the B operand's bytes of k = 64 half + 8 c + 0..7 and + 32
//   power   [step][token] the block's power of two (with the weights' 1/16 and the top digit's 256^(PARTS-1))
//   sums    [step][group][col] -16 sum X
// As fp16 operands
//   digits  [step][t][c][token, of an odd number] of 16 bytes: the values of k = 32 t + 8 c + 0, 4, 1, 5, 2, 6, 3, 7
//           (an odd number: neighbouring lanes store neighbouring k, and meet different banks)
//   power   [step][token] the block's power of two
struct XImage {
    uint8_t* digits;
    float* power;
    int* sums;
};

// Bytes of a block's 256 k: digits, power and sums.
__host__ __device__ constexpr int64_t digit_bytes(int64_t parts, int64_t m) { return parts == 1 ? 512 * (m | 1) : 256 * parts * m; }
__host__ __device__ constexpr int64_t table_bytes(int64_t parts, int64_t m, int64_t per, bool zeros) {
    return 8 * m + (zeros && parts > 1 ? 8 * per * parts * m : 0);
}

// Bytes of a chunk in LDS and in the image.
__host__ __device__ constexpr int64_t chunk_bytes(int64_t blocks, int64_t parts, int64_t m, int64_t per, bool zeros) {
    return (blocks * (digit_bytes(parts, m) + table_bytes(parts, m, per, zeros)) + 15) / 16 * 16;
}

__device__ __forceinline__ XImage x_image(uint8_t* at, int blocks, int parts, int m) {
    XImage x;
    x.digits = at;
    x.power = reinterpret_cast<float*>(at + digit_bytes(parts, m) * blocks);
    x.sums = reinterpret_cast<int*>(x.power + 2 * blocks * m);
    return x;
}

// One piece (eight values; piece kc of the chunk, 16 to a block in 16 neighbouring lanes) of a token.
template <int PARTS, int PER, bool ZEROS>
__device__ __forceinline__ void x_store(const XUnit<PARTS>& r, const XImage& x, int type, int m, int token, int kc) {
    if constexpr (PARTS == 1) {
        u32x4 h;  // values i and i + 4 side by side, as their codes come out of the weights
#pragma unroll
        for (int i = 0; i < 4; i++) h[i] = __builtin_amdgcn_perm(r.u[2 + i / 2], r.u[i / 2], i & 1 ? 0x07060302u : 0x05040100u);
        float power = 1.f;
        if (type == ELEM_BF16) {
            typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
            u16x2 most = {0, 0};
#pragma unroll
            for (int i = 0; i < 4; i++) most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2, h[i] & 0x7fff7fffu));
            int big = max(most[0], most[1]);
            big = max(big, dpp_i<0xB1>(big));
            big = max(big, dpp_i<0x4E>(big));
            big = max(big, dpp_i<0x141>(big));
            big = max(big, dpp_i<0x140>(big));
            const int e = max(big >> 7, 1) - 127;  // |v| < 2^(e + 1)
            power = big >= 0x7f80 ? NAN : __builtin_ldexpf(1.f, e - 14);
#pragma unroll
            for (int i = 0; i < 4; i++)
                h[i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(__builtin_ldexpf(__uint_as_float(h[i] << 16), 14 - e),
                                                                               __builtin_ldexpf(__uint_as_float(h[i] & 0xffff0000u), 14 - e)));
        }
        *reinterpret_cast<u32x4*>(x.digits + (kc * (m | 1) + token) * 16) = h;
        if ((kc & 15) == 0) x.power[(kc >> 4) * m + token] = power;
        return;
    }
    const int cols = PARTS * m;
    float v[8];
    if constexpr (PARTS == 4) {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = __uint_as_float(r.u[i]);
    } else if (type == ELEM_F16) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            v[2 * i] = f16lo(r.u[i]);
            v[2 * i + 1] = f16hi(r.u[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            v[2 * i] = __uint_as_float(r.u[i] << 16);
            v[2 * i + 1] = __uint_as_float(r.u[i] & 0xffff0000u);
        }
    }
    // the block's largest magnitude, as bits: NaN and infinity are the largest
    int big = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) big = max(big, static_cast<int>(__float_as_uint(v[i]) & 0x7fffffffu));
    big = max(big, dpp_i<0xB1>(big));
    big = max(big, dpp_i<0x4E>(big));
    big = max(big, dpp_i<0x141>(big));
    big = max(big, dpp_i<0x140>(big));
    const int e = max(big >> 23, 1) - 127;  // |v| < 2^(e + 1)
    constexpr int BITS = PARTS == 4 ? 29 : 21;
    constexpr uint32_t BIAS = PARTS == 4 ? 0x80808080u : 0x00808080u;
    // byte h of X + BIAS is digit h, offset by 128
    uint32_t d[8];
#pragma unroll
    for (int i = 0; i < 8; i++)
        d[i] = (static_cast<uint32_t>(static_cast<int>(__builtin_rintf(__builtin_ldexpf(v[i], BITS - e)))) + BIAS) ^ BIAS;
    uint32_t* at = reinterpret_cast<uint32_t*>(x.digits) +
                   (static_cast<int64_t>((kc >> 4) * 8 + ((kc >> 3) & 1) * 4 + (kc & 3)) * cols + PARTS * token) * 4 + ((kc >> 2) & 1) * 2;
    // bytes h of four values: pairs by v_perm, then pairs of pairs
    const auto gather = [](uint32_t a, uint32_t b, uint32_t c, uint32_t f, uint32_t* out) {
        const uint32_t ab01 = __builtin_amdgcn_perm(b, a, 0x05010400u), ab23 = __builtin_amdgcn_perm(b, a, 0x07030602u);
        const uint32_t cf01 = __builtin_amdgcn_perm(f, c, 0x05010400u), cf23 = __builtin_amdgcn_perm(f, c, 0x07030602u);
        out[0] = __builtin_amdgcn_perm(cf01, ab01, 0x05040100u);
        out[1] = __builtin_amdgcn_perm(cf01, ab01, 0x07060302u);
        out[2] = __builtin_amdgcn_perm(cf23, ab23, 0x05040100u);
        out[3] = __builtin_amdgcn_perm(cf23, ab23, 0x07060302u);
    };
    uint32_t even[4], odd[4];  // the codes of even and odd k come out of the weights apart
    gather(d[0], d[2], d[4], d[6], even);
    gather(d[1], d[3], d[5], d[7], odd);
#pragma unroll
    for (int h = 0; h < PARTS; h++) {
        *reinterpret_cast<u32x2*>(at + 4 * h) = u32x2{even[h], odd[h]};
        if constexpr (ZEROS) {
            int s = sdot4(even[h], 0x01010101u, sdot4(odd[h], 0x01010101u, 0));
            s += dpp_i<0xB1>(s);
            s += dpp_i<0x4E>(s);
            if (PER <= 2) s += dpp_i<0x141>(s);
            if (PER == 1) s += dpp_i<0x140>(s);
            if ((kc & (16 / PER - 1)) == 0) x.sums[((kc >> 4) * PER + (kc & 15) * PER / 16) * cols + PARTS * token + h] = -16 * s;
        }
    }
    if ((kc & 15) == 0)
        x.power[(kc >> 4) * m + token] = big >= 0x7f800000 ? NAN : __builtin_ldexpf(1.f, e - BITS - 4 + 8 * (PARTS - 1));
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

// What a wave loads of one block.
template <int PER, bool ZEROS>
struct WBlock {
    u32x4 q[2];
    half8_t s[PER];  // group g's four at 4 (g & 1) of s[g >> 1]
    uint32_t z[PER];  // group g's four at bit 16 (g & 1) of z[g >> 1]
};

// x of a launch as digits into the workspace, one thread per piece.
template <int PER, bool ZEROS, int PARTS>
__global__ void __launch_bounds__(256) g4_image_kernel(G4Args a) {
    const int t = static_cast<int>(blockIdx.y);
    const int64_t at = first_item();
    if (at >= a.l.blocks * 32) return;
    const int64_t z = at / (a.chunk * 32);
    const int64_t left = a.l.blocks - z * a.chunk;
    const int blocks = static_cast<int>(left < a.chunk ? left : a.chunk);
    const XImage x = x_image(a.image + z * chunk_bytes(a.chunk, PARTS, a.m, PER, ZEROS), blocks, PARTS, a.m);
    x_store<PARTS, PER, ZEROS>(x_load<PARTS, false>(a, t, at * 8), x, a.x_type, a.m, t,
                               static_cast<int>(at - z * a.chunk * 32));
}

// Where a workgroup has its activations from: its own arithmetic, or the image.
enum { G4_SELF, G4_COPY };

constexpr int G4_DEPTH = 2;  // blocks in flight per wave

// Kernels that take the registers of 8 waves a CU, not 16.
__host__ __device__ constexpr bool g4_wide(int parts, int nt, int per, bool zeros) {
    return nt > 1 || (per == 4 && (zeros || parts == 1));
}

// PARTS 0: a.parts (no code but the staging depends on it).
template <int PER, bool ZEROS, int PARTS, int NT, int MODE>
__global__ void __launch_bounds__(64 * G4_WAVES, g4_wide(PARTS, NT, PER, ZEROS) ? 2 : 4) g4_gemv_kernel(G4Args a) {
    constexpr int DEPTH = NT == 3 && PER == 4 && ZEROS ? 1 : G4_DEPTH;  // (two do not fit the registers)
    extern __shared__ uint4 lds[];
    const int tid = static_cast<int>(threadIdx.x), lane = tid & 63, n = lane & 15, c = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int waves = static_cast<int>(blockDim.x) >> 6, threads = static_cast<int>(blockDim.x);
    const int parts = PARTS ? PARTS : a.parts, m = a.m, cols = parts * m;
    const int ks = a.ks, sub = wave % ks, local = wave / ks, per_group = waves / ks;
    const int kz = a.kz, z = static_cast<int>(blockIdx.x);
    const int turn = static_cast<int>(blockIdx.y), turns = static_cast<int>(gridDim.y);
    const int64_t row_blocks = a.l.blocks, first = static_cast<int64_t>(z) * a.chunk;
    const int tiles = static_cast<int>(a.l.tiles);
    const int blocks = static_cast<int>(row_blocks - first < a.chunk ? row_blocks - first : a.chunk);
    float4_t* red = reinterpret_cast<float4_t*>(lds);  // [wave][nt][lane]
    uint8_t* const mine = reinterpret_cast<uint8_t*>(lds + waves * NT * 64);
    const XImage x = x_image(mine, blocks, parts, m);

    int col[NT], token[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) {
        col[t] = t * 16 + n < cols ? t * 16 + n : cols - 1;
        token[t] = col[t] / parts;
    }

    // Loads of the ring: a block or tile past the last is outside of its
    // buffer and reads nothing.  (A branch around a load would make the
    // compiler wait for all loads in flight.)
    const uint32_t bytes = static_cast<uint32_t>(a.l.bytes), vo = static_cast<uint32_t>(lane) * 16;
    auto load = [&](int tile, int block, WBlock<PER, ZEROS>& r) __attribute__((always_inline)) {
        const bool in = tile < tiles;
        const __amdgpu_buffer_rsrc_t w = make_rsrc(a.w + (in ? (static_cast<int64_t>(tile) * row_blocks + first) * bytes : 0),
                                                   in ? static_cast<uint32_t>(blocks) * bytes : 0u);
        const uint32_t at = static_cast<uint32_t>(block) * bytes;
        const auto ld = [&](uint32_t o) __attribute__((always_inline)) {
            return __builtin_amdgcn_raw_buffer_load_b128(w, static_cast<int>(at + o), 0, 2);
        };
        r.q[0] = ld(vo);
        r.q[1] = ld(1024 + vo);
#pragma unroll
        for (int g = 0; g < PER; g++) r.s[g] = __builtin_bit_cast(half8_t, ld(2048 + c * (16 * PER) + 16 * g));
        if constexpr (ZEROS) {
            const uint32_t zo = 2048 + 64 * PER + (PARTS == 1 ? n >> 2 : c) * (4 * PER);
            if constexpr (PER == 4) {
                const u32x4 v = ld(zo);
#pragma unroll
                for (int g = 0; g < 4; g++) r.z[g] = v[g];
            } else if constexpr (PER == 2) {
                const u32x2 v = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(w, static_cast<int>(at + zo), 0, 2));
                r.z[0] = v[0];
                r.z[1] = v[1];
            } else {
                r.z[0] = __builtin_amdgcn_raw_buffer_load_b32(w, static_cast<int>(at + zo), 0, 2);
            }
        }
        __builtin_amdgcn_sched_barrier(0);  // slot after slot, as they are waited for
    };
    float4_t acc[NT];
    // Half `from` of a block with fp16 operands.  A code q is made from the bits
    // of 1024 + q, or where it lies four bits higher of 1024 + 16 q, and its zero
    // point taken off, two at a time and exactly.
    auto multiply_half = [&](const WBlock<PER, ZEROS>& r, int from, int at) __attribute__((always_inline)) {
        const int step = 2 * at + from;
        const uint4* xs = reinterpret_cast<const uint4*>(x.digits) + (step * 16 + c) * (m | 1) + col[0];
        half8_t xv[4];
#pragma unroll
        for (int t = 0; t < 4; t++) xv[t] = __builtin_bit_cast(half8_t, xs[4 * t * (m | 1)]);
        const float f = x.power[step * m + token[0]];
        float4_t p[PER];
#pragma unroll
        for (int t = 0; t < 4; t++) {
            const int g = t * PER / 4, gb = from * PER + g;
            uint32_t low = 0xe408e408u, high = 0xd480d480u;  // -(1024 + z), -(64 + z)
            if constexpr (ZEROS) {
                const uint32_t zz = ((r.z[gb >> 1] >> ((gb & 1) * 16 + (n & 3) * 4)) & 15) * 0x10001u;
                low ^= zz;
                high ^= zz << 4;
            }
            half8_t wv;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint32_t word = r.q[from][t] >> (i & 2) * 4;
                const uint32_t bits = i & 1 ? (word & 0x00f000f0u) ^ 0x64806480u : (word & 0x000f000fu) ^ 0x64086408u;
                const half2_t v = __builtin_bit_cast(half2_t, bits);
                const half2_t w = i & 1 ? __builtin_elementwise_fma(v, half2_t{0x1p-4f16, 0x1p-4f16}, __builtin_bit_cast(half2_t, high))
                                        : v + __builtin_bit_cast(half2_t, low);
                wv[2 * i] = w[0];
                wv[2 * i + 1] = w[1];
            }
            const float4_t before = t * PER % 4 == 0 ? float4_t{0.f, 0.f, 0.f, 0.f} : p[g];
            p[g] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wv, xv[t], before, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            float sum = 0.f;
#pragma unroll
            for (int g = 0; g < PER; g++) {
                const int gb = from * PER + g;
                sum = __builtin_fmaf(static_cast<float>(r.s[gb >> 1][(gb & 1) * 4 + i]), p[g][i], sum);
            }
            acc[0][i] = __builtin_fmaf(f, sum, acc[0][i]);
        }
    };
    // H halves of a block from half `from` on.
    auto multiply = [&](auto halves, const WBlock<PER, ZEROS>& r, int from, int at) __attribute__((always_inline)) {
        constexpr int H = decltype(halves)::value;
        const int4_t zero = {0, 0, 0, 0};
        // With few columns all operands are requested first, then all products,
        // then the sums: a wave has little else to fill these latencies with.
        constexpr bool EARLY = NT == 1 || (NT == 2 && PER == 1);
        int4_t xe[H][2][EARLY ? NT : 1];
        float fe[H][EARLY ? NT : 1];
        int se[H][EARLY ? NT : 1][PER];
        const auto x_of = [&](int e, int h, int u) __attribute__((always_inline)) {
            return __builtin_bit_cast(int4_t, reinterpret_cast<const uint4*>(x.digits)[((2 * at + from + e) * 8 + 4 * h + c) * cols + col[u]]);
        };
        const auto f_of = [&](int e, int u) __attribute__((always_inline)) { return x.power[(2 * at + from + e) * m + token[u]]; };
        const auto s_of = [&](int e, int u, int g) __attribute__((always_inline)) {
            return ZEROS ? x.sums[((2 * at + from + e) * PER + g) * cols + col[u]] : 0;
        };
        if constexpr (EARLY) {
#pragma unroll
            for (int e = 0; e < H; e++)
#pragma unroll
                for (int u = 0; u < NT; u++) {
                    xe[e][0][u] = x_of(e, 0, u);
                    xe[e][1][u] = x_of(e, 1, u);
                    fe[e][u] = f_of(e, u);
#pragma unroll
                    for (int g = 0; g < PER; g++) se[e][u][g] = s_of(e, u, g);
                }
        }
        int4_t wv[H][2];
#pragma unroll
        for (int e = 0; e < H; e++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                constexpr uint32_t HIGH = 0xf0f0f0f0u;
                const uint32_t q0 = r.q[from + e][2 * h], q1 = r.q[from + e][2 * h + 1];
                wv[e][h] = int4_t{static_cast<int>(q0 << 4 & HIGH), static_cast<int>(q0 & HIGH),
                                  static_cast<int>(q1 << 4 & HIGH), static_cast<int>(q1 & HIGH)};
            }
#pragma unroll
        for (int u = 0; u < NT; u++) {
            int4_t p[H][PER];
#pragma unroll
            for (int e = 0; e < H; e++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const int4_t xv = EARLY ? xe[e][h][EARLY ? u : 0] : x_of(e, h, u);
                    if constexpr (PER == 4) {
                        const auto pair = [](int lo, int hi) {
                            return static_cast<long>(static_cast<uint64_t>(static_cast<uint32_t>(hi)) << 32 | static_cast<uint32_t>(lo));
                        };
#pragma unroll
                        for (int t = 0; t < 2; t++)
                            p[e][2 * h + t] = __builtin_amdgcn_mfma_i32_16x16x32_i8(pair(wv[e][h][2 * t], wv[e][h][2 * t + 1]),
                                                                                   pair(xv[2 * t], xv[2 * t + 1]), zero, 0, 0, 0);
                    } else {
                        int4_t& to = p[e][PER == 1 ? 0 : h];
                        to = __builtin_amdgcn_mfma_i32_16x16x64_i8(wv[e][h], xv, PER == 1 && h == 1 ? to : zero, 0, 0, 0);
                    }
                }
#pragma unroll
            for (int e = 0; e < H; e++) {
                const float f = EARLY ? fe[e][EARLY ? u : 0] : f_of(e, u);
                float sum[4];
#pragma unroll
                for (int g = 0; g < PER; g++) {
                    const int gb = (from + e) * PER + g;  // of the block
                    const int sx = EARLY ? se[e][EARLY ? u : 0][g] : s_of(e, u, g);
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        int q = p[e][g][i];
                        if (ZEROS) q += __mul24(static_cast<int>(__builtin_amdgcn_sbfe(r.z[gb >> 1], (gb & 1) * 16 + 4 * i, 4)), sx);
                        const float s = static_cast<float>(r.s[gb >> 1][(gb & 1) * 4 + i]);
                        sum[i] = g == 0 ? s * static_cast<float>(q) : __builtin_fmaf(s, static_cast<float>(q), sum[i]);
                    }
                }
                // (s p) f: f p by itself may leave fp32's range where W x does not
#pragma unroll
                for (int i = 0; i < 4; i++) acc[u][i] = __builtin_fmaf(f, sum[i], acc[u][i]);
            }
            if (PER == 4 && NT == 3) __builtin_amdgcn_sched_barrier(0);  // three at once do not fit the registers
        }
    };

    // The wave's blocks of a tile: sub, sub + ks, ..., in rounds of DEPTH; the
    // last round loads the next tile's first ones.
    const int rounds = (blocks + ks * DEPTH - 1) / (ks * DEPTH);
    const int hop = turns * per_group;
    int tile = turn * per_group + local;
    WBlock<PER, ZEROS> ring[DEPTH];
    const auto fill = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int d = 0; d < DEPTH; d++) load(tile, sub + d * ks, ring[d]);
    };
    // x first, as loads come back in order: what a thread cannot hold, then the
    // rest of it on the way together with the ring's first round.
    if constexpr (MODE == G4_SELF) {
        // Digits take long code, which a launch fetches anew: two at a time (one, two
        // and four: 4096 x 4096, one token 6.3, 5.9 and 6.1 us).
        constexpr int HELD = PARTS == 1 ? 8 : 2;
        XUnit<PARTS> held[HELD];
        const int pieces = blocks * 32, units = pieces * m;  // of a token, of all
        const int64_t k0 = first * GROUP4_K;
        const float share = 1.f / static_cast<float>(pieces);
        // u / pieces: u < 2^14, so half a piece is more than the rounding
        const auto token_of = [&](int u) __attribute__((always_inline)) {
            return m == 1 ? 0 : static_cast<int>((static_cast<float>(u) + 0.5f) * share);
        };
        const auto get = [&](int base) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < HELD; i++) {
                const int u = base + i * threads + tid, v = u < units ? u : units - 1, t = token_of(v);
                held[i] = x_load<PARTS, true>(a, t, k0 + static_cast<int64_t>(v - t * pieces) * 8);
            }
        };
        const auto put = [&](int base) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < HELD; i++) {
                const int u = base + i * threads + tid;
                if (u >= units) continue;
                const int t = token_of(u), kc = u - t * pieces;
                const int64_t at = k0 + kc * 8;
                if (at + 8 > a.k) x_shift<PARTS>(held[i], static_cast<int>(at >= a.k ? 8 : at + 8 - a.k));
                x_store<PARTS, PER, ZEROS>(held[i], x, a.x_type, m, t, kc);
            }
        };
        if (a.k >= 8) {
            int base = 0;
#pragma unroll 1
            for (; base + HELD * threads < units; base += HELD * threads) {
                get(base);
                put(base);
            }
            get(base);
            fill();
            put(base);
        } else {
            for (int u = tid; u < units; u += threads) {
                const int t = u / pieces, kc = u - t * pieces;
                x_store<PARTS, PER, ZEROS>(x_load<PARTS, false>(a, t, kc * 8), x, a.x_type, m, t, kc);
            }
            fill();
        }
    } else {
        constexpr int HELD = 8;
        const u32x4* from = reinterpret_cast<const u32x4*>(a.image + z * chunk_bytes(a.chunk, parts, m, PER, ZEROS));
        u32x4* to = reinterpret_cast<u32x4*>(mine);
        const int count = static_cast<int>(chunk_bytes(blocks, parts, m, PER, ZEROS) / 16);
        u32x4 held[HELD];
        const auto get = [&](int base) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < HELD; i++) {
                const int u = base + i * threads + tid;
                held[i] = from[u < count ? u : count - 1];
            }
        };
        const auto put = [&](int base) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < HELD; i++) {
                const int u = base + i * threads + tid;
                if (u < count) to[u] = held[i];
            }
        };
        int base = 0;
        for (; base + HELD * threads < count; base += HELD * threads) {
            get(base);
            put(base);
        }
        get(base);
        fill();
        put(base);
    }
    lds_barrier();
    for (int grp = turn; grp < a.groups; grp += turns, tile += hop) {
#pragma unroll
        for (int t = 0; t < NT; t++) acc[t] = float4_t{0.f, 0.f, 0.f, 0.f};
        for (int i = 0; i < rounds; i++) {
            const int s = i * ks * DEPTH + sub;
            const bool last = i + 1 == rounds;
            const int next = last ? tile + hop : tile, from = last ? sub : s + DEPTH * ks;
#pragma unroll
            for (int d = 0; d < DEPTH; d++) {
                if (tile < tiles && s + d * ks < blocks) {
                    if constexpr (PARTS == 1) {
                        multiply_half(ring[d], 0, s + d * ks);
                        multiply_half(ring[d], 1, s + d * ks);
                    } else if constexpr (NT == 1 && PER == 1) {
                        multiply(std::integral_constant<int, 2>{}, ring[d], 0, s + d * ks);
                    } else {
                        multiply(std::integral_constant<int, 1>{}, ring[d], 0, s + d * ks);
                        __builtin_amdgcn_sched_barrier(0);  // (both halves at once do not fit the registers)
                        multiply(std::integral_constant<int, 1>{}, ring[d], 1, s + d * ks);
                    }
                }
                load(next, from + d * ks, ring[d]);
            }
        }
        // y: a token's digits of a tile's waves, added in order.  A wave that has
        // a tile by itself reads what it wrote.
#pragma unroll
        for (int t = 0; t < NT; t++) red[(wave * NT + t) * 64 + lane] = acc[t];
        if (ks > 1) lds_barrier();
        const float* rf = reinterpret_cast<const float*>(red);
        const int outs = (ks > 1 ? per_group : 1) * 16 * m;
        for (int o = ks > 1 ? tid : lane; o < outs; o += ks > 1 ? threads : 64) {
            const int r = o & 15, tt = ks > 1 ? (o >> 4) % per_group : local, t = ks > 1 ? (o >> 4) / per_group : o >> 4;
            const int64_t row = (static_cast<int64_t>(grp) * per_group + tt) * 16 + r;
            float total = 0.f;
            for (int h = 0; h < parts; h++) {
                const int cc = parts * t + h;
                float sum = 0.f;
                for (int v = 0; v < ks; v++)
                    sum += rf[(((tt * ks + v) * NT + (cc >> 4)) * 64 + (r >> 2) * 16 + (cc & 15)) * 4 + (r & 3)];
                total = __builtin_fmaf(total, 0x1p-8f, sum);  // digit h is worth 256 times digit h - 1
            }
            float* y = kz > 1 ? a.partial + static_cast<int64_t>(z) * m * a.rows : a.y;
            if (row < a.rows) y[static_cast<int64_t>(t) * a.rows + row] = total;
        }
        if (ks > 1) lds_barrier();  // red is free
    }
}

// y = the chunks' sums, added in order.  (Joined by the last workgroup of a
// tile instead, the fences around its count write back and drop a die's whole
// L2 each time: 4096 x 14336, eight tokens, 37 us.)
__global__ void __launch_bounds__(256) g4_join_kernel(const float* partial, float* y, int64_t n, int kz) {
    for (int64_t i = first_item(); i < n; i += item_stride()) {
        float total = partial[i];
        for (int z = 1; z < kz; z++) total += partial[z * n + i];
        y[i] = total;
    }
}

constexpr int64_t G4_LDS = 160 << 10;  // of a CU
// Activations that every workgroup turns into digits itself; more are made once,
// by a launch of their own, and copied (itself and once: 4096 x 4096, one token
// 5.9 and 7.8 us, four 9.2 and 9.7; 4096 x 8192, three 10.8 and 10.7; 4096 x
// 14336, two 14.3 and 13.2).
constexpr int64_t G4_SELF_VALUES = 16384;
constexpr int G4_COLS = 48;  // columns of a launch, at most

// How a launch of m tokens runs.
struct G4Plan {
    int mode, parts, nt, ks, waves;
    int64_t kz, chunk, groups;
    int64_t lds;
    int64_t partial, workspace;  // byte offset of the chunks' sums behind the image, bytes in all
};

G4Plan g4_plan(const Group4Layout& l, int64_t rows, int64_t m, int x_type, bool has_zeros) {
    G4Plan p{};
    // Tokens of 16 bits as fp16 operands: from the sixth on, whose digits take a
    // second set of columns (six to sixteen tokens of 14336 x 4096: 20 us as
    // digits, 13.3 so); and fp16 tokens from the third where what a workgroup
    // stages counts for more than what it decodes, at up to four row tiles a CU
    // (digits and fp16: 14336 x 4096, two tokens 9.3 and 9.9 us, four 10.5 and
    // 10.1; 4096 x 4096, three 8.2 and 6.4; 4096 x 14336, five 15.2 and 13.7;
    // 128256 x 4096, five 56.8 and 62.8).  bf16 tokens take longer to stage
    // (three 10.0 and 10.7, five of 4096 x 14336 15.1 and 16.0).
    p.parts = x_type == ELEM_F32 ? 4 : m > 5 || (x_type == ELEM_F16 && m > 2 && l.tiles <= 4 * num_cus()) ? 1 : 3;
    p.nt = static_cast<int>((p.parts * m + 15) / 16);
    // Chunks of k whose digits fit into LDS beside the sums.
    const int64_t room = G4_LDS - G4_WAVES * p.nt * 1024 - 16, block = digit_bytes(p.parts, m) + table_bytes(p.parts, m, l.per, has_zeros);
    const int64_t fit = room / block;  // 146 blocks of one fp32 token, 10 of twelve
    p.kz = (l.blocks + fit - 1) / fit;
    // where there are several, as many as give every CU a workgroup (4096 x 14336, eight tokens as
    // digits: 3 chunks 21.3 us, 4 18.8)
    const int64_t even = (4 * num_cus() + l.tiles - 1) / l.tiles;
    // or all of them the same number (nine fp32 tokens, groups of 32: 5 chunks 53.7 us, 8 31.9)
    if (p.kz > 1) p.kz = even <= 8 ? (p.kz + even - 1) / even * even : p.kz < 8 ? 8 : p.kz;
    // and where the row tiles leave CUs without work, if there is enough of it to
    // pay for the launch that joins them (whole and split: 549 x 12800, one token
    // 12.3 us and 9.0; 1024 x 4096, four 9.0 and 7.6, but two 6.5 and 6.9)
    if (p.kz == 1 && m * l.blocks >= 48) {
        const int64_t idle = num_cus() / l.tiles, pairs = l.blocks / 2, most = idle < pairs ? idle : pairs;
        p.kz = most < 1 ? 1 : most < 8 ? most : 8;
    }
    if (p.kz > l.blocks) p.kz = l.blocks;
    p.chunk = (l.blocks + p.kz - 1) / p.kz;
    p.kz = (l.blocks + p.chunk - 1) / p.chunk;
    p.mode = p.parts == 1 || (p.nt == 1 && m * p.chunk * GROUP4_K <= G4_SELF_VALUES) ? G4_SELF : G4_COPY;
    // A tile is shared by as many waves as leave each four blocks, up to eight
    // waves a CU: more of them cost more in x staged and sums joined than they
    // bring in loads in flight (14336 x 4096, one token: ks 1 to 8 take 9.7,
    // 9.3, 10.5 and 14.0 us; 4096 x 4096: 9.2, 6.9, 6.1 and 6.6).
    p.ks = 1;
    while (p.ks < G4_WAVES && l.tiles * p.kz * p.ks * 2 <= 8 * num_cus() && p.chunk >= 8 * p.ks) p.ks *= 2;
    // workgroups of four waves where eight would leave a quarter of the CUs without one
    p.waves = p.ks <= 4 && l.tiles * p.kz * p.ks < 6 * num_cus() ? 4 : G4_WAVES;
    p.groups = (l.tiles * p.ks + p.waves - 1) / p.waves;
    p.lds = p.waves * p.nt * 1024 + chunk_bytes(p.chunk, p.parts, m, l.per, has_zeros);
    p.workspace = p.mode == G4_SELF ? 0 : p.kz * chunk_bytes(p.chunk, p.parts, m, l.per, has_zeros);
    if (p.kz > 1) {
        p.partial = p.workspace;
        p.workspace += (p.kz * m * rows * 4 + 15) / 16 * 16;
    }
    return p;
}

template <int PER, bool ZEROS>
int g4_launch(const G4Args& a, const G4Plan& p, dim3 grid, hipStream_t st) {
    const uint32_t threads = 64 * p.waves, lds = static_cast<uint32_t>(p.lds);
    if (p.mode == G4_SELF) {
        if (a.parts == 1) g4_gemv_kernel<PER, ZEROS, 1, 1, G4_SELF><<<grid, threads, lds, st>>>(a);
        else if (a.parts == 4) g4_gemv_kernel<PER, ZEROS, 4, 1, G4_SELF><<<grid, threads, lds, st>>>(a);
        else g4_gemv_kernel<PER, ZEROS, 3, 1, G4_SELF><<<grid, threads, lds, st>>>(a);
    } else {
        const dim3 pieces(static_cast<uint32_t>((a.l.blocks * 32 + 255) / 256), static_cast<uint32_t>(a.m));
        if (a.parts == 4) g4_image_kernel<PER, ZEROS, 4><<<pieces, 256, 0, st>>>(a);
        else g4_image_kernel<PER, ZEROS, 3><<<pieces, 256, 0, st>>>(a);
        if (const int rc = check_launch("vb_group4_gemv"); rc != OK) return rc;
        if (p.nt == 1) g4_gemv_kernel<PER, ZEROS, 0, 1, G4_COPY><<<grid, threads, lds, st>>>(a);
        else if (p.nt == 2) g4_gemv_kernel<PER, ZEROS, 0, 2, G4_COPY><<<grid, threads, lds, st>>>(a);
        else g4_gemv_kernel<PER, ZEROS, 0, 3, G4_COPY><<<grid, threads, lds, st>>>(a);
    }
    if (p.kz > 1) {
        if (const int rc = check_launch("vb_group4_gemv"); rc != OK) return rc;
        g4_join_kernel<<<item_blocks(a.rows * a.m), 256, 0, st>>>(a.partial, a.y, a.rows * a.m, a.kz);
    }
    return check_launch("vb_group4_gemv");
}

int g4_run(G4Args a, bool has_zeros, uint8_t* workspace, hipStream_t st) {
    const G4Plan p = g4_plan(a.l, a.rows, a.m, a.x_type, has_zeros);
    a.image = workspace;
    a.partial = reinterpret_cast<float*>(workspace + p.partial);
    a.parts = p.parts;
    a.ks = p.ks;
    a.kz = static_cast<int32_t>(p.kz);
    a.chunk = static_cast<int32_t>(p.chunk);
    a.groups = static_cast<int32_t>(p.groups);
    // as many workgroups as are resident at once (16 waves a CU or 8), a share for every chunk
    const int64_t fit = G4_LDS / p.lds, want = (g4_wide(p.parts, p.nt, a.l.per, has_zeros) ? 8 : 16) / p.waves;
    const int64_t most = ((fit < want ? fit : want) * num_cus() + p.kz - 1) / p.kz;
    const dim3 grid(static_cast<uint32_t>(p.kz), static_cast<uint32_t>(p.groups < most ? p.groups : most));
    if (a.l.per == 1) return has_zeros ? g4_launch<1, true>(a, p, grid, st) : g4_launch<1, false>(a, p, grid, st);
    if (a.l.per == 2) return has_zeros ? g4_launch<2, true>(a, p, grid, st) : g4_launch<2, false>(a, p, grid, st);
    return has_zeros ? g4_launch<4, true>(a, p, grid, st) : g4_launch<4, false>(a, p, grid, st);
}

// Tokens of a launch of m, in even shares.
int64_t g4_slab(int64_t m, int x_type) {
    const int64_t slab = G4_COLS / (x_type == ELEM_F32 ? 4 : 3), launches = (m + slab - 1) / slab;
    return (m + launches - 1) / launches;
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
    g4_pack_codes_kernel<<<item_blocks(l.tiles * l.blocks * 512), 256, 0, st>>>(packed, static_cast<uint8_t*>(w), l,
                                                                                  rows, k);
    if (const int rc = check_launch("vb_group4_pack"); rc != OK) return rc;
    g4_pack_groups_kernel<<<item_blocks(l.tiles * l.blocks), 256, 0, st>>>(
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

int64_t vb_group4_workspace(int64_t m, int64_t rows, int64_t k, int32_t group, int32_t has_zeros, int32_t x_type) {
    Group4Layout l;
    if (m < 0 || !elem_type(x_type) || !group4_layout(rows, k, group, has_zeros != 0, &l)) return -1;
    if (m == 0) return 0;
    const int64_t slab = g4_slab(m, x_type), rest = m % slab;  // the last launch may be smaller
    const int64_t need = g4_plan(l, rows, slab, x_type, has_zeros != 0).workspace;
    const int64_t last = rest > 0 ? g4_plan(l, rows, rest, x_type, has_zeros != 0).workspace : 0;
    return last > need ? last : need;
}

int vb_group4_gemv(const void* w, int64_t rows, int64_t k, int32_t group, int32_t has_zeros, const void* x,
                   int32_t x_type, int64_t x_ld, int64_t m, float* y, void* workspace, size_t workspace_bytes,
                   void* stream) {
    Group4Layout l;
    if (const int rc = layout_of("vb_group4_gemv", rows, k, group, has_zeros, &l); rc != OK) return rc;
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
    const int64_t need = vb_group4_workspace(m, rows, k, group, has_zeros, x_type);
    if (static_cast<int64_t>(workspace_bytes) < need ||
        (need > 0 && (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16 != 0))) {
        set_error("vb_group4_gemv: workspace of %zu bytes (16-byte aligned) is below the %lld needed", workspace_bytes,
                  static_cast<long long>(need));
        return E_INVAL;
    }
    const int64_t slab = g4_slab(m, x_type);
    for (int64_t t = 0; t < m; t += slab) {
        G4Args a{};
        a.w = static_cast<const uint8_t*>(w);
        a.l = l;
        a.x = static_cast<const uint8_t*>(x) + t * x_ld * elem_bytes(x_type);
        a.y = y + t * rows;
        a.x_ld = x_ld;
        a.rows = rows;
        a.k = k;
        a.x_type = x_type;
        a.m = static_cast<int32_t>(m - t < slab ? m - t : slab);
        if (const int rc = g4_run(a, has_zeros != 0, static_cast<uint8_t*>(workspace), as_stream(stream)); rc != OK) return rc;
    }
    return OK;
}

}  // extern "C"
