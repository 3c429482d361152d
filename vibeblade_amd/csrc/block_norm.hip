// The seam between two blocks of a decoder, one pass over its rows:
//
//   p = b / sqrt(mean(b^2) + eps) * post_w   (p = b without post_w)
//   y = x + scale * gate * p                 (the residual stream)
//   n = y / sqrt(mean(y^2) + eps) * pre_w    (the next block's input)
//
// b is a block's output, x the stream before it.  Sums, the scale factors and
// y as n is computed from it are fp32 whatever the tensors' types; y and n are
// rounded once, to the nearest, as they are stored.
//
// A workgroup takes a row, and a thread its share of it into registers, in
// pieces of four values: the branch, the stream and the gate are requested
// together, the two sums go over the workgroup, and every value is read and
// written once.  Rows longer than the registers of a workgroup are read again
// for each sum (seam_long_kernel).
//
// Memory bounds it: fp32 rows run at 6.0 to 6.5 TB/s of what is read and written
// (4096 x 8192 86 us, 8192 x 4096 with fp16 n 73), 16-bit ones at 5.2 to 5.8
// (8192 x 4096 46 us), rows of odd length at 4.9 (7001 x 5121, a full gate: 103
// us; 7001 x 5120 82).  One row of 4096 takes 3.4 us in a graph, of which a
// launch is 1.9.
#include "elem_types.hpp"
#include "vb_internal.hpp"
#include "../../include/vbhip.h"

namespace vb {
namespace {

struct SeamArgs {
    const void* b;
    const void* x;
    void* y;
    void* n;
    const float* post_w;
    const float* pre_w;
    const void* gate;
    int64_t b_ld, x_ld, y_ld, n_ld, gate_row, gate_col;
    int64_t rows, dim;
    int32_t b_type, x_type, n_type, gate_type;
    float scale, eps;
};

// Where element i of a tensor is.
__device__ __forceinline__ uint8_t* elem_at(const void* p, int64_t i, int type) {
    return static_cast<uint8_t*>(const_cast<void*>(p)) + i * (type == ELEM_F32 ? 4 : 2);
}

// ---- four neighbouring values; rows begin at any element ---------------------
// (a row is the same in all of a wave: one address and an offset of 32 bits a lane)

template <int TYPE>
struct Piece {
    uint32_t u[TYPE == ELEM_F32 ? 4 : 2];
};

// ONCE: past the caches' usual order, as this launch is the last to read it
// (8192 x 4096 fp32: 84 to 78 us, 4096 x 8192: 106 to 88).
template <int TYPE, bool ONCE = false>
__device__ __forceinline__ Piece<TYPE> piece_ld(const void* p, uint32_t i) {
    Piece<TYPE> r;
    if constexpr (TYPE == ELEM_F32) {
        typedef uint32_t v4 __attribute__((ext_vector_type(4), aligned(4)));
        const v4* q = reinterpret_cast<const v4*>(static_cast<const uint8_t*>(p) + i * 4);
        const v4 v = ONCE ? __builtin_nontemporal_load(q) : *q;
#pragma unroll
        for (int j = 0; j < 4; j++) r.u[j] = v[j];
    } else {
        typedef uint32_t v2 __attribute__((ext_vector_type(2), aligned(2)));
        const v2* q = reinterpret_cast<const v2*>(static_cast<const uint8_t*>(p) + i * 2);
        const v2 v = ONCE ? __builtin_nontemporal_load(q) : *q;
        r.u[0] = v[0];
        r.u[1] = v[1];
    }
    return r;
}

template <int TYPE>
__device__ __forceinline__ float piece_at(const Piece<TYPE>& r, int j) {
    if constexpr (TYPE == ELEM_F32) return __uint_as_float(r.u[j]);
    else if constexpr (TYPE == ELEM_F16) return j & 1 ? f16hi(r.u[j >> 1]) : f16lo(r.u[j >> 1]);
    else return __uint_as_float(j & 1 ? r.u[j >> 1] & 0xffff0000u : r.u[j >> 1] << 16);
}

template <int TYPE>
__device__ __forceinline__ void piece_st(void* p, uint32_t i, const float* v) {
    if constexpr (TYPE == ELEM_F32) {
        typedef float v4 __attribute__((ext_vector_type(4), aligned(4)));
        *reinterpret_cast<v4*>(static_cast<uint8_t*>(p) + i * 4) = v4{v[0], v[1], v[2], v[3]};
    } else {
        typedef uint32_t v2 __attribute__((ext_vector_type(2), aligned(2)));
        uint32_t u[2];
#pragma unroll
        for (int j = 0; j < 2; j++) {
            if constexpr (TYPE == ELEM_F16) {
                typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
                u[j] = __builtin_bit_cast(uint32_t, half2_t{static_cast<_Float16>(v[2 * j]), static_cast<_Float16>(v[2 * j + 1])});
            } else {
                u[j] = f32_bf16x2(v[2 * j], v[2 * j + 1]);
            }
        }
        *reinterpret_cast<v2*>(static_cast<uint8_t*>(p) + i * 2) = v2{u[0], u[1]};
    }
}

// The workgroup's sum of v, in every thread (waves added in order); part: of this sum alone.
template <int WAVES>
__device__ __forceinline__ float wg_sum(float v, float* part) {
    v = wave_sum_dpp(v);
    if constexpr (WAVES == 1) return v;
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = part[0];
#pragma unroll
    for (int i = 1; i < WAVES; i++) s += part[i];
    return s;
}

// Four neighbouring values of the gate as they lie (gate_col 1), or its one value of the row.
__device__ __forceinline__ Piece<ELEM_F32> gate_ld(const SeamArgs& a, const void* gate, uint32_t at) {
    Piece<ELEM_F32> g;
    if (a.gate_col == 0) {
        g.u[0] = __float_as_uint(elem_ld(gate, 0, a.gate_type));
    } else if (a.gate_type == ELEM_F32) {
        g = piece_ld<ELEM_F32, true>(gate, at);
    } else {
        const Piece<ELEM_F16> h = piece_ld<ELEM_F16, true>(gate, at);
        g.u[0] = h.u[0];
        g.u[1] = h.u[1];
    }
    return g;
}

__device__ __forceinline__ float gate_at(const SeamArgs& a, const Piece<ELEM_F32>& g, int j) {
    if (a.gate_col == 0) return __uint_as_float(g.u[0]);
    if (a.gate_type == ELEM_F32) return __uint_as_float(g.u[j]);
    const uint32_t w = g.u[j >> 1];
    if (a.gate_type == ELEM_F16) return j & 1 ? f16hi(w) : f16lo(w);
    return __uint_as_float(j & 1 ? w & 0xffff0000u : w << 16);
}

// Values skip.. of a piece (all of it as one store).
template <int TYPE>
__device__ __forceinline__ void piece_put(void* p, uint32_t i, const float* v, int skip) {
    if (skip == 0) {
        piece_st<TYPE>(p, i, v);
    } else {
#pragma unroll
        for (int j = 1; j < 4; j++)
            if (j >= skip) elem_st(p, i + j, TYPE, v[j]);
    }
}

// Rows of at least 4 and over 256 * WAVES * (PIECES - 1) values, up to 256 *
// WAVES * PIECES: all but a thread's last piece are whole.  The row's last
// piece is moved back to end with it; its first values are another thread's,
// and are neither summed nor stored again.
template <int BT, int XT, int WAVES, int PIECES>
__global__ void __launch_bounds__(64 * WAVES) seam_kernel(SeamArgs a) {
    // the weights come with the rest (8192 x 4096 fp32 78 us and 73, 7001 x 5120 91 and 81), where that leaves
    // the registers for as many workgroups (eight waves, three pieces: 101 us and 106)
    constexpr bool EARLY = WAVES <= 4 || (WAVES == 8 && PIECES <= 2);
    __shared__ float part[2][WAVES];
    const int dim = static_cast<int>(a.dim);
    const int begin = static_cast<int>(threadIdx.x) * 4, last = begin + (PIECES - 1) * 256 * WAVES;
    // how many values of a piece are not its own (4: there is no piece)
    const int last_skip = last >= dim ? 4 : last + 4 <= dim ? 0 : last + 4 - dim;
    const auto skip = [&](int k) { return k < PIECES - 1 ? 0 : last_skip; };
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const uint8_t* rb = elem_at(a.b, row * a.b_ld, BT);
        const uint8_t* rx = elem_at(a.x, row * a.x_ld, XT);
        const uint8_t* rg = elem_at(a.gate, row * a.gate_row, a.gate_type);
        uint8_t* ry = elem_at(a.y, row * a.y_ld, XT);
        uint8_t* rn = elem_at(a.n, row * a.n_ld, a.n_type);
        // a piece's first value (made anew in each turn: an address a piece would take the registers of half a row)
        uint32_t start = begin, end = last + 4 <= dim ? last : dim - 4;
        asm volatile("" : "+v"(start), "+v"(end));
        const auto at = [&](int k) { return k < PIECES - 1 ? start + k * 256 * WAVES : end; };
        Piece<ELEM_F32> g[PIECES];
        Piece<BT> b[PIECES];
        Piece<XT> x[PIECES];
        if (a.gate) {
#pragma unroll
            for (int k = 0; k < PIECES; k++) g[k] = gate_ld(a, rg, at(k));
        }
#pragma unroll
        for (int k = 0; k < PIECES; k++) b[k] = piece_ld<BT, true>(rb, at(k));
#pragma unroll
        for (int k = 0; k < PIECES; k++) x[k] = piece_ld<XT, true>(rx, at(k));
        Piece<ELEM_F32> post[EARLY ? PIECES : 1], pre[EARLY ? PIECES : 1];
        if constexpr (EARLY) {
#pragma unroll
            for (int k = 0; k < PIECES; k++) {
                if (a.post_w) post[k] = piece_ld<ELEM_F32>(a.post_w, at(k));
                if (a.pre_w) pre[k] = piece_ld<ELEM_F32>(a.pre_w, at(k));
            }
        }
        float inv = a.scale;
        if (a.post_w) {
            float s = 0.f;
#pragma unroll
            for (int k = 0; k < PIECES; k++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float v = piece_at<BT>(b[k], j);
                    s += j >= skip(k) ? v * v : 0.f;
                }
            inv = 1.f / sqrtf(wg_sum<WAVES>(s, part[0]) / static_cast<float>(dim) + a.eps);
        }
        float y[PIECES][4];
        float s = 0.f;
#pragma unroll
        for (int k = 0; k < PIECES; k++) {
            float p[4];
#pragma unroll
            for (int j = 0; j < 4; j++) p[j] = piece_at<BT>(b[k], j) * inv;
            if (a.post_w) {
                const Piece<ELEM_F32> w = EARLY ? post[EARLY ? k : 0] : piece_ld<ELEM_F32>(a.post_w, at(k));
#pragma unroll
                for (int j = 0; j < 4; j++) p[j] *= piece_at<ELEM_F32>(w, j) * a.scale;
            }
            if (a.gate) {
#pragma unroll
                for (int j = 0; j < 4; j++) p[j] *= gate_at(a, g[k], j);
            }
#pragma unroll
            for (int j = 0; j < 4; j++) {
                y[k][j] = piece_at<XT>(x[k], j) + p[j];
                s += j >= skip(k) ? y[k][j] * y[k][j] : 0.f;
            }
        }
        // (y may be x: all of the row is read before the barrier, and stored behind it)
        if (a.pre_w) s = wg_sum<WAVES>(s, part[1]);
        else __syncthreads();
        const float inv2 = 1.f / sqrtf(s / static_cast<float>(dim) + a.eps);
#pragma unroll
        for (int k = 0; k < PIECES; k++) {
            if (skip(k) == 4) continue;
            piece_put<XT>(ry, at(k), y[k], skip(k));
            if (a.pre_w) {
                const Piece<ELEM_F32> w = EARLY ? pre[EARLY ? k : 0] : piece_ld<ELEM_F32>(a.pre_w, at(k));
                float n[4];
#pragma unroll
                for (int j = 0; j < 4; j++) n[j] = y[k][j] * inv2 * piece_at<ELEM_F32>(w, j);
                if (a.n_type == ELEM_F32) piece_put<ELEM_F32>(rn, at(k), n, skip(k));
                else if (a.n_type == ELEM_F16) piece_put<ELEM_F16>(rn, at(k), n, skip(k));
                else piece_put<ELEM_BF16>(rn, at(k), n, skip(k));
            }
        }
        if (WAVES > 1) __syncthreads();  // the sums are read
    }
}

constexpr int LONG_WAVES = 16;

// Rows of any length: read again for every sum.
__global__ void __launch_bounds__(64 * LONG_WAVES) seam_long_kernel(SeamArgs a) {
    __shared__ float part[2][LONG_WAVES];
    constexpr int STEP = 64 * LONG_WAVES;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const int64_t bo = row * a.b_ld, xo = row * a.x_ld, yo = row * a.y_ld, no = row * a.n_ld, go = row * a.gate_row;
        float inv = 1.f;
        if (a.post_w) {
            float s = 0.f;
            for (int64_t i = threadIdx.x; i < a.dim; i += STEP) {
                const float v = elem_ld(a.b, bo + i, a.b_type);
                s += v * v;
            }
            inv = 1.f / sqrtf(wg_sum<LONG_WAVES>(s, part[0]) / static_cast<float>(a.dim) + a.eps);
        }
        auto value = [&](int64_t i) {
            float p = elem_ld(a.b, bo + i, a.b_type) * inv;
            if (a.post_w) p *= a.post_w[i];
            p *= a.scale;
            if (a.gate) p *= elem_ld(a.gate, go + i * a.gate_col, a.gate_type);
            return elem_ld(a.x, xo + i, a.x_type) + p;
        };
        float inv2 = 1.f;
        if (a.pre_w) {
            float s = 0.f;
            for (int64_t i = threadIdx.x; i < a.dim; i += STEP) {
                const float v = value(i);
                s += v * v;
            }
            inv2 = 1.f / sqrtf(wg_sum<LONG_WAVES>(s, part[1]) / static_cast<float>(a.dim) + a.eps);
        }
        for (int64_t i = threadIdx.x; i < a.dim; i += STEP) {
            const float v = value(i);
            elem_st(a.y, yo + i, a.x_type, v);
            if (a.pre_w) elem_st(a.n, no + i, a.n_type, v * inv2 * a.pre_w[i]);
        }
        __syncthreads();  // the sums are read
    }
}

template <int BT, int XT>
void seam_launch(const SeamArgs& a, hipStream_t st) {
    const uint32_t grid = static_cast<uint32_t>(a.rows < (1 << 20) ? a.rows : 1 << 20);  // fewer than 2^32 threads
    // Few rows (a CU or less for each) are on their way soonest with sixteen
    // waves and short shares.  With many, bytes in flight count: as few waves as
    // hold a row in up to seven pieces a thread, and lengths that leave few
    // threads idle (bf16, eight waves and two pieces against the many's: 8192 x
    // 2560 49 us and 35, 16384 x 2048 73 and 51, 65536 x 512 113 and 44, 8192 x
    // 4096 55 and 46; six pieces half of whose last is there, 7001 x 6144: 66 and
    // 60, seven, 5000 x 7168: 59 and 52, but 7001 x 5121 101 and 105).  Between
    // them eight waves (512 x 4096 6.7 us, four 7.3; 1024 rows 10.9 and 9.8).
    // Over 7168 eight waves again (4096 x 8192 fp32: 86 us, four 89), and sixteen
    // where eight no longer fit twice (2048 x 16384: eight 97 us, sixteen 86).
    const bool few = a.rows <= num_cus(), many = a.rows > 2 * num_cus();
    const int64_t d = a.dim;
    const auto within = [d](int64_t waves, int64_t pieces) { return d <= 256 * waves * pieces; };
    if (d < 4 || !within(16, 4)) seam_long_kernel<<<grid, 64 * LONG_WAVES, 0, st>>>(a);
    else if (within(1, 1)) seam_kernel<BT, XT, 1, 1><<<grid, 64, 0, st>>>(a);
    else if (many && within(1, 2)) seam_kernel<BT, XT, 1, 2><<<grid, 64, 0, st>>>(a);
    else if (many && within(1, 3)) seam_kernel<BT, XT, 1, 3><<<grid, 64, 0, st>>>(a);
    else if (many && within(2, 2)) seam_kernel<BT, XT, 2, 2><<<grid, 128, 0, st>>>(a);
    else if (many && within(2, 3)) seam_kernel<BT, XT, 2, 3><<<grid, 128, 0, st>>>(a);
    else if (many && within(4, 2)) seam_kernel<BT, XT, 4, 2><<<grid, 256, 0, st>>>(a);
    else if (many && within(2, 5)) seam_kernel<BT, XT, 2, 5><<<grid, 128, 0, st>>>(a);
    else if (many && within(4, 3)) seam_kernel<BT, XT, 4, 3><<<grid, 256, 0, st>>>(a);
    else if (many && within(4, 4)) seam_kernel<BT, XT, 4, 4><<<grid, 256, 0, st>>>(a);
    else if (many && within(4, 5)) seam_kernel<BT, XT, 4, 5><<<grid, 256, 0, st>>>(a);
    else if (many && d > 5632 && within(4, 6)) seam_kernel<BT, XT, 4, 6><<<grid, 256, 0, st>>>(a);
    else if (many && d > 6656 && within(4, 7)) seam_kernel<BT, XT, 4, 7><<<grid, 256, 0, st>>>(a);
    else if (within(4, 1)) seam_kernel<BT, XT, 4, 1><<<grid, 256, 0, st>>>(a);
    else if (few && within(16, 1)) seam_kernel<BT, XT, 16, 1><<<grid, 1024, 0, st>>>(a);
    else if (few && within(16, 2)) seam_kernel<BT, XT, 16, 2><<<grid, 1024, 0, st>>>(a);
    else if (few && within(16, 3)) seam_kernel<BT, XT, 16, 3><<<grid, 1024, 0, st>>>(a);
    else if (within(8, 1)) seam_kernel<BT, XT, 8, 1><<<grid, 512, 0, st>>>(a);
    else if (within(8, 2)) seam_kernel<BT, XT, 8, 2><<<grid, 512, 0, st>>>(a);
    else if (within(8, 3)) seam_kernel<BT, XT, 8, 3><<<grid, 512, 0, st>>>(a);
    else if (within(8, 4)) seam_kernel<BT, XT, 8, 4><<<grid, 512, 0, st>>>(a);
    else if (within(8, 5)) seam_kernel<BT, XT, 8, 5><<<grid, 512, 0, st>>>(a);
    else if (within(8, 6)) seam_kernel<BT, XT, 8, 6><<<grid, 512, 0, st>>>(a);
    else if (!few && within(8, 7)) seam_kernel<BT, XT, 8, 7><<<grid, 512, 0, st>>>(a);
    else seam_kernel<BT, XT, 16, 4><<<grid, 1024, 0, st>>>(a);
}

template <int BT>
void seam_launch_x(const SeamArgs& a, hipStream_t st) {
    if (a.x_type == ELEM_F32) seam_launch<BT, ELEM_F32>(a, st);
    else if (a.x_type == ELEM_F16) seam_launch<BT, ELEM_F16>(a, st);
    else seam_launch<BT, ELEM_BF16>(a, st);
}

}  // namespace
}  // namespace vb

using namespace vb;

extern "C" int vb_block_norm(const void* branch, int32_t branch_type, int64_t branch_ld, const float* post_w,
                             const void* gate, int32_t gate_type, int64_t gate_row, int64_t gate_col, float scale,
                             const void* x, int32_t x_type, int64_t x_ld, void* y, int64_t y_ld, const float* pre_w,
                             void* n, int32_t n_type, int64_t n_ld, int64_t rows, int64_t dim, float eps,
                             void* stream) {
    if (!elem_type(branch_type) || !elem_type(x_type) || (gate && !elem_type(gate_type)) || (pre_w && !elem_type(n_type))) {
        set_error("vb_block_norm: element types are 0 (fp32), 1 (fp16) and 2 (bf16)");
        return E_INVAL;
    }
    if (rows < 0 || rows > 0x7fffffff || dim <= 0 || dim > 0x7fffffff || !(eps >= 0.f) ||
        (rows > 0 && (!branch || !x || !y || (pre_w && !n)))) {
        set_error("vb_block_norm: bad arguments (rows=%lld, dim=%lld)", static_cast<long long>(rows),
                  static_cast<long long>(dim));
        return E_INVAL;
    }
    if (rows > 1 && (branch_ld < 0 || x_ld < 0 || y_ld < dim || (pre_w && n_ld < dim))) {
        set_error("vb_block_norm: a negative row stride, or one of y or n below dim=%lld", static_cast<long long>(dim));
        return E_INVAL;
    }
    if (gate && (gate_row < 0 || gate_col < 0 || gate_col > 1)) {
        set_error("vb_block_norm: gate strides (%lld, %lld): a row stride of 0 or more, a column stride of 0 or 1",
                  static_cast<long long>(gate_row), static_cast<long long>(gate_col));
        return E_INVAL;
    }
    if (rows == 0) return OK;
    const SeamArgs a{branch, x,      y,        n,   post_w,      pre_w,  gate,   branch_ld, x_ld,  y_ld, n_ld,
                     gate_row, gate_col, rows, dim, branch_type, x_type, n_type, gate_type, scale, eps};
    if (branch_type == ELEM_F32) seam_launch_x<ELEM_F32>(a, as_stream(stream));
    else if (branch_type == ELEM_F16) seam_launch_x<ELEM_F16>(a, as_stream(stream));
    else seam_launch_x<ELEM_BF16>(a, as_stream(stream));
    return check_launch("vb_block_norm");
}
