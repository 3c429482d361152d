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
// One workgroup per row.
#include "vb_common.hpp"
#include "elem_types.hpp"
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

constexpr int SEAM_THREADS = 256;

// The workgroup's sum of v, in every thread (waves added in order).
__device__ __forceinline__ float wg_sum(float v, float* part) {
    v = wave_sum_dpp(v);
    __syncthreads();  // the last sum's readers are done
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = part[0];
    for (int i = 1; i < SEAM_THREADS / 64; i++) s += part[i];
    return s;
}

__device__ __forceinline__ void seam_row(const SeamArgs& a, int64_t row, float* part) {
    const int64_t bo = row * a.b_ld, xo = row * a.x_ld, yo = row * a.y_ld, no = row * a.n_ld, go = row * a.gate_row;
    float inv = 1.f;
    if (a.post_w) {
        float s = 0.f;
        for (int64_t i = threadIdx.x; i < a.dim; i += SEAM_THREADS) {
            const float v = elem_ld(a.b, bo + i, a.b_type);
            s += v * v;
        }
        inv = 1.f / sqrtf(wg_sum(s, part) / static_cast<float>(a.dim) + a.eps);
    }
    auto value = [&](int64_t i) {
        float p = elem_ld(a.b, bo + i, a.b_type);
        if (a.post_w) p = p * inv * a.post_w[i];
        if (a.gate) p *= elem_ld(a.gate, go + i * a.gate_col, a.gate_type);
        return elem_ld(a.x, xo + i, a.x_type) + a.scale * p;
    };
    float inv2 = 1.f;
    if (a.pre_w) {
        float s = 0.f;
        for (int64_t i = threadIdx.x; i < a.dim; i += SEAM_THREADS) {
            const float v = value(i);
            s += v * v;
        }
        inv2 = 1.f / sqrtf(wg_sum(s, part) / static_cast<float>(a.dim) + a.eps);
    }
    for (int64_t i = threadIdx.x; i < a.dim; i += SEAM_THREADS) {
        const float v = value(i);
        elem_st(a.y, yo + i, a.x_type, v);
        if (a.pre_w) elem_st(a.n, no + i, a.n_type, v * inv2 * a.pre_w[i]);
    }
}

__global__ void __launch_bounds__(SEAM_THREADS) seam_kernel(SeamArgs a) {
    __shared__ float part[SEAM_THREADS / 64];
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) seam_row(a, row, part);
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
    const uint32_t grid = static_cast<uint32_t>(rows < (1 << 20) ? rows : 1 << 20);  // fewer than 2^32 threads
    seam_kernel<<<dim3(grid), dim3(SEAM_THREADS), 0, as_stream(stream)>>>(a);
    return check_launch("vb_block_norm");
}
