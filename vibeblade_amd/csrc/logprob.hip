// Log probabilities of given tokens from rows of logits, with each row's
// entropy and its most likely alternatives.  With z the logits of a row over
// the temperature T, m their maximum and
//
//   S = sum of exp(z_i - m) over all i but one place of the maximum,
//
// the row's log-sum-exp is m + log1p(S): the term 1 of the maximum is kept
// apart, so the log probability -log1p(S) of a nearly certain token keeps
// its digits.  Then
//
//   lp(t) = z_t - m - log1p(S)
//   H     = log1p(S) - sum_i exp(z_i - m) (z_i - m) / (1 + S)
//
// Maximum, sums and results are fp32.  The alternatives are ordered by the
// logits themselves (not over T), equal logits by the lower id.
//
// A row that a mask leaves empty (all logits -inf) has lp = -inf and H = 0; a
// -inf logit is never named (id -1, lp -inf).  A row with a NaN or a +inf has
// NaN for lp, H and the alternatives' log probabilities.
//
// One workgroup per row.
#include "elem_types.hpp"
#include "../../include/vbhip.h"

namespace vb {
namespace {

constexpr int LP_THREADS = 256;
constexpr int LP_MAX_TOP = 64;

struct LpArgs {
    const void* z;
    const void* tokens;
    float* lp;
    float* entropy;
    int32_t* top_ids;
    float* top_lp;
    int64_t ld, rows;
    int32_t vocab, type, token_bytes, n_tokens, top;
    float inv_t;
};

// A value's place in the order of the alternatives: larger first, equal
// values by the lower index.  0: none (NaN, -inf).
__device__ __forceinline__ uint64_t order_key(float v, uint32_t i) {
    if (!(v > -INFINITY)) return 0;
    const uint32_t u = __float_as_uint(v + 0.f);  // -0 is 0
    const uint32_t o = u & 0x80000000u ? ~u : u | 0x80000000u;
    return static_cast<uint64_t>(o) << 32 | (0xffffffffu - i);
}

__device__ __forceinline__ uint64_t umax(uint64_t a, uint64_t b) { return a > b ? a : b; }

__device__ void logprob_row(const LpArgs& a, int64_t row) {
    __shared__ float part[3][LP_THREADS / 64];
    __shared__ uint64_t best[LP_THREADS / 64];
    const int64_t base = row * a.ld;
    const int wave = threadIdx.x >> 6;
    auto key_max = [&](uint64_t below) {  // the largest key under `below`, in every thread
        uint64_t k = 0;
        for (int i = threadIdx.x; i < a.vocab; i += LP_THREADS) {
            const uint64_t o = order_key(elem_ld(a.z, base + i, a.type), i);
            if (o < below) k = umax(k, o);
        }
        for (int off = 32; off >= 1; off >>= 1) k = umax(k, __shfl_xor(k, off, 64));
        __syncthreads();
        if ((threadIdx.x & 63) == 0) best[wave] = k;
        __syncthreads();
        k = best[0];
        for (int w = 1; w < LP_THREADS / 64; w++) k = umax(k, best[w]);
        return k;
    };
    auto index_of = [](uint64_t k) { return static_cast<int>(0xffffffffu - static_cast<uint32_t>(k)); };
    uint64_t k = key_max(~0ull);
    const int at = k ? index_of(k) : -1;
    const float top = k ? elem_ld(a.z, base + at, a.type) : -INFINITY, m = k ? top : 0.f;
    float s = 0.f, t = 0.f;
    for (int i = threadIdx.x; i < a.vocab; i += LP_THREADS) {
        const float d = elem_ld(a.z, base + i, a.type) - m;
        if (i == at) continue;
        const float e = __expf(d * a.inv_t);
        s += e;
        t += e * fmaxf(d, -3.0e38f);
    }
    s = wave_sum_dpp(s);
    t = wave_sum_dpp(t);
    if ((threadIdx.x & 63) == 0) {
        part[0][wave] = s;
        part[1][wave] = t;
    }
    __syncthreads();
    s = part[0][0];
    t = part[1][0];
    for (int w = 1; w < LP_THREADS / 64; w++) {
        s += part[0][w];
        t += part[1][w];
    }
    if (top == INFINITY) s = t = NAN;
    const bool empty = !k && s == 0.f;
    const float rest = log1pf(s);
    auto lp_of = [&](float v) { return empty ? -INFINITY : (v - m) * a.inv_t - rest; };
    if (a.entropy && threadIdx.x == 0) a.entropy[row] = empty ? 0.f : rest - t * a.inv_t / (1.f + s);
    for (int j = threadIdx.x; j < a.n_tokens; j += LP_THREADS) {
        const int64_t p = row * a.n_tokens + j;
        const int64_t id = a.token_bytes == 8 ? static_cast<const int64_t*>(a.tokens)[p]
                                              : static_cast<const int32_t*>(a.tokens)[p];
        a.lp[p] = id >= 0 && id < a.vocab ? lp_of(elem_ld(a.z, base + id, a.type)) : 0.f;
    }
    for (int j = 0; j < a.top; j++) {
        if (threadIdx.x == 0) {
            a.top_ids[row * a.top + j] = k ? index_of(k) : -1;
            a.top_lp[row * a.top + j] = s != s ? NAN : k ? lp_of(elem_ld(a.z, base + index_of(k), a.type)) : -INFINITY;
        }
        if (k && j + 1 < a.top) k = key_max(k);
    }
}

__global__ void __launch_bounds__(LP_THREADS) logprob_kernel(LpArgs a) {
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        logprob_row(a, row);
        __syncthreads();  // its sums are read
    }
}

}  // namespace
}  // namespace vb

using namespace vb;

extern "C" {

int64_t vb_token_logprobs_workspace(int64_t rows, int64_t vocab, int32_t top) {
    if (rows < 0 || rows > 0x7fffffff || vocab <= 0 || vocab > 0x7fffffff || top < 0 || top > LP_MAX_TOP) return -1;
    return 0;
}

int vb_token_logprobs(const void* logits, int32_t type, int64_t ld, int64_t rows, int64_t vocab, float temperature,
                      const void* tokens, int32_t token_bytes, int32_t n_tokens, float* logprobs, float* entropy,
                      int32_t top, int32_t* top_ids, float* top_logprobs, void* workspace, size_t workspace_bytes,
                      void* stream) {
    if (!elem_type(type)) {
        set_error("vb_token_logprobs: element types are 0 (fp32), 1 (fp16) and 2 (bf16)");
        return E_INVAL;
    }
    const int64_t need = vb_token_logprobs_workspace(rows, vocab, top);
    if (need < 0 || n_tokens < 0 || (rows > 1 && ld < 0)) {
        set_error("vb_token_logprobs: bad arguments (rows=%lld, vocab=%lld, ld=%lld, n_tokens=%d, top=%d of at most %d)",
                  static_cast<long long>(rows), static_cast<long long>(vocab), static_cast<long long>(ld), n_tokens,
                  top, LP_MAX_TOP);
        return E_INVAL;
    }
    if (!(temperature >= 1e-30f && temperature <= 1e30f)) {  // its reciprocal is a normal number
        set_error("vb_token_logprobs: temperature must be in [1e-30, 1e30]");
        return E_INVAL;
    }
    if (rows > 0 && (!logits || (n_tokens > 0 && (!tokens || !logprobs || (token_bytes != 4 && token_bytes != 8))) ||
                     (top > 0 && (!top_ids || !top_logprobs)))) {
        set_error("vb_token_logprobs: null pointer, or token ids of %d bytes (4 or 8)", token_bytes);
        return E_INVAL;
    }
    if (static_cast<int64_t>(workspace_bytes) < need || (need > 0 && (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16))) {
        set_error("vb_token_logprobs: workspace of %zu bytes (16-byte aligned) is below the %lld needed",
                  workspace_bytes, static_cast<long long>(need));
        return E_INVAL;
    }
    if (rows == 0) return OK;
    const LpArgs a{logits, tokens, logprobs, entropy, top_ids, top_logprobs, ld, rows, static_cast<int32_t>(vocab), type,
                   token_bytes, n_tokens, top, 1.f / temperature};
    const uint32_t grid = static_cast<uint32_t>(rows < (1 << 20) ? rows : 1 << 20);  // fewer than 2^32 threads
    logprob_kernel<<<dim3(grid), dim3(LP_THREADS), 0, as_stream(stream)>>>(a);
    return check_launch("vb_token_logprobs");
}

}  // extern "C"
