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
// One pass over the logits.  A wave walks over a slice of a row, 16 logits a
// lane at a time, with its running maximum m, S and the entropy's sum (each
// lane's share of them, relative to the wave's m).  The alternatives hang on a
// threshold that at least `top` logits of the row reach: at first the top-th
// largest of the lanes' maxima over the workgroup's first batches, found by
// bisection.  A batch whose every lane stays at or below it costs one
// comparison; otherwise the logits that reach it are appended to a buffer in
// LDS.  When that fills, its best `top` are ranked (each entry counts those
// before it) and the threshold rises.  The waves' buffers, and the lists of a
// row's slices where there are few rows, are joined and ranked once.
//
// Memory bounds many rows (512 x 128256 fp32 41 us, 6.4 TB/s, with five
// alternatives 45; 1500 x 151669 bf16 73, 6.2 TB/s); few rows wait for the two
// launches, and with alternatives for the threshold and the ranking in each
// (1 x 128256: 5.7 us, with twenty 11.8).  No vector register is spilled; with
// alternatives 46 scalar ones are kept in lanes of vector registers.
#include <type_traits>

#include "elem_types.hpp"
#include "vb_internal.hpp"
#include "../../include/vbhip.h"

namespace vb {
namespace {

constexpr int LP_WAVES = 4;
constexpr int LP_THREADS = 64 * LP_WAVES;
constexpr int LP_MAX_TOP = 64;
constexpr int LP_MAX_VOCAB = 1 << 28; // a slice's offsets are 32 bits
constexpr int LP_MAX_SPLIT = 64;      // slices of a row, one per lane of the wave that joins them
constexpr int LP_BATCH = 16;          // logits of a lane at a time
constexpr int LP_BUF = 128;           // candidates of a wave: 64 kept, 64 new
// |c m| up to which sums are kept relative to c m rounded: its rounding is an
// exponent of at most 1/2 there, which costs no range (from 2^31 on it may be 128
// and more, and a term no number of fp32's).  The form for larger ones takes an
// instruction more a logit.
constexpr float LP_NEAR = 0x1p24f;

struct LpArgs {
    const void* z;
    const void* tokens;
    float* lp;
    float* entropy;
    int32_t* top_ids;
    float* top_lp;
    float4* stats;    // [row][split]: m, S, sum (workspace)
    uint64_t* keys;   // [row][place][split]
    int64_t ld, rows;
    int32_t vocab, token_bytes, n_tokens, top, splits;
    float c, inv_t;   // log2(e) / T, 1 / T
};

// A value's place in the order of the alternatives: larger first, equal
// values by the lower index.  0: none (NaN, -inf).
__device__ __forceinline__ uint32_t order_bits(float v) {
    const uint32_t u = __float_as_uint(v + 0.f);  // -0 is 0
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float order_value(uint32_t o) { return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o); }
__device__ __forceinline__ float order_floor(uint32_t o) { return o > 0x007fffffu ? order_value(o) : -INFINITY; }  // (-inf's)
__device__ __forceinline__ uint64_t order_key(float v, uint32_t i) {
    return v > -INFINITY ? static_cast<uint64_t>(order_bits(v)) << 32 | (0xffffffffu - i) : 0;
}
__device__ __forceinline__ int key_index(uint64_t k) { return static_cast<int>(0xffffffffu - static_cast<uint32_t>(k)); }
__device__ __forceinline__ float key_value(uint64_t k) { return order_value(static_cast<uint32_t>(k >> 32)); }

// The largest value of a wave, in every lane.
__device__ __forceinline__ float wave_max(float v) {
    const auto dpp = [](float x, auto ctrl, auto rows) {
        return __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(x), __float_as_int(x), decltype(ctrl)::value,
                                                          decltype(rows)::value, 0xF, false));
    };
    using std::integral_constant;
    v = fmaxf(v, dpp(v, integral_constant<int, 0xB1>{}, integral_constant<int, 0xF>{}));   // quad_perm [1,0,3,2]
    v = fmaxf(v, dpp(v, integral_constant<int, 0x4E>{}, integral_constant<int, 0xF>{}));   // quad_perm [2,3,0,1]
    v = fmaxf(v, dpp(v, integral_constant<int, 0x141>{}, integral_constant<int, 0xF>{}));  // row_half_mirror
    v = fmaxf(v, dpp(v, integral_constant<int, 0x140>{}, integral_constant<int, 0xF>{}));  // row_mirror
    v = fmaxf(v, dpp(v, integral_constant<int, 0x142>{}, integral_constant<int, 0xA>{}));  // row_bcast:15 into rows 1, 3
    v = fmaxf(v, dpp(v, integral_constant<int, 0x143>{}, integral_constant<int, 0xC>{}));  // row_bcast:31 into rows 2, 3
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}

// A value that at least n of the lanes' order bits reach (NV a lane, 0: none)
// and about as few as possible; 0 where there are fewer than n.
template <int NV>
__device__ __forceinline__ uint32_t reached_by(const uint32_t (&o)[NV], int n) {
    uint32_t at = 0;
    for (int bit = 31; bit >= 12; bit--) {
        const uint32_t up = at | 1u << bit;
        int count = 0;
#pragma unroll
        for (int i = 0; i < NV; i++) count += __popcll(__ballot(o[i] >= up));
        if (count >= n) at = up;
        if (count >= n && count <= n + (n >> 2)) break;
    }
    return at;
}

__device__ __forceinline__ int lanes_below(uint64_t mask) {
    return __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(mask >> 32), __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(mask), 0));
}

// LDS of one wave: what its lanes wrote is read by the others.
__device__ __forceinline__ void wave_lds_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// A wave's best n candidates (the same in every lane, but for the buffer).
struct Best {
    uint64_t* buf;
    int n, count;
    float tau;  // no candidate below it is wanted

    // The n best of the buffer, in order.
    __device__ __forceinline__ void rank() {
        wave_lds_fence();
        const int lane = static_cast<int>(threadIdx.x) & 63;
        const uint64_t a = lane < count ? buf[lane] : 0, b = lane + 64 < count ? buf[lane + 64] : 0;
        if (lane >= count) buf[lane] = 0;  // (the loop below reads whole groups)
        if (lane + 64 >= count) buf[lane + 64] = 0;
        wave_lds_fence();
        int ra = 0, rb = 0;
        if (count <= 64) {
            for (int i = 0; i < count; i += 8) {
                uint64_t k[8];
#pragma unroll
                for (int j = 0; j < 8; j++) k[j] = buf[i + j];
#pragma unroll
                for (int j = 0; j < 8; j++) ra += k[j] > a;
            }
        } else {
            for (int i = 0; i < count; i += 8) {
                uint64_t k[8];
#pragma unroll
                for (int j = 0; j < 8; j++) k[j] = buf[i + j];
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    ra += k[j] > a;
                    rb += k[j] > b;
                }
            }
        }
        wave_lds_fence();
        if (lane < count && ra < n) buf[ra] = a;
        if (lane + 64 < count && rb < n) buf[rb] = b;
        wave_lds_fence();
        count = count < n ? count : n;
        tau = count == n ? fmaxf(tau, key_value(buf[n - 1])) : tau;
    }

    __device__ __forceinline__ void append(uint64_t key, bool in) {
        const uint64_t mask = __ballot(in);
        if (!mask) return;
        if (count > LP_BUF - 64) rank();
        if (in) buf[count + lanes_below(mask)] = key;
        count += __popcll(mask);
    }
};

// Maximum and sums of a set of logits: S without one place of the maximum, and
// sum e^(z - m) (z - m), in units of log2.
struct Stat {
    float m, s, t;
};

// The lanes' sets as one, in every lane (an empty one: m = -inf, s = t = 0, or
// NaN where it held one).
__device__ __forceinline__ Stat join(Stat v, float c) {
    const float m = wave_max(v.m);
    const int owner = __ffsll(static_cast<unsigned long long>(__ballot(v.m == m))) - 1;
    const int lane = static_cast<int>(threadIdx.x) & 63;
    if (lane != owner && v.m > -INFINITY) {
        const float d = (v.m - m) * c, f = __builtin_amdgcn_exp2f(d);
        v.t = f * (v.t + fmaxf(d, -1e30f) * (v.s + 1.f));
        v.s = f * (v.s + 1.f);
    }
    return Stat{m, wave_sum_dpp(v.s), wave_sum_dpp(v.t)};
}

// What a row's results are made from.
struct RowResult {
    bool empty;
    float m, s, t, rest, inv_t;
    __device__ __forceinline__ RowResult(Stat v, float inv_t_) : m(v.m), s(v.s), t(v.t), inv_t(inv_t_) {
        if (m == INFINITY) s = t = NAN;
        empty = m == -INFINITY && s == 0.f;
        rest = log1pf(s);
    }
    __device__ __forceinline__ float lp(float z) const {
        // (halves, as z - m itself may leave fp32's range)
        return empty ? -INFINITY : (0.5f * z - 0.5f * m) * (2.f * inv_t) - rest;
    }
    __device__ __forceinline__ float entropy() const { return empty ? 0.f : rest - t * 0.693147180559945f / (1.f + s); }
};

template <int TYPE>
__device__ __forceinline__ float logit(const LpArgs& a, int64_t i) {
    return elem_ld(a.z, i, TYPE);
}

// A row's outputs by one wave; best: its alternatives in order.
template <int TYPE>
__device__ __forceinline__ void write_row(const LpArgs& a, int64_t row, const RowResult& r, const uint64_t* best, int count) {
    const int lane = static_cast<int>(threadIdx.x) & 63;
    if (a.entropy && lane == 0) a.entropy[row] = r.entropy();
    for (int j = lane; j < a.n_tokens; j += 64) {
        const int64_t p = row * a.n_tokens + j;
        const int64_t id = a.token_bytes == 8 ? static_cast<const int64_t*>(a.tokens)[p]
                                              : static_cast<const int32_t*>(a.tokens)[p];
        a.lp[p] = id >= 0 && id < a.vocab ? r.lp(logit<TYPE>(a, row * a.ld + id)) : 0.f;
    }
    if (lane < a.top) {
        const uint64_t k = lane < count ? best[lane] : 0;
        a.top_ids[row * a.top + lane] = k ? key_index(k) : -1;
        a.top_lp[row * a.top + lane] = r.s != r.s ? NAN : k ? r.lp(key_value(k)) : -INFINITY;
    }
}

template <int TYPE, bool LIST>
struct Walk {
    static constexpr int V = TYPE == ELEM_F32 ? 4 : 8;  // logits of a 16-byte load
    static constexpr int U = LP_BATCH / V;              // loads of a batch
    const LpArgs& a;
    Best best;
    float m, s, t;  // m: the wave's; s, t: the lane's sums, relative to `ref`
    float tau;      // no candidate at or below it
    float ref;      // c m, rounded: a term is 2^(c z - ref), one instruction for the exponent
    bool far;       // |c m| from LP_NEAR on: ref is 0, a term is 2^(c (z - m))
    bool masked;    // a term with z = -inf was met: 0 (-inf) is kept out of t

    __device__ __forceinline__ Walk(const LpArgs& a_, uint64_t* buf)
        : a(a_), best{buf, a_.top, 0, -INFINITY}, m(-INFINITY), s(0.f), t(0.f), tau(-INFINITY), ref(0.f), far(false), masked(false) {}

    // Logit r of the batch, and its index in the row.
    __device__ __forceinline__ static int index_of(int base, int r) {
        return base + (r / V * 64 + (static_cast<int>(threadIdx.x) & 63)) * V + r % V;
    }

    __device__ __forceinline__ void above(float (&v)[LP_BATCH], float cm, int base) {
        if (LIST && __any(cm > tau)) {
            const float least = fmaxf(best.tau, -3.402823466e38f);  // -inf is never a candidate
            int more = 0;
            bool ranked = true;
#pragma unroll
            for (int g = 0; g < LP_BATCH; g += 4) {  // most fours have none
                const uint64_t any = __ballot(fmaxf(fmaxf(v[g], v[g + 1]), fmaxf(v[g + 2], v[g + 3])) >= least);
                more += 4 * __popcll(any);
            }
            if (best.count + more > LP_BUF) {
                more = 0;
#pragma unroll
                for (int r = 0; r < LP_BATCH; r++) more += __popcll(__ballot(v[r] >= least));
            }
            if (best.count + more <= LP_BUF) {
#pragma unroll
                for (int g = 0; g < LP_BATCH; g += 4) {
                    if (!__any(fmaxf(fmaxf(v[g], v[g + 1]), fmaxf(v[g + 2], v[g + 3])) >= least)) continue;
#pragma unroll
                    for (int r = g; r < g + 4; r++) {
                        const uint64_t reach = __ballot(v[r] >= least);
                        if (!reach) continue;
                        if (v[r] >= least)
                            best.buf[best.count + lanes_below(reach)] = order_key(v[r], static_cast<uint32_t>(index_of(base, r)));
                        best.count += __popcll(reach);
                    }
                }
                ranked = best.count >= 2 * best.n && best.count >= 24;
            } else {
                uint32_t left = 0;
#pragma unroll
                for (int r = 0; r < LP_BATCH; r++) left |= v[r] >= least ? 1u << r : 0u;
                while (__any(left != 0)) {
                    const int r = __ffs(left) - 1;
                    float x = v[0];
#pragma unroll
                    for (int i = 1; i < LP_BATCH; i++) x = r == i ? v[i] : x;
                    best.append(order_key(x, static_cast<uint32_t>(index_of(base, r))), left != 0 && x >= best.tau);
                    left &= left - 1;
                }
            }
            if (ranked) {
                best.rank();
                if (best.count == best.n) tau = best.tau;  // equal values further on come after these
            }
        }
        if (__any(cm > m)) {
            const float top = wave_max(cm);
            // one place of the new maximum leaves the sums, the old one joins them
            const float now = top * a.c;
            const bool out_of = !(fabsf(now) < LP_NEAR);
            if (m > -INFINITY) {
                // the old reference and the old maximum, from the new reference
                const float back_at = out_of ? (m - top) * a.c : __builtin_fmaf(m, a.c, -now);
                const float d = far ? back_at : out_of ? __builtin_fmaf(-top, a.c, ref) : ref - now;
                const float f = __builtin_amdgcn_exp2f(d), dd = fmaxf(d, -1e30f), dm = fmaxf(back_at, -1e30f);
                const float back = (threadIdx.x & 63) == 0 ? __builtin_amdgcn_exp2f(dm) : 0.f;
                t = f * (t + dd * s) + back * dm;
                s = f * s + back;
            }
            m = top;
            ref = out_of ? 0.f : now;
            far = out_of;
            const int owner = __ffsll(static_cast<unsigned long long>(__ballot(cm == top))) - 1;
            bool out = (static_cast<int>(threadIdx.x) & 63) == owner;
            const float gone = far ? -INFINITY : (ref - 300.f) / a.c;  // its term is 0
#pragma unroll
            for (int r = 0; r < LP_BATCH; r++) {
                const bool hit = out && v[r] == top;
                v[r] = hit ? gone : v[r];
                out = out && !hit;
            }
            if (!LIST) tau = m;
        }
    }

    __device__ __forceinline__ void batch(float (&v)[LP_BATCH], int base) {
        float cm = v[0];
#pragma unroll
        for (int r = 1; r < LP_BATCH; r++) cm = fmaxf(cm, v[r]);
        if (__any(cm > fminf(tau, m))) above(v, cm, base);
        if (!far && !masked) {
            float s1 = s, t1 = t;
#pragma unroll
            for (int r = 0; r < LP_BATCH; r++) {
                const float d = __builtin_fmaf(v[r], a.c, -ref), e = __builtin_amdgcn_exp2f(d);
                s1 += e;
                t1 = __builtin_fmaf(e, d, t1);
            }
            if (!__any(t1 != t1)) {
                s = s1;
                t = t1;
                return;
            }
            masked = true;
        }
        const float from = far ? m : 0.f;
#pragma unroll
        for (int r = 0; r < LP_BATCH; r++) {
            const float d = __builtin_fmaf(v[r] - from, a.c, -ref), e = __builtin_amdgcn_exp2f(d);
            s += e;
            t = __builtin_fmaf(e, fmaxf(d, -1e30f), t);  // e is 0 below (and NaN for a NaN)
        }
    }

    // The wave's set, relative to m itself.
    __device__ __forceinline__ Stat stat() const {
        const float lo = far || !(m > -INFINITY) ? 0.f : __builtin_fmaf(m, a.c, -ref), f = __builtin_amdgcn_exp2f(-lo);
        return Stat{m, wave_sum_dpp(s * f), wave_sum_dpp((t - lo * s) * f)};
    }

    // The workgroup's 16-byte units [u0, u1) from unit 0 at `body`, whose first
    // logit has index i0: its waves take batches in turn.  With a list every wave
    // of the workgroup calls this, as they share their first batches' maxima in
    // `maxima`.
    __device__ __forceinline__ void run(const void* body, int u0, int u1, int i0, uint32_t (*maxima)[64]) {
        const int lane = static_cast<int>(threadIdx.x) & 63;
        const int count = u1 > u0 ? u1 - u0 : 0;
        const __amdgpu_buffer_rsrc_t r = make_rsrc(static_cast<const uint8_t*>(body) + static_cast<int64_t>(count ? u0 : 0) * 16,
                                                   static_cast<uint32_t>(count) * 16u);
        u32x4 raw[U];
        const auto load = [&](int at) __attribute__((always_inline)) {  // units past the last read nothing
#pragma unroll
            for (int u = 0; u < U; u++)
                raw[u] = __builtin_amdgcn_raw_buffer_load_b128(r, static_cast<int>(static_cast<uint32_t>(at + u * 64 + lane) * 16u), 0, 2);
        };
        const auto decode = [&](float (&v)[LP_BATCH], int at) __attribute__((always_inline)) {
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const uint32_t w = raw[u][i];
                    if constexpr (TYPE == ELEM_F32) {
                        v[u * V + i] = __uint_as_float(w);
                    } else if constexpr (TYPE == ELEM_F16) {
                        v[u * V + 2 * i] = f16lo(w);
                        v[u * V + 2 * i + 1] = f16hi(w);
                    } else {
                        v[u * V + 2 * i] = __uint_as_float(w << 16);
                        v[u * V + 2 * i + 1] = __uint_as_float(w & 0xffff0000u);
                    }
                }
            if (at + 64 * U > count) {
#pragma unroll
                for (int k = 0; k < LP_BATCH; k++)
                    if (at + k / V * 64 + lane >= count) v[k] = -INFINITY;
            }
        };
        const int begin = static_cast<int>(threadIdx.x >> 6) * 64 * U, step = LP_WAVES * 64 * U;
        load(begin);
        if constexpr (LIST) {
            float v[LP_BATCH];
            decode(v, begin);
            float cm = v[0];
#pragma unroll
            for (int k = 1; k < LP_BATCH; k++) cm = fmaxf(cm, v[k]);
            maxima[threadIdx.x >> 6][lane] = cm > -INFINITY ? order_bits(cm) : 0;
            __syncthreads();
            uint32_t o[LP_WAVES];
#pragma unroll
            for (int k = 0; k < LP_WAVES; k++) o[k] = maxima[k][lane];
            const uint32_t at = reached_by(o, best.n);
            best.tau = order_floor(at);
            // the value below (of 0 not -0): what equals the threshold is a candidate
            tau = order_floor(at == 0x80000000u ? at - 2 : at - (at > 0));
        }
        for (int at = __builtin_amdgcn_readfirstlane(begin); at < count; at += step) {
            float v[LP_BATCH];
            decode(v, at);
            load(at + step);
            batch(v, i0 + (u0 + at) * V);
        }
    }
};

// Workgroup: a slice of a row.  16-byte units from the row's first aligned one
// on; the logits before and behind them (fewer than a unit's each) are joined
// at the end as sets of one.
template <int TYPE, bool LIST>
__global__ void __launch_bounds__(LP_THREADS) logprob_kernel(LpArgs a) {
    using W = Walk<TYPE, LIST>;
    constexpr int SIZE = TYPE == ELEM_F32 ? 4 : 2;
    __shared__ uint64_t bufs[LIST ? LP_WAVES : 1][LP_BUF];
    __shared__ int counts[LP_WAVES];
    __shared__ uint32_t maxima[LP_WAVES][64];
    __shared__ Stat stats[LP_WAVES];
    const int lane = static_cast<int>(threadIdx.x) & 63;
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
    for (int64_t item = blockIdx.x; item < a.rows * a.splits; item += gridDim.x) {
        const int64_t row = item / a.splits;
        const int split = static_cast<int>(item % a.splits);
        const uint8_t* z = static_cast<const uint8_t*>(a.z) + row * a.ld * SIZE;
        int head = static_cast<int>((16 - (reinterpret_cast<uintptr_t>(z) & 15)) & 15) / SIZE;
        head = head < a.vocab ? head : a.vocab;
        const int units = (a.vocab - head) / W::V;
        const int each = ((units + a.splits - 1) / a.splits + 63) / 64 * 64;
        const int64_t u0 = static_cast<int64_t>(split) * each, u1 = u0 + each < units ? u0 + each : units;
        W w(a, bufs[LIST ? wave : 0]);
        w.run(z + head * SIZE, static_cast<int>(u0 < units ? u0 : units), static_cast<int>(u1), head, maxima);
        const Stat mine = w.stat();
        if (lane == 0) {
            stats[wave] = mine;
            counts[wave] = w.best.count;
        }
        __syncthreads();
        if (wave == 0) {
            // lanes 0-3: the waves; from lane 4 on: single logits
            const int tail = head + units * W::V, single = lane - LP_WAVES;
            const int singles = split == 0 ? head + (a.vocab - tail) : 0;
            const int at = single < head ? single : tail + single - head;
            Stat v{-INFINITY, 0.f, 0.f};
            if (lane < LP_WAVES) {
                v = stats[lane];
            } else if (single < singles) {
                const float x = logit<TYPE>(a, row * a.ld + at);
                if (x > -INFINITY) v.m = x;
                else if (x != x) v.s = v.t = NAN;
            }
            const Stat all = join(v, a.c);
            if constexpr (LIST) {
                for (int k = 1; k < LP_WAVES; k++)
                    for (int i = 0; i < counts[k]; i += 64) {
                        const uint64_t key = i + lane < counts[k] ? bufs[k][i + lane] : 0;
                        w.best.append(key, key != 0 && key_value(key) >= w.best.tau);
                    }
                const bool one = single >= 0 && single < singles && v.m > -INFINITY;
                w.best.append(order_key(v.m, static_cast<uint32_t>(at)), one && v.m >= w.best.tau);
                w.best.rank();
            }
            if (a.splits == 1) {
                write_row<TYPE>(a, row, RowResult(all, a.inv_t), bufs[0], LIST ? w.best.count : 0);
            } else {
                if (lane == 0) a.stats[item] = make_float4(all.m, all.s, all.t, 0.f);
                if (LIST && lane < a.top)
                    a.keys[(row * a.top + lane) * a.splits + split] = lane < w.best.count ? bufs[0][lane] : 0;
            }
        }
        __syncthreads();  // bufs and stats are free
    }
}

// One wave: the slices of a row.  Their lists are in order and lie place by
// place, so once no slice's candidate of a place is wanted none behind it is.
// Eight candidates a lane come at once (slice by slice, four places at a time:
// eight rows of 32003 with 64 alternatives 25.9 us a call, so 18.2; 200 rows of
// 32000 with 20 alternatives 22.2 and 19.1).
template <int TYPE, bool LIST>
__global__ void __launch_bounds__(64) logprob_join_kernel(LpArgs a) {
    __shared__ uint64_t buf[LP_BUF];
    const int lane = static_cast<int>(threadIdx.x);
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        constexpr int BATCH = 8;
        uint64_t key[BATCH];
        const uint64_t* list = a.keys + row * a.top * a.splits;
        const int total = a.top * a.splits;
        const auto load = [&](int base) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < BATCH; i++) key[i] = base + i * 64 + lane < total ? list[base + i * 64 + lane] : 0;
        };
        if constexpr (LIST) load(0);
        Stat v{-INFINITY, 0.f, 0.f};
        if (lane < a.splits) {
            const float4 p = a.stats[row * a.splits + lane];
            v = Stat{p.x, p.y, p.z};
        }
        const Stat all = join(v, a.c);
        Best best{buf, a.top, 0, -INFINITY};
        if constexpr (LIST) {
            // At least `top` candidates reach the q-th of every slice, q slices'
            // worth of them being enough, or (q = 1) a bisection of the firsts.
            const int q = (a.top + a.splits - 1) / a.splits;
            const uint64_t qth = lane < a.splits ? list[(q - 1) * a.splits + lane] : 0;
            const uint32_t o[1] = {static_cast<uint32_t>(qth >> 32)};
            const uint32_t at = reached_by(o, q == 1 ? a.top : a.splits);
            best.tau = order_floor(at);
            for (int base = 0; base < total;) {
                uint64_t k = key[0];
#pragma unroll 1
                for (int i = 0; i < BATCH && base + i * 64 < total; i++) {
                    best.append(k, k != 0 && key_value(k) >= best.tau);
#pragma unroll
                    for (int j = 1; j < BATCH; j++) k = i + 1 == j ? key[j] : k;
                }
                // the last place that is here from every slice
                if (!__any(lane >= 64 - a.splits && key[BATCH - 1] != 0 && key_value(key[BATCH - 1]) >= best.tau)) break;
                base += 64 * BATCH;
                load(base);
            }
            best.rank();
        }
        write_row<TYPE>(a, row, RowResult(all, a.inv_t), buf, best.count);
        wave_lds_fence();
    }
}

// Slices of a row.  A row is one workgroup's from two rows a CU on, as slices
// have a threshold and a list each and the launch that joins them (512 x 128256
// fp32, five alternatives: 45 us whole, 49 halved, 52 in four; without a list
// 41, 44, 46); fewer rows make three workgroups a CU (256 rows, five
// alternatives: 36 us with one, 30 with two to four; 64, twenty: 23 with two, 22
// with three, 21 with four, 23 with eight).  Each wave has a batch or more.
int64_t lp_splits(int64_t rows, int64_t vocab) {
    if (rows <= 0 || rows >= 2 * num_cus()) return 1;
    const int64_t want = (3 * num_cus() + rows - 1) / rows;
    const int64_t most = (vocab + LP_THREADS * LP_BATCH - 1) / (LP_THREADS * LP_BATCH);
    const int64_t n = want < most ? want : most;
    return n < LP_MAX_SPLIT ? n : LP_MAX_SPLIT;
}

template <int TYPE>
int lp_launch(const LpArgs& a, hipStream_t st) {
    const int64_t items = a.rows * a.splits;
    const uint32_t grid = static_cast<uint32_t>(items < (1 << 20) ? items : 1 << 20);  // fewer than 2^32 threads
    if (a.top > 0) logprob_kernel<TYPE, true><<<grid, LP_THREADS, 0, st>>>(a);
    else logprob_kernel<TYPE, false><<<grid, LP_THREADS, 0, st>>>(a);
    if (a.splits > 1) {
        if (const int rc = check_launch("vb_token_logprobs"); rc != OK) return rc;
        const uint32_t rows = static_cast<uint32_t>(a.rows < (1 << 20) ? a.rows : 1 << 20);
        if (a.top > 0) logprob_join_kernel<TYPE, true><<<rows, 64, 0, st>>>(a);
        else logprob_join_kernel<TYPE, false><<<rows, 64, 0, st>>>(a);
    }
    return check_launch("vb_token_logprobs");
}

}  // namespace
}  // namespace vb

using namespace vb;

extern "C" {

int64_t vb_token_logprobs_workspace(int64_t rows, int64_t vocab, int32_t top) {
    if (rows < 0 || rows > 0x7fffffff || vocab <= 0 || vocab > LP_MAX_VOCAB || top < 0 || top > LP_MAX_TOP) return -1;
    const int64_t splits = lp_splits(rows, vocab);
    return splits > 1 ? rows * splits * (16 + 8 * top) : 0;
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
    LpArgs a{};
    a.z = logits;
    a.tokens = tokens;
    a.lp = logprobs;
    a.entropy = entropy;
    a.top_ids = top_ids;
    a.top_lp = top_logprobs;
    a.ld = ld;
    a.rows = rows;
    a.vocab = static_cast<int32_t>(vocab);
    a.token_bytes = token_bytes;
    a.n_tokens = n_tokens;
    a.top = top;
    a.splits = static_cast<int32_t>(lp_splits(rows, vocab));
    a.c = 1.4426950408889634f / temperature;
    a.inv_t = 1.f / temperature;
    a.stats = static_cast<float4*>(workspace);
    a.keys = reinterpret_cast<uint64_t*>(a.stats + rows * a.splits);
    if (type == ELEM_F32) return lp_launch<ELEM_F32>(a, as_stream(stream));
    if (type == ELEM_F16) return lp_launch<ELEM_F16>(a, as_stream(stream));
    return lp_launch<ELEM_BF16>(a, as_stream(stream));
}

}  // extern "C"
