// Verification of drafted tokens against a target's logits, from given random
// numbers.  Of a sequence with k drafted tokens d_j, the target's logits of
// k + 1 positions and a drafter's of k, let
//
//   p_j = softmax(target_j / T)      q_j = softmax(draft_j / T')
//
// (without the drafter's logits q_j is 1 at d_j).  With u_j in [0, 1), d_j is
// accepted while u_j q_j(d_j) < p_j(d_j).  At the first that is not, a token
// from max(p_j - q_j, 0) (from p_j, where that is 0 everywhere) takes its
// place; behind k accepted ones a token from p_k follows.  That token is the
// first i with C_i > u C_V, C_i the sum of the weights up to i and u the
// sequence's last random number: the tokens are distributed as the target's own.
//
// Exponentials and sums are 64 bits, those of whole slices and those within them
// by the same 2^x of eleven points (nine have an error of 1.1e-12).  A token is an
// id, found by comparing a random number with a sum over a vocabulary; in fp32 the
// order of the additions would decide about one in a hundred of them.
//
//   stats    (row, slice): the maximum and the sum of 2^(c (z - max)), c =
//            log2(e) / T, of each slice of each row that a decision may need
//   decide   (sequence), with a drafter's logits: what is accepted, and what the
//            token is drawn from
//   rest     (sequence, slice), with a drafter's logits: the slice's sum of the
//            weights that the token is drawn by
//   token    one workgroup a sequence: the slice that the random number falls
//            into, then the place in it (without a drafter's logits the decision
//            is made here, and the slices' sums are those of stats)
//
// The terms' arithmetic (25 instructions a logit, seventeen of them 64-bit) bounds
// many rows before the memory does (64 sequences of 4 drafts over 128256 fp32 ids:
// stats 66 us, 4.5 TB/s; without the terms it takes 52, without the loads 61; nine
// points of 2^x take 61), the residual by its two terms a logit
// (19 us for 64 rows and rows of drafts); few rows wait for launches and for one
// workgroup's chain of loads, sums over waves and barriers (one sequence 4.8 + 8
// us, eight of 32003 ids 7.2 + 3.1 + 4.7 + 6.6).
//
// A row with a NaN or +inf (target's or drafter's) ends the sequence at its
// position: its token is -1, as it is where a mask leaves the target nothing.
// An id outside the vocabulary ends the drafts there, as a length does.
#include "elem_types.hpp"
#include "vb_internal.hpp"
#include "wave64.hpp"
#include "../../include/vbhip.h"

namespace vb {
namespace {

constexpr int VF_MAX_DRAFTS = 63;    // one a lane, and one lane more
constexpr int VF_MAX_SLICES = 64;    // one a lane
constexpr int VF_MAX_VOCAB = 1 << 28;
constexpr int VF_THREADS = 256;      // of the passes over rows
constexpr int VF_PIECE = 8;          // logits of a thread at a time
constexpr int VF_WIDE = 1024;        // threads of a sequence's last step
constexpr double LOG2E = 1.4426950408889634;

struct Source;
struct VerifyArgs {
    const void* target;
    const void* draft;
    const void* drafted;
    const int32_t* lengths;
    const float* u;
    int32_t* tokens;
    int32_t* accepted;
    double2* stats;  // [sequence][row][slice]: maximum, sum
    double* rest;    // [sequence][slice]
    Source* sources;  // [sequence]
    int64_t target_seq, target_row, draft_seq, draft_row, drafted_row, u_row;
    int32_t seqs, drafts, vocab, token_bytes, slices, slice, rests, rest_slice;
    double c, cd;  // log2(e) / T of the target and of the drafter
};

// Drafts of a sequence that count: up to its length and the first id outside
// the vocabulary.  Every wave of a workgroup computes the same.
__device__ __forceinline__ int drafts_of(const VerifyArgs& a, int seq) {
    const int lane = static_cast<int>(threadIdx.x) & 63;
    const int given = a.lengths ? a.lengths[seq] : a.drafts;
    bool in = lane < a.drafts && lane < given;
    if (in) {
        const int64_t p = seq * a.drafted_row + lane;
        const int64_t id = a.token_bytes == 8 ? static_cast<const int64_t*>(a.drafted)[p]
                                              : static_cast<const int32_t*>(a.drafted)[p];
        in = id >= 0 && id < a.vocab;
    }
    return __ffsll(static_cast<unsigned long long>(~__ballot(in))) - 1;
}

__device__ __forceinline__ int drafted_id(const VerifyArgs& a, int seq, int j) {
    const int64_t p = seq * a.drafted_row + j;
    return a.token_bytes == 8 ? static_cast<int>(static_cast<const int64_t*>(a.drafted)[p])
                              : static_cast<const int32_t*>(a.drafted)[p];
}

// VF_PIECE logits from an address of any whole element.
template <int TYPE>
struct Logits {
    float v[VF_PIECE];
    __device__ __forceinline__ void load(const void* z, int64_t i) {
        if constexpr (TYPE == ELEM_F32) {
            typedef float v4 __attribute__((ext_vector_type(4), aligned(4)));
            const v4* p = reinterpret_cast<const v4*>(static_cast<const float*>(z) + i);
            const v4 a = p[0], b = p[1];
#pragma unroll
            for (int j = 0; j < 4; j++) v[j] = a[j], v[4 + j] = b[j];
        } else {
            typedef uint32_t v4 __attribute__((ext_vector_type(4), aligned(2)));
            const v4 a = *reinterpret_cast<const v4*>(static_cast<const uint16_t*>(z) + i);
#pragma unroll
            for (int j = 0; j < VF_PIECE; j++) {
                const uint32_t h = a[j >> 1] >> 16 * (j & 1) & 0xffffu;
                v[j] = TYPE == ELEM_BF16 ? __uint_as_float(h << 16)
                                         : static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(h)));
            }
        }
    }
    // the first n of them, -inf behind
    __device__ __forceinline__ void load(const void* z, int64_t i, int n) {
        if (n >= VF_PIECE) return load(z, i);
#pragma unroll
        for (int j = 0; j < VF_PIECE; j++) v[j] = j < n ? elem_ld(z, i + j, TYPE) : -INFINITY;
    }
    // VF_PIECE of the logits [i, end) of a row at z[at], i the same in all of a
    // workgroup, by lanes side by side: an instruction's 16 bytes a lane are one run.
    __device__ __forceinline__ void spread(const void* z, int64_t at, int i, int end) {
        if constexpr (TYPE == ELEM_F32) {
            typedef float v4 __attribute__((ext_vector_type(4), aligned(4)));
            const float* p = static_cast<const float*>(z) + at;
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int k = i + h * 4 * VF_THREADS + 4 * static_cast<int>(threadIdx.x);
                if (k + 4 <= end) {
                    const v4 a = __builtin_nontemporal_load(reinterpret_cast<const v4*>(p + k));
#pragma unroll
                    for (int j = 0; j < 4; j++) v[4 * h + j] = a[j];
                } else {
#pragma unroll
                    for (int j = 0; j < 4; j++) v[4 * h + j] = k + j < end ? p[k + j] : -INFINITY;
                }
            }
        } else {
            const int k = i + VF_PIECE * static_cast<int>(threadIdx.x);
            load(z, at + k, end - k);
        }
    }
    __device__ __forceinline__ float largest() const {
        float m = v[0];
#pragma unroll
        for (int j = 1; j < VF_PIECE; j++) m = fmaxf(m, v[j]);
        return m;
    }
};

// 2^(c (z - m)); 0 for z = -inf (m finite).
__device__ __forceinline__ double term(const Exp2& exp2, float z, double m, double c) {
    return exp2((static_cast<double>(z) - m) * c);
}

// Sum over a workgroup of up to 16 waves, in every thread; buf: one place a wave.
__device__ __forceinline__ double group_sum(double v, double* buf) {
    const int wave = static_cast<int>(threadIdx.x) >> 6, waves = static_cast<int>(blockDim.x) >> 6;
    v = wave_sum64(v);
    __syncthreads();
    buf[wave] = v;
    __syncthreads();
    const int lane = static_cast<int>(threadIdx.x) & 63;
    return wave_sum64(lane < waves ? buf[lane] : 0.0);
}

// ---- stats ------------------------------------------------------------------

template <int TYPE>
__global__ void __launch_bounds__(VF_THREADS) verify_stats_kernel(VerifyArgs a) {
    const Exp2 exp2;
    __shared__ float tops[VF_THREADS / 64];
    __shared__ double sums[VF_THREADS / 64];
    const int rows = a.drafts + 1 + (a.draft ? a.drafts : 0);
    const int lane = static_cast<int>(threadIdx.x) & 63, wave = static_cast<int>(threadIdx.x) >> 6;
    for (int64_t item = blockIdx.x; item < static_cast<int64_t>(a.seqs) * rows * a.slices; item += gridDim.x) {
        const int slice = static_cast<int>(item % a.slices), row = static_cast<int>(item / a.slices % rows);
        const int seq = static_cast<int>(item / a.slices / rows);
        const int count = drafts_of(a, seq);
        const bool of_target = row <= a.drafts;
        const int j = of_target ? row : row - a.drafts - 1;
        if (j > count || (!of_target && j == count)) continue;  // no decision asks for it
        const void* z = of_target ? a.target : a.draft;
        const int64_t at = of_target ? seq * a.target_seq + j * a.target_row : seq * a.draft_seq + j * a.draft_row;
        const double c = of_target ? a.c : a.cd;
        const int begin = slice * a.slice, end = a.vocab - begin < a.slice ? a.vocab : begin + a.slice;
        // The lane's sum is relative to the largest of its first logits: only a logit
        // that is 2^450 times that (or the first one after nothing but -inf) moves the
        // reference.  fp32 rounds the border up by half a step at most, and by no more
        // than the 450: exponents stay below 901 (from 1024 on there is no 2^x), and a
        // term of up to 2^450 is good to 2^-45, the fma's rounding.  What is stored is
        // relative to the slice's largest logit: terms of a row by its maximum are at
        // most 1 and its sum at most the vocabulary, so products of the two stay finite.
        double ref = 0.0, at_ref = 0.0, sum = 0.0;  // at_ref: c ref, rounded; a term is 2^(c z - at_ref), one fma for the exponent
        float top = -INFINITY, limit = -INFINITY;
        bool bad = false, far = false;  // far: rounding c ref may cost that much; a term is 2^(c (z - ref))
        Logits<TYPE> next;
        next.spread(z, at, begin, end);
        for (int i = begin; i < end; i += VF_THREADS * VF_PIECE) {
            const Logits<TYPE> l = next;
            const int ahead = i + VF_THREADS * VF_PIECE;
            if (ahead < end) next.spread(z, at, ahead, end);
            const float most = l.largest();
#pragma unroll
            for (int j = 0; j < VF_PIECE; j++) bad = bad || !(l.v[j] < INFINITY);
            if (most > limit) {
                const double to = static_cast<double>(most);
                sum = limit > -INFINITY ? sum * exp2(far ? (ref - to) * c : __builtin_fma(-to, c, at_ref)) : 0.0;
                ref = to;
                at_ref = to * c;
                if (!(fabs(at_ref) < 0x1p40)) {
                    far = true;
                    at_ref = 0.0;
                } else {
                    far = false;
                }
                limit = fminf(static_cast<float>(to + 450.0 / c), 3.402823466e38f);
            }
            top = fmaxf(top, most);
            double part = 0.0;
            if (!__any(far)) {
#pragma unroll
                for (int j = 0; j < VF_PIECE; j++) part += exp2.normal(__builtin_fma(static_cast<double>(l.v[j]), c, -at_ref));
            } else {
#pragma unroll 1
                for (int j = 0; j < VF_PIECE; j++) {
                    float z_j = l.v[0];
#pragma unroll
                    for (int k = 1; k < VF_PIECE; k++) z_j = j == k ? l.v[k] : z_j;
                    part += exp2.normal(far ? (static_cast<double>(z_j) - ref) * c : __builtin_fma(static_cast<double>(z_j), c, -at_ref));
                }
            }
            sum += top > -INFINITY ? part : 0.0;
        }
        const float all = wave_largest(top);
        sum = wave_sum64(top > -INFINITY ? sum * exp2(far ? (ref - static_cast<double>(all)) * c
                                                          : __builtin_fma(-static_cast<double>(all), c, at_ref)) : 0.0);
        if (__any(bad)) sum = NAN;
        if (lane == 0) {
            tops[wave] = all;
            sums[wave] = sum;
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            float m = tops[0];
            for (int w = 1; w < VF_THREADS / 64; w++) m = fmaxf(m, tops[w]);
            double s = 0.0;
            for (int w = 0; w < VF_THREADS / 64; w++)
                s += sums[w] != sums[w] ? NAN : tops[w] > -INFINITY ? sums[w] * term(exp2, tops[w], m, c) : 0.0;
            a.stats[item] = make_double2(static_cast<double>(m), s);
        }
        __syncthreads();
    }
}

// ---- the decision -------------------------------------------------------------

// A row's maximum and sum from its slices, by a wave, in every lane.
__device__ __forceinline__ double2 row_stats(const Exp2& exp2, const VerifyArgs& a, int seq, int row, double c) {
    const int lane = static_cast<int>(threadIdx.x) & 63;
    const int rows = a.drafts + 1 + (a.draft ? a.drafts : 0);
    double2 v = make_double2(-INFINITY, 0.0);
    if (lane < a.slices) v = a.stats[(static_cast<int64_t>(seq) * rows + row) * a.slices + lane];
    const double m = wave_largest(v.x);
    const double s = v.y != v.y ? NAN : v.x > -INFINITY ? v.y * exp2((v.x - m) * c) : 0.0;
    return make_double2(m, wave_sum64(s));
}

// What a sequence's token is drawn from.
struct Source {
    int accepted;  // drafted tokens
    bool bad;      // the token is -1
    bool refused;  // from max(p - q, 0), else from p
    int without;   // q is 1 at this id (no drafter's logits), or -1
    int64_t p, q;  // rows: first logit
    double pm, qm, ratio;  // their maxima; the sum of p's terms over that of q's (0: q has none)
    double ps;             // the sum of p's terms
};

// max(p - q, 0).  Of equal p and q the roundings of two sums may leave some 2^-52
// p, which is no weight.
__device__ __forceinline__ double left_of(double p, double q) {
    const double r = p - q;
    return r > 0x1p-45 * p ? r : 0.0;
}

// Weight of id i, before the sum of them all divides it: p's term, less q's by
// p's sum.  (A row of nothing but -inf has the maximum 0.)
template <int TYPE>
__device__ __forceinline__ double weight(const Exp2& exp2, const VerifyArgs& a, const Source& s, bool refused, int i, float zp, float zq) {
    const double r = term(exp2, zp, s.pm, a.c);
    if (refused && a.draft) return left_of(r, term(exp2, zq, s.qm, a.cd) * s.ratio);
    return refused && i == s.without ? 0.0 : r;
}

// Weights of ids i ... i + n - 1 (n up to VF_PIECE; 0 behind).
template <int TYPE>
struct Weights {
    double w[VF_PIECE], sum;
    __device__ __forceinline__ Weights(const Exp2& exp2, const VerifyArgs& a, const Source& s, bool refused, int i, int n) {
        Logits<TYPE> p, q;
        if (n > 0) p.load(a.target, s.p + i, n);
        if (n > 0 && refused && a.draft) q.load(a.draft, s.q + i, n);
        sum = 0.0;
#pragma unroll
        for (int j = 0; j < VF_PIECE; j++) {
            w[j] = n > 0 ? weight<TYPE>(exp2, a, s, refused, i + j, p.v[j], q.v[j]) : 0.0;
            sum += w[j];
        }
    }
};

// The decision of a sequence, by a workgroup: a wave a position.
struct Decision {
    double2 p[VF_MAX_DRAFTS + 1], q[VF_MAX_DRAFTS + 1];  // rows' maxima and sums
    int id[VF_MAX_DRAFTS + 1], verdict[VF_MAX_DRAFTS + 1];
};
template <int TYPE>
__device__ __forceinline__ Source decide(const Exp2& exp2, const VerifyArgs& a, int seq, Decision& d) {
    const int wave = static_cast<int>(threadIdx.x) >> 6, waves = static_cast<int>(blockDim.x) >> 6;
    const int lane = static_cast<int>(threadIdx.x) & 63;
    const int count = drafts_of(a, seq);
    // 0: accepted, 1: refused, 2: a row that holds NaN or +inf
    for (int j = wave; j <= count; j += waves) {
        int id = -1, verdict = 1;
        float zp = -INFINITY, zq = -INFINITY, u = 0.f;
        if (j < count) {
            id = drafted_id(a, seq, j);
            zp = elem_ld(a.target, seq * a.target_seq + j * a.target_row + id, TYPE);
            if (a.draft) zq = elem_ld(a.draft, seq * a.draft_seq + j * a.draft_row + id, TYPE);
            u = a.u[seq * a.u_row + j];
        }
        const double2 p = row_stats(exp2, a, seq, j, a.c);
        double2 q = make_double2(0.0, 1.0);
        double qd = 1.0;
        if (j < count && a.draft) {
            q = row_stats(exp2, a, seq, a.drafts + 1 + j, a.cd);
            qd = zq > -INFINITY ? term(exp2, zq, q.x, a.cd) : 0.0;
        }
        const double pd = zp > -INFINITY ? term(exp2, zp, p.x, a.c) : 0.0;
        if (p.y != p.y || q.y != q.y) verdict = 2;
        else if (j < count && static_cast<double>(u) * qd * p.y < pd * (q.y > 0.0 ? q.y : 1.0)) verdict = 0;
        if (lane == 0) {
            d.p[j] = p;
            d.q[j] = q;
            d.id[j] = id;
            d.verdict[j] = verdict;
        }
    }
    __syncthreads();
    Source s{};
    const uint64_t stops = __ballot(lane >= count || d.verdict[lane < count ? lane : 0] != 0);
    s.accepted = __ffsll(static_cast<unsigned long long>(stops)) - 1;
    const double2 p = d.p[s.accepted], q = d.q[s.accepted];
    s.bad = d.verdict[s.accepted] == 2 || !(p.y > 0.0);  // (or nothing is left)
    s.refused = s.accepted < count;
    s.without = s.refused && !a.draft ? d.id[s.accepted] : -1;
    s.p = seq * a.target_seq + s.accepted * a.target_row;
    s.pm = p.x;
    s.ps = p.y;
    s.q = seq * a.draft_seq + s.accepted * a.draft_row;
    s.qm = q.x > -INFINITY ? q.x : 0.0;
    s.ratio = q.y > 0.0 ? p.y / q.y : 0.0;
    return s;
}

// ---- rest ---------------------------------------------------------------------

template <int TYPE>
__global__ void __launch_bounds__(VF_WIDE) verify_decide_kernel(VerifyArgs a) {
    const Exp2 exp2;
    __shared__ Decision d;
    for (int seq = static_cast<int>(blockIdx.x); seq < a.seqs; seq += static_cast<int>(gridDim.x)) {
        const Source s = decide<TYPE>(exp2, a, seq, d);
        if (threadIdx.x == 0) a.sources[seq] = s;
        __syncthreads();
    }
}

template <int TYPE>
__global__ void __launch_bounds__(VF_THREADS) verify_rest_kernel(VerifyArgs a) {
    const Exp2 exp2;
    __shared__ double sums[VF_THREADS / 64];
    for (int64_t item = blockIdx.x; item < static_cast<int64_t>(a.seqs) * a.rests; item += gridDim.x) {
        const int slice = static_cast<int>(item % a.rests), seq = static_cast<int>(item / a.rests);
        const Source s = a.sources[seq];
        const int begin = slice * a.rest_slice;
        const int end = a.vocab - begin < a.rest_slice ? a.vocab : begin + a.rest_slice;
        double sum = 0.0;
        if (!s.bad)
            for (int i = begin; i < end; i += VF_THREADS * VF_PIECE) {
                Logits<TYPE> p, q;
                p.spread(a.target, s.p, i, end);
                if (s.refused) q.spread(a.draft, s.q, i, end);
#pragma unroll
                for (int j = 0; j < VF_PIECE; j++) sum += weight<TYPE>(exp2, a, s, s.refused, 0, p.v[j], q.v[j]);
            }
        sum = group_sum(sum, sums);
        if (threadIdx.x == 0) a.rest[item] = sum;
    }
}

// ---- token --------------------------------------------------------------------

// The sum of the lanes up to each.
__device__ __forceinline__ double lanes_up_to(double v) {
    const int lane = static_cast<int>(threadIdx.x) & 63;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const double u = __shfl_up(v, o, 64);
        v += lane >= o ? u : 0.0;
    }
    return v;
}

// Of the lanes' parts v, with `upto` their sums up to each: the first that ends
// past the goal, or (by rounding, or at a random number of 1) the last that is
// not 0; -1: all are 0.
__device__ __forceinline__ int part_of(double v, double upto, double goal) {
    const uint64_t some = __ballot(v > 0.0), past = __ballot(v > 0.0 && upto > goal);
    return past ? __ffsll(static_cast<unsigned long long>(past)) - 1
                : some ? 63 - __clzll(static_cast<long long>(some)) : -1;
}

// The first id of [begin, end) whose sum of weights, from `carry` on, exceeds
// `goal`; the last id of a weight where rounding leaves none; -1 without weights.
// By a workgroup of VF_WIDE threads, a piece a thread at a time.
template <int TYPE>
__device__ __forceinline__ int locate(const Exp2& exp2, const VerifyArgs& a, const Source& s, bool refused, int begin, int end, double carry,
                                      double goal, double* buf, int* found) {
    constexpr int WAVES = VF_WIDE / 64;
    const int lane = static_cast<int>(threadIdx.x) & 63, wave = static_cast<int>(threadIdx.x) >> 6;
    int last = -1;
    for (int i0 = begin; i0 < end; i0 += VF_WIDE * VF_PIECE) {
        const int i = i0 + static_cast<int>(threadIdx.x) * VF_PIECE;
        const Weights<TYPE> w(exp2, a, s, refused, i, end - i);
        const double upto = lanes_up_to(w.sum);
        __syncthreads();  // (buf is free)
        if (lane == 63) buf[wave] = upto;
        if (threadIdx.x == 0) *found = -1;
        __syncthreads();
        const double mine = lane < WAVES ? buf[lane] : 0.0, waves = carry + lanes_up_to(mine);
        const int owner = part_of(mine, waves, goal);
        if (owner == wave) {
            const double before = owner > 0 ? lane_value(waves, owner - 1) : carry;
            const int who = part_of(w.sum, before + upto, goal);
            if (lane == who) {
                double at = before + upto - w.sum;
                int id = -1;
#pragma unroll
                for (int j = 0; j < VF_PIECE; j++) {
                    const bool open = id < 0 || !(at > goal);
                    at += w.w[j];
                    if (open && w.w[j] > 0.0) id = i + j;
                }
                *found = id;
            }
        }
        __syncthreads();
        if (*found >= 0) last = *found;
        carry = lane_value(waves, 63);
        if (carry > goal && last >= 0) break;
    }
    return last;
}

template <int TYPE>
__global__ void __launch_bounds__(VF_WIDE) verify_token_kernel(VerifyArgs a) {
    const Exp2 exp2;
    __shared__ Decision d;
    __shared__ double buf[VF_WIDE / 64];
    __shared__ int found;
    const int lane = static_cast<int>(threadIdx.x) & 63;
    const int rows = a.drafts + 1 + (a.draft ? a.drafts : 0);
    for (int seq = static_cast<int>(blockIdx.x); seq < a.seqs; seq += static_cast<int>(gridDim.x)) {
        const Source s = a.draft ? a.sources[seq] : decide<TYPE>(exp2, a, seq, d);
        const double u = static_cast<double>(a.u[seq * a.u_row + a.drafts]);
        int token = -1;
        if (!s.bad) {
            // each slice's weights, one a lane: summed by the pass before, or the target's own sums
            const int slices = a.draft ? a.rests : a.slices, size = a.draft ? a.rest_slice : a.slice;
            double part = 0.0;
            if (lane < slices) {
                if (a.draft) {
                    part = a.rest[static_cast<int64_t>(seq) * slices + lane];
                } else {
                    const double2 p = a.stats[(static_cast<int64_t>(seq) * rows + s.accepted) * slices + lane];
                    part = p.x > -INFINITY ? p.y * exp2((p.x - s.pm) * a.c) : 0.0;
                }
            }
            if (s.without >= 0) {  // the slice of the refused token, without it (the difference of sums would lose digits)
                const int slice = s.without / size, begin = slice * size, end = a.vocab - begin < size ? a.vocab : begin + size;
                double sum = 0.0;
                for (int i = begin + static_cast<int>(threadIdx.x) * VF_PIECE; i < end; i += VF_WIDE * VF_PIECE)
                    sum += Weights<TYPE>(exp2, a, s, true, i, end - i).sum;
                sum = group_sum(sum, buf);
                part = lane == slice ? sum : part;
            }
            const double upto = lanes_up_to(part), total = lane_value(upto, 63);
            if (total > 0.0) {
                const double goal = u * total;
                const int owner = part_of(part, upto, goal);
                const int begin = owner * size, end = a.vocab - begin < size ? a.vocab : begin + size;
                token = locate<TYPE>(exp2, a, s, s.refused, begin, end, owner > 0 ? lane_value(upto, owner - 1) : 0.0, goal, buf, &found);
            } else {  // nothing is left of p behind q: from p itself
                token = locate<TYPE>(exp2, a, s, false, 0, a.vocab, 0.0, u * s.ps, buf, &found);
            }
        }
        for (int j = static_cast<int>(threadIdx.x); j <= a.drafts; j += VF_WIDE)
            a.tokens[static_cast<int64_t>(seq) * (a.drafts + 1) + j] =
                j < s.accepted ? drafted_id(a, seq, j) : j == s.accepted ? token : -1;
        if (threadIdx.x == 0) a.accepted[seq] = s.accepted;
        __syncthreads();
    }
}

struct VerifyPlan {
    int64_t slices, slice, rests, rest_slice, workspace;
};

// Slices of a row: for the sums of rows at most eight workgroups a CU, about as many
// as are resident (64 sequences have three slices a row; four were 2 us slower), for
// the residual sixteen (22 us with four, 18 with sixteen), and whole pieces of a
// workgroup.
VerifyPlan verify_plan(int64_t seqs, int64_t drafts, int64_t vocab, bool draft) {
    const int64_t rows = seqs * (drafts + 1 + (draft ? drafts : 0));
    const auto cut = [&](int64_t n, int64_t groups, int64_t* slices, int64_t* slice) {
        const int64_t most = (vocab + VF_THREADS * VF_PIECE - 1) / (VF_THREADS * VF_PIECE);
        int64_t want = groups * num_cus() / (n > 0 ? n : 1);
        want = want < 1 ? 1 : want < VF_MAX_SLICES ? want : VF_MAX_SLICES;
        want = want < most ? want : most;
        *slice = ((vocab + want - 1) / want + VF_PIECE - 1) / VF_PIECE * VF_PIECE;
        *slices = (vocab + *slice - 1) / *slice;
    };
    VerifyPlan p{};
    cut(rows, 8, &p.slices, &p.slice);
    cut(seqs, 16, &p.rests, &p.rest_slice);
    if (!draft) p.rests = 0;
    p.workspace = rows * p.slices * 16 + (draft ? seqs * (p.rests * 8 + static_cast<int64_t>(sizeof(Source))) : 0);
    return p;
}

template <int TYPE>
int verify_launch(const VerifyArgs& a, hipStream_t st) {
    const auto grid = [](int64_t n) { return static_cast<uint32_t>(n < (1 << 20) ? n : 1 << 20); };
    verify_stats_kernel<TYPE><<<grid(static_cast<int64_t>(a.seqs) * (a.drafts + 1 + (a.draft ? a.drafts : 0)) * a.slices),
                                VF_THREADS, 0, st>>>(a);
    if (const int rc = check_launch("vb_verify_draft"); rc != OK) return rc;
    if (a.draft) {
        verify_decide_kernel<TYPE><<<grid(a.seqs), VF_WIDE, 0, st>>>(a);
        if (const int rc = check_launch("vb_verify_draft"); rc != OK) return rc;
        verify_rest_kernel<TYPE><<<grid(static_cast<int64_t>(a.seqs) * a.rests), VF_THREADS, 0, st>>>(a);
        if (const int rc = check_launch("vb_verify_draft"); rc != OK) return rc;
    }
    verify_token_kernel<TYPE><<<grid(a.seqs), VF_WIDE, 0, st>>>(a);
    return check_launch("vb_verify_draft");
}

}  // namespace
}  // namespace vb

using namespace vb;

extern "C" {

int64_t vb_verify_draft_workspace(int64_t n_seqs, int32_t n_drafts, int64_t vocab, int32_t has_draft) {
    if (n_seqs < 0 || n_seqs > 1 << 24 || n_drafts < 0 || n_drafts > VF_MAX_DRAFTS || vocab <= 0 || vocab > VF_MAX_VOCAB)
        return -1;
    if (n_seqs == 0) return 0;
    return verify_plan(n_seqs, n_drafts, vocab, has_draft != 0 && n_drafts > 0).workspace;
}

int vb_verify_draft(const void* target, int32_t type, int64_t target_seq, int64_t target_row, const void* draft,
                    int64_t draft_seq, int64_t draft_row, const void* drafted, int32_t token_bytes, int64_t drafted_row,
                    const int32_t* lengths, const float* uniforms, int64_t uniforms_row, int64_t n_seqs, int32_t n_drafts,
                    int64_t vocab, float temperature, float draft_temperature, int32_t* tokens, int32_t* accepted,
                    void* workspace, size_t workspace_bytes, void* stream) {
    if (n_drafts == 0) draft = nullptr;
    const int64_t need = vb_verify_draft_workspace(n_seqs, n_drafts, vocab, draft != nullptr);
    if (!elem_type(type) || need < 0 || target_seq < 0 || target_row < 0 || draft_seq < 0 || draft_row < 0 ||
        drafted_row < 0 || uniforms_row < 0) {
        set_error("vb_verify_draft: bad arguments (type %d, %lld sequences, %d of at most %d drafts, vocab=%lld, or a "
                  "negative stride)", type, static_cast<long long>(n_seqs), n_drafts, VF_MAX_DRAFTS,
                  static_cast<long long>(vocab));
        return E_INVAL;
    }
    if (!(temperature >= 1e-30f && temperature <= 1e30f && draft_temperature >= 1e-30f && draft_temperature <= 1e30f)) {
        set_error("vb_verify_draft: temperatures must be in [1e-30, 1e30]");
        return E_INVAL;
    }
    if (n_seqs == 0) return OK;
    if (!target || !uniforms || !tokens || !accepted || (n_drafts > 0 && (!drafted || (token_bytes != 4 && token_bytes != 8)))) {
        set_error("vb_verify_draft: null pointer, or token ids of %d bytes (4 or 8)", token_bytes);
        return E_INVAL;
    }
    if (static_cast<int64_t>(workspace_bytes) < need || !workspace || reinterpret_cast<uintptr_t>(workspace) % 16 != 0) {
        set_error("vb_verify_draft: workspace of %zu bytes (16-byte aligned) is below the %lld needed", workspace_bytes,
                  static_cast<long long>(need));
        return E_INVAL;
    }
    const VerifyPlan p = verify_plan(n_seqs, n_drafts, vocab, draft != nullptr);
    VerifyArgs a{};
    a.target = target;
    a.draft = draft;
    a.drafted = drafted;
    a.lengths = lengths;
    a.u = uniforms;
    a.tokens = tokens;
    a.accepted = accepted;
    a.target_seq = target_seq;
    a.target_row = target_row;
    a.draft_seq = draft_seq;
    a.draft_row = draft_row;
    a.drafted_row = drafted_row;
    a.u_row = uniforms_row;
    a.seqs = static_cast<int32_t>(n_seqs);
    a.drafts = n_drafts;
    a.vocab = static_cast<int32_t>(vocab);
    a.token_bytes = token_bytes;
    a.slices = static_cast<int32_t>(p.slices);
    a.slice = static_cast<int32_t>(p.slice);
    a.rests = static_cast<int32_t>(p.rests);
    a.rest_slice = static_cast<int32_t>(p.rest_slice);
    a.c = LOG2E / static_cast<double>(temperature);
    a.cd = LOG2E / static_cast<double>(draft_temperature);
    a.stats = static_cast<double2*>(workspace);
    a.rest = reinterpret_cast<double*>(a.stats + n_seqs * (n_drafts + 1 + (draft ? n_drafts : 0)) * p.slices);
    a.sources = reinterpret_cast<Source*>(a.rest + n_seqs * p.rests);
    if (type == ELEM_F32) return verify_launch<ELEM_F32>(a, as_stream(stream));
    if (type == ELEM_F16) return verify_launch<ELEM_F16>(a, as_stream(stream));
    return verify_launch<ELEM_BF16>(a, as_stream(stream));
}

}  // extern "C"
