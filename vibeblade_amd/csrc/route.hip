// Experts of every token from a router's logits z (E a token):
//
//   s_e = softmax(z)_e  or  sigmoid(z_e)
//   c_e = s_e + b_e     or, without a bias, z_e (of the same order)
//   of `groups` groups of consecutive experts the `kept` best ones stay, by the
//   largest c of each, or by the sum of its two largest s + b
//   the top k of their experts by (c descending, id ascending)
//   w_e = scale * s_e / (renorm ? sum of the chosen s : 1)
//
// Scores, choices and group sums are compared in 64 bits: which of two experts
// comes first is an id, and no two programs agree on it where c is rounded to
// fp32 (of 16384 tokens of 256 experts one or two have two choices within 2^-23).
//
// An expert whose logit (or bias) is -inf is never chosen: where there are not
// enough others the id is -1 and the weight 0.  A token with a NaN logit (or
// choice), or +inf under softmax, has ids -1 and weights NaN.
//
// One wave a token.  The lanes hold the experts in order: 64 / G' lanes a group
// (G' = the number of groups, rounded up to a power of two) and V experts a
// lane, so that a group's lanes are a butterfly of their own and a lower lane
// has lower ids.  A lane sorts its choices; a round takes the largest of the
// lanes' first ones (a maximum needs no id beside it) and the lowest lane that
// holds it.
//
// Instructions bound many tokens (16384 of 256 experts, sigmoid, bias, 4 of 8
// groups, top 8: 24.5 us, 740 vector instructions a token, four fifths of the
// issue slots; the logits alone are 3 us of memory), and one wave's chain of them
// few (one token of 128 experts 2.9 us, 16 of 256 5.3, of which a launch is 1.9).
// The choices in 64 bits throughout take 34 us for the 16384; unsorted, looked
// through every round, 32.
#include "elem_types.hpp"
#include "vb_internal.hpp"
#include "wave64.hpp"
#include "../../include/vbhip.h"

namespace vb {
namespace {

constexpr int ROUTE_WAVES = 4;
constexpr int ROUTE_MAX_EXPERTS = 512;  // at most 16 a lane, whatever the groups
constexpr int ROUTE_MAX = 64;           // groups, and experts of a token: one a lane
constexpr double LOG2E = 1.4426950408889634;

struct RouteArgs {
    const void* z;
    const float* bias;
    int32_t* ids;
    float* w;
    int64_t ld, tokens;
    int32_t experts, topk, groups, kept, size, shift;  // size: experts of a group; 1 << shift: its lanes
    bool sigmoid, top2, renorm;
    float scale;
};

// v of the lane 1 << s away within the eight, from DPP where there is one.
template <typename T>
__device__ __forceinline__ T lane_across(T v, int s) {
    switch (s) {
        case 0: return dpp_or_self<0xB1>(v);   // quad_perm [1,0,3,2]
        case 1: return dpp_or_self<0x4E>(v);   // quad_perm [2,3,0,1]
        case 2: return dpp_or_self<0x141>(v);  // row_half_mirror: quads are alike by now
        case 3: return dpp_or_self<0x140>(v);  // row_mirror: so are eights
        default: return __shfl_xor(v, 1 << s, 64);
    }
}

__device__ __forceinline__ float smaller(float a, float b) { return fminf(a, b); }
__device__ __forceinline__ double smaller(double a, double b) { return fmin(a, b); }

// The sum of the two largest (a >= b) of a group's 1 << shift lanes, in each of
// them.  -inf: none; one alone counts for itself.
template <typename T>
__device__ __forceinline__ T group_top2(T a, T b, int shift) {
#pragma unroll
    for (int s = 0; s < 6; s++) {
        if (s >= shift) break;
        const T oa = lane_across(a, s), ob = lane_across(b, s);
        b = larger(smaller(a, oa), larger(b, ob));
        a = larger(a, oa);
    }
    return a + (b > -INFINITY ? b : T(0));
}

template <typename T>
__device__ __forceinline__ T group_largest(T v, int shift) {
#pragma unroll
    for (int s = 0; s < 6; s++) {
        if (s >= shift) break;
        v = larger(v, lane_across(v, s));
    }
    return v;
}

// Whether the lane's group is among the `kept` best by `mine` (equal ones: the lower group).
template <typename T>
__device__ __forceinline__ bool group_stays(const RouteArgs& a, T mine, int group) {
    int before = 0;
    for (int g = 0; g < a.groups; g++) {
        const T other = lane_value(mine, g << a.shift);
        before += other > mine || (other == mine && g < group);
    }
    return before < a.kept;
}

// What the lanes take in the rounds: lane r the r-th expert.
struct Taken {
    int id = -1;
};

// The order of floats as that of unsigned numbers (-0 is 0), and back.
__device__ __forceinline__ uint32_t order_bits(float v) {
    const uint32_t u = __float_as_uint(v + 0.f);
    return u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float order_value(uint32_t o) { return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o); }
constexpr uint32_t ORDER_NONE = 0x007fffffu;  // of -inf

template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp_max_u(uint32_t v) {
    const uint32_t u = __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, false);
    return u > v ? u : v;
}
__device__ __forceinline__ uint32_t wave_largest_u(uint32_t v) {
    v = dpp_max_u<0xB1, 0xF>(v);
    v = dpp_max_u<0x4E, 0xF>(v);
    v = dpp_max_u<0x141, 0xF>(v);
    v = dpp_max_u<0x140, 0xF>(v);
    v = dpp_max_u<0x142, 0xA>(v);
    v = dpp_max_u<0x143, 0xC>(v);
    return __builtin_amdgcn_readlane(v, 63);
}

// The lane's choices in descending order, equal ones by the lower place.
template <int V>
struct Sorted {
    uint32_t key[V];
    int at[V];
    __device__ __forceinline__ explicit Sorted(const float (&c)[V]) {
#pragma unroll
        for (int v = 0; v < V; v++) key[v] = order_bits(c[v]), at[v] = v;
#pragma unroll
        for (int n = V - 1; n > 0; n--)  // neighbours only: equal ones keep their order
#pragma unroll
            for (int v = 0; v < n; v++) {
                const bool swap = key[v + 1] > key[v];
                const uint32_t k = swap ? key[v] : key[v + 1];
                const int i = swap ? at[v] : at[v + 1];
                key[v] = swap ? key[v + 1] : key[v];
                at[v] = swap ? at[v + 1] : at[v];
                key[v + 1] = k;
                at[v + 1] = i;
            }
    }
};

// As `take` below, from sorted choices: a round's is the largest of the lanes'
// first ones, and the lane that gave it moves up its others.
template <int V>
__device__ __forceinline__ float take_sorted(const RouteArgs& a, Sorted<V>& c, int base, int rounds, Taken& out) {
    const int lane = static_cast<int>(threadIdx.x) & 63;
    float gap = INFINITY, last = INFINITY;
    for (int r = 0; r < rounds; r++) {
        const uint32_t best = wave_largest_u(c.key[0]);
        if (best <= ORDER_NONE) break;  // no expert is left
        const float value = order_value(best);
        gap = fminf(gap, last - value);
        last = value;
        const int owner = __ffsll(static_cast<unsigned long long>(__ballot(c.key[0] == best))) - 1;
        const int chosen = __builtin_amdgcn_readlane(base + c.at[0], owner);
        out.id = lane == r && r < a.topk ? chosen : out.id;
        if (lane == owner) {
#pragma unroll
            for (int v = 0; v + 1 < V; v++) c.key[v] = c.key[v + 1], c.at[v] = c.at[v + 1];
            c.key[V - 1] = 0;
        }
    }
    return gap;
}

// `rounds` rounds over the choices c (of which the first a.topk count); the
// smallest difference of one round's choice to the next.
template <int V, typename T>
__device__ __forceinline__ T take(const RouteArgs& a, T (&c)[V], int base, int rounds, Taken& out) {
    const int lane = static_cast<int>(threadIdx.x) & 63;
    T gap = INFINITY, last = INFINITY;
    for (int r = 0; r < rounds; r++) {
        T most = c[0];
#pragma unroll
        for (int v = 1; v < V; v++) most = larger(most, c[v]);
        const T best = wave_largest(most);
        if (best == -INFINITY) break;  // no expert is left
        gap = smaller(gap, last - best);
        last = best;
        const int owner = __ffsll(static_cast<unsigned long long>(__ballot(most == best))) - 1;
        int at = 0;
#pragma unroll
        for (int v = V - 1; v >= 0; v--) at = c[v] == best ? v : at;
        if (lane == owner) {
#pragma unroll
            for (int v = 0; v < V; v++) c[v] = v == at ? -INFINITY : c[v];
        }
        const int chosen = __builtin_amdgcn_readlane(base + at, owner);
        out.id = lane == r && r < a.topk ? chosen : out.id;
    }
    return gap;
}

// Choices in fp32: sorted where a lane has few.
template <int V>
__device__ __forceinline__ float take_fp32(const RouteArgs& a, float (&c)[V], int base, int rounds, Taken& out) {
    if constexpr (V <= 4) {
        Sorted<V> s(c);
        return take_sorted<V>(a, s, base, rounds, out);
    } else {
        return take<V, float>(a, c, base, rounds, out);
    }
}

// What groups go by, in every lane of each: the largest of the choices c, or the
// sum of the two largest values.
template <int V, typename T>
__device__ __forceinline__ T group_score(const RouteArgs& a, const T (&c)[V], const T (&value)[V]) {
    if (a.top2) {
        T x = -INFINITY, y = -INFINITY;
#pragma unroll
        for (int v = 0; v < V; v++) {
            y = larger(y, smaller(x, value[v]));
            x = larger(x, value[v]);
        }
        return group_top2(x, y, a.shift);
    }
    T most = c[0];
#pragma unroll
    for (int v = 1; v < V; v++) most = larger(most, c[v]);
    return group_largest(most, a.shift);
}

// SCORED: choices are scores with a bias, or groups go by sums of scores.  These
// are first taken in fp32, which is enough where no two that are compared lie
// within its error (`sure`; of scores of 256 experts two do in one token of
// several hundred), and in 64 bits where they do.  Choices that are logits are
// exact in fp32.
template <int TYPE, int V, bool SCORED>
__global__ void __launch_bounds__(64 * ROUTE_WAVES) route_kernel(RouteArgs a) {
    const Exp2 exp2;
    const int lane = static_cast<int>(threadIdx.x) & 63;
    const int group = lane >> a.shift, first = (lane & ((1 << a.shift) - 1)) * V;
    const int here = group < a.groups && a.size > first ? (a.size - first < V ? a.size - first : V) : 0;
    const int base = group * a.size + first;
    float b[V];
#pragma unroll
    for (int v = 0; v < V; v++) b[v] = SCORED && a.bias && v < here ? a.bias[base + v] : 0.f;
    // Two choices' difference: scores are at most 1 and less than 2e-6 off (an
    // exponent's rounding costs at most x e^-x half steps, a sum of 512 terms 22 of
    // them), the sum with a bias half a step of itself.  The sum of two past 2^126
    // may be no fp32 number, and an infinity is equal to any other: never sure.
    float off = 0.f;
    if constexpr (SCORED) {
        float most = 0.f;
#pragma unroll
        for (int v = 0; v < V; v++) most = fabsf(b[v]) < INFINITY ? fmaxf(most, fabsf(b[v])) : most;
        off = __builtin_fmaf(4.f * wave_largest(most), 0x1p-24f, 4e-6f + 0x1p-22f);  // (4 * 2^126 is infinite)
    }
    for (int64_t token = static_cast<int64_t>(blockIdx.x) * ROUTE_WAVES + (threadIdx.x >> 6); token < a.tokens;
         token += static_cast<int64_t>(gridDim.x) * ROUTE_WAVES) {
        float z[V];
#pragma unroll
        for (int v = 0; v < V; v++) z[v] = v < here ? elem_ld(a.z, token * a.ld + base + v, TYPE) : -INFINITY;
        bool bad = false;
        float top = -INFINITY;
#pragma unroll
        for (int v = 0; v < V; v++) {
            bad = bad || z[v] != z[v];
            top = fmaxf(top, z[v]);
        }
        if (!a.sigmoid) {
            top = wave_largest(top);
            bad = bad || top == INFINITY;
        }
        // softmax: relative to the largest logit, the sum kept apart
        const auto score = [&](float x) __attribute__((always_inline)) {
            if (a.sigmoid) {
                const double e = exp2(-fabs(static_cast<double>(x)) * LOG2E);
                return (x >= 0.f ? 1.0 : e) / (1.0 + e);
            }
            return exp2((static_cast<double>(x) - static_cast<double>(top)) * LOG2E);
        };
        double sum = 1.0;
        const auto total = [&]() __attribute__((always_inline)) {
            double part = 0.0;
#pragma unroll
            for (int v = 0; v < V; v++) part += z[v] > -INFINITY ? score(z[v]) : 0.0;
            return wave_sum64(part);
        };
        Taken taken;
        if constexpr (SCORED) {
            float c[V], value[V], sum32 = 1.f;
            if (!a.sigmoid) {
                float part = 0.f;
#pragma unroll
                for (int v = 0; v < V; v++) {
                    value[v] = __builtin_amdgcn_exp2f((z[v] - top) * static_cast<float>(LOG2E));
                    part += z[v] > -INFINITY ? value[v] : 0.f;
                }
                sum32 = __builtin_amdgcn_rcpf(wave_sum_dpp(part));
            }
#pragma unroll
            for (int v = 0; v < V; v++) {
                const float s = a.sigmoid ? __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-z[v] * static_cast<float>(LOG2E)))
                                          : value[v] * sum32;
                value[v] = z[v] > -INFINITY ? s + b[v] : -INFINITY;
                bad = bad || value[v] != value[v];
                c[v] = a.bias ? value[v] : z[v];
            }
            bool sure = true;
            if (a.kept < a.groups) {
                const float mine = group_score<V, float>(a, c, value);
                const bool stays = group_stays(a, mine, group);
                // the least group that stays, and the best of those that do not; logits are exact
                const float in = -wave_largest(stays ? -mine : -INFINITY), out = wave_largest(stays || group >= a.groups ? -INFINITY : mine);
                sure = !(in - out <= (a.top2 ? 2.f * off : a.bias ? off : -1.f));
#pragma unroll
                for (int v = 0; v < V; v++) c[v] = stays ? c[v] : -INFINITY;
            }
            const float gap = take_fp32<V>(a, c, base, a.bias ? a.topk + 1 : a.topk, taken);
            if (a.bias) sure = sure && gap > off;
            if (__any(bad || !sure)) {
                taken = Taken{};
                double c[V], value[V];
                if (!a.sigmoid) sum = total();
#pragma unroll
                for (int v = 0; v < V; v++) {
                    value[v] = z[v] > -INFINITY ? score(z[v]) / sum + static_cast<double>(b[v]) : -INFINITY;
                    bad = bad || value[v] != value[v];
                    c[v] = a.bias ? value[v] : static_cast<double>(z[v]);
                }
                if (a.kept < a.groups) {
                    const bool stays = group_stays(a, group_score<V, double>(a, c, value), group);
#pragma unroll
                    for (int v = 0; v < V; v++) c[v] = stays ? c[v] : -INFINITY;
                }
                if (!__any(bad)) take<V, double>(a, c, base, a.topk, taken);
            }
        } else {
            float c[V];
#pragma unroll
            for (int v = 0; v < V; v++) c[v] = z[v];
            if (a.kept < a.groups) {
                const bool stays = group_stays(a, group_score<V, float>(a, c, c), group);
#pragma unroll
                for (int v = 0; v < V; v++) c[v] = stays ? c[v] : -INFINITY;
            }
            if (!__any(bad)) take_fp32<V>(a, c, base, a.topk, taken);
        }
        const bool none = __any(bad);
        double w = !none && taken.id >= 0 ? score(elem_ld(a.z, token * a.ld + taken.id, TYPE)) : 0.0;
        if (a.renorm) sum = wave_sum64(w);
        else if (!a.sigmoid) sum = total();
        w = w > 0.0 ? w / sum : 0.0;  // (all chosen scores 0: weights 0)
        if (lane < a.topk) {
            a.ids[token * a.topk + lane] = none ? -1 : taken.id;
            a.w[token * a.topk + lane] = none ? NAN : static_cast<float>(static_cast<double>(a.scale) * w);
        }
    }
}

template <int TYPE, int V>
int route_launch(const RouteArgs& a, hipStream_t st) {
    const int64_t want = (a.tokens + ROUTE_WAVES - 1) / ROUTE_WAVES;
    const uint32_t grid = static_cast<uint32_t>(want < (1 << 20) ? want : 1 << 20);
    if (a.bias || (a.top2 && a.kept < a.groups)) route_kernel<TYPE, V, true><<<grid, 64 * ROUTE_WAVES, 0, st>>>(a);
    else route_kernel<TYPE, V, false><<<grid, 64 * ROUTE_WAVES, 0, st>>>(a);
    return check_launch("vb_route_experts");
}

template <int TYPE>
int route_type(const RouteArgs& a, hipStream_t st) {
    const int each = (a.size + (1 << a.shift) - 1) >> a.shift;  // experts of a lane
    if (each <= 1) return route_launch<TYPE, 1>(a, st);
    if (each <= 2) return route_launch<TYPE, 2>(a, st);
    if (each <= 4) return route_launch<TYPE, 4>(a, st);
    if (each <= 8) return route_launch<TYPE, 8>(a, st);
    return route_launch<TYPE, 16>(a, st);
}

}  // namespace
}  // namespace vb

using namespace vb;

extern "C" int vb_route_experts(const void* logits, int32_t type, int64_t ld, int64_t n_tokens, int32_t n_exp,
                                int32_t topk, int32_t scores, const float* bias, int32_t groups, int32_t groups_kept,
                                int32_t group_score, int32_t renorm, float scale, int32_t* out_idx, float* out_w,
                                void* stream) {
    if (!elem_type(type) || n_tokens < 0 || n_tokens > 0x7fffffff || n_exp <= 0 || n_exp > ROUTE_MAX_EXPERTS ||
        (n_tokens > 1 && ld < 0)) {
        set_error("vb_route_experts: bad arguments (type %d, %lld tokens, row stride %lld, %d of at most %d experts)",
                  type, static_cast<long long>(n_tokens), static_cast<long long>(ld), n_exp, ROUTE_MAX_EXPERTS);
        return E_INVAL;
    }
    if (groups < 1 || groups > ROUTE_MAX || n_exp % groups != 0 || groups_kept < 1 || groups_kept > groups ||
        topk < 1 || topk > ROUTE_MAX || topk > groups_kept * (n_exp / groups)) {
        set_error("vb_route_experts: %d experts a token (at most %d) from %d of %d groups (at most %d) of %d experts",
                  topk, ROUTE_MAX, groups_kept, groups, ROUTE_MAX, n_exp);
        return E_INVAL;
    }
    if ((scores != 0 && scores != 1) || (group_score != 0 && group_score != 1) || !(fabsf(scale) < INFINITY)) {
        set_error("vb_route_experts: scores %d and group_score %d are 0 or 1, the scale (%g) is finite", scores,
                  group_score, static_cast<double>(scale));
        return E_INVAL;
    }
    if (n_tokens == 0) return OK;
    if (!logits || !out_idx || !out_w) {
        set_error("vb_route_experts: null pointer");
        return E_INVAL;
    }
    RouteArgs a{};
    a.z = logits;
    a.bias = bias;
    a.ids = out_idx;
    a.w = out_w;
    a.ld = ld;
    a.tokens = n_tokens;
    a.experts = n_exp;
    a.topk = topk;
    // groups that all stay decide nothing
    a.groups = groups_kept < groups ? groups : 1;
    a.kept = groups_kept < groups ? groups_kept : 1;
    a.size = n_exp / a.groups;
    a.shift = 6;
    while ((64 >> a.shift) < a.groups) a.shift--;
    a.sigmoid = scores == 1;
    a.top2 = group_score == 1;
    a.renorm = renorm != 0;
    a.scale = scale;
    if (type == ELEM_F32) return route_type<ELEM_F32>(a, as_stream(stream));
    if (type == ELEM_F16) return route_type<ELEM_F16>(a, as_stream(stream));
    return route_type<ELEM_BF16>(a, as_stream(stream));
}
