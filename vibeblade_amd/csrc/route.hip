// Experts of every token from a router's logits z (E a token):
//
//   s_e = softmax(z)_e  or  sigmoid(z_e)
//   c_e = s_e + b_e     or, without a bias, z_e (of the same order)
//   of `groups` groups of consecutive experts the `kept` best ones stay, by the
//   largest c of each, or by the sum of its two largest s + b
//   the top k of their experts by (c descending, id ascending)
//   w_e = scale * s_e / (renorm ? sum of the chosen s : 1)
//
// Scores, choices and group sums are 64 bits: which of two experts comes first
// is an id, and no two programs agree on it where c is rounded to fp32 (of
// 16384 tokens of 256 experts one or two have two choices within 2^-23).
//
// An expert whose logit (or bias) is -inf is never chosen: where there are not
// enough others the id is -1 and the weight 0.  A token with a NaN logit (or
// choice), or +inf under softmax, has ids -1 and weights NaN.
//
// One wave a token.  The lanes hold the experts in order: 64 / G' lanes a group
// (G' = the number of groups, rounded up to a power of two) and V experts a
// lane, so that a group's lanes are a butterfly of their own and a lower lane
// has lower ids.  A round takes the wave's largest choice (a maximum needs no
// id beside it), then the lowest lane that holds it, then its first place.
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

// The sum of the two largest (a >= b) of a group's 1 << shift lanes, in each of
// them.  -inf: none; one alone counts for itself.
__device__ __forceinline__ double group_top2(double a, double b, int shift) {
    for (int s = 0; s < shift; s++) {
        const double oa = __shfl_xor(a, 1 << s, 64), ob = __shfl_xor(b, 1 << s, 64);
        b = fmax(fmin(a, oa), fmax(b, ob));
        a = fmax(a, oa);
    }
    return a + (b > -INFINITY ? b : 0.0);
}

template <typename T>
__device__ __forceinline__ T group_largest(T v, int shift) {
    for (int s = 0; s < shift; s++) v = larger(v, __shfl_xor(v, 1 << s, 64));
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

// T: what the choice is held in, float where it is the logit itself and double
// where it is a score with a bias, or groups go by sums of scores.
template <int TYPE, int V, typename T>
__global__ void __launch_bounds__(64 * ROUTE_WAVES) route_kernel(RouteArgs a) {
    constexpr bool SCORED = sizeof(T) == 8;
    const Exp2 exp2;
    const int lane = static_cast<int>(threadIdx.x) & 63;
    const int group = lane >> a.shift, first = (lane & ((1 << a.shift) - 1)) * V;
    const int here = group < a.groups && a.size > first ? (a.size - first < V ? a.size - first : V) : 0;
    const int base = group * a.size + first;
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
        double s[V], sum = 1.0;
        if (SCORED || (!a.sigmoid && !a.renorm)) {
            double part = 0.0;
#pragma unroll
            for (int v = 0; v < V; v++) {
                s[v] = z[v] > -INFINITY ? score(z[v]) : 0.0;
                part += s[v];
            }
            if (!a.sigmoid) sum = wave_sum64(part);
        }
        T c[V];
        if constexpr (SCORED) {
            double value[V];
#pragma unroll
            for (int v = 0; v < V; v++) {
                const float b = a.bias && v < here ? a.bias[base + v] : 0.f;
                value[v] = z[v] > -INFINITY ? (a.sigmoid ? s[v] : s[v] / sum) + static_cast<double>(b) : -INFINITY;
                bad = bad || value[v] != value[v];
                c[v] = a.bias ? value[v] : static_cast<double>(z[v]);
            }
            if (a.kept < a.groups) {
                T mine;
                if (a.top2) {
                    double x = -INFINITY, y = -INFINITY;
#pragma unroll
                    for (int v = 0; v < V; v++) {
                        y = fmax(y, fmin(x, value[v]));
                        x = fmax(x, value[v]);
                    }
                    mine = group_top2(x, y, a.shift);
                } else {
                    mine = c[0];
#pragma unroll
                    for (int v = 1; v < V; v++) mine = larger(mine, c[v]);
                    mine = group_largest(mine, a.shift);
                }
                const bool stays = group_stays(a, mine, group);
#pragma unroll
                for (int v = 0; v < V; v++) c[v] = stays ? c[v] : -INFINITY;
            }
        } else {
#pragma unroll
            for (int v = 0; v < V; v++) c[v] = z[v];
            if (a.kept < a.groups) {
                T mine = c[0];
#pragma unroll
                for (int v = 1; v < V; v++) mine = larger(mine, c[v]);
                const bool stays = group_stays(a, group_largest(mine, a.shift), group);
#pragma unroll
                for (int v = 0; v < V; v++) c[v] = stays ? c[v] : -INFINITY;
            }
        }
        int id = -1;
        float mine_z = -INFINITY;
        const bool none = __any(bad);
        if (!none) {
            for (int r = 0; r < a.topk; r++) {
                T most = c[0];
#pragma unroll
                for (int v = 1; v < V; v++) most = larger(most, c[v]);
                const T best = wave_largest(most);
                if (best == -INFINITY) break;  // no expert is left
                const int owner = __ffsll(static_cast<unsigned long long>(__ballot(most == best))) - 1;
                int at = 0;
                float zat = z[0];
#pragma unroll
                for (int v = V - 1; v >= 0; v--) {
                    at = c[v] == best ? v : at;
                    zat = c[v] == best ? z[v] : zat;
                }
#pragma unroll
                for (int v = 0; v < V; v++) c[v] = lane == owner && v == at ? -INFINITY : c[v];
                const int chosen = __builtin_amdgcn_readlane(base + at, owner);
                const float chosen_z = lane_value(zat, owner);
                if (lane == r) {
                    id = chosen;
                    mine_z = chosen_z;
                }
            }
        }
        double w = id >= 0 ? score(mine_z) : 0.0;
        if (a.renorm) sum = wave_sum64(w);
        w = w > 0.0 ? w / sum : 0.0;  // (all chosen scores 0: weights 0)
        if (lane < a.topk) {
            a.ids[token * a.topk + lane] = id;
            a.w[token * a.topk + lane] = none ? NAN : static_cast<float>(static_cast<double>(a.scale) * w);
        }
    }
}

template <int TYPE, int V>
int route_launch(const RouteArgs& a, hipStream_t st) {
    const int64_t want = (a.tokens + ROUTE_WAVES - 1) / ROUTE_WAVES;
    const uint32_t grid = static_cast<uint32_t>(want < (1 << 20) ? want : 1 << 20);
    if (a.bias || (a.top2 && a.kept < a.groups)) route_kernel<TYPE, V, double><<<grid, 64 * ROUTE_WAVES, 0, st>>>(a);
    else route_kernel<TYPE, V, float><<<grid, 64 * ROUTE_WAVES, 0, st>>>(a);
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
