/*
 * moe_route_scores.hip - the experts of each token and their weights, for the routers that qlin_moe_route_dev does not cover: softmax or
 * sigmoid scores, a bias on the choice, groups of experts, weights renormalised or not.
 *
 *   s_e = exp(x_e - max) / sum exp(x - max)   or   1 / (1 + exp(-x_e))
 *   c_e = s_e + bias_e; without a bias the experts' order is that of their logits
 *   the n_group_used groups with the largest sum of their group_top largest c stay, of those the top_k largest c are chosen;
 *   equal ones by index; w_e = scale s_e (divided by the chosen ones' sum).
 *
 * The choice is the one of 64-bit values, also where two experts lie next to each other. Logits are read once and 8 top_k bytes a token written: 16384
 * tokens of 256 experts, 17.8 MB, would take 3.5 us at the 5.12 TB/s of a copy. What takes the time is the choice itself, one place after the other, each a
 * chain of some 15 dependent moves and comparisons, and the order of a lane's experts: a wave of its own for a token took 78 us there, 16 lanes for a token take 18 us (sigmoid, a
 * bias, 4 of 8 groups, 8 places; 24 us for 16 places, 106 for 17 by a wave to a token). Vector instructions are issued in 76% of the busy cycles there, 1470 by a wave (four
 * tokens). A single token takes 4.8 us, of which 2 are the launch.
 *   moe_route_row_kernel (16 lanes to a token) takes up to 512 experts and 16 places, where groups are 1, 2, 4 or 8 whole lanes: 35 us for 16384
 * tokens of 512 experts; moe_route_any_kernel (a wave to a token) all else: 96 us for 528 experts.
 */
#include "qlin_device.h"
#include "qlin_internal.h"

#include <cfloat>
#include <type_traits>

namespace qlin {

namespace {

struct Bf16 { uint16_t bits; };
__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(_Float16 v) { return (float)v; }
__device__ __forceinline__ float to_f32(Bf16 v) { return __uint_as_float((uint32_t)v.bits << 16); }

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) v += __shfl_xor(v, off, 64);
    return v;
}
/* the largest of the lanes' (v, i), of equal ones the one with the lowest i; every lane gets it */
__device__ __forceinline__ void wave_best(double &v, int &i) {
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) {
        const double ov = __shfl_xor(v, off, 64);
        const int oi = __shfl_xor(i, off, 64);
        if (ov > v || (ov == v && oi < i)) {
            v = ov;
            i = oi;
        }
    }
}

/* a logit's score; max and sum belong to the softmax */
__device__ __forceinline__ double score_of(int kind, double x, double max, double sum) {
    if (kind == 0) return (x == max ? 1.0 : exp(x - max)) / sum; /* infinities share the weight */
    const double e = exp(-fabs(x));
    return (x >= 0 ? 1.0 : e) / (1.0 + e);
}
/* What renormalised weights are made of: the chosen scores over exp(base), which the division takes out again. The base is the largest of the chosen logits, in a
 * sigmoid only below 0, where a score is exp(x) / (1 + exp(x)): so one term is between 1/2 and 1 however small the scores themselves are (all
 * of them below fp32 from logits of -104 down, or in a softmax whose largest logits a bias took out). Scores are 64-bit values: from e^-745.13 down they are 0,
 * and a token all of whose chosen scores are has the weights 0, which an infinite base gives. max is the softmax's. */
__device__ __forceinline__ float base_of(int kind, float largest, float max) {
    if ((kind == 0 ? largest - max : largest) < -745.1332f) return INFINITY;
    return kind == 0 ? largest : fminf(largest, 0.0f);
}
__device__ __forceinline__ double over_base(int kind, double x, double base) {
    const double e = x == base ? 1.0 : exp(x - base); /* infinities share the weight */
    if (kind == 0) return e;
    return x >= 0 ? 1.0 / (1.0 + exp(-x)) : e / (1.0 + exp(x));
}

/* A token by one wave, its experts' 64-bit values in LDS: any number of experts, places and groups. Bound by the chain of a place: six moves of a
 * 64-bit value and an index between lanes (1 token of 128 experts, 17 places: 17 us). */
template <class X>
__global__ void __launch_bounds__(64)
moe_route_any_kernel(RouteCall c) {
    extern __shared__ double key[]; /* [n_expert], then [n_group] */
    double *of_group = key + c.n_expert;
    const int lane = threadIdx.x;
    const X *x = static_cast<const X *>(c.logits) + (size_t)blockIdx.x * c.ld;
    const size_t out = (size_t)blockIdx.x * c.top_k;
    const double none = -INFINITY;
    double max = none, sum = 0.0;
    for (int e = lane; e < c.n_expert; e += 64) {
        const double v = to_f32(x[e]);
        key[e] = v > none ? v : none; /* (a NaN compares false) */
        max = fmax(max, key[e]);
    }
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) max = fmax(max, __shfl_xor(max, off, 64));
    if (c.score == 0) {
        for (int e = lane; e < c.n_expert; e += 64)
            if (key[e] > none) sum += key[e] == max ? 1.0 : exp(key[e] - max);
        sum = wave_sum(sum);
    }
    if (c.bias)
        for (int e = lane; e < c.n_expert; e += 64) {
            const double v = key[e] > none ? score_of(c.score, key[e], max, sum) + (double)c.bias[e] : none;
            key[e] = v > none ? v : none;
        }
    __syncthreads();
    if (c.n_group_used < c.n_group) {
        const int per = c.n_expert / c.n_group;
        for (int g = lane; g < c.n_group; g += 64) {
            double first = none, second = none;
            for (int e = g * per; e < (g + 1) * per; e++) {
                const double v = key[e];
                second = fmax(second, fmin(first, v));
                first = fmax(first, v);
            }
            if (c.group_top > 1 && first > none) {
                if (!c.bias) {
                    first = score_of(c.score, first, max, sum);
                    if (second > none) second = score_of(c.score, second, max, sum);
                }
                if (second > none) first += second;
            }
            of_group[g] = first;
        }
        __syncthreads();
        for (int n = 0; n < c.n_group_used; n++) {
            double best = none;
            int at = 0x7FFFFFFF;
            for (int g = lane; g < c.n_group; g += 64)
                if (of_group[g] > best) {
                    best = of_group[g];
                    at = g;
                }
            wave_best(best, at);
            if (at == 0x7FFFFFFF) break; /* uniform: no group is left with an expert */
            __syncthreads();
            if (lane == 0) of_group[at] = NAN; /* stays */
            __syncthreads();
        }
        for (int e = lane; e < c.n_expert; e += 64) {
            const double v = of_group[e / per];
            if (v == v) key[e] = none;
        }
        __syncthreads();
    }
    float largest = -INFINITY; /* of the chosen logits */
    for (int n = 0; n < c.top_k; n++) {
        double best = none;
        int at = 0x7FFFFFFF;
        for (int e = lane; e < c.n_expert; e += 64)
            if (key[e] > best) {
                best = key[e];
                at = e;
            }
        wave_best(best, at);
        const bool found = at != 0x7FFFFFFF;
        double w = 0.0;
        if (found) {
            const float logit = to_f32(x[at]);
            largest = fmaxf(largest, logit);
            if (!c.renorm) w = score_of(c.score, (double)logit, max, sum) * (double)c.scale;
            if ((at & 63) == lane) key[at] = none; /* its own to look at in the next round */
        }
        if ((n & 63) == lane) {
            c.idx[out + n] = found ? at : -1;
            c.w[out + n] = (float)w;
        }
    }
    if (!c.renorm) return;
    const double base = base_of(c.score, largest, (float)max);
    double total = 0.0;
    auto places = [&](auto see) { /* the lane's own that hold an expert, which it wrote itself */
        for (int n = lane; n < c.top_k; n += 64) {
            const int at = c.idx[out + n];
            if (at >= 0) see(n, over_base(c.score, (double)to_f32(x[at]), base));
        }
    };
    places([&](int, double s) { total += s; });
    total = wave_sum(total);
    places([&](int n, double s) { c.w[out + n] = total > 0.0 ? (float)(s / total * (double)c.scale) : 0.0f; });
}

/* ------------------------------------------------------------------ up to 512 experts and 16 places */

template <int CTRL> __device__ __forceinline__ int mov(int v) { return __builtin_amdgcn_mov_dpp(v, CTRL, 0xf, 0xf, true); }
template <int CTRL> __device__ __forceinline__ float mov(float v) { return __int_as_float(mov<CTRL>(__float_as_int(v))); }
template <int CTRL> __device__ __forceinline__ double mov(double v) { return __hiloint2double(mov<CTRL>(__double2hiint(v)), mov<CTRL>(__double2loint(v))); }
constexpr int kSwap1 = 0xB1, kSwap2 = 0x4E, kMirror8 = 0x141, kMirror16 = 0x140; /* the four moves after which each of 16 lanes has seen all others */
template <class T, class F> __device__ __forceinline__ T row_all(T v, F f) {
    v = f(v, mov<kSwap1>(v));
    v = f(v, mov<kSwap2>(v));
    v = f(v, mov<kMirror8>(v));
    return f(v, mov<kMirror16>(v));
}
__device__ __forceinline__ float row_max(float v) { return row_all(v, [](float a, float b) { return fmaxf(a, b); }); }
__device__ __forceinline__ float row_sum(float v) { return row_all(v, [](float a, float b) { return a + b; }); }
__device__ __forceinline__ double row_sum(double v) { return row_all(v, [](double a, double b) { return a + b; }); }

/* exp in 64 bits for arguments up to 0, to about 2^-52: 2^n exp(r), r to degree 12 of its series; 0 below the least number */
__device__ __forceinline__ double exp_to_one(double x) {
    if (!(x > -745.2)) return 0.0;
    const double n = rint(x * 1.4426950408889634);
    double r = fma(n, -0.6931471805599453, x);
    r = fma(n, -2.3190468138462996e-17, r);
    double p = 1.0 / 479001600;
    p = fma(p, r, 1.0 / 39916800);
    p = fma(p, r, 1.0 / 3628800);
    p = fma(p, r, 1.0 / 362880);
    p = fma(p, r, 1.0 / 40320);
    p = fma(p, r, 1.0 / 5040);
    p = fma(p, r, 1.0 / 720);
    p = fma(p, r, 1.0 / 120);
    p = fma(p, r, 1.0 / 24);
    p = fma(p, r, 1.0 / 6);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0);
    return ldexp(p, (int)n);
}
__device__ __forceinline__ double quotient(double a, double b) { /* b from 1 up */
    double r = __builtin_amdgcn_rcp(b);
    r = fma(fma(-b, r, 1.0), r, r);
    r = fma(fma(-b, r, 1.0), r, r);
    const double q = a * r;
    return fma(fma(-b, q, a), r, q);
}

/* keeps what is computed of x in the branch that asks for it: the compiler would do it for every token, ahead of a loop */
__device__ __forceinline__ float here(float x) {
    asm volatile("" : "+v"(x));
    return x;
}

/* 16 lanes to a token, N experts to a lane in registers (its next `per`), a place of the result in each of the 16 lanes.
 *   Without a bias the experts' order is that of their logits, which fp32 holds. With one, values are computed in fp32, and where one lies so close to
 * the largest that their errors could change the order (`away`), those that do are computed once more in 64 bits: the choice is always the one of
 * 64-bit values, and hardly a wave has to. Groups go the same way, by the sum of their largest values.
 *   A pick: the lanes' largest, the largest of 16 lanes by four moves between lanes, the first lane and in it the first expert that has it. */
template <class X, int N, bool BIAS>
__global__ void __launch_bounds__(256, N <= 16 ? 4 : 2)
moe_route_row_kernel(RouteCall c, int per, int group_lanes) {
    const int lane = threadIdx.x & 15;
    const long long row = (long long)blockIdx.x * 16 + threadIdx.x / 16;
    if (row - (threadIdx.x & 48) / 16 >= c.n_tok) return; /* none of the wave's */
    const bool there = row < c.n_tok;
    const X *x = static_cast<const X *>(c.logits) + (size_t)(there ? row : c.n_tok - 1) * c.ld;
    const int e0 = lane * per, n = c.n_expert - e0 < per ? c.n_expert - e0 : per; /* the lane's experts: e0 .. e0 + n - 1 */
    const float none = -INFINITY;
    float v[N], key[N];
    constexpr int kVec = 16 / sizeof(X);
    const bool whole = c.n_expert % per == 0;
    if (per % kVec == 0 && whole && ((uintptr_t)c.logits & 15) == 0 && (size_t)c.ld * sizeof(X) % 16 == 0) {
        struct alignas(16) Vec { X v[kVec]; };
#pragma unroll
        for (int j = 0; j < N; j += kVec) {
            Vec w = {};
            if (j < n) w = *reinterpret_cast<const Vec *>(x + e0 + j);
#pragma unroll
            for (int i = 0; i < kVec && j + i < N; i++) v[j + i] = j + i < n ? to_f32(w.v[i]) : none;
        }
    } else {
#pragma unroll
        for (int j = 0; j < N; j++) v[j] = j < n ? to_f32(x[e0 + j]) : none;
    }
    if constexpr (BIAS) {
        if (per % 4 == 0 && whole && ((uintptr_t)c.bias & 15) == 0) {
#pragma unroll
            for (int j = 0; j < N; j += 4) {
                float4 w = {};
                if (j < n) w = *reinterpret_cast<const float4 *>(c.bias + e0 + j);
                key[j] = w.x;
                key[j + 1] = w.y;
                key[j + 2] = w.z;
                key[j + 3] = w.w;
            }
        } else {
#pragma unroll
            for (int j = 0; j < N; j++) key[j] = j < n ? c.bias[e0 + j] : none;
        }
    }
    float most = none;
#pragma unroll
    for (int j = 0; j < N; j++) {
        v[j] = v[j] > none ? v[j] : none; /* (a NaN compares false) */
        most = fmaxf(most, v[j]);
    }
    most = row_max(most);
    constexpr float kLog2e = 1.44269504088896341f;
    auto power = [&](float x) { return x == most ? 1.0f : __builtin_amdgcn_exp2f((x - most) * kLog2e); }; /* (infinities share) */
    float sum = 1.0f; /* of the softmax */
    if (c.score == 0) {
        sum = 0.0f;
#pragma unroll
        for (int j = 0; j < N; j++) sum += v[j] > none ? power(v[j]) : 0.0f;
        sum = row_sum(sum);
    }
    /* in 64 bits; every lane of the row takes part in the sum */
    auto below = [&](float x) { return x == most ? 0.0 : (double)x - (double)most; };
    auto sum64 = [&]() {
        double s = 1.0;
        if (c.score == 0) {
            s = 0.0;
#pragma unroll
            for (int j = 0; j < N; j++) {
                const float x = here(v[j]);
                s += x > none ? exp_to_one(below(x)) : 0.0;
            }
            s = row_sum(s);
        }
        return s;
    };
    auto score64 = [&](float x, double sum64) { /* of an expert that is there */
        const double e = exp_to_one(c.score == 0 ? below(x) : -fabs((double)x));
        return quotient(c.score == 0 || x < 0.0f ? e : 1.0, c.score == 0 ? sum64 : 1.0 + e);
    };
    /* how far an fp32 value may be from another to be taken for it: twice their error. A sigmoid's is below 4e-7 (argument, exponential and reciprocal), a
     * softmax's 2e-6 of itself (the sum's most of all), and no score is above 1 / sum; adding the bias rounds by 2^-24 */
    float away = 0.0f;
    /* (and the lowest value that is one: experts that are not there have -infinity, which a lowest value less that would be) */
    auto threshold = [&](float m) { return !BIAS || m == INFINITY ? m : fmaxf(m - (away + 2.4e-7f * fabsf(m)), -FLT_MAX); };
    if constexpr (BIAS) {
        const float inverse = __builtin_amdgcn_rcpf(sum);
        away = c.score == 0 ? 4e-6f * inverse : 8e-7f;
        auto values = [&](auto score) {
#pragma unroll
            for (int j = 0; j < N; j++) {
                const float value = score(v[j]) + key[j];
                key[j] = v[j] > none && value > none ? value : none;
            }
        };
        if (c.score == 0) values([&](float x) { return power(x) * inverse; });
        else values([&](float x) { return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * -kLog2e)); });
    } else {
#pragma unroll
        for (int j = 0; j < N; j++) key[j] = v[j];
    }
    /* the lane's four largest in order, equal ones by index, and which they are; `gone` has a bit for each that is picked */
    float top = none, next = none, third = none, fourth = none;
    int at = 0, next_at = 0, third_at = 0, fourth_at = 0;
    uint32_t gone = 0;
    auto rank = [&](auto some_gone) {
        top = next = third = fourth = none;
#pragma unroll
        for (int j = 0; j < N; j++) {
            const float k = decltype(some_gone)::value && (gone >> j) & 1 ? none : key[j];
            const bool a = k > top, b = k > next, d = k > third, e = k > fourth;
            fourth_at = d ? third_at : e ? j : fourth_at;
            third_at = b ? next_at : d ? j : third_at;
            next_at = a ? at : b ? j : next_at;
            at = a ? j : at;
            fourth = __builtin_amdgcn_fmed3f(third, fourth, k);
            third = __builtin_amdgcn_fmed3f(next, third, k);
            next = __builtin_amdgcn_fmed3f(top, next, k);
            top = fmaxf(top, k);
        }
    };
    rank(std::false_type{});
    if (group_lanes) {
        bool kept;
        float first = top, second = next; /* of the group */
        auto join = [&](auto &a, auto &b, auto c, auto d) {
            b = fmax(fmin(a, c), fmax(b, d));
            a = fmax(a, c);
        };
        auto join_lanes = [&](auto &a, auto &b) {
            if (group_lanes > 1) join(a, b, mov<kSwap1>(a), mov<kSwap1>(b));
            if (group_lanes > 2) join(a, b, mov<kSwap2>(a), mov<kSwap2>(b));
            if (group_lanes > 4) join(a, b, mov<kMirror8>(a), mov<kMirror8>(b));
        };
        join_lanes(first, second);
        auto look = [&](auto see) { /* at the other groups of the row, and the lane of each */
#define QLIN_LOOK(N_) \
    if ((N_) % group_lanes == 0) see([](auto w) { return mov<0x120 + (N_)>(w); });
            QLIN_LOOK(1) QLIN_LOOK(2) QLIN_LOOK(3) QLIN_LOOK(4) QLIN_LOOK(5) QLIN_LOOK(6) QLIN_LOOK(7) QLIN_LOOK(8)
            QLIN_LOOK(9) QLIN_LOOK(10) QLIN_LOOK(11) QLIN_LOOK(12) QLIN_LOOK(13) QLIN_LOOK(14) QLIN_LOOK(15)
#undef QLIN_LOOK
        };
        bool close = false;
        if (BIAS) {
            const bool two = c.group_top > 1 && second > none;
            const float worth = two ? first + second : first;
            const float size = row_max(first > none ? fabsf(first) + (two ? fabsf(second) : 0.0f) : 0.0f), apart = 2.0f * away + 5e-7f * size;
            int surely = 0, maybe = 0;
            look([&](auto other) {
                const float w = other(worth);
                surely += w - worth > apart ? 1 : 0;
                maybe += w - worth >= -apart ? 1 : 0;
            });
            kept = surely < c.n_group_used;
            close = first > none && (!(apart < INFINITY) || (kept && maybe >= c.n_group_used));
        }
        if (!BIAS || __ballot(close)) { /* by 64-bit values, equal ones by index */
            double a = top, b = next;
            double s64 = 1.0;
            if (BIAS || c.group_top > 1) s64 = sum64();
            if constexpr (BIAS) {
                a = b = none;
                const float least = next > none ? threshold(next) : top > none ? threshold(top) : INFINITY;
#pragma unroll
                for (int j = 0; j < N; j++)
                    if (__ballot(key[j] >= least)) {
                        const double d = key[j] >= least ? score64(here(v[j]), s64) + (double)c.bias[e0 + j] : (double)none;
                        b = fmax(b, fmin(a, d));
                        a = fmax(a, d);
                    }
            }
            join_lanes(a, b);
            double worth = a;
            if (c.group_top > 1 && a > (double)none) {
                if constexpr (!BIAS) {
                    worth = score64((float)a, s64);
                    if (b > (double)none) worth += score64((float)b, s64);
                } else if (b > (double)none) {
                    worth += b;
                }
            }
            int before = 0;
            look([&](auto other) {
                const double w = other(worth);
                const int from = other(lane); /* (with all lanes) */
                before += w > worth || (w == worth && from < lane) ? 1 : 0;
            });
            kept = before < c.n_group_used;
        }
        if (!kept) {
            gone = ~0u;
            top = next = third = fourth = none;
        }
    }
    int pick = -1; /* of place `lane` */
    const int shift = threadIdx.x & 48; /* the row's 16 bits of a ballot */
    auto of_row = [&](bool b) { return (uint32_t)(__ballot(b) >> shift) & 0xFFFFu; };
    int left_in_list = 4;
    constexpr int kRankAt = BIAS ? 1 : 0; /* (where values may be close, the one behind the first has to be known) */
    for (int k = 0; k < c.top_k; k++) {
        const float m = row_max(top);
        uint32_t lanes;
        bool looked = false; /* at all experts once more */
        int which = at;
        if constexpr (BIAS) {
            const float least = threshold(m);
            lanes = of_row(top >= least);
            looked = __ballot(next >= least || (lanes & (lanes - 1))); /* several that could be the largest */
            if (looked) {
                double best = none;
                const double s64 = sum64();
#pragma unroll
                for (int j = 0; j < N; j++) {
                    const bool may = key[j] >= least && !((gone >> j) & 1);
                    if (__ballot(may)) {
                        const double d = may ? score64(here(v[j]), s64) + (double)c.bias[e0 + j] : (double)none;
                        which = d > best ? j : which;
                        best = fmax(best, d);
                    }
                }
                const double row_best = row_all(best, [](double a, double b) { return fmax(a, b); });
                lanes = of_row(best > (double)none && best == row_best);
            }
        } else {
            lanes = of_row(top == m && m > none);
        }
        const int winner = __builtin_ctz(lanes | 0x10000u); /* 16: nothing is left */
        const int chosen = __shfl(e0 + which, winner & 15, 16);
        if (lane == k) pick = winner < 16 ? chosen : -1;
        const bool mine = winner == lane;
        if (mine) {
            gone |= 1u << which;
            left_in_list--;
        }
        if (looked || (N > 4 && __ballot(left_in_list <= kRankAt))) {
            rank(std::true_type{});
            left_in_list = 4;
        } else {
            top = mine ? next : top;
            next = mine ? third : next;
            third = mine ? fourth : third;
            fourth = mine ? none : fourth;
            at = mine ? next_at : at;
            next_at = mine ? third_at : next_at;
            third_at = mine ? fourth_at : third_at;
        }
    }
    float w = 0.0f;
    const float p = pick >= 0 ? to_f32(x[pick]) : none;
    const float base = c.renorm ? base_of(c.score, row_max(p), most) : c.score == 0 ? most : 0.0f;
    if (pick >= 0) { /* as over_base, in fp32 */
        const float e = expf(c.score != 0 ? -fabsf(p) : p == base ? 0.0f : p - base);
        if (c.score == 0) {
            w = c.renorm ? e : e / sum;
        } else {
            float over = p >= 0.0f ? 1.0f : e;
            if (base != 0.0f) over = expf(p - base);
            w = over / (1.0f + e);
        }
    }
    if (c.renorm) {
        const float total = row_sum(w);
        if (total > 0.0f) w /= total;
    }
    if (there && lane < c.top_k) {
        c.idx[row * c.top_k + lane] = pick;
        c.w[row * c.top_k + lane] = w * c.scale;
    }
}

template <class X, int N> void launch_rows(const RouteCall &c, int per, int group_lanes) {
    const dim3 grid((uint32_t)(((long long)c.n_tok + 15) / 16)), block(256);
    if (c.bias)
        hipLaunchKernelGGL((moe_route_row_kernel<X, N, true>), grid, block, 0, c.stream, c, per, group_lanes);
    else
        hipLaunchKernelGGL((moe_route_row_kernel<X, N, false>), grid, block, 0, c.stream, c, per, group_lanes);
}

template <class X> hipError_t launch_route(const RouteCall &c) {
    const int per = (c.n_expert + 15) / 16, of_group = c.n_expert / c.n_group;
    /* lanes to a group: 0 where all groups stay, else a power of two */
    const int group_lanes = c.n_group_used == c.n_group ? 0 : of_group % per ? -1 : of_group / per;
    if (c.top_k > 16 || per > 32 || (group_lanes && group_lanes != 1 && group_lanes != 2 && group_lanes != 4 && group_lanes != 8)) {
        const size_t lds = ((size_t)c.n_expert + c.n_group) * sizeof(double);
        hipLaunchKernelGGL(moe_route_any_kernel<X>, dim3(c.n_tok), dim3(64), lds, c.stream, c);
    } else if (per <= 4) {
        launch_rows<X, 4>(c, per, group_lanes);
    } else if (per <= 8) {
        launch_rows<X, 8>(c, per, group_lanes);
    } else if (per <= 16) {
        launch_rows<X, 16>(c, per, group_lanes);
    } else {
        launch_rows<X, 32>(c, per, group_lanes);
    }
    return hipGetLastError();
}

}  // namespace

hipError_t launch_moe_route_scores(uint32_t type, const RouteCall &c) {
    return type == T_F32 ? launch_route<float>(c) : type == T_F16 ? launch_route<_Float16>(c) : launch_route<Bf16>(c);
}

}  // namespace qlin
