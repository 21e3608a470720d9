/*
 * moe_route_scores.hip - the experts of each token and their weights, for the routers that qlin_moe_route_dev does not cover: softmax or
 * sigmoid scores, a bias on the choice, groups of experts, weights renormalised or not.
 *
 *   s_e = exp(x_e - max) / sum exp(x - max)   or   1 / (1 + exp(-x_e))
 *   c_e = s_e + bias_e; without a bias the experts' order is that of their logits
 *   the n_group_used groups with the largest sum of their group_top largest c stay, of those the top_k largest c are chosen;
 *   equal ones by index; w_e = scale s_e (divided by the chosen ones' sum).
 *
 * Scores and c are 64-bit here: the choice is the definition's also where two experts lie next to each other.
 */
#include "qlin_device.h"
#include "qlin_internal.h"

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

/* One wave per token, the experts' 64-bit values in LDS. */
template <class X>
__global__ void __launch_bounds__(64)
moe_route_scores_kernel(RouteCall c) {
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
    double total = 0.0;
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
        double s = 0.0;
        if (found) {
            s = score_of(c.score, (double)to_f32(x[at]), max, sum);
            if ((at & 63) == lane) key[at] = none; /* its own to look at in the next round */
        }
        total += s;
        if ((n & 63) == lane) {
            c.idx[out + n] = found ? at : -1;
            c.w[out + n] = (float)(c.renorm ? s : s * (double)c.scale);
        }
    }
    if (c.renorm && total > 0.0) /* what a lane wrote, with the chosen scores once more in 64 bits */
        for (int n = lane; n < c.top_k; n += 64) {
            const int at = c.idx[out + n];
            if (at >= 0) c.w[out + n] = (float)(score_of(c.score, (double)to_f32(x[at]), max, sum) / total * (double)c.scale);
        }
}

}  // namespace

hipError_t launch_moe_route_scores(uint32_t type, const RouteCall &c) {
    const size_t lds = ((size_t)c.n_expert + c.n_group) * sizeof(double);
    const dim3 grid(c.n_tok), block(64);
    if (type == T_F32)
        hipLaunchKernelGGL(moe_route_scores_kernel<float>, grid, block, lds, c.stream, c);
    else if (type == T_F16)
        hipLaunchKernelGGL(moe_route_scores_kernel<_Float16>, grid, block, lds, c.stream, c);
    else
        hipLaunchKernelGGL(moe_route_scores_kernel<Bf16>, grid, block, lds, c.stream, c);
    return hipGetLastError();
}

}  // namespace qlin
