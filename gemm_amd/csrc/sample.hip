/*
 * sample.hip - the next token of each sequence from its logits: temperature, top-k, top-p and min-p, and a random number that the
 * caller has drawn.
 *
 * Tokens stand in the order of their logits, largest first, equal ones by index; NaN and -infinity are not there. With T the
 * temperature, a token weighs w = exp((l - max l) / T). Top-k keeps the first k tokens, top-p the shortest run of those whose weights
 * reach p times their sum, min-p of those the tokens with w >= m (the largest has 1). The pick is the first kept token at which the
 * running sum of weights exceeds u times the sum of the kept.
 *
 * Nothing is sorted. A cut ("the k-th", "where the sum reaches s") is found by its value: floats map to unsigned keys of the same
 * order, and of the keys' 11 + 11 + 10 bits each pass over the row fixes the next by a histogram of counts and weights. Tokens
 * that share the value at a cut weigh the same, so how many of them stay is a division, and which one is picked a count by index.
 *
 * Weights are exp in 64 bits, as 64-bit integers of 2^-shift with shift such that a row of the largest weight does not overflow
 * (2^-45 at 152k tokens): borders between tokens lie closer to each other than fp32 sums resolve, and integer sums do not depend on
 * their order, so the same call gives the same token. A token below half a unit has no weight and is never picked, as one of 10^5 such
 * tokens would be once in 10^8 calls.
 */
#include "qlin_device.h"
#include "qlin_internal.h"

namespace qlin {

namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;

struct Bf16 { uint16_t bits; };
__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(_Float16 v) { return (float)v; }
__device__ __forceinline__ float to_f32(Bf16 v) { return __uint_as_float((uint32_t)v.bits << 16); }

constexpr float kMinusInf = -__builtin_inff();
__device__ __forceinline__ bool is_there(float v) { return v > kMinusInf; } /* false for NaN */

/* larger floats have larger keys, both zeros the same; 0 is no float's */
__device__ __forceinline__ uint32_t key_of(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k); }

struct Weights {
    float max;
    double per_t; /* 1 / T */
    double unit;  /* 2^shift */
    __device__ double real(float v) const {
        if (v == max) return 1.0;
        if (max == -kMinusInf) return 0.0;
        return exp(((double)v - (double)max) * per_t);
    }
    __device__ uint64_t operator()(float v) const { return (uint64_t)__double2ull_rn(real(v) * unit); }
};

struct Sum { uint32_t count; uint64_t weight; };
__device__ __forceinline__ Sum operator+(Sum a, Sum b) { return {a.count + b.count, a.weight + b.weight}; }

__device__ __forceinline__ uint64_t shfl_u64(uint64_t v, int from) {
    return (uint64_t)__shfl((uint32_t)(v >> 32), from, 64) << 32 | __shfl((uint32_t)v, from, 64);
}

struct Shared {
    uint32_t count[2048];
    uint64_t weight[2048];
    Sum wave[kWaves];
    float wave_max[kWaves];
    uint32_t digit;
    Sum above;
    int picked;
};

__device__ float max_of_workgroup(float v, Shared &s) {
    for (int off = 32; off; off >>= 1) v = fmaxf(v, __shfl_xor(v, off, 64));
    if ((threadIdx.x & 63) == 0) s.wave_max[threadIdx.x >> 6] = v;
    __syncthreads();
    v = s.wave_max[0];
    for (int w = 1; w < kWaves; w++) v = fmaxf(v, s.wave_max[w]);
    __syncthreads();
    return v;
}

/* sum of all threads' v, in every thread; `before`: of the threads before this one */
__device__ Sum sum_of_workgroup(Sum v, Shared &s, Sum *before) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    Sum run = v;
    for (int off = 1; off < 64; off <<= 1) {
        const Sum o = {(uint32_t)__shfl((int)run.count, max(lane - off, 0), 64), shfl_u64(run.weight, max(lane - off, 0))};
        if (lane >= off) run = run + o;
    }
    if (lane == 63) s.wave[wave] = run;
    __syncthreads();
    Sum total = {0, 0}, earlier = {0, 0};
    for (int w = 0; w < kWaves; w++) {
        if (w == wave) earlier = total;
        total = total + s.wave[w];
    }
    if (before) *before = {earlier.count + run.count - v.count, earlier.weight + run.weight - v.weight};
    __syncthreads();
    return total;
}

/* The value at which the running sum down the order reaches `target` (of counts or of weights; the row's sum does): its key, and the
 * sum over larger ones */
struct Cut { uint32_t key; Sum above; };
template <bool BY_WEIGHT, class T> __device__ Cut find_cut(const T *x, int n, const Weights &w, uint64_t target, Shared &s) {
    Cut c = {0, {0, 0}};
    for (int pass = 0; pass < 3; pass++) {
        const int low = pass == 0 ? 21 : pass == 1 ? 10 : 0, bins = pass == 2 ? 1024 : 2048;
        for (int i = threadIdx.x; i < 2048; i += kThreads) s.count[i] = 0, s.weight[i] = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < n; i += kThreads) {
            const float v = to_f32(x[i]);
            if (!is_there(v)) continue;
            const uint32_t k = key_of(v);
            if (pass && (pass == 1 ? k >> 21 : k >> 10) != c.key) continue;
            const uint32_t d = (k >> low) & (bins - 1);
            atomicAdd(&s.count[d], 1u);
            if (const uint64_t m = w(v)) atomicAdd((unsigned long long *)&s.weight[d], (unsigned long long)m);
        }
        __syncthreads();
        const int hi = 2047 - 2 * threadIdx.x; /* two bins per thread, the largest first */
        const Sum a = {s.count[hi], s.weight[hi]}, b = {s.count[hi - 1], s.weight[hi - 1]};
        Sum before;
        (void)sum_of_workgroup(a + b, s, &before);
        before = before + c.above;
        const Sum mid = before + a, after = mid + b;
        auto reached = [&](const Sum &v) { return (BY_WEIGHT ? v.weight : (uint64_t)v.count) >= target; };
        if (!reached(before) && reached(after)) {
            s.digit = reached(mid) ? hi : hi - 1;
            s.above = reached(mid) ? before : mid;
        }
        __syncthreads();
        c.key = c.key << (pass == 2 ? 10 : 11) | s.digit;
        c.above = s.above;
        __syncthreads();
    }
    return c;
}

/* index of the nth (from 1) element of value key k */
template <class T> __device__ int nth_of_value(const T *x, int n, uint32_t k, uint32_t nth, Shared &s) {
    const int per = (n + kWaves - 1) / kWaves, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int lo = min(wave * per, n), hi = min(lo + per, n);
    auto is = [&](int i) { return i < hi && is_there(to_f32(x[i])) && key_of(to_f32(x[i])) == k; };
    uint32_t mine = 0;
    for (int i = lo; i < hi; i += 64) mine += __popcll(__ballot(is(i + lane)));
    if (lane == 0) s.wave[wave].count = mine;
    __syncthreads();
    uint32_t before = 0;
    for (int w = 0; w < wave; w++) before += s.wave[w].count;
    if (before < nth && nth <= before + mine) {
        uint32_t seen = before;
        for (int i = lo; i < hi; i += 64) {
            const uint64_t b = __ballot(is(i + lane));
            const uint32_t upto = seen + __popcll(b & ((1ull << lane) - 1)) + 1; /* (of a lane that is one) */
            if ((b >> lane & 1) && upto == nth) s.picked = i + lane;
            seen += __popcll(b);
        }
    }
    __syncthreads();
    return s.picked;
}

template <class T>
__global__ void __launch_bounds__(kThreads)
sample_kernel(const T *__restrict__ logits, int n, size_t ld, const float *__restrict__ temperature, const int32_t *__restrict__ top_k,
              const float *__restrict__ top_p, const float *__restrict__ min_p, const float *__restrict__ u, int32_t *__restrict__ ids,
              float *__restrict__ probs, int shift) {
    __shared__ Shared s;
    const int seq = blockIdx.x;
    const T *x = logits + (size_t)seq * ld;
    const float t = temperature ? temperature[seq] : 1.0f;
    const int k = top_k ? top_k[seq] : 0;
    const float p = top_p ? top_p[seq] : 1.0f;
    const float m = min_p && min_p[seq] > 0.0f ? fminf(min_p[seq], 1.0f) : 0.0f;

    float best = kMinusInf;
    for (int i = threadIdx.x; i < n; i += kThreads) {
        const float v = to_f32(x[i]);
        if (is_there(v)) best = fmaxf(best, v);
    }
    Weights w;
    w.max = max_of_workgroup(best, s);
    if (!is_there(w.max)) {
        if (threadIdx.x == 0) {
            ids[seq] = -1;
            if (probs) probs[seq] = 0.0f;
        }
        return;
    }
    if (!(t > 0.0f) || k == 1) {
        const int at = nth_of_value(x, n, key_of(w.max), 1, s);
        if (threadIdx.x == 0) {
            ids[seq] = at;
            if (probs) probs[seq] = 1.0f;
        }
        return;
    }
    w.per_t = 1.0 / (double)t;
    w.unit = (double)(1ull << shift);

    Sum all = {0, 0};
    for (int i = threadIdx.x; i < n; i += kThreads) {
        const float v = to_f32(x[i]);
        if (is_there(v)) all = all + Sum{1, w(v)};
    }
    all = sum_of_workgroup(all, s, nullptr);

    uint32_t last = 0; /* key of the last kept token's value (0: everything is kept) */
    uint64_t total = all.weight;
    if (k > 0 && (uint32_t)k < all.count) {
        const Cut c = find_cut<false>(x, n, w, (uint64_t)k, s);
        last = c.key;
        total = c.above.weight + (k - c.above.count) * w(value_of(c.key));
    }
    if (p < 1.0f) {
        const uint64_t target = min(max((uint64_t)ceil(fmax((double)p, 0.0) * (double)total), (uint64_t)1), total);
        const Cut c = find_cut<true>(x, n, w, target, s);
        const uint64_t each = w(value_of(c.key)); /* not 0: the sum grows here */
        last = c.key;
        total = c.above.weight + (target - c.above.weight + each - 1) / each * each;
    }
    if (m > 0.0f && (last == 0 || w.real(value_of(last)) < (double)m)) {
        Sum kept = {0, 0};
        for (int i = threadIdx.x; i < n; i += kThreads) {
            const float v = to_f32(x[i]);
            if (is_there(v) && (v == w.max || (key_of(v) > last && w.real(v) >= (double)m))) kept = kept + Sum{1, w(v)};
        }
        total = sum_of_workgroup(kept, s, nullptr).weight;
    }
    const float draw = u[seq];
    uint64_t target = draw > 0.0f ? (uint64_t)fmin((double)draw * (double)total, 9.0e18) : 0;
    target = min(target, total - 1) + 1;
    const Cut c = find_cut<true>(x, n, w, target, s);
    const uint64_t each = w(value_of(c.key));
    const int at = nth_of_value(x, n, c.key, (uint32_t)((target - c.above.weight + each - 1) / each), s);
    if (threadIdx.x == 0) {
        ids[seq] = at;
        if (probs) probs[seq] = (float)((double)each / (double)total);
    }
}

template <class T> hipError_t sample(const SampleCall &c) {
    int shift = 62; /* n << shift stays below 2^63 */
    while (shift > 0 && ((uint64_t)c.n_vocab >> (62 - shift)) > 1) shift--;
    sample_kernel<T><<<c.n_seq, kThreads, 0, c.stream>>>(static_cast<const T *>(c.logits), c.n_vocab, (size_t)c.ld, c.temperature, c.top_k, c.top_p, c.min_p, c.u,
                                                        c.ids, c.probs, shift);
    return hipGetLastError();
}

}  // namespace

size_t sample_workspace_bytes(int n_seq, int n_vocab) {
    (void)n_seq;
    (void)n_vocab;
    return 0;
}

hipError_t launch_sample(uint32_t type, const SampleCall &c) {
    if (type == T_F32) return sample<float>(c);
    return type == T_F16 ? sample<_Float16>(c) : sample<Bf16>(c);
}

}  // namespace qlin
