/*
 * sample.hip - the next token of each sequence from its logits: temperature, top-k, top-p and min-p, and a random number that the
 * caller has drawn.
 *
 * Tokens stand in the order of their logits, largest first, equal ones by index; NaN and -infinity are not there. With T the
 * temperature, a token weighs w = exp((l - max l) / T). Top-k keeps the first k tokens, top-p the shortest run of those whose weights
 * reach p times their sum, min-p of those the tokens with w >= m (the largest has 1). The pick is the first kept token at which the
 * running sum of weights exceeds u times the sum of the kept.
 *
 * A row is not sorted. Its tokens fall into 2048 bins by their distance from the largest logit, in bins of 1/64 of the temperature (of
 * 1/2040 of the row's range where that is finer); what is further away than 2046 bins weighs less than 1.3e-14 and is not counted.
 * Sums over the bins say in which bin a cut lies - the k-th token, p times the sum, the smallest weight, u times the sum - or, as
 * long as an earlier cut inside a bin leaves a sum open, in which few of them. Only the tokens of those bins are listed and sorted (from
 * one to a few hundred of 150000), and the cuts are made exactly on the list. With top_k of up to 1024 all kept tokens fit the list, and the
 * bins hold counts instead of weights; with top_k of up to 512 what the threads read largest says enough, and the bins hold only that.
 *   One pass over the row finds the largest and smallest logit, one fills the bins, one lists; the second and third read from LDS and the
 * caches what the first brought, and a row with top_k up to 512 makes the first alone.
 *
 * Weights and sums are 64-bit: the borders between tokens lie closer to each other than fp32 sums resolve, and the token is to be the
 * one that the definition gives. A bin's weight is exp(centre) times the sum of exp(offset from the centre), offsets up to 1/128, so
 * that a token costs a polynomial of degree 4 instead of an exponential; the sum is of integers of 2^-40, which do not depend on
 * the order of the additions: the same call gives the same token. A bin's sum is off by 2^-41 of itself for the rounding and 2.4e-13 for
 * the polynomial (of n tokens above 2^21, whose sums must stay within 64 bits, by 2^-62 to 2^-61 n), and all sums lack what is too far down
 * for a bin, at most 1.3e-14 n.
 *   A list that overflows leaves the row to sample_by_value, which takes three passes over it for each cut: rows of equal logits, of 16-bit
 * logits so large that few values lie near the top, of which a finite mask leaves the others a few bins. 256 rows of 128256 bf16
 * logits of one value 0.5 to 0.8 ms, around -30 instead of 0 0.3 ms, 0.46 with top-p (by 64-bit integer weights of the whole row 1.0 to
 * 2.4, 0.48 and 0.86).
 *
 * What bounds it, 256 rows of 128256 bf16 logits without filters, 67 us, by the clock in the kernel: 11 us for the first pass (6 TB/s), 21 for
 * the bins (14 64-bit vector instructions and an LDS addition per token), 14 for the list (what LDS does not hold of the row comes from the
 * last-level cache again), 9 for sums, sort and cuts, which are chains of a few hundred instructions; the rest is how far the workgroups'
 * starts and ends lie apart. With top_k 40, 24 us: 9 for the first pass, 2 for the bins of the threads' largest, 3 for the list, 5 for the
 * rest. A row alone is bound by what one compute unit loads and executes (9 rows of 151936 fp32 logits with top_k 40 19 us, one 22 with the
 * two launches that such a row leaves empty, 16 bf16 rows without top_k 55, one 36 by several workgroups).
 */
#include "qlin_device.h"
#include "qlin_internal.h"

namespace qlin {

namespace {

constexpr int kThreads = kSampleThreads, kWaves = kThreads / 64;

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

/* values that are the same in all lanes, into scalar registers: a row's bins and cuts would otherwise hold half of the 128 vector registers
 * that 1024 threads have each */
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)v); }
__device__ __forceinline__ float uniform(float v) { return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(v))); }
__device__ __forceinline__ double uniform(double v) {
    const uint64_t b = (uint64_t)__double_as_longlong(v);
    return __longlong_as_double((long long)((uint64_t)uniform((uint32_t)(b >> 32)) << 32 | uniform((uint32_t)b)));
}

/* a sequence's settings */
struct Settings {
    float t, p, m, u;
    int k;
};
__device__ __forceinline__ Settings settings_of(const SampleCall &c, int seq) {
    Settings s;
    s.t = c.temperature ? c.temperature[seq] : 1.0f;
    s.k = c.top_k ? c.top_k[seq] : 0;
    s.p = c.top_p ? c.top_p[seq] : 1.0f;
    s.m = c.min_p && c.min_p[seq] > 0.0f ? fminf(c.min_p[seq], 1.0f) : 0.0f;
    const float u = c.u[seq];
    s.u = u > 0.0f ? u : 0.0f;
    return s;
}
constexpr int kFewOfThreads = 512; /* top_k up to which the threads' largest logits bound it */
__device__ __forceinline__ bool takes_first(const Settings &s) { return !(s.t > 0.0f) || s.k == 1; }
__device__ __forceinline__ bool by_largest(const Settings &s) { return s.k > 1 && s.k <= kFewOfThreads; }

__device__ __forceinline__ uint64_t shfl_u64(uint64_t v, int from) {
    return (uint64_t)__shfl((uint32_t)(v >> 32), from, 64) << 32 | __shfl((uint32_t)v, from, 64);
}
__device__ __forceinline__ double shfl_up_f64(double v, int by) { return __shfl_up(v, by, 64); }

struct Sum { uint32_t count; uint64_t weight; };
__device__ __forceinline__ Sum operator+(Sum a, Sum b) { return {a.count + b.count, a.weight + b.weight}; }

constexpr int kBins = 2048, kListed = 2048, kTopList = 1024; /* bins; tokens of a list; top_k up to which a list holds all kept */

struct Shared {
    union {
        uint64_t weight[kBins]; /* sums of 2^-bits exp(offset); afterwards, as doubles, running sums of weights */
        double upto[kBins];
    };
    __attribute__((aligned(16))) uint32_t count[kBins]; /* afterwards running sums */
    uint64_t list[kListed];
    union {
        double run[kListed];     /* running sums of the list's weights */
        uint64_t sorted[kListed];
    };
    Sum wave[kWaves];
    double wave_f64[kWaves];
    uint32_t wave_u32[kWaves];
    float wave_max[kWaves], wave_min[kWaves];
    uint32_t digit, n_list, best, found[2], least[10];
    Sum above;
    int picked;
};

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

/* ------------------------------------------------------------------ a row by bins */

/* This thread's share of elements lo .. hi - 1 of x, in vectors of 16 bytes from the first to the last address on 16; an element before or
 * behind those is a vector of its own, whose other places hold NaN. One load ahead of its use: four waves per SIMD cover the rest, and
 * vectors handed on from register to register are instructions (256 rows without filters 65.5 us, four loads ahead 68). fn(values, index of
 * the first) is called from one place: a workgroup runs most of this file's code once, and what it has not run yet comes from memory, 64
 * bytes at a time. Unrolled over four vectors, the pass that lists tokens took 15 us instead of 6, most of it for its own instructions. */
template <class T> constexpr int kPer = 16 / sizeof(T);
template <class T> struct alignas(16) Vec { T v[kPer<T>]; };
/* The first vectors of a row, which its first pass leaves in LDS for the next ones, each thread its own: 96 KB of the 160 that a workgroup of
 * 1024 threads has to itself (its registers leave no room for another). 256 rows of 128256 bf16 logits without filters 66 -> 62.5 us. */
constexpr int kKept = 6 * kThreads;
struct Kept { uint4 *at; int n; };
template <class T> struct Vectors {
    static constexpr int N = kPer<T>;
    const T *x;
    int lo, first, vecs, behind, all, kept;
    const uint4 *in_lds;
    __device__ Vectors(const T *p, int begin, int end, Kept k = {nullptr, 0}) : x(p), lo(begin), in_lds(k.at) {
        const int skip = (int)(((16 - (reinterpret_cast<uintptr_t>(x + lo) & 15)) & 15) / sizeof(T));
        first = min(lo + skip, end), vecs = (end - first) / N, behind = first + vecs * N;
        all = vecs + (first - lo) + (end - behind);
        kept = min(k.n, vecs);
    }
    __device__ int index(int i) const { return i < vecs ? first + i * N : i < vecs + first - lo ? lo + i - vecs : behind + i - vecs - (first - lo); }
    __device__ Vec<T> load(int i) const {
        Vec<T> v;
        if (i < kept) {
            const uint4 bits = in_lds[i];
            __builtin_memcpy(&v, &bits, 16);
            return v;
        }
        if (i < vecs) return *reinterpret_cast<const Vec<T> *>(x + first + i * N);
        const uint32_t nan = sizeof(T) == 4 ? 0x7FC00000u : 0x7FFF7FFFu; /* of either 16-bit type */
        *reinterpret_cast<uint4 *>(&v) = {nan, nan, nan, nan};
        if (i < all) v.v[0] = x[index(i)];
        return v;
    }
};
template <class T, class F> __device__ __forceinline__ void for_vectors(const T *x, int lo, int hi, Kept kept, F fn) {
    constexpr int N = kPer<T>;
    const Vectors<T> vec(x, lo, hi, kept);
    int i = threadIdx.x;
    Vec<T> a = vec.load(i);
#pragma unroll 1
    for (; i < vec.all; i += kThreads) {
        float v[N];
#pragma unroll
        for (int j = 0; j < N; j++) v[j] = to_f32(a.v[j]);
        a = vec.load(i + kThreads);
        fn(v, vec.index(i));
    }
}
template <class T, class F> __device__ __forceinline__ void for_each(const T *x, int lo, int hi, Kept kept, F fn) {
    for_vectors(x, lo, hi, kept, [&](const float (&v)[kPer<T>], int at) {
#pragma unroll
        for (int j = 0; j < kPer<T>; j++) fn(v[j], at + j);
    });
}
/* fn(value, index) for the few elements that pass a cheap test */
template <class T, class P, class F> __device__ __forceinline__ void for_each_of(const T *x, int lo, int hi, Kept kept, P test, F fn) {
    for_vectors(x, lo, hi, kept, [&](const float (&v)[kPer<T>], int at) {
        uint32_t passed = 0;
#pragma unroll
        for (int j = 0; j < kPer<T>; j++) passed |= test(v[j]) ? 1u << j : 0u;
        while (passed) {
            const int j = __builtin_ctz(passed);
            passed &= passed - 1;
            fn(to_f32(x[at + j]), at + j);
        }
    });
}

struct Range { float max, min; };
__device__ __forceinline__ Range range_of_workgroup(Range r, Shared &s) {
    for (int off = 32; off; off >>= 1) {
        r.max = fmaxf(r.max, __shfl_xor(r.max, off, 64));
        r.min = fminf(r.min, __shfl_xor(r.min, off, 64));
    }
    if ((threadIdx.x & 63) == 0) s.wave_max[threadIdx.x >> 6] = r.max, s.wave_min[threadIdx.x >> 6] = r.min;
    __syncthreads();
    for (int w = 0; w < kWaves; w++) r.max = fmaxf(r.max, s.wave_max[w]), r.min = fminf(r.min, s.wave_min[w]);
    __syncthreads();
    return {uniform(r.max), uniform(r.min)};
}
/* The range of what for_vectors would give this thread; without MIN its largest alone. Four loads ahead, each into the registers that
 * were just used: one row is bound by its vector instructions here, of which handing vectors on took a third (151936 fp32 logits, top_k
 * 40: 25.6 -> 22.1 us; eight ahead spill). */
template <bool MIN, class T> __device__ __forceinline__ Range range_of_share(const T *x, int lo, int hi, Kept keep = {nullptr, 0}) {
    constexpr int kAhead = 4;
    const Vectors<T> vec(x, lo, hi, keep);
    Range r = {kMinusInf, -kMinusInf};
    auto take = [&](float v) {
        r.max = fmaxf(r.max, v); /* (NaN is not taken) */
        if constexpr (MIN) r.min = fminf(r.min, is_there(v) ? v : -kMinusInf);
    };
    const int behind = vec.vecs + ((int)(threadIdx.x - (unsigned)vec.vecs) & (kThreads - 1)); /* of this thread's, the first that is no whole vector */
    if (behind < vec.all) take(to_f32(x[vec.index(behind)]));
    int i = threadIdx.x;
    if (i >= vec.vecs) return r;
    const Vec<T> *from = reinterpret_cast<const Vec<T> *>(x + vec.first);
    Vec<T> a[kAhead];
#pragma unroll
    for (int d = 0; d < kAhead; d++) a[d] = from[i + d * kThreads < vec.vecs ? i + d * kThreads : i];
#pragma unroll 1
    for (; i < vec.vecs; i += kAhead * kThreads) {
#pragma unroll
        for (int d = 0; d < kAhead; d++) {
#pragma unroll
            for (int j = 0; j < kPer<T>; j++) take(to_f32(a[d].v[j]));
            if (i + d * kThreads < vec.kept) __builtin_memcpy(&keep.at[i + d * kThreads], &a[d], 16);
            const int next = i + (kAhead + d) * kThreads;
            if (next < vec.vecs) a[d] = from[next]; /* (else the same again, which changes nothing) */
        }
    }
    return r;
}

/* the bins of a row whose largest logit is finite */
constexpr double kTicks = 4503599627370496.0; /* 2^52 */
struct Grid {
    float max;
    double per_t;  /* 1 / T */
    double scale;  /* bins per unit of logits */
    double step;   /* a bin in units of the exponent: at most 1/64 */
    double unit, per_unit; /* 2^bits: of the sums of exp(offset); its inverse */
    double c1, c2, c3, c4; /* unit exp(-step f) in powers of f */
    __device__ Grid(const Range &r, float t, int n) : max(r.max), per_t(1.0 / (double)t) {
        const double span = (double)r.max - (double)r.min;
        scale = fmax(64.0 * per_t, span > 0.0 ? 2040.0 / span : 0.0);
        if (!(scale > 0.0)) scale = 1.0;
        scale = fmin(scale, 1e250); /* (a temperature of 1e-45) */
        step = fmin(per_t / scale, 1.0 / 64);
        int bits = 40; /* n << bits stays below 2^62 */
        while (bits > 0 && ((uint64_t)n >> (61 - bits)) > 0) bits--;
        unit = (double)(1ull << bits);
        max = uniform(max), per_t = uniform(per_t), scale = uniform(scale), step = uniform(step);
        per_unit = 1.0 / unit;
        c1 = -step * unit, c2 = 0.5 * step * step * unit, c3 = -step * step * step * unit / 6, c4 = step * step * step * step * unit / 24;
    }
    __device__ Grid scalar() const { /* (the arguments of a function that is not inlined come in vector registers) */
        Grid g = *this;
        g.max = uniform(max), g.per_t = uniform(per_t), g.scale = uniform(scale), g.step = uniform(step), g.unit = uniform(unit), g.per_unit = uniform(per_unit);
        g.c1 = uniform(c1), g.c2 = uniform(c2), g.c3 = uniform(c3), g.c4 = uniform(c4);
        return g;
    }
    /* The bin of a value is its distance from the largest in bins, rounded: the sum with 2^52 rounds at 1 and holds it in its lower half.
     * One rounding, so that it never falls from a logit to a smaller one. NaN where the value is; infinite for -infinity. */
    __device__ __forceinline__ double distance(float v) const { return (double)max - (double)v; }
    __device__ __forceinline__ double ticks(double distance) const { return fma(distance, scale, kTicks); }
    static __device__ __forceinline__ bool counts(double ticks) { return ticks < kTicks + (kBins - 1); }
    static __device__ __forceinline__ int bin(double ticks) { return (int)__double_as_longlong(ticks); }
    __device__ __forceinline__ int bin_of(float v) const { /* kBins: not counted */
        const double t = ticks(distance(v));
        return counts(t) ? bin(t) : kBins;
    }
    /* exp(centre of the bin - distance), by a polynomial of degree 4 (2.4e-13 at the bin's edge), as an integer of 1 / unit: the last of
     * the sums rounds as above. (Eight 64-bit operations; with the conversions to an integer and back, which take four times an
     * addition, a pass took a quarter longer.) */
    __device__ __forceinline__ uint64_t offset_weight(double distance, double ticks) const {
        const double f = fma(distance, scale, kTicks - ticks); /* from the centre, in bins */
        double e = fma(f, c4, c3);
        e = fma(e, f, c2);
        e = fma(e, f, c1);
        e = fma(e, f, unit + kTicks);
        return (uint64_t)__double_as_longlong(e) & 0x000FFFFFFFFFFFFFull;
    }
    /* floats below (above) every value of the bins up to (from) `bin` */
    __device__ float value_below(int bin) const { return __double2float_rd((double)max - ((double)bin + 1.0) / scale); }
    __device__ float value_above(int bin) const { return __double2float_ru((double)max - ((double)bin - 1.0) / scale); }
    __device__ double weight(float v) const { return exp(((double)v - (double)max) * per_t); }
};
constexpr int kLastBin = kBins - 2;

/* what the bins hold: counts where the list will hold all kept tokens, else weights, and both where top_k is larger than that */
struct Holds { bool counts, weights; };
__device__ __forceinline__ Holds holds_for(const Settings &s) { return {s.k > 0, s.k <= 0 || s.k > kTopList}; }

__device__ __forceinline__ void into_bin(float v, const Grid &g, bool counts, bool weights, Shared &s) {
    const double d = g.distance(v), t = g.ticks(d);
    if (!g.counts(t)) return;
    if (weights) atomicAdd((unsigned long long *)&s.weight[g.bin(t)], (unsigned long long)g.offset_weight(d, t));
    if (counts) atomicAdd(&s.count[g.bin(t)], 1u);
}
template <class T> __device__ __forceinline__ void fill_bins(const T *x, int lo, int hi, Kept kept, const Grid &g, const Holds &h, Shared &s) {
    if (!h.weights) for_each(x, lo, hi, kept, [&](float v, int) { into_bin(v, g, true, false, s); });
    else if (!h.counts) for_each(x, lo, hi, kept, [&](float v, int) { into_bin(v, g, false, true, s); });
    else for_each(x, lo, hi, kept, [&](float v, int) { into_bin(v, g, true, true, s); });
}

/* counts and weights to running sums */
__device__ void sum_bins(const Grid &g, const Holds &h, Shared &s) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, b = 2 * threadIdx.x;
    if (h.weights) {
        const double a0 = (double)s.weight[b] * g.per_unit * exp(-(double)b * g.step);
        const double a1 = b + 1 > kLastBin ? 0.0 : (double)s.weight[b + 1] * g.per_unit * exp(-((double)b + 1.0) * g.step);
        double run = a0 + a1;
        for (int off = 1; off < 64; off <<= 1) {
            const double o = shfl_up_f64(run, off);
            if (lane >= off) run += o;
        }
        if (lane == 63) s.wave_f64[wave] = run;
        __syncthreads();
        double before = 0.0;
        for (int w = 0; w < wave; w++) before += s.wave_f64[w];
        /* (both are the same sum and a1: within a pair no sum falls; from pair to pair one may, by a rounding) */
        s.upto[b + 1] = before + run;
        s.upto[b] = before + run - a1;
    }
    if (h.counts) {
        const uint32_t a0 = s.count[b], a1 = s.count[b + 1];
        uint32_t run = a0 + a1;
        for (int off = 1; off < 64; off <<= 1) {
            const uint32_t o = __shfl_up(run, off, 64);
            if (lane >= off) run += o;
        }
        if (lane == 63) s.wave_u32[wave] = run;
        __syncthreads();
        uint32_t before = 0;
        for (int w = 0; w < wave; w++) before += s.wave_u32[w];
        s.count[b] = before + run - a1;
        s.count[b + 1] = before + run;
    }
    __syncthreads();
}

/* The first bin of which `one` holds, and the first of which `other` holds; kLastBin + 1 if there is none. The tests are of running sums,
 * which fall by a rounding here and there: what holds of a bin need not of the next, and of several firsts the least counts. All threads of
 * the workgroup call it. */
struct Pair { int one, other; };
template <class F, class G> __device__ Pair first_bins(Shared &s, F one, G other) {
    if (threadIdx.x < 2) s.found[threadIdx.x] = kLastBin + 1;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 2; e++) {
        const int b = 2 * threadIdx.x + e;
        if (b <= kLastBin && one(b) && (b == 0 || !one(b - 1))) atomicMin(&s.found[0], (uint32_t)b);
        if (b <= kLastBin && other(b) && (b == 0 || !other(b - 1))) atomicMin(&s.found[1], (uint32_t)b);
    }
    __syncthreads();
    const Pair r = {uniform((int)s.found[0]), uniform((int)s.found[1])};
    __syncthreads();
    return r;
}
template <class F> __device__ int first_bin(Shared &s, F one) { return first_bins(s, one, [](int) { return false; }).one; }

/* The bins to list. Each cut has a run of bins in which it may lie, empty (hi < lo) where it does not cut. */
struct Run { int lo, hi; };
constexpr int kNowhere = 1 << 30;
struct Wanted {
    Run k, p, m, u;
    Run run[4];     /* the same in order; an empty one begins at kNowhere */
    int from[4];    /* where the bins that are listed without a gap begin, of each run */
    double before[4]; /* sums of weights of the bins before that */
    double total, m_total; /* of all bins; of those up to the end of m's */
    uint32_t k_before; /* tokens of the bins before k's */
    bool all;       /* the list holds every kept token (run[0] from bin 0) */
};
/* (no index that is not a constant: an array that has one lies in memory, which took 20 us of every row) */
__device__ __forceinline__ void order_runs(Wanted &w) {
    w.run[0] = w.k, w.run[1] = w.p, w.run[2] = w.m, w.run[3] = w.u;
#pragma unroll
    for (int r = 0; r < 4; r++)
        if (w.run[r].hi < w.run[r].lo) w.run[r] = {kNowhere, -1};
    auto by_start = [&](Run &a, Run &b) {
        if (b.lo < a.lo) {
            const Run t = a;
            a = b;
            b = t;
        }
    };
    by_start(w.run[0], w.run[1]);
    by_start(w.run[2], w.run[3]);
    by_start(w.run[0], w.run[2]);
    by_start(w.run[1], w.run[3]);
    by_start(w.run[1], w.run[2]);
    w.from[0] = w.run[0].lo;
    int reach = w.run[0].hi;
#pragma unroll
    for (int r = 1; r < 4; r++) {
        const bool joins = w.run[r].lo <= reach + 1;
        w.from[r] = joins ? w.from[r - 1] : w.run[r].lo;
        reach = joins ? max(reach, w.run[r].hi) : w.run[r].hi;
    }
}
/* The bins in which min-p may cut; empty: it cuts nothing that has a weight. The weights and the logarithm are rounded, by less than 1e-15 of
 * the exponent and 1e-15: a part of a bin, but many bins where logits lie closer together than 64-bit weights tell apart. */
__device__ __forceinline__ Run min_p_bins(const Grid &g, float m) {
    const double at = -log((double)m), off = 1e-15 * (at + 1.0), lo = (at - off) / g.step - 1.0, hi = (at + off) / g.step + 1.0;
    if (!(lo < kBins)) return {0, -1};
    return {uniform((int)fmax(lo, 0.0)), uniform((int)fmin(hi, (double)kLastBin))};
}
__device__ Wanted wanted_bins(const Grid &g, const Settings &set, const Holds &h, Shared &s) {
    const double slack = 1e-11 + 2.0 * g.per_unit; /* of the sums' rounding: half a unit for each of a bin's tokens, which may all go one way */
    const Run none = {0, -1};
    Wanted w = {};
    w.k = w.p = w.m = w.u = none;
    w.all = !h.weights;
    if (w.all) {
        w.k = {0, min(first_bin(s, [&](int b) { return s.count[b] >= (uint32_t)set.k; }), kLastBin)};
        order_runs(w);
        return w;
    }
    auto before = [&](int b) { return b > 0 ? uniform(s.upto[b - 1]) : 0.0; };
    const double everything = uniform(s.upto[kLastBin]);
    double lo = everything, hi = lo; /* between which the sum of the kept lies */
    if (set.k > 0) {
        const int b = first_bin(s, [&](int i) { return s.count[i] >= (uint32_t)set.k; });
        if (b <= kLastBin) w.k = {b, b}, lo = before(b), hi = uniform(s.upto[b]);
    }
    if (set.p < 1.0f) {
        const double p = fmax((double)set.p, 0.0), at_least = p * lo * (1.0 - slack), at_most = p * hi * (1.0 + slack);
        const Pair f = first_bins(s, [&](int i) { return s.upto[i] >= at_least; }, [&](int i) { return s.upto[i] >= at_most; });
        w.p = {min(f.one, kLastBin), min(f.other, kLastBin)};
        lo = fmin(lo, before(w.p.lo));
        hi = fmin(hi, uniform(s.upto[w.p.hi]));
    }
    if (set.m > 0.0f) {
        w.m = min_p_bins(g, set.m);
        if (w.m.hi >= w.m.lo) {
            lo = fmin(lo, before(w.m.lo));
            hi = fmin(hi, uniform(s.upto[w.m.hi]));
        }
    }
    /* of top-p and min-p the one that cuts off more is enough, where that is clear */
    if (w.p.hi >= w.p.lo && w.m.hi >= w.m.lo) {
        if (w.m.hi < w.p.lo) w.p = none;
        else if (w.p.hi < w.m.lo) w.m = none;
    }
    const double u = (double)set.u, at_least = u * lo * (1.0 - slack), at_most = u * hi * (1.0 + slack); /* (u < 1: some bin is past both) */
    const Pair f = first_bins(s, [&](int i) { return s.upto[i] > at_least; }, [&](int i) { return s.upto[i] > at_most; });
    w.u = {min(f.one, kLastBin), min(max(f.one, f.other), kLastBin)};
    order_runs(w);
#pragma unroll
    for (int r = 0; r < 4; r++) w.before[r] = w.from[r] < kNowhere ? before(w.from[r]) : 0.0;
    w.total = everything;
    w.m_total = w.m.hi >= w.m.lo ? uniform(s.upto[w.m.hi]) : 0.0;
    w.k_before = w.k.hi >= w.k.lo && w.k.lo > 0 ? uniform(s.count[w.k.lo - 1]) : 0;
    return w;
}

/* ascending order of these is the order of the tokens */
__device__ __forceinline__ uint64_t entry_of(float v, int i) { return (uint64_t)(~key_of(v)) << 32 | (uint32_t)i; }
__device__ __forceinline__ float entry_value(uint64_t e) { return value_of(~(uint32_t)(e >> 32)); }

__device__ __forceinline__ bool is_wanted(int bin, const Wanted &w) {
    bool in = false;
#pragma unroll
    for (int r = 0; r < 4; r++) in = in || (bin >= w.run[r].lo && bin <= w.run[r].hi);
    return in;
}
/* Whether a value can lie in a wanted bin, by floats a little outside of the first bins without a gap, and of all behind them. */
struct Bounds {
    float low0, high0, low1, high1;
    __device__ Bounds(const Grid &g, const Wanted &w) {
        int end = w.run[0].hi, start = kNowhere, last = -1;
#pragma unroll
        for (int r = 1; r < 4; r++) {
            const bool joins = w.from[r] == w.from[0];
            if (joins) end = max(end, w.run[r].hi);
            else start = min(start, w.run[r].lo), last = max(last, w.run[r].hi);
        }
        low0 = uniform(g.value_below(end)), high0 = uniform(w.run[0].lo == 0 ? g.max : g.value_above(w.run[0].lo));
        low1 = uniform(start < kNowhere ? g.value_below(last) : -kMinusInf), high1 = uniform(start < kNowhere ? g.value_above(start) : kMinusInf);
    }
    __device__ __forceinline__ bool operator()(float v) const { return (v >= low0 && v <= high0) || (v >= low1 && v <= high1); }
};
__device__ __forceinline__ void add_to_list(uint64_t e, Shared &s) {
    const uint32_t at = atomicAdd(&s.n_list, 1u);
    if (at < kListed) s.list[at] = e;
}
/* fn(entry) for the tokens of the wanted bins */
template <class F> __device__ __forceinline__ void if_wanted(float v, int i, const Grid &g, const Wanted &w, F fn) {
    const int bin = g.bin_of(v);
    if (bin < kBins && is_wanted(bin, w)) fn(entry_of(v, i));
}
template <class T, class F> __device__ __forceinline__ void for_each_wanted(const T *x, int lo, int hi, Kept kept, const Grid &g, const Wanted &w, F fn) {
    const Bounds bounds(g, w);
    for_each_of(x, lo, hi, kept, bounds, [&](float v, int i) { if_wanted(v, i, g, w, fn); });
}

__device__ __forceinline__ uint64_t shfl_xor_u64(uint64_t v, int by) {
    return (uint64_t)__shfl_xor((uint32_t)(v >> 32), by, 64) << 32 | __shfl_xor((uint32_t)v, by, 64);
}
/* s.list[0 .. n) into order: a bitonic network over `size` entries (a power of two, E per thread: entry e * kThreads + thread), its
 * short exchanges between the lanes of a wave, the longer ones through LDS, alternating between two buffers, one barrier each */
template <int E> __device__ void sort_network(int n, int size, Shared &s) {
    const int t = threadIdx.x;
    uint64_t v[E];
    if (t < size) {
#pragma unroll
        for (int e = 0; e < E; e++) v[e] = e * kThreads + t < n ? s.list[e * kThreads + t] : ~0ull;
    }
    uint64_t *buffer = s.sorted;
    for (int k = 2; k <= size; k <<= 1)
        for (int j = k >> 1; j; j >>= 1) {
            if (E == 2 && j == kThreads) {
                const uint64_t a = v[0], b = v[E - 1]; /* (k is the whole size: ascending) */
                v[0] = min(a, b), v[E - 1] = max(a, b);
                continue;
            }
            uint64_t o[E];
            if (j >= 64) {
                if (t < size) {
#pragma unroll
                    for (int e = 0; e < E; e++) buffer[e * kThreads + t] = v[e];
                }
                __syncthreads();
                if (t < size) {
#pragma unroll
                    for (int e = 0; e < E; e++) o[e] = buffer[e * kThreads + (t ^ j)];
                }
                buffer = buffer == s.sorted ? s.list : s.sorted;
            } else if (t < size) {
#pragma unroll
                for (int e = 0; e < E; e++) o[e] = shfl_xor_u64(v[e], j);
            }
            if (t < size) {
#pragma unroll
                for (int e = 0; e < E; e++) {
                    const bool smaller = ((t & j) == 0) == (((e * kThreads + t) & k) == 0);
                    v[e] = smaller ? min(v[e], o[e]) : max(v[e], o[e]);
                }
            }
        }
    if (size > 64) __syncthreads();
    if (t < size) {
#pragma unroll
        for (int e = 0; e < E; e++) s.list[e * kThreads + t] = v[e];
    }
    if (size > 64) __syncthreads(); /* up to 64 entries are wave 0's alone, as is their pick */
    else __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
}
__device__ void sort_list(int n, Shared &s) {
    int size = 64;
    while (size < n) size <<= 1;
    if (size > kThreads) sort_network<2>(n, size, s);
    else sort_network<1>(n, size, s);
}

/* The cuts on the sorted list, E entries per thread of `WAVES` waves: one wave for up to 64 entries, which then needs no barrier, else
 * all. */
constexpr int kOneWave = 64;
template <int WAVES, int E> __device__ __forceinline__ void pick_with(int n, const Grid &g, const Settings &set, const Wanted &w, int32_t *id, float *prob, Shared &s) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i0 = E * threadIdx.x;
    double *weight = s.upto; /* the entries' (the bins' sums have gone into w) */
    auto meet = [&] {
        if constexpr (WAVES > 1) __syncthreads();
        else __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    };
    /* the least of the waves' least entries for which a test holds, n if there is none; each call has a place of its own */
    if (threadIdx.x < 10) s.least[threadIdx.x] = (uint32_t)n;
    double wt[E], run = 0.0;
    int bin[E];
#pragma unroll
    for (int e = 0; e < E; e++) {
        const bool there = i0 + e < n;
        const float value = there ? entry_value(s.list[i0 + e]) : 0.0f;
        wt[e] = there ? g.weight(value) : 0.0;
        bin[e] = there ? g.bin_of(value) : kBins;
        weight[i0 + e] = wt[e];
        run += wt[e];
    }
    for (int off = 1; off < 64; off <<= 1) {
        const double o = shfl_up_f64(run, off);
        if (lane >= off) run += o;
    }
    double ahead = 0.0;
    if constexpr (WAVES > 1) {
        if (lane == 63) s.wave_f64[wave] = run;
        meet();
        for (int v = 0; v < wave; v++) ahead += s.wave_f64[v];
    }
    s.run[i0 + E - 1] = ahead + run;
    if constexpr (E == 2) s.run[i0] = ahead + run - wt[1];
    meet();
    int calls = 0;
    auto first = [&](Run where, auto test) {
        int best = n;
#pragma unroll
        for (int e = E - 1; e >= 0; e--) {
            const uint64_t holds = __ballot(i0 + e < n && bin[e] >= where.lo && bin[e] <= where.hi && test(i0 + e, wt[e], e));
            if (holds) best = min(best, E * (wave * 64 + (int)__builtin_ctzll(holds)) + e);
        }
        if constexpr (WAVES > 1) {
            if (lane == 0 && best < n) atomicMin(&s.least[calls], (uint32_t)best);
            meet();
            best = uniform((int)s.least[calls]);
        }
        calls++;
        return best;
    };
    auto any = [](int, double, int) { return true; };
    /* running sum over the row minus running sum over the list, by run of bins */
    double base[4] = {0.0, 0.0, 0.0, 0.0};
    if (!w.all) {
#pragma unroll
        for (int r = 0; r < 4; r++)
            if (w.from[r] < kNowhere) {
                const int at = first({w.from[r], kBins}, any);
                base[r] = uniform(w.before[r] - (at > 0 ? s.run[at - 1] : 0.0));
            }
    }
    auto sum_to = [&](int i, int b) { /* running sum at entry i, of bin b */
        double off = base[0];
#pragma unroll
        for (int r = 1; r < 4; r++)
            if (b >= w.run[r].lo) off = base[r];
        return s.run[i] + off;
    };
    double sums[E];
#pragma unroll
    for (int e = 0; e < E; e++) sums[e] = i0 + e < n ? sum_to(i0 + e, bin[e]) : 0.0;
    auto sum_at = [&](int i) { return sum_to(i, g.bin_of(entry_value(s.list[i]))); };
    const Run everywhere = {0, kBins};
    int kept = n; /* list entries from here on are cut off (those between the runs lie on the right side by construction) */
    double total = w.all ? s.run[n - 1] : w.total;
    if (w.all) {
        kept = min(set.k, n);
        total = s.run[kept - 1];
    } else if (w.k.hi >= w.k.lo) {
        const uint32_t at = (uint32_t)set.k - w.k_before; /* of the bin's tokens, from 1 */
        kept = min(first(w.k, any) + (int)at, n);
        total = sum_to(kept - 1, w.k.lo);
    }
    if (w.all ? set.p < 1.0f : w.p.hi >= w.p.lo) {
        const double target = fmax((double)set.p, 0.0) * total;
        const int i = first(w.all ? everywhere : w.p, [&](int, double, int e) { return sums[e] >= target; });
        if (i < kept) {
            kept = i + 1;
            total = sum_at(i);
        }
    }
    if (w.all ? set.m > 0.0f : w.m.hi >= w.m.lo) {
        const int i = first(w.all ? everywhere : w.m, [&](int, double weight, int) { return weight < (double)set.m; });
        const int from = i < n || w.all ? i : first({w.m.hi + 1, kBins}, any);
        if (i < n && i < kept) total = fmin(total, sum_at(i) - weight[i]);
        else if (i >= n && !w.all) total = fmin(total, w.m_total);
        kept = min(kept, from); /* (what lies behind the bins of this cut is lighter) */
    }
    const double target = (double)set.u * total;
    int i = first(w.all ? everywhere : w.u, [&](int at, double weight, int e) { return at < kept && weight > 0.0 && sums[e] > target; });
    if (i >= n) { /* the last border rounded away: the last kept token that weighs anything, which is before the first that does not */
        const int none = first(everywhere, [&](int at, double weight, int) { return at >= kept || !(weight > 0.0); });
        i = max(none - 1, 0);
    }
    if (threadIdx.x == 0) {
        *id = (int32_t)(uint32_t)s.list[i];
        if (prob) *prob = (float)(weight[i] / total);
    }
}
/* s.list[0 .. n), in any order, to the pick. A longer list of all kept tokens is itself a row of which bins say where the cuts lie (k = 1000:
 * sorting all of them took 15 us). */
__device__ void clear_bins(Shared &s) {
    for (int i = threadIdx.x; i < kBins; i += kThreads) s.weight[i] = 0, s.count[i] = 0;
}
__device__ void pick_from_list(int n, const Grid &g, const Settings &set, Wanted w, int32_t *id, float *prob, Shared &s) {
    if (w.all && n > kOneWave) {
        const Holds both = {true, true};
        __syncthreads();
        clear_bins(s);
        if (threadIdx.x == 0) s.n_list = 0;
        __syncthreads();
        uint64_t entry[kListed / kThreads];
#pragma unroll
        for (int e = 0; e < kListed / kThreads; e++) {
            const int i = threadIdx.x + e * kThreads;
            entry[e] = i < n ? s.list[i] : 0; /* (no token's: its value is NaN) */
            if (i < n) into_bin(entry_value(entry[e]), g, true, true, s);
        }
        __syncthreads();
        sum_bins(g, both, s);
        w = wanted_bins(g, set, both, s);
#pragma unroll
        for (int e = 0; e < kListed / kThreads; e++)
            if ((int)threadIdx.x + e * kThreads < n && is_wanted(g.bin_of(entry_value(entry[e])), w)) s.list[atomicAdd(&s.n_list, 1u)] = entry[e];
        __syncthreads();
        n = uniform((int)s.n_list);
    }
    sort_list(n, s);
    if (n > kOneWave) pick_with<kWaves, 2>(n, g, set, w, id, prob, s);
    else if (threadIdx.x < 64) pick_with<1, 1>(n, g, set, w, id, prob, s);
}

/* ------------------------------------------------------------------ a row by values
 * Where the bins of the cuts hold more tokens than a list, a cut is searched for in its bin by the bits of the values: three passes over the
 * row, each with sums by 11 (10) of the bits. Weights are the bins', multiples of 2^-40 of the bin's own, so that a tail far below
 * the largest logit is as sharp as its head (integers of the whole row's weights put 6 to 87 % of the picks from a flat tail 21
 * temperatures down on a neighbour). */

/* the first bin with tokens of which `test` holds (kBins: none) */
template <class F> __device__ int first_filled(Shared &s, F test) {
    if (threadIdx.x == 0) s.found[0] = kBins;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 2; e++) {
        const int b = 2 * threadIdx.x + e;
        if (b <= kLastBin && s.count[b] > (b ? s.count[b - 1] : 0) && test(b)) atomicMin(&s.found[0], (uint32_t)b);
    }
    __syncthreads();
    const int r = uniform((int)s.found[0]);
    __syncthreads();
    return r;
}

/* what the bins before `bin` weigh, and what 1 of its own sums does */
__device__ __forceinline__ double before_bin(int bin, Shared &s) { return bin > 0 ? uniform(s.upto[bin - 1]) : 0.0; }
__device__ __forceinline__ double unit_of_bin(int bin, const Grid &g) { return g.per_unit * exp(-(double)bin * g.step); }

/* A thread's additions to sums by bin or digit, those that follow each other to the same place as one: of a row of one value all threads' go to
 * one place, and wait for each other there (128256 equal logits 1050 -> 310 us). */
struct Additions {
    uint32_t *count;
    uint64_t *weight;
    int at = -1;
    Sum held = {0, 0};
    __device__ __forceinline__ void flush() {
        if (at < 0) return;
        atomicAdd(&count[at], held.count);
        atomicAdd((unsigned long long *)&weight[at], (unsigned long long)held.weight);
    }
    __device__ __forceinline__ void add(int to, uint64_t w) {
        if (to != at) {
            flush();
            at = to, held = {0, 0};
        }
        held = held + Sum{1, w};
    }
};

/* where the kept end: with the bin, or inside it at `upto` of its sum; the sum of all kept */
struct End {
    int bin;
    uint64_t upto;
    double total;
};
/* the end that min-p makes: its lightest token is in one of `bins`, or those before them stay and no more */
template <class T> __device__ __forceinline__ End end_by_min_p(const T *x, int n, const Grid &g, float m, Run bins, Shared &s) {
    const Kept nothing = {nullptr, 0};
    if (threadIdx.x == 0) s.best = ~0u;
    __syncthreads();
    uint32_t least = ~0u;
    for_each(x, 0, n, nothing, [&](float v, int) {
        const int b = g.bin_of(v);
        if (b >= bins.lo && b <= bins.hi && g.weight(v) >= (double)m) least = min(least, key_of(v));
    });
    if (least != ~0u) atomicMin(&s.best, least);
    __syncthreads();
    least = uniform(s.best);
    if (least == ~0u) { /* (never from bin 0 on: the largest token stays) */
        const uint32_t heavier = uniform(s.count[bins.lo - 1]);
        const int b = first_filled(s, [&](int i) { return s.count[i] >= heavier; });
        return {b, ~0ull, uniform(s.upto[b])};
    }
    const int bin = g.bin_of(value_of(least));
    Sum kept = {0, 0};
    for_each(x, 0, n, nothing, [&](float v, int) {
        const double d = g.distance(v), t = g.ticks(d);
        if (g.counts(t) && g.bin(t) == bin && key_of(v) >= least) kept = kept + Sum{1, g.offset_weight(d, t)};
    });
    kept = sum_of_workgroup(kept, s, nullptr);
    return {bin, kept.weight, before_bin(bin, s) + unit_of_bin(bin, g) * (double)kept.weight};
}

/* The value in a bin, which has tokens, at which the bin's running sum reaches `target` (a number of tokens, or a sum in the bin's unit; at
 * least 1), its last one if none does: its key, which of its tokens it is (from 1), what each weighs, and the bin's sum with that token */
struct Cut {
    uint32_t key, nth;
    uint64_t each, upto;
};
template <class T> __device__ __forceinline__ Cut find_cut(const T *x, int n, const Grid &g, int bin, bool by_weight, uint64_t target, Shared &s) {
    uint64_t *weight = s.list;
    uint32_t *count = reinterpret_cast<uint32_t *>(s.sorted);
    uint32_t key = 0;
    Sum above = {0, 0};
#pragma unroll 1
    for (int pass = 0; pass < 3; pass++) {
        const int low = pass == 0 ? 21 : pass == 1 ? 10 : 0, known = pass == 0 ? 32 : low + (pass == 1 ? 11 : 10), digits = pass == 2 ? 1024 : 2048;
        for (int i = threadIdx.x; i < 2048; i += kThreads) count[i] = 0, weight[i] = 0;
        __syncthreads();
        Additions sums = {count, weight};
        for_each(x, 0, n, Kept{nullptr, 0}, [&](float v, int) {
            const double d = g.distance(v), t = g.ticks(d);
            if (!g.counts(t) || g.bin(t) != bin) return;
            const uint32_t k = key_of(v);
            if (pass && k >> known != key) return;
            sums.add((k >> low) & (digits - 1), g.offset_weight(d, t));
        });
        sums.flush();
        __syncthreads();
        const int hi = 2047 - 2 * threadIdx.x; /* two digits per thread, the largest first */
        const Sum a = {count[hi], weight[hi]}, b = {count[hi - 1], weight[hi - 1]};
        Sum before;
        const Sum all = sum_of_workgroup(a + b, s, &before);
        if (pass == 0) target = min(target, by_weight ? all.weight : (uint64_t)all.count);
        before = before + above;
        const Sum mid = before + a, after = mid + b;
        auto reached = [&](const Sum &v) { return (by_weight ? v.weight : (uint64_t)v.count) >= target; };
        if (!reached(before) && reached(after)) {
            s.digit = reached(mid) ? hi : hi - 1;
            s.above = reached(mid) ? before : mid;
        }
        __syncthreads();
        key = key << (known - low) | uniform(s.digit);
        above = s.above;
        __syncthreads();
    }
    const double d = g.distance(value_of(key));
    const uint64_t each = g.offset_weight(d, g.ticks(d));
    const uint32_t nth = by_weight ? (uint32_t)((target - above.weight + each - 1) / each) : (uint32_t)target - above.count;
    return {key, nth, each, above.weight + nth * each};
}

/* the whole row, whose largest logit is finite, from bins of its own */
template <class T> __device__ __noinline__ void sample_by_value(const T *x, int n, Settings set, Grid grid, int32_t *id, float *prob, Shared &s) {
    const Grid g = grid.scalar();
    clear_bins(s);
    __syncthreads();
    Additions sums = {s.count, s.weight};
    for_each(x, 0, n, Kept{nullptr, 0}, [&](float v, int) {
        const double d = g.distance(v), t = g.ticks(d);
        if (g.counts(t)) sums.add(g.bin(t), g.offset_weight(d, t));
    });
    sums.flush();
    __syncthreads();
    sum_bins(g, Holds{true, true}, s);
    const uint32_t tokens = uniform(s.count[kLastBin]);
    End end = {first_filled(s, [&](int b) { return s.count[b] >= tokens; }), ~0ull, 0.0};
    end.total = uniform(s.upto[end.bin]);
    enum Step { top_k, top_p, min_p, pick };
#pragma unroll 1
    for (int step = top_k; step <= pick; step++) {
        int bin = end.bin;
        uint64_t goal = end.upto;
        if (step == top_k) {
            if (set.k <= 0 || (uint32_t)set.k >= tokens) continue;
            bin = first_filled(s, [&](int b) { return s.count[b] >= (uint32_t)set.k; });
            goal = (uint32_t)set.k - (bin > 0 ? uniform(s.count[bin - 1]) : 0);
        } else if (step == min_p) {
            const Run bins = set.m > 0.0f ? min_p_bins(g, set.m) : Run{0, -1};
            if (bins.hi < bins.lo) continue;
            const End m = end_by_min_p(x, n, g, set.m, bins, s);
            if (m.bin < end.bin || (m.bin == end.bin && m.upto < end.upto)) end = m;
            continue;
        } else { /* the first kept token at which the running sum reaches p times the sum, or is past u times the sum */
            if (step == top_p && !(set.p < 1.0f)) continue;
            const double target = (step == top_p ? fmax((double)set.p, 0.0) : (double)set.u) * end.total;
            if (target < end.total) {
                bin = min(first_filled(s, [&](int b) { return step == top_p ? s.upto[b] >= target : s.upto[b] > target; }), end.bin);
                const double in_bin = fmax(target - before_bin(bin, s), 0.0) / unit_of_bin(bin, g);
                goal = max((uint64_t)fmin(step == top_p ? ceil(in_bin) : floor(in_bin) + 1.0, 9.0e18), (uint64_t)1); /* (a bin's sum is below 2^62.1) */
                if (bin == end.bin) goal = min(goal, end.upto);
            }
        }
        const Cut c = find_cut(x, n, g, bin, step != top_k, goal, s);
        const double unit = unit_of_bin(bin, g);
        if (step == pick) {
            const int at = nth_of_value(x, n, c.key, c.nth, s);
            if (threadIdx.x == 0) {
                *id = at;
                if (prob) *prob = (float)(unit * (double)c.each / end.total);
            }
        }
        end = {bin, c.upto, before_bin(bin, s) + unit * (double)c.upto};
    }
}

/* a row whose largest logits are infinite: each of them weighs 1, the others nothing */
template <class T> __device__ __noinline__ void sample_infinities(const T *x, int n, Settings set, int32_t *id, float *prob, Shared &s) {
    Sum mine = {0, 0};
    for_each(x, 0, n, Kept{nullptr, 0}, [&](float v, int) { mine.count += v == -kMinusInf; });
    uint32_t kept = sum_of_workgroup(mine, s, nullptr).count;
    if (set.k > 0) kept = min(kept, (uint32_t)set.k);
    if (set.p < 1.0f) kept = max((uint32_t)ceil(fmax((double)set.p, 0.0) * kept), 1u);
    const double target = (double)set.u * kept;
    const int at = nth_of_value(x, n, key_of(-kMinusInf), target < kept ? (uint32_t)target + 1 : kept, s);
    if (threadIdx.x == 0) {
        *id = at;
        if (prob) *prob = (float)(1.0 / kept);
    }
}

__device__ __forceinline__ void nothing_there(int32_t *id, float *prob) {
    if (threadIdx.x == 0) {
        *id = -1;
        if (prob) *prob = 0.0f;
    }
}

/* A row to the pick: from its bins, where they are `filled` or are here; or where the threads' largest logits have been `counted` (`mine` is
 * this thread's) from those. */
enum class Bins { empty, filled, counted };
template <class T> __device__ __forceinline__ void finish_row(const T *x, int n, Kept kept, const Grid &g, float mine, Bins bins, const Settings &set, int32_t *id, float *prob, Shared &s) {
    const Holds holds = holds_for(set);
    if (g.max == -kMinusInf) return sample_infinities(x, n, set, id, prob, s);
    if (bins == Bins::empty) {
        fill_bins(x, 0, n, kept, g, holds, s);
        __syncthreads();
    }
    if (bins != Bins::counted) sum_bins(g, holds, s);
    const Wanted w = wanted_bins(g, set, holds, s);
    if (bins == Bins::counted) {
        /* only what those threads read whose largest logit is wanted is looked at again: their vectors, dealt to all threads (for
         * k = 40 some 720 vectors of 16032; a pass over all of them takes 12 us where all compute units make one) */
        uint32_t *of = reinterpret_cast<uint32_t *>(s.sorted);
        const Bounds bounds(g, w);
        if (mine >= bounds.low0) of[atomicAdd(&s.digit, 1u)] = threadIdx.x;
        __syncthreads();
        const Vectors<T> vec(x, 0, n);
        const int rounds = (vec.all + kThreads - 1) / kThreads, tasks = uniform((int)s.digit) * rounds;
        for (int q = threadIdx.x; q < tasks; q += kThreads) {
            const int i = (int)of[q / rounds] + q % rounds * kThreads;
            const Vec<T> v = vec.load(i);
#pragma unroll
            for (int j = 0; j < kPer<T>; j++)
                if (bounds(to_f32(v.v[j]))) if_wanted(to_f32(v.v[j]), vec.index(i) + j, g, w, [&](uint64_t e) { add_to_list(e, s); });
        }
    } else {
        for_each_wanted(x, 0, n, kept, g, w, [&](uint64_t e) { add_to_list(e, s); });
    }
    __syncthreads();
    /* (a u of 1 or more takes the last token with a weight: sums do not find its bin, to which it adds next to nothing) */
    const uint32_t listed = set.u >= 1.0f ? kListed + 1 : uniform(s.n_list);
    if (listed > kListed) return sample_by_value(x, n, set, g, id, prob, s);
    pick_from_list((int)listed, g, set, w, id, prob, s);
}

/* a row by one workgroup */
template <class T> __device__ __forceinline__ void whole_row(const T *x, int n, const Settings &set, int32_t *id, float *prob, Shared &s) {
    __shared__ uint4 keep[kKept];
    if (threadIdx.x == 0) s.best = (uint32_t)n, s.n_list = 0, s.digit = 0;
    clear_bins(s);
    const bool first = takes_first(set);
    bool largest = first || by_largest(set), counted = false;
    float mine = kMinusInf;
    /* The k-th largest of the threads' own largest logits is not above the k-th of all. For a k that is small beside the threads it is
     * close below (of 128256 logits and k = 512 some 700 are as large), so that bins of those alone, over the range of those alone, say
     * what to list. Where fewer than k threads have one within the bins, all tokens are counted. */
#pragma unroll 1
    for (;; largest = false) {
        Range r;
        if (largest) {
            mine = range_of_share<false>(x, 0, n).max;
            r = {mine, is_there(mine) ? mine : -kMinusInf};
        } else {
            r = range_of_share<true>(x, 0, n, Kept{keep, kKept});
        }
        r = range_of_workgroup(r, s);
        if (!is_there(r.max)) return nothing_there(id, prob);
        if (first) {
            if (mine == r.max) /* few threads have it */
                for_each_of(x, 0, n, Kept{nullptr, 0}, [&](float v) { return v == r.max; }, [&](float, int i) { atomicMin(&s.best, (uint32_t)i); });
            __syncthreads();
            if (threadIdx.x == 0) {
                *id = (int32_t)s.best;
                if (prob) *prob = 1.0f;
            }
            return;
        }
        const Grid g(r, set.t, n);
        if (largest && r.max < -kMinusInf) {
            if (is_there(mine)) into_bin(mine, g, true, false, s);
            __syncthreads();
            sum_bins(g, holds_for(set), s);
            counted = uniform(s.count[kLastBin]) >= (uint32_t)set.k;
            __syncthreads();
            if (!counted) {
                clear_bins(s);
                __syncthreads();
                continue;
            }
        }
        return finish_row(x, n, Kept{keep, counted ? 0 : kKept}, g, mine, counted ? Bins::counted : Bins::empty, set, id, prob, s);
    }
}

template <class T> __global__ void __launch_bounds__(kThreads) sample_row_kernel(const T *__restrict__ logits, SampleCall c) {
    __shared__ Shared s;
    const int seq = blockIdx.x;
    whole_row(logits + (size_t)seq * c.ld, c.n_vocab, settings_of(c, seq), c.ids + seq, c.probs ? c.probs + seq : nullptr, s);
}

/* ------------------------------------------------------------------ few sequences
 * Rows that have to be put into bins, by several workgroups each: their ranges, their bins, and the rest by one workgroup, in a launch
 * each. Other rows are the first launch's first workgroup's alone. (What comes after the bins was spread over the workgroups too, the
 * list by one launch and the pick by another, or by the last to finish: what a launch gains over 12 us it loses by starting, and fences
 * between the dies' L2s took 40 to 60 us where 32 sequences met them; with the eight at most that this route has now it was not measured.) */

constexpr int kMaxParts = 16;
struct Part { float max, min; };
struct Row { /* of the workspace */
    uint64_t weight[kBins];
    uint32_t count[kBins];
    Part part[kMaxParts];
    uint64_t unused[16];
};
static_assert(sizeof(Row) % 256 == 0, "rows start on 256 bytes");
__device__ __forceinline__ bool by_parts(const Settings &s) { return !takes_first(s) && !by_largest(s); }
struct Share { int lo, hi; };
__device__ __forceinline__ Share share_of(int n, int parts, int part) {
    const int per = ((n + parts - 1) / parts + 63) & ~63; /* (rows on 16 bytes stay so) */
    return {min(part * per, n), min((part + 1) * per, n)};
}

template <class T> __global__ void __launch_bounds__(kThreads) sample_parts_kernel(const T *__restrict__ logits, SampleCall c, int parts) {
    __shared__ Shared s;
    const int seq = blockIdx.x / (unsigned)parts, part = blockIdx.x - seq * parts;
    const T *x = logits + (size_t)seq * c.ld;
    const Settings set = settings_of(c, seq);
    if (!by_parts(set)) {
        if (part == 0) whole_row(x, c.n_vocab, set, c.ids + seq, c.probs ? c.probs + seq : nullptr, s);
        return;
    }
    Row *row = static_cast<Row *>(c.workspace) + seq;
    for (int i = part * kThreads + threadIdx.x; i < kBins; i += parts * kThreads) row->weight[i] = 0, row->count[i] = 0;
    const Share sh = share_of(c.n_vocab, parts, part);
    const Range r = range_of_workgroup(range_of_share<true>(x, sh.lo, sh.hi), s);
    if (threadIdx.x == 0) row->part[part] = {r.max, r.min};
}

/* the row's range, in every thread: a lane loads one part's */
__device__ Range range_of_parts(const Row *row, int parts) {
    const Part mine = row->part[min((int)threadIdx.x & (kMaxParts - 1), parts - 1)];
    Range r = {mine.max, mine.min};
#pragma unroll
    for (int off = kMaxParts / 2; off; off >>= 1) {
        r.max = fmaxf(r.max, __shfl_xor(r.max, off, 64));
        r.min = fminf(r.min, __shfl_xor(r.min, off, 64));
    }
    return {uniform(r.max), uniform(r.min)};
}

template <class T> __global__ void __launch_bounds__(kThreads) sample_bins_kernel(const T *__restrict__ logits, SampleCall c, int parts) {
    __shared__ Shared s;
    const int seq = blockIdx.x / (unsigned)parts, part = blockIdx.x - seq * parts;
    const Settings set = settings_of(c, seq);
    if (!by_parts(set)) return;
    Row *row = static_cast<Row *>(c.workspace) + seq;
    const Range r = range_of_parts(row, parts);
    if (!is_there(r.max) || r.max == -kMinusInf) return;
    const Grid g(r, set.t, c.n_vocab);
    clear_bins(s);
    __syncthreads();
    const Share sh = share_of(c.n_vocab, parts, part);
    fill_bins(logits + (size_t)seq * c.ld, sh.lo, sh.hi, Kept{nullptr, 0}, g, holds_for(set), s);
    __syncthreads();
    for (int i = threadIdx.x; i < kBins; i += kThreads) {
        if (const uint64_t w = s.weight[i]) atomicAdd((unsigned long long *)&row->weight[i], (unsigned long long)w);
        if (const uint32_t k = s.count[i]) atomicAdd(&row->count[i], k);
    }
}

template <class T> __global__ void __launch_bounds__(kThreads) sample_finish_kernel(const T *__restrict__ logits, SampleCall c, int parts) {
    __shared__ Shared s;
    const int seq = blockIdx.x;
    const Settings set = settings_of(c, seq);
    if (!by_parts(set)) return;
    const Row *row = static_cast<const Row *>(c.workspace) + seq;
    const T *x = logits + (size_t)seq * c.ld;
    int32_t *id = c.ids + seq;
    float *prob = c.probs ? c.probs + seq : nullptr;
    const Range r = range_of_parts(row, parts);
    if (!is_there(r.max)) return nothing_there(id, prob);
    for (int i = threadIdx.x; i < kBins; i += kThreads) s.weight[i] = row->weight[i], s.count[i] = row->count[i];
    if (threadIdx.x == 0) s.n_list = 0;
    __syncthreads();
    finish_row(x, c.n_vocab, Kept{nullptr, 0}, Grid(r, set.t, c.n_vocab), 0.0f, Bins::filled, set, id, prob, s);
}

/* Workgroups per sequence: 1 = the kernel of one, else the three launches. Of 128256 bf16 logits, rows that need bins (no top_k) take 51, 53
 * and 57 us by one workgroup each for 1, 4 and 16 sequences, 36, 39 and 47 by parts; rows that do not (top_k 40) 16 and 20, for the
 * two launches more; 16 sequences with settings of all kinds 57 and 70. Of 32003 logits a row takes 24 us at most by one. The rule follows
 * sizes alone, as the settings are on the GPU. */
int parts_for(int n_seq, int n_vocab) {
    if (n_seq > 8 || n_vocab < 65536) return 1;
    return kMaxParts;
}

template <class T> hipError_t sample(const SampleCall &c) {
    const T *x = static_cast<const T *>(c.logits);
    const int parts = parts_for(c.n_seq, c.n_vocab);
    if (parts == 1) {
        sample_row_kernel<T><<<c.n_seq, kThreads, 0, c.stream>>>(x, c);
    } else {
        sample_parts_kernel<T><<<c.n_seq * parts, kThreads, 0, c.stream>>>(x, c, parts);
        sample_bins_kernel<T><<<c.n_seq * parts, kThreads, 0, c.stream>>>(x, c, parts);
        sample_finish_kernel<T><<<c.n_seq, kThreads, 0, c.stream>>>(x, c, parts);
    }
    return hipGetLastError();
}

}  // namespace

size_t sample_workspace_bytes(int n_seq, int n_vocab) {
    const int parts = parts_for(n_seq, n_vocab);
    return parts == 1 ? 0 : (size_t)n_seq * sizeof(Row);
}

hipError_t launch_sample(uint32_t type, const SampleCall &c) {
    if (type == T_F32) return sample<float>(c);
    return type == T_F16 ? sample<_Float16>(c) : sample<Bf16>(c);
}

}  // namespace qlin
