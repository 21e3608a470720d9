/*
 * lora.hip - low-rank adapters of many requests beside a shared projection.
 *
 *   out[t, r] = Y[t, r] + scale_a sum_k B_a[r, k] h[t, k],   h[t, k] = sum_c A_a[k, c] X[t, c],   a = ids[t]
 *
 * for one to three tensors that share X, or, of two tensors (gate and up), out = silu(first) * second. A token whose id names no
 * adapter keeps its Y.
 *
 * Two launches: the first makes h (fp32, in the workspace, as partial sums over parts of the columns), the second adds the parts up
 * in their order and makes the results. Both go by tiles of 64 tokens. A wave holds one id per lane and finds the tile's classes,
 * tokens that share an adapter, by ballots; the tokens of a class are packed into groups of 16 columns of the matrix instruction, so
 * that an adapter is read once for all of them, whatever the order of the tokens. `slots` workgroups share a tile's classes: for a
 * decoding batch, in which nearly every token has its own adapter, one each.
 *   Products: where the adapter and X are of one 16-bit type the first launch multiplies them on v_mfma_f32_16x16x32 of that type
 * (products exact, sums fp32); every other pair is widened to fp32 and goes through v_mfma_f32_16x16x4_f32, and so does h times B,
 * since h rounded to 16 bits would cost results in F32 their precision.
 */
#include "qlin_device.h"
#include "qlin_internal.h"

#include <type_traits>

#include "mxfp4.h"

namespace qlin {

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

struct Bf16 { uint16_t bits; };
__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(_Float16 v) { return (float)v; }
__device__ __forceinline__ float to_f32(Bf16 v) { return __uint_as_float((uint32_t)v.bits << 16); }

template <class T, int N> struct alignas(sizeof(T) * N < 16 ? sizeof(T) * N : 16) Vec { T v[N]; };

template <class A, class B> struct Same { static constexpr bool value = false; };
template <class A> struct Same<A, A> { static constexpr bool value = true; };

constexpr int kTile = kLoraTile; /* tokens of a tile */
constexpr int kShrinkWaves = kLoraShrinkThreads / 64, kExpandWaves = kLoraExpandThreads / 64;

/* A wave's lanes read from LDS what others of its lanes wrote, and write it anew: one wave's requests to LDS stay in order, and this keeps the
 * compiler from changing it. No instruction. */
__device__ __forceinline__ void wave_meets() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

/* addresses that come out of a table are global ones: without this the loads would ask LDS as well */
template <class T> using Global = const T __attribute__((address_space(1))) *;

/* N elements p[at..], zeros from `end` on; VEC: p + at on the vector's alignment, at and end multiples of N */
template <class T, int N, bool VEC> __device__ __forceinline__ Vec<T, N> load(const T *p, int at, int end) {
    Vec<T, N> e = {};
    if constexpr (VEC) {
        typedef uint32_t Words __attribute__((ext_vector_type(sizeof(T) * N / 4 < 4 ? sizeof(T) * N / 4 : 4)));
        constexpr int kPieces = sizeof(T) * N / sizeof(Words);
        struct { Words w[kPieces]; } raw = {};
        if (at < end) {
#pragma unroll
            for (int i = 0; i < kPieces; i++) raw.w[i] = ((Global<Words>)(p + at))[i];
        }
        e = __builtin_bit_cast(Vec<T, N>, raw);
    } else {
        const Global<T> g = (Global<T>)p;
#pragma unroll
        for (int i = 0; i < N; i++)
            if (at + i < end) {
                if constexpr (Same<T, Bf16>::value) e.v[i].bits = ((Global<uint16_t>)p)[at + i];
                else e.v[i] = g[at + i];
            }
    }
    return e;
}

__device__ __forceinline__ bool on(const void *p, size_t bytes) { return ((uintptr_t)p & (bytes - 1)) == 0; }

/* an adapter as the kernels take it: rank 0 where the table's entry cannot be used */
struct Entry {
    const void *A, *B;
    int rank;
    float scale;
};
__device__ __forceinline__ Entry entry_of(const LoraEntry *table, int id, int max_rank) {
    if (id < 0 || !table) return {nullptr, nullptr, 0, 0.0f}; /* (no table where a tensor has no rows) */
    const LoraEntry *v = table + id;
    const void *A = v->A, *B = v->B;
    const int rank = v->rank;
    return {A, B, A && B && rank > 0 && rank <= max_rank ? rank : 0, v->scale};
}
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ const void *uniform(const void *p) {
    const uint64_t v = (uint64_t)p;
    return (const void *)((uint64_t)(uint32_t)uniform((int)(v >> 32)) << 32 | (uint32_t)uniform((int)v));
}

/* A group: up to 16 tokens of a tile that share an id, with what the second launch needs of their adapters. The first launch writes them. */
struct alignas(16) Group {
    int32_t id, n; /* n 0: none */
    uint8_t token[16];
    int32_t unused[2];
    struct {
        const void *B;
        int32_t rank;
        float scale;
    } of[3];
};
static_assert(sizeof(Group) == kLoraGroupBytes, "as the workspace is sized");

/* The tokens of a tile by adapter, found by the workgroup's first 256 threads, a token each. Tokens that share an id (-1 for one outside of the table)
 * are a class, in order, and a class is cut into groups of G; a token is the first of a group where a multiple of G tokens before it share its
 * id, which all threads count together. */
template <int G> struct Tile {
    struct Shared {
        alignas(16) int id[kTile];
        int equal[kShrinkWaves * 64 / kTile][kTile]; /* earlier tokens with the same id, by quarters of the tile */
        int before[kTile], first[kTile], list[G], in_wave[4];
        Entry entry[kTile];
    };
    int id, before;
    __device__ int find(Shared &s, const LoraCall &c, const LoraEntry *table, int tile) {
        const int t = threadIdx.x % kTile, quarter = threadIdx.x / kTile;
        const long long left = (long long)c.n_tok - (long long)tile * kTile;
        const int here = left < kTile ? (int)left : kTile;
        id = -2;
        Entry e = {nullptr, nullptr, 0, 0.0f};
        if (threadIdx.x < kTile) {
            if (t < here) {
                const int v = c.ids[(size_t)tile * kTile + t];
                id = v >= 0 && v < c.n_adapter ? v : -1;
                e = entry_of(table, id, c.max_rank);
            }
            s.id[t] = id;
        }
        __syncthreads();
        const int mine = s.id[t], low = 64 * quarter, word = __builtin_amdgcn_readfirstlane(t / 64);
        int equal = 0;
        if (quarter <= word)
            for (int j = 0; j < 64 && low + j < here; j += 4) {
                const int4 v = *reinterpret_cast<const int4 *>(&s.id[low + j]);
                equal += (v.x == mine && low + j < t) + (v.y == mine && low + j + 1 < t) + (v.z == mine && low + j + 2 < t) + (v.w == mine && low + j + 3 < t);
            }
        s.equal[quarter][t] = equal;
        __syncthreads();
        before = 0;
        uint64_t firsts = 0;
        if (threadIdx.x < kTile) {
#pragma unroll
            for (int q = 0; q < kShrinkWaves * 64 / kTile; q++) before += s.equal[q][t];
            s.before[t] = before;
            s.entry[t] = e;
            firsts = __ballot(id != -2 && before % G == 0);
            s.in_wave[t / 64] = __popcll(firsts);
        }
        __syncthreads();
        int start = 0, all = 0;
#pragma unroll
        for (int w = 0; w < kTile / 64; w++) {
            if (w < t / 64) start += s.in_wave[w];
            all += s.in_wave[w];
        }
        if (threadIdx.x < kTile && (firsts >> (t & 63)) & 1) s.first[start + __builtin_amdgcn_mbcnt_hi((uint32_t)(firsts >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)firsts, 0))] = t;
        __syncthreads();
        return all;
    }
    /* the tokens of the group that token t0 is the first of, into the list; their number */
    __device__ int gather(Shared &s, int t0) {
        if (threadIdx.x < kTile) {
            const int place = before - s.before[t0];
            const bool in = id == s.id[t0] && place >= 0 && place < G;
            if (in) s.list[place] = threadIdx.x;
            s.in_wave[threadIdx.x / 64] = __popcll(__ballot(in));
        }
        __syncthreads();
        return s.in_wave[0] + s.in_wave[1] + s.in_wave[2] + s.in_wave[3];
    }
};

/* ------------------------------------------------------------------ h = A x */

/* acc += w . x over 32 columns, eight to a lane */
template <class W, class X> __device__ __forceinline__ f32x4 multiply(const Vec<W, 8> &w, const Vec<X, 8> &x, f32x4 acc) {
    if constexpr (Same<W, Bf16>::value && Same<X, Bf16>::value) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, w), __builtin_bit_cast(bf16x8, x), acc, 0, 0, 0);
    } else if constexpr (Same<W, _Float16>::value && Same<X, _Float16>::value) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, w), __builtin_bit_cast(f16x8, x), acc, 0, 0, 0);
    } else { /* the e-th of a lane's eight columns with the e-th of the other lanes': any order of columns does, the same on both sides */
#pragma unroll
        for (int e = 0; e < 8; e++) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(to_f32(w.v[e]), to_f32(x.v[e]), acc, 0, 0, 0);
        return acc;
    }
}

/* a stage: U x 32 columns, as a fragment each per group of 16 ranks or tokens; WHOLE: all of its columns are there */
template <class W, class X, int RT, int NJ, int U> struct Stage {
    Vec<W, 8> w[U][RT];
    Vec<X, 8> x[U][NJ];
    template <bool WHOLE> __device__ __forceinline__ void fetch(const W *const (&a)[RT], const X *const (&t)[NJ], int stage, int n_cols) {
        const int at = 32 * U * stage + 8 * ((threadIdx.x & 63) >> 4), end = WHOLE ? 0x7FFFFFFF : n_cols;
#pragma unroll
        for (int j = 0; j < NJ; j++)
#pragma unroll
            for (int u = 0; u < U; u++) x[u][j] = load<X, 8, true>(t[j], at + 32 * u, end);
#pragma unroll
        for (int i = 0; i < RT; i++)
#pragma unroll
            for (int u = 0; u < U; u++) w[u][i] = load<W, 8, true>(a[i], at + 32 * u, end);
    }
    __device__ __forceinline__ void add_to(f32x4 (&acc)[NJ][RT]) const {
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int j = 0; j < NJ; j++)
#pragma unroll
                for (int i = 0; i < RT; i++) acc[j][i] = multiply(w[u][i], x[u][j], acc[j][i]);
    }
};
/* 64 columns, a whole line of 128 bytes of a row in 16 bits, where two such stages leave the registers of four waves per SIMD */
template <class W, class X, int RT, int NJ> constexpr int stage_steps() { return (RT * sizeof(W) + NJ * sizeof(X)) <= 8 ? 2 : 1; }

/* sums over steps [k0, k1) of 32 columns for RT groups of 16 ranks and NJ groups of 16 tokens; k0 even; rows of A from its rank on give sums that are
 * not looked at */
template <class W, class X, int RT, int NJ>
__device__ __forceinline__ void shrink_sums(bool vec, const W *A, int rank0, int rank, const X *const (&x)[NJ], int n_cols, int k0, int k1, f32x4 (&acc)[NJ][RT]) {
    const int lane = threadIdx.x & 63;
    const W *a[RT];
#pragma unroll
    for (int i = 0; i < RT; i++) {
        const int row = rank0 + 16 * i + (lane & 15);
        a[i] = A + (size_t)(row < rank ? row : rank - 1) * n_cols;
    }
    if (vec) { /* the next stage is on its way while one is multiplied; behind the last one it is that once more */
        constexpr int U = stage_steps<W, X, RT, NJ>();
        const int whole = n_cols / (32 * U), all = (k1 + U - 1) / U, end = all < whole ? all : whole;
        Stage<W, X, RT, NJ, U> s[2];
        int k = k0 / U;
        if (k < end) {
            s[0].template fetch<true>(a, x, k, n_cols);
            for (;;) {
                s[1].template fetch<true>(a, x, k + 1 < end ? k + 1 : k, n_cols);
                s[0].add_to(acc);
                if (++k == end) break;
                s[0].template fetch<true>(a, x, k + 1 < end ? k + 1 : k, n_cols);
                s[1].add_to(acc);
                if (++k == end) break;
            }
        }
        if (end < all) {
            s[0].template fetch<false>(a, x, end, n_cols);
            s[0].add_to(acc);
        }
    } else { /* rows that do not lie on 16 bytes: element by element, eight at a time */
        const int end = 32 * k1 < n_cols ? 32 * k1 : n_cols;
#pragma unroll 1
        for (int first = 32 * k0; first < end; first += 32) {
            const int at = first + 8 * (lane >> 4);
#pragma unroll
            for (int i = 0; i < RT; i++) {
                const Vec<W, 8> w = load<W, 8, false>(a[i], at, n_cols);
#pragma unroll
                for (int j = 0; j < NJ; j++) acc[j][i] = multiply(w, load<X, 8, false>(x[j], at, n_cols), acc[j][i]);
            }
        }
    }
}

template <class W, class X, int RT, int NJ>
__global__ void __launch_bounds__(64 * kShrinkWaves)
lora_shrink_kernel(LoraCall c, LoraPlan p) {
    __shared__ f32x4 red[kShrinkWaves][NJ * RT][64];
    __shared__ typename Tile<16 * NJ>::Shared shared;
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    /* workgroups b and b + 8 share a die: the tensors of the same tokens, one after the other */
    uint32_t b = blockIdx.x % 8 + blockIdx.x / 8 / c.n_mat * 8;
    const int mat = blockIdx.x / 8 % c.n_mat;
    if (b >= p.shrink_units()) return;
    const int part = b % p.parts; b /= p.parts;
    const int slot = b % p.shrink_slots; b /= p.shrink_slots;
    const int block = b % p.rank_blocks, tile = b / p.rank_blocks;
    const X *x0 = static_cast<const X *>(c.X);
    const int rank0 = block * 16 * RT;
    const int pairs = (c.n_cols + 63) / 64, share = part * kShrinkWaves + wv, shares = p.parts * kShrinkWaves;
    const int k0 = 2 * (int)((long long)pairs * share / shares), k1 = 2 * (int)((long long)pairs * (share + 1) / shares);
    const bool x_vec = c.n_cols % 8 == 0 && on(c.X, 16) && (size_t)c.ldx * sizeof(X) % 16 == 0;
    Group *records = static_cast<Group *>(c.workspace) + (size_t)tile * p.groups;
    Tile<16 * NJ> tokens;
    const int all = tokens.find(shared, c, mat == 0 ? c.m[0].adapters : mat == 1 ? c.m[1].adapters : c.m[2].adapters, tile);
    for (int s = slot; s * NJ < p.groups; s += p.shrink_slots) {
        if (s >= all) { /* the second launch looks at every record */
            if (part == 0 && block == 0 && mat == 0 && threadIdx.x < NJ) records[s * NJ + threadIdx.x].n = 0;
            continue;
        }
        const int t0 = uniform(shared.first[s]), n = uniform(tokens.gather(shared, t0));
        const Entry e = {uniform(shared.entry[t0].A), uniform(shared.entry[t0].B), uniform(shared.entry[t0].rank), shared.entry[t0].scale};
        size_t token[NJ];
#pragma unroll
        for (int j = 0; j < NJ; j++) {
            const int q = 16 * j + (lane & 15);
            token[j] = (size_t)tile * kTile + (q < n ? shared.list[q] : t0);
            if (part == 0 && block == 0 && wv == 0 && lane < 16) {
                Group &r = records[s * NJ + j];
                if (mat == 0) r.token[lane] = (uint8_t)(token[j] % kTile);
                if (lane == 0) {
                    if (mat == 0) r.n = n - 16 * j > 16 ? 16 : n - 16 * j > 0 ? n - 16 * j : 0;
                    r.of[mat].B = e.B;
                    r.of[mat].rank = e.rank;
                    r.of[mat].scale = e.scale;
                }
            }
        }
        if (e.rank > rank0) { /* else no adapter, or none of its ranks here: nothing is read of h either */
            const X *x[NJ];
#pragma unroll
            for (int j = 0; j < NJ; j++) x[j] = x0 + token[j] * c.ldx;
            f32x4 acc[NJ][RT] = {};
            if (k0 < k1) shrink_sums<W, X, RT, NJ>(x_vec && on(e.A, 16), static_cast<const W *>(e.A), rank0, e.rank, x, c.n_cols, k0, k1, acc);
            /* the waves' sums, added in the waves' order */
#pragma unroll
            for (int j = 0; j < NJ; j++)
#pragma unroll
                for (int i = 0; i < RT; i++) red[wv][j * RT + i][lane] = acc[j][i];
            __syncthreads();
            for (int f = wv; f < NJ * RT; f += kShrinkWaves) {
                const int j = f / RT, i = f % RT;
                f32x4 v = red[0][f][lane];
#pragma unroll
                for (int w = 1; w < kShrinkWaves; w++) v += red[w][f][lane];
                const int r = rank0 + 16 * i + 4 * (lane >> 4);
#pragma unroll
                for (int q = 0; q < 4; q++)
                    if (r + q >= e.rank) v[q] = 0.0f;
                const size_t t = (j > 0 ? token[NJ - 1] : token[0]) + (size_t)mat * c.n_tok;
                if (16 * j + (lane & 15) >= n || r >= p.rank_pad) continue;
                char *h = static_cast<char *>(c.workspace) + p.h_at;
                if (p.split) {
                    v *= e.scale;
                    bf16x4 three[3];
#pragma unroll
                    for (int q = 0; q < 4; q++) {
                        three[0][q] = (__bf16)v[q];
                        const float rest = v[q] - (float)three[0][q];
                        three[1][q] = (__bf16)rest;
                        three[2][q] = (__bf16)(rest - (float)three[1][q]);
                    }
                    uint16_t *to = reinterpret_cast<uint16_t *>(h) + (t * p.rank_pad + r / 16 * 16) * 3 + r % 16;
#pragma unroll
                    for (int q = 0; q < 3; q++) *reinterpret_cast<bf16x4 *>(to + 16 * q) = three[q];
                } else {
                    *reinterpret_cast<f32x4 *>(reinterpret_cast<float *>(h) + ((size_t)part * c.n_mat * c.n_tok + t) * p.rank_pad + r) = v;
                }
            }
        }
        __syncthreads();
    }
}

/* ------------------------------------------------------------------ Y + B h */

/* four consecutive elements of a row, T float or the bits of a 16-bit type; WHOLE: all four are there, on the vector's alignment */
template <class T, bool WHOLE> __device__ __forceinline__ f32x4 load4(const void *base, size_t at, int left, bool bf16) {
    const T *p = static_cast<const T *>(base) + at;
    Vec<T, 4> v = {};
    if constexpr (WHOLE) {
        v = *reinterpret_cast<const Vec<T, 4> *>(p);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (i < left) v.v[i] = p[i];
    }
    f32x4 y;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (sizeof(T) == 4) y[i] = v.v[i];
        else y[i] = bf16 ? to_f32(Bf16{v.v[i]}) : to_f32(__builtin_bit_cast(_Float16, v.v[i]));
    }
    return y;
}
/* the one rounding of a result in 16 bits: to the nearest, ties to even */
template <class T, bool WHOLE> __device__ __forceinline__ void store4(void *base, size_t at, int left, bool bf16, f32x4 y) {
    T *p = static_cast<T *>(base) + at;
    Vec<T, 4> v;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (sizeof(T) == 4) v.v[i] = y[i];
        else v.v[i] = bf16 ? __builtin_bit_cast(uint16_t, (__bf16)y[i]) : __builtin_bit_cast(uint16_t, (_Float16)y[i]);
    }
    if constexpr (WHOLE) {
        *reinterpret_cast<Vec<T, 4> *>(p) = v;
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (i < left) p[i] = v.v[i];
    }
}

/* acc += B h over an adapter's ranks, for MT groups of 16 rows x 16 tokens; h: the lane's token in the workspace, of which the parts are
 * added in their order */
template <class W, int MT, bool VEC>
__device__ __forceinline__ void expand_sums(const Entry &e, int row0, int n_rows, const float *h, size_t part, int parts, f32x4 (&acc)[MT]) {
    const int lane = threadIdx.x & 63, g = lane >> 4;
    const W *b[MT];
#pragma unroll
    for (int i = 0; i < MT; i++) {
        const int row = row0 + 16 * i + (lane & 15);
        b[i] = static_cast<const W *>(e.B) + (size_t)(row < n_rows ? row : n_rows - 1) * e.rank;
    }
    for (int r = 4 * g; r < e.rank + 4 * g; r += 16) {
        Vec<W, 4> w[MT];
#pragma unroll
        for (int i = 0; i < MT; i++) w[i] = load<W, 4, VEC>(b[i], r, e.rank);
        f32x4 v = *reinterpret_cast<const f32x4 *>(h + r);
        for (int s = 1; s < parts; s += 4) { /* (four on their way at a time) */
            f32x4 more[4];
#pragma unroll
            for (int q = 0; q < 4; q++) more[q] = *reinterpret_cast<const f32x4 *>(h + (s + q < parts ? s + q : 0) * part + r);
#pragma unroll
            for (int q = 0; q < 4; q++)
                if (s + q < parts) v += more[q];
        }
        v *= e.scale;
#pragma unroll
        for (int q = 0; q < 4; q++)
#pragma unroll
            for (int i = 0; i < MT; i++) acc[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(to_f32(w[i].v[q]), v[q], acc[i], 0, 0, 0);
    }
}

/* the same where the workspace holds scale h as three numbers in bf16, whose sum it is: 16 first parts of 16 ranks, their second and their third
 * ones. The first instruction takes first parts in its first 16 columns and second parts in the others, the second one third parts, with
 * the same 16 columns of B on both halves: the products are exact. */
template <int MT, bool VEC>
__device__ __forceinline__ void expand_split(const Entry &e, int row0, int n_rows, const uint16_t *h, f32x4 (&acc)[MT]) {
    const int lane = threadIdx.x & 63, g = lane >> 4;
    const Bf16 *b[MT];
#pragma unroll
    for (int i = 0; i < MT; i++) {
        const int row = row0 + 16 * i + (lane & 15);
        b[i] = static_cast<const Bf16 *>(e.B) + (size_t)(row < n_rows ? row : n_rows - 1) * e.rank;
    }
    for (int r = 0; r < e.rank; r += 16) {
        Vec<Bf16, 8> w[MT];
#pragma unroll
        for (int i = 0; i < MT; i++) w[i] = load<Bf16, 8, VEC>(b[i], r + 8 * (g & 1), e.rank);
        const bf16x8 v = *reinterpret_cast<const bf16x8 *>(h + 3 * r + 8 * g);
        bf16x8 rest = *reinterpret_cast<const bf16x8 *>(h + 3 * r + 32 + 8 * (g & 1));
        if (g > 1) rest = bf16x8{};
#pragma unroll
        for (int i = 0; i < MT; i++) acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, w[i]), rest, acc[i], 0, 0, 0);
#pragma unroll
        for (int i = 0; i < MT; i++) acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, w[i]), v, acc[i], 0, 0, 0);
    }
}

/* a wave: 16 MT rows of one tensor or, PAIR, of gate and up; T, O: Y's and the result's type, float or the bits of a 16-bit one. The sums come
 * out of the matrix instruction with a lane's four rows 16 tokens apart; they go through LDS, so that Y is read and results are written in
 * runs of a token's 16 MT rows. */
template <class W, class T, class O, int MT, bool PAIR, bool SPLIT>
__global__ void __launch_bounds__(64 * kExpandWaves)
lora_expand_kernel(LoraCall c, LoraPlan p) {
    constexpr int MATS = PAIR ? 2 : 1, kRows = 16 * MT, kStride = kRows + 4; /* (a token's run behind the one before: other banks) */
    constexpr int kLanes = kRows / 4, kRuns = 64 / kLanes, kSteps = 16 / kRuns; /* lanes of a run, runs at a time */
    __shared__ float turn[kExpandWaves][16 * kStride];
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int mat = 0, block = blockIdx.x % p.row_blocks_all;
    const int unit = blockIdx.x / p.row_blocks_all, slot = unit % p.expand_slots, tile = unit / p.expand_slots;
    LoraTensor m = c.m[0];
    if (!PAIR) {
        if (block >= p.row_blocks[0]) {
            block -= p.row_blocks[0];
            mat = 1;
            m = c.m[1];
            if (block >= p.row_blocks[1]) {
                block -= p.row_blocks[1];
                mat = 2;
                m = c.m[2];
            }
        }
    }
    const int row0 = (block * kExpandWaves + wv) * kRows;
    if (row0 >= m.n_rows) return;
    const bool y_bf16 = c.y_type == T_BF16, o_bf16 = c.out_type == T_BF16;
    const bool whole = row0 + kRows <= m.n_rows && on(m.Y, 4 * sizeof(T)) && (!PAIR || on(c.m[1].Y, 4 * sizeof(T))) && m.ldy % 4 == 0 && on(m.out, 4 * sizeof(O)) && m.ldo % 4 == 0;
    const size_t part = (size_t)c.n_mat * c.n_tok * p.rank_pad;
    const int row = 4 * (lane % kLanes), left = m.n_rows - row0 - row; /* of the run */
    const char *hs = static_cast<const char *>(c.workspace) + p.h_at;
    for (int u = slot; u < p.groups; u += p.expand_slots) {
        const Group *group = static_cast<const Group *>(c.workspace) + (size_t)tile * p.groups + u;
        const int n = uniform(group->n);
        if (n == 0) continue;
        const size_t token = (size_t)tile * kTile + group->token[lane & 15]; /* (behind the group's tokens: the first) */
        size_t run[kSteps]; /* the tokens of the lane's runs */
#pragma unroll
        for (int s = 0; s < kSteps; s++) run[s] = (size_t)tile * kTile + group->token[s * kRuns + lane / kLanes];
        Entry of[MATS];
#pragma unroll
        for (int a = 0; a < MATS; a++) of[a] = {nullptr, uniform(group->of[mat + a].B), uniform(group->of[mat + a].rank), group->of[mat + a].scale};
        f32x4 y[MATS][kSteps];
        auto load_all = [&](auto w) {
#pragma unroll
            for (int s = 0; s < kSteps; s++) {
                y[0][s] = load4<T, decltype(w)::value>(m.Y, run[s] * m.ldy + row0 + row, left, y_bf16);
                if constexpr (PAIR) y[1][s] = load4<T, decltype(w)::value>(c.m[1].Y, run[s] * m.ldy + row0 + row, left, y_bf16);
            }
        };
        if (whole) load_all(std::true_type{});
        else load_all(std::false_type{});
#pragma unroll
        for (int a = 0; a < MATS; a++) {
            const Entry e = of[a];
            if (e.rank == 0) continue;
            f32x4 acc[MT] = {};
            const size_t h_at = ((size_t)(mat + a) * c.n_tok + token) * p.rank_pad;
            if constexpr (SPLIT) {
                const uint16_t *h = reinterpret_cast<const uint16_t *>(hs) + 3 * h_at;
                if (e.rank % 8 == 0 && on(e.B, 16))
                    expand_split<MT, true>(e, row0, m.n_rows, h, acc);
                else
                    expand_split<MT, false>(e, row0, m.n_rows, h, acc);
            } else {
                const float *h = reinterpret_cast<const float *>(hs) + h_at;
                if (e.rank % 4 == 0 && on(e.B, 4 * sizeof(W)))
                    expand_sums<W, MT, true>(e, row0, m.n_rows, h, part, p.parts, acc);
                else
                    expand_sums<W, MT, false>(e, row0, m.n_rows, h, part, p.parts, acc);
            }
            wave_meets();
#pragma unroll
            for (int i = 0; i < MT; i++) *reinterpret_cast<f32x4 *>(&turn[wv][(lane & 15) * kStride + 16 * i + 4 * (lane >> 4)]) = acc[i];
            wave_meets();
#pragma unroll
            for (int s = 0; s < kSteps; s++) y[a][s] += *reinterpret_cast<const f32x4 *>(&turn[wv][(s * kRuns + lane / kLanes) * kStride + row]);
        }
        if constexpr (PAIR) {
#pragma unroll
            for (int s = 0; s < kSteps; s++)
#pragma unroll
                for (int r = 0; r < 4; r++) y[0][s][r] = mxfp4::silu_mul(y[0][s][r], y[MATS - 1][s][r]);
        }
        auto store_all = [&](auto w) {
#pragma unroll
            for (int s = 0; s < kSteps; s++)
                if (s * kRuns + lane / kLanes < n) store4<O, decltype(w)::value>(m.out, run[s] * m.ldo + row0 + row, left, o_bf16, y[0][s]);
        };
        if (whole) store_all(std::true_type{});
        else store_all(std::false_type{});
    }
}

template <class W, class X, int RT> void launch_shrink(const LoraCall &c, const LoraPlan &p) {
    const dim3 grid((uint32_t)p.shrink_workgroups()), block(kLoraShrinkThreads);
    if (p.token_groups == 1)
        hipLaunchKernelGGL((lora_shrink_kernel<W, X, RT, 1>), grid, block, 0, c.stream, c, p);
    else
        hipLaunchKernelGGL((lora_shrink_kernel<W, X, RT, 2>), grid, block, 0, c.stream, c, p);
}
template <class W, class X> void launch_shrink(const LoraCall &c, const LoraPlan &p) {
    if (p.rank_tiles == 1) launch_shrink<W, X, 1>(c, p);
    else if (p.rank_tiles == 2) launch_shrink<W, X, 2>(c, p);
    else launch_shrink<W, X, 4>(c, p);
}

template <class W, class T, class O, bool PAIR> void launch_expand(const LoraCall &c, const LoraPlan &p) {
    const dim3 grid((uint32_t)p.expand_workgroups()), block(kLoraExpandThreads);
    if constexpr (Same<W, Bf16>::value) {
        if (p.split) {
            hipLaunchKernelGGL((lora_expand_kernel<W, T, O, 4, PAIR, true>), grid, block, 0, c.stream, c, p);
            return;
        }
    }
    if (p.row_tiles == 1)
        hipLaunchKernelGGL((lora_expand_kernel<W, T, O, 1, PAIR, false>), grid, block, 0, c.stream, c, p);
    else
        hipLaunchKernelGGL((lora_expand_kernel<W, T, O, 4, PAIR, false>), grid, block, 0, c.stream, c, p);
}
template <class W, bool PAIR> void launch_expand(const LoraCall &c, const LoraPlan &p) {
    const bool y32 = c.y_type == T_F32, o32 = c.out_type == T_F32;
    if (y32 && o32) launch_expand<W, float, float, PAIR>(c, p);
    else if (y32) launch_expand<W, float, uint16_t, PAIR>(c, p);
    else if (o32) launch_expand<W, uint16_t, float, PAIR>(c, p);
    else launch_expand<W, uint16_t, uint16_t, PAIR>(c, p);
}

template <class W> hipError_t launch_both(const LoraCall &c, const LoraPlan &p) {
    if (c.x_type == T_F32) launch_shrink<W, float>(c, p);
    else if (c.x_type == T_F16) launch_shrink<W, _Float16>(c, p);
    else launch_shrink<W, Bf16>(c, p);
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
    if (c.pair) launch_expand<W, true>(c, p);
    else launch_expand<W, false>(c, p);
    return hipGetLastError();
}

}  // namespace

/* 16 ranks, 32 or 64 to a workgroup */
static int lora_rank_tiles(int max_rank) { return max_rank <= 16 ? 1 : max_rank <= 32 ? 2 : 4; }
static int lora_token_groups(int n_tok) { return n_tok >= 1024 ? 2 : 1; }

/* how many parts the columns are cut into: enough workgroups for the chip, as far as their number is known without the ids, and at
 * least 64 columns for a wave; the second launch reads every part of h again for each of its rows' workgroups */
static int lora_parts(int n_mat, int max_rank, int n_cols, int n_tok) {
    const int rt = lora_rank_tiles(max_rank);
    const long long tokens = 16ll * lora_token_groups(n_tok), groups = (n_tok + tokens - 1) / tokens * n_mat * ((max_rank + 16 * rt - 1) / (16 * rt));
    const long long want = groups >= 96 ? 1 : 256 / groups, most = n_cols / (64 * kShrinkWaves);
    const long long parts = want < most ? want : most;
    return (int)(parts > 8 ? 8 : parts < 1 ? 1 : parts);
}

/* the groups of every tile, of which there are at most as many as tokens, or half of them twice as many; then h in fp32 for each part, or, of
 * one part, as three numbers in bf16 */
static size_t lora_records(int n_tok, int groups) { return ((size_t)n_tok + kTile - 1) / kTile * groups * sizeof(Group); }
size_t lora_workspace_bytes(int n_mat, int max_rank, int n_cols, int n_tok) {
    const int parts = lora_parts(n_mat, max_rank, n_cols, n_tok);
    return lora_records(n_tok, (n_tok < kTile ? n_tok : kTile) * lora_token_groups(n_tok)) + (size_t)n_mat * n_tok * ((max_rank + 15) / 16 * 16) * (parts == 1 ? 6 : 4 * (size_t)parts);
}

LoraPlan lora_plan(const LoraCall &c) {
    LoraPlan p;
    p.tiles = (int)(((long long)c.n_tok + kTile - 1) / kTile);
    p.rank_pad = (c.max_rank + 15) / 16 * 16;
    p.rank_tiles = lora_rank_tiles(c.max_rank);
    p.rank_blocks = (c.max_rank + 16 * p.rank_tiles - 1) / (16 * p.rank_tiles);
    p.token_groups = lora_token_groups(c.n_tok);
    p.parts = lora_parts(c.n_mat, c.max_rank, c.n_cols, c.n_tok);
    p.split = p.parts == 1 && c.lora_type == T_BF16;
    p.row_tiles = c.n_tok <= 8 && !p.split ? 1 : 4;
    p.n_mat = c.n_mat;
    p.row_blocks_all = 0;
    for (int i = 0; i < 3; i++) {
        const int rows = 16 * kExpandWaves * p.row_tiles;
        p.row_blocks[i] = i < c.n_mat && (i == 0 || !c.pair) ? (int)(((long long)c.m[i].n_rows + rows - 1) / rows) : 0;
        p.row_blocks_all += p.row_blocks[i];
    }
    /* a workgroup for each group of tokens that a tile can have, unless that makes too many, but then one for each that a prompt of one adapter has */
    const int tokens = c.n_tok < kTile ? c.n_tok : kTile, size = 16 * p.token_groups;
    const long long classes = c.n_adapter + 1ll < tokens ? c.n_adapter + 1ll : tokens, bound = (tokens - classes) / size + classes, full = (tokens + size - 1) / size;
    auto slots = [&](long long bound, long long full, long long others, long long most) {
        const long long want = others > 0 && most / others > full ? most / others : full;
        return (int)(want < bound ? want : bound);
    };
    p.groups = (int)bound * p.token_groups;
    p.h_at = lora_records(c.n_tok, p.groups);
    p.shrink_slots = slots(bound, full, (long long)p.tiles * p.n_mat * p.rank_blocks * p.parts, 1024);
    p.expand_slots = slots(p.groups, full * p.token_groups, (long long)p.tiles * p.row_blocks_all, 16384);
    return p;
}

hipError_t launch_lora(const LoraCall &c, const LoraPlan &p) {
    return c.lora_type == T_F32 ? launch_both<float>(c, p) : c.lora_type == T_F16 ? launch_both<_Float16>(c, p) : launch_both<Bf16>(c, p);
}

}  // namespace qlin
