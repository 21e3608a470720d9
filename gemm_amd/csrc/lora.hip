/*
 * lora.hip - low-rank adapters of many requests beside a shared projection.
 *
 *   out[t, r] = Y[t, r] + scale_a sum_k B_a[r, k] h[t, k],   h[t, k] = sum_c A_a[k, c] X[t, c],   a = ids[t]
 *
 * for one to three tensors that share X, or, of two tensors (gate and up), out = silu(first) * second. A token whose id names no
 * adapter keeps its Y.
 *
 * What has to move: X once, each adapter's A and B once, Y and the result once (2048 tokens, gate and up of 14336 rows, 322 MB: 63 us at the
 * 5.12 TB/s of a copy). Multiplications are few, 4 max_rank to a result.
 *
 * A few tokens (lora_few_kernel): one launch. A workgroup takes 1024 results of a token and makes h for itself. Where the workgroups' reads of A add up to
 * little that costs less than a second launch and h in memory: 1 token beside Q, K and V of 4096 columns, rank 16: 5.0 us, 7.4 + 4.1 in two launches; 24
 * tokens: 8.3 us, 7.9 + 4.9; 48 tokens: 9.9, 9.0 + 4.9; 4 tokens beside gate and up of 14336 rows, rank 32: 20.3, 7.4 + 5.9. The limits (kFewBytes) are no more than
 * roughly where the two ways meet, and beyond them are calls that one launch would serve better: 48 tokens of rank 32: 15.4, taken are 9.8 + 6.3; 4 tokens of 14336
 * columns, 4096 rows, rank 16: 9.6, taken 7.5 + 4.2; 1 token of rank 128: 10.3 (with twice the LDS), taken 10.9 + 4.4, where 22 tokens are better off with two, 19.7 and 10.5 + 6.0.
 *
 * Any number of them: two launches, by tiles of 256 tokens.
 *   lora_shrink_kernel makes h. A workgroup finds the tile's classes, tokens that share an adapter, packs the tokens of a class into groups of 16 (or
 * 32), the columns of the matrix instruction, so that an adapter is read once for them whatever the order of the tokens, and takes one group of one tensor, or a
 * few; its 16 waves share the columns and add their sums in order. It also writes a record of each group, from which the second launch knows all
 * that it needs with one load. 2048 tokens, Q, K and V of 4096 columns, rank 64: 27 us; X comes three times, twice from L2.
 *   lora_expand_kernel: a wave takes 64 rows of a tensor (or of gate and up) and a group, and writes results in runs of 128 to 256 bytes of a token. 2048
 * tokens, gate and up of 14336 rows, 305 MB: 66 us, 90% of a copy's rate.
 *   Products: where the adapter and X are of one 16-bit type the first launch multiplies them on v_mfma_f32_16x16x32 of that type
 * (products exact, sums fp32); every other pair is widened to fp32 and goes through v_mfma_f32_16x16x4_f32, and so does h times B,
 * since h rounded to 16 bits would cost results in F32 their precision. Of bf16 adapters and many tokens scale h is cut into three bf16 numbers, which hold its 24
 * bits, and goes through the bf16 instruction three times, the products exact again: 23 us for the second launch of the case above, 29 with fp32.
 *   No atomics: the same call gives the same bits.
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

/* N elements p[at..], zeros from `end` on, at any element's address; WHOLE: at and end are multiples of N */
template <class T, int N, bool WHOLE> __device__ __forceinline__ Vec<T, N> load(const T *p, int at, int end) {
    typedef uint32_t Words __attribute__((ext_vector_type(sizeof(T) * N / 4 < 4 ? sizeof(T) * N / 4 : 4)));
    typedef Words Anywhere __attribute__((aligned(sizeof(T))));
    constexpr int kPieces = sizeof(T) * N / sizeof(Words);
    struct { Words w[kPieces]; } raw = {};
    if (WHOLE ? at < end : at + N <= end) {
#pragma unroll
        for (int i = 0; i < kPieces; i++) raw.w[i] = ((Global<Anywhere>)(p + at))[i];
    }
    Vec<T, N> e = __builtin_bit_cast(Vec<T, N>, raw);
    if (!WHOLE && at < end && at + N > end) {
#pragma unroll
        for (int i = 0; i < N - 1; i++)
            if (at + i < end) {
                if constexpr (Same<T, Bf16>::value) e.v[i].bits = ((Global<uint16_t>)p)[at + i];
                else e.v[i] = ((Global<T>)p)[at + i];
            }
    }
    return e;
}

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
    int32_t n;      /* 0: none */
    int32_t place;  /* of its first token among the tile's tokens sorted by id */
    uint8_t token[16];
    int32_t to_16_bytes[2];
    struct {
        const void *B;
        int32_t rank;
        float scale;
    } of[3];
};
static_assert(sizeof(Group) == kLoraGroupBytes, "as the workspace is sized");

/* Where the workspace holds h of a group: its tokens stand next to each other, in the order in which the lanes of the second launch take
 * them. In fp32: piece 4 c + g of 16 bytes per token, ranks 16 c + 4 g to + 3, for each part. As three numbers in bf16: piece 12 c + 4 k + g,
 * the k-th numbers of ranks 32 c + 8 g to + 7. */
__device__ __forceinline__ size_t piece_at(size_t first, int pieces, int piece, int n, int q) { return (first * pieces + (size_t)piece * n + q) * 16; }

/* The tokens of a tile by adapter, found by a whole workgroup: tokens that share an id (-1 for one outside of the table) are a class, a class is cut into
 * groups of G tokens in order. Each token counts the tokens with a lower id and those with the same one, a quarter of them on each of four waves; from
 * that it knows its place among the tokens sorted by id, and whether it is the first of a group. */
template <int G> struct Tile {
    static constexpr int kQuarters = kShrinkWaves * 64 / kTile, kFewRuns = 12;
    alignas(16) int id[kTile];
    int counts[kQuarters][kTile]; /* lower << 20 | same << 10 | same and earlier, of the tokens' own quarter */
    int in_wave[kTile / 64];
    uint8_t token[kTile], first[kTile], size[kTile]; /* the sorted tokens; where each group begins, and its number of tokens */
    Entry entry[kTile];
    int groups;

    __device__ void find(const LoraCall &c, const LoraEntry *table, int tile) {
        const int t = threadIdx.x % kTile, quarter = threadIdx.x / kTile, word = uniform(t / 64);
        const long long left = (long long)c.n_tok - (long long)tile * kTile;
        const int here = left < kTile ? (int)left : kTile;
        Entry e = {nullptr, nullptr, 0, 0.0f};
        if (threadIdx.x < kTile) {
            int mine = 0x7FFFFFFF; /* behind the last token */
            if (t < here) {
                const int v = c.ids[(size_t)tile * kTile + t];
                mine = v >= 0 && v < c.n_adapter ? v : -1;
                e = entry_of(table, mine, c.max_rank);
            }
            id[t] = mine;
        }
        __syncthreads();
        /* ids by words of 64 tokens, and how often a token's is another than the one's before */
        typedef int Ids __attribute__((ext_vector_type(kTile / 64))); /* (arrays would come to lie in memory) */
        const int lane = t & 63;
        Ids v;
        int runs = 0;
#pragma unroll
        for (int w = 0; w < kTile / 64; w++) {
            v[w] = id[64 * w + lane];
            runs += __popcll(__ballot(v[w] != id[64 * w + lane > 0 ? 64 * w + lane - 1 : 0]));
        }
        int place = 0, before = 0, all = 0, g = 0, total = 0;
        bool is_first = false;
        if (runs <= kFewRuns) { /* prompts: class by class in the order of their first tokens, by each of the first four waves */
            if (threadIdx.x < kTile) {
                int placed = 0;
                for (int w = 0; w < kTile / 64; w++) {
                    const int ids_here = w == 0 ? v[0] : w == 1 ? v[1] : w == 2 ? v[2] : v[3];
                    for (uint64_t rest = __ballot(64 * w + lane < here); rest;) {
                        const int which = __builtin_amdgcn_readlane(ids_here, __builtin_ctzll(rest));
                        int n = 0, earlier = 0, in_earlier_words = 0;
                        uint64_t own = 0;
#pragma unroll
                        for (int u = 0; u < kTile / 64; u++) {
                            const uint64_t same = __ballot(v[u] == which);
                            if (u == word) {
                                own = same;
                                earlier = n + __builtin_amdgcn_mbcnt_hi((uint32_t)(same >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)same, 0));
                            }
                            if (u < w) in_earlier_words += __popcll(same);
                            if (u == w) rest &= ~same;
                            n += __popcll(same);
                        }
                        if (in_earlier_words) continue; /* done there */
                        if ((own >> lane) & 1) {
                            place = placed + earlier;
                            before = earlier;
                            all = n;
                            g = total + earlier / G;
                        }
                        placed += n;
                        total += (n + G - 1) / G;
                    }
                }
                is_first = t < here && before % G == 0;
            }
        } else {
            const int mine = id[t], low = 64 * quarter, high = here < low + 64 ? here : low + 64;
            int lower = 0, same = 0, earlier = 0;
            if (64 * word < here) {
#pragma unroll 4
                for (int j = low; j < high; j += 4) {
                    const int4 v = *reinterpret_cast<const int4 *>(&id[j]);
                    lower += (v.x < mine) + (v.y < mine) + (v.z < mine) + (v.w < mine);
                    same += (v.x == mine) + (v.y == mine) + (v.z == mine) + (v.w == mine);
                    if (word == quarter) earlier += (v.x == mine && j < t) + (v.y == mine && j + 1 < t) + (v.z == mine && j + 2 < t) + (v.w == mine && j + 3 < t);
                }
            }
            counts[quarter][t] = lower << 20 | same << 10 | earlier;
            __syncthreads();
            uint64_t firsts = 0;
            if (threadIdx.x < kTile) {
#pragma unroll
                for (int q = 0; q < kQuarters; q++) {
                    const int n = counts[q][t], equal = n >> 10 & 1023;
                    place += n >> 20;
                    all += equal;
                    before += q < word ? equal : n & 1023; /* (0 but for the own quarter) */
                }
                place += before;
                is_first = t < here && before % G == 0;
                firsts = __ballot(is_first);
                if (lane == 0) in_wave[word] = __popcll(firsts);
            }
            __syncthreads();
            if (threadIdx.x < kTile) {
                g = __builtin_amdgcn_mbcnt_hi((uint32_t)(firsts >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)firsts, 0));
#pragma unroll
                for (int w = 0; w < kTile / 64; w++) {
                    g += w < word ? in_wave[w] : 0;
                    total += in_wave[w];
                }
            }
        }
        if (threadIdx.x < kTile) {
            if (t < here) token[place] = (uint8_t)t;
            if (is_first) {
                first[g] = (uint8_t)place;
                size[g] = (uint8_t)(all - before < G ? all - before : G);
            }
            entry[t] = e;
            if (t == 0) groups = total;
        }
        __syncthreads();
    }
};

/* ------------------------------------------------------------------ h = A x */

template <class W, class X> constexpr bool native() { return Same<W, X>::value && sizeof(W) == 2; }

/* acc += w . x over 32 columns, eight to a lane */
template <class W, class X> __device__ __forceinline__ f32x4 multiply(const Vec<W, 8> &w, const Vec<X, 8> &x, f32x4 acc) {
    if constexpr (native<W, X>() && Same<W, Bf16>::value) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, w), __builtin_bit_cast(bf16x8, x), acc, 0, 0, 0);
    } else if constexpr (native<W, X>()) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, w), __builtin_bit_cast(f16x8, x), acc, 0, 0, 0);
    } else { /* the e-th of a lane's columns with the e-th of the other lanes': any order of columns does, the same on both sides */
#pragma unroll
        for (int e = 0; e < 8; e++) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(to_f32(w.v[e]), to_f32(x.v[e]), acc, 0, 0, 0);
        return acc;
    }
}

/* 16 rows of C columns as they come from memory, the lanes along the rows, and as the instruction takes them, lane & 15 to a row: through LDS. (Loads by
 * lane & 15 would touch 16 lines of memory at every 16 lanes, at a fourth of the rate.) A row's pieces of 16 bytes are turned by the row, so that
 * 16 lanes reach all banks both ways. */
template <class T, int C> struct Rows16 {
    static constexpr int kPieces = C * sizeof(T) / 16, kLoads = kPieces / 4, kRowsPerLoad = 64 / kPieces;
    typedef uint32_t Piece __attribute__((ext_vector_type(4)));
    Piece v[kLoads];
    static __device__ __forceinline__ int row(int load) { return kRowsPerLoad * load + (threadIdx.x & 63) / kPieces; }
    static __device__ __forceinline__ int column() { return (threadIdx.x & 63) % kPieces * (16 / (int)sizeof(T)); }
    static __device__ __forceinline__ int place(int row, int piece) { return row * kPieces + ((piece ^ (kPieces == 8 ? row >> 1 : row >> 2)) & (kPieces - 1)); }
    __device__ __forceinline__ void put(Piece *turn) const {
#pragma unroll
        for (int i = 0; i < kLoads; i++) turn[place(row(i), (threadIdx.x & 63) % kPieces)] = v[i];
    }
    /* columns 32 u + 8 g to + 7 of row lane & 15, g = lane >> 4 */
    static __device__ __forceinline__ Vec<T, 8> get(const Piece *turn, int u) {
        constexpr int kPer = sizeof(T) / 2;
        const int lane = threadIdx.x & 63;
        struct { Piece p[kPer]; } e;
#pragma unroll
        for (int i = 0; i < kPer; i++) e.p[i] = turn[place(lane & 15, (4 * u + (lane >> 4)) * kPer + i)];
        return __builtin_bit_cast(Vec<T, 8>, e);
    }
};

/* columns of a step: whole lines of 128 bytes, where the registers of four waves per SIMD hold two steps */
template <class W, class X, int RT, int NJ> constexpr int columns() { return native<W, X>() && RT + NJ <= 4 ? 64 : 32; }
constexpr int kTurnBytes = 2 * 16 * 128; /* of a wave, for two of its operands in turn */

/* a step on its way; WHOLE: all of its columns are there, else from where `from` stands some are not */
template <class W, class X, int RT, int NJ> struct Step {
    static constexpr int C = columns<W, X, RT, NJ>();
    typedef Rows16<W, C> RowsW;
    typedef Rows16<X, C> RowsX;
    RowsW w[RT];
    RowsX x[NJ];
    struct From { /* the rows' addresses */
        const W *w[RT][RowsW::kLoads];
        const X *x[NJ][RowsX::kLoads];
    };
    template <bool WHOLE, class T, class R> static __device__ __forceinline__ void fetch_rows(R &r, const T *const (&from)[R::kLoads], int at, int n_cols) {
#pragma unroll
        for (int l = 0; l < R::kLoads; l++) r.v[l] = __builtin_bit_cast(typename R::Piece, load<T, 16 / sizeof(T), WHOLE>(from[l], at, WHOLE ? 0x7FFFFFFF : n_cols - R::column()));
    }
    template <bool WHOLE> __device__ __forceinline__ void fetch(const From &from, int step, int n_cols) {
#pragma unroll
        for (int j = 0; j < NJ; j++) fetch_rows<WHOLE>(x[j], from.x[j], C * step, n_cols);
#pragma unroll
        for (int i = 0; i < RT; i++) fetch_rows<WHOLE>(w[i], from.w[i], C * step, n_cols);
    }
    __device__ __forceinline__ void add_to(f32x4 (&acc)[NJ][RT], char *turn) const {
        Vec<X, 8> b[NJ][C / 32];
#pragma unroll
        for (int j = 0; j < NJ; j++) {
            typename RowsX::Piece *to = reinterpret_cast<typename RowsX::Piece *>(turn + j % 2 * (kTurnBytes / 2));
            wave_meets();
            x[j].put(to);
            wave_meets();
#pragma unroll
            for (int u = 0; u < C / 32; u++) b[j][u] = RowsX::get(to, u);
        }
#pragma unroll
        for (int i = 0; i < RT; i++) {
            typename RowsW::Piece *to = reinterpret_cast<typename RowsW::Piece *>(turn + (NJ + i) % 2 * (kTurnBytes / 2));
            wave_meets();
            w[i].put(to);
            wave_meets();
#pragma unroll
            for (int u = 0; u < C / 32; u++) {
                const Vec<W, 8> a = RowsW::get(to, u);
#pragma unroll
                for (int j = 0; j < NJ; j++) acc[j][i] = multiply(a, b[j][u], acc[j][i]);
            }
        }
    }
};

/* sums over columns [k0, k1) for RT groups of 16 ranks and NJ groups of 16 tokens, the n that list names; what comes of ranks and tokens that are not there is
 * not looked at */
template <class W, class X, int RT, int NJ>
__device__ __forceinline__ void shrink_sums(const W *A, int rank0, int rank, const X *X0, int ldx, const uint8_t *list, int n, int n_cols, int k0, int k1,
                                            char *turn, f32x4 (&acc)[NJ][RT]) {
    /* the next step is on its way while one is multiplied; behind the last one it is that once more */
    typedef Step<W, X, RT, NJ> S;
    typename S::From from;
#pragma unroll
    for (int i = 0; i < RT; i++)
#pragma unroll
        for (int l = 0; l < S::RowsW::kLoads; l++) {
            const int r = rank0 + 16 * i + S::RowsW::row(l);
            from.w[i][l] = A + (size_t)(r < rank ? r : rank - 1) * n_cols + S::RowsW::column();
        }
#pragma unroll
    for (int j = 0; j < NJ; j++)
#pragma unroll
        for (int l = 0; l < S::RowsX::kLoads; l++) {
            const int q = 16 * j + S::RowsX::row(l);
            from.x[j][l] = X0 + (size_t)list[q < n ? q : 0] * ldx + S::RowsX::column();
        }
    const int whole = n_cols / S::C, last = (k1 + S::C - 1) / S::C, end = last < whole ? last : whole;
    int k = k0 / S::C;
    S s[2];
    if (k < end) {
        s[0].template fetch<true>(from, k, n_cols);
        for (; k + 2 <= end; k += 2) {
            s[1].template fetch<true>(from, k + 1, n_cols);
            __builtin_amdgcn_sched_barrier(0); /* (the compiler would fetch where it multiplies) */
            s[0].add_to(acc, turn);
            s[0].template fetch<true>(from, k + 2 < end ? k + 2 : k + 1, n_cols);
            __builtin_amdgcn_sched_barrier(0);
            s[1].add_to(acc, turn);
        }
        if (k < end) s[0].add_to(acc, turn);
    }
    if (end < last && S::C * end < n_cols) {
        s[0].template fetch<false>(from, end, n_cols);
        s[0].add_to(acc, turn);
    }
}

/* The leading eight bits of a number, or the eight-bit number next below where it has no more: something of its sign is left behind them in any case, and a
 * number cut into three in bf16 (24 bits are eight, eight and eight) has none that is 0. An infinite element of B times each of the three is then the infinity that it is times the
 * number, not the NaN of infinity times 0. The last of an infinity's three is one; 0 is 0 in all three; bf16 has no last one for numbers below 2^-110. */
__device__ __forceinline__ float leading(float v) { return __uint_as_float((__float_as_uint(v) - (v != 0.0f ? 1 : 0)) & 0xFFFF0000u); }

template <class W, class X, int RT, int NJ>
__global__ void __launch_bounds__(64 * kShrinkWaves)
lora_shrink_kernel(LoraCall c, LoraPlan p) {
    __shared__ union { /* a wave's own operands on their way, then every wave's sums */
        char turn[kShrinkWaves][kTurnBytes];
        f32x4 sum[kShrinkWaves][NJ * RT][64];
    } u;
    __shared__ Tile<16 * NJ> tokens;
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    /* workgroups b and b + 8 share a die: the tensors of the same tokens, one after the other */
    uint32_t b = blockIdx.x % 8 + blockIdx.x / 8 / c.n_mat * 8;
    const int mat = blockIdx.x / 8 % c.n_mat;
    if (b >= p.shrink_units()) return;
    const int part = b % p.parts; b /= p.parts;
    const int slot = b % p.shrink_slots; b /= p.shrink_slots;
    const int block = b % p.rank_blocks, tile = b / p.rank_blocks;
    const X *x0 = static_cast<const X *>(c.X) + (size_t)tile * kTile * c.ldx;
    const int rank0 = block * 16 * RT;
    const int pieces = (c.n_cols + 63) / 64, share = part * kShrinkWaves + wv, shares = p.parts * kShrinkWaves;
    const int k0 = 64 * (int)((long long)pieces * share / shares), k1 = 64 * (int)((long long)pieces * (share + 1) / shares);
    Group *records = static_cast<Group *>(c.workspace) + (size_t)tile * p.groups;
    tokens.find(c, mat == 0 ? c.m[0].adapters : mat == 1 ? c.m[1].adapters : c.m[2].adapters, tile);
    for (int s = slot; s * NJ < p.groups; s += p.shrink_slots) {
        if (s >= tokens.groups) { /* the second launch looks at every record */
            if (part == 0 && block == 0 && mat == 0 && threadIdx.x < NJ) records[s * NJ + threadIdx.x].n = 0;
            continue;
        }
        const int place = uniform(tokens.first[s]), n = uniform(tokens.size[s]), t0 = uniform(tokens.token[place]);
        const uint8_t *list = tokens.token + place;
        const Entry e = {uniform(tokens.entry[t0].A), uniform(tokens.entry[t0].B), uniform(tokens.entry[t0].rank), tokens.entry[t0].scale};
        if (part == 0 && block == 0 && wv < NJ) {
            Group &r = records[s * NJ + wv];
            const int here = n - 16 * wv > 16 ? 16 : n - 16 * wv > 0 ? n - 16 * wv : 0;
            if (mat == 0 && lane < 16) r.token[lane] = list[lane < here ? 16 * wv + lane : 0]; /* (behind its tokens: the first) */
            if (lane == 0) {
                if (mat == 0) {
                    r.n = here;
                    r.place = place + 16 * wv;
                }
                r.of[mat].B = e.B;
                r.of[mat].rank = e.rank;
                r.of[mat].scale = e.scale;
            }
        }
        if (e.rank > rank0) { /* else no adapter, or none of its ranks here: nothing is read of h either */
            f32x4 acc[NJ][RT] = {};
            if (k0 < k1)
                shrink_sums<W, X, RT, NJ>(static_cast<const W *>(e.A), rank0, e.rank, x0, c.ldx, list, n, c.n_cols, k0, k1, u.turn[wv], acc);
            /* the waves' sums, added in the waves' order */
            __syncthreads();
#pragma unroll
            for (int j = 0; j < NJ; j++)
#pragma unroll
                for (int i = 0; i < RT; i++) u.sum[wv][j * RT + i][lane] = acc[j][i];
            __syncthreads();
            for (int f = wv; f < NJ * RT; f += kShrinkWaves) {
                const int j = f / RT, i = f % RT, here = n - 16 * j < 16 ? n - 16 * j : 16;
                f32x4 v = u.sum[0][f][lane];
#pragma unroll
                for (int w = 1; w < kShrinkWaves; w++) v += u.sum[w][f][lane];
                const int r = rank0 + 16 * i + 4 * (lane >> 4), q = lane & 15;
#pragma unroll
                for (int d = 0; d < 4; d++)
                    if (r + d >= e.rank) v[d] = 0.0f;
                if (q >= here || r >= p.rank_pad) continue;
                const size_t first = (size_t)tile * kTile + place + 16 * j;
                char *h = static_cast<char *>(c.workspace) + p.h_at;
                if (p.split) {
                    v *= e.scale;
                    bf16x4 three[3];
#pragma unroll
                    for (int d = 0; d < 4; d++) {
                        const float first = leading(v[d]), rest = v[d] - first, second = leading(rest);
                        three[0][d] = (__bf16)first;
                        three[1][d] = (__bf16)second;
                        three[2][d] = (__bf16)(rest - second);
                    }
                    const int pieces = (p.rank_pad + 31) / 32 * 12, piece = r / 32 * 12 + r % 32 / 8;
#pragma unroll
                    for (int d = 0; d < 3; d++)
                        *reinterpret_cast<bf16x4 *>(h + piece_at(first + (size_t)mat * c.n_tok, pieces, piece + 4 * d, here, q) + r % 8 * 2) = three[d];
                } else {
                    const size_t of_part = ((size_t)part * c.n_mat + mat) * c.n_tok;
                    *reinterpret_cast<f32x4 *>(h + piece_at(of_part + first, p.rank_pad / 4, r / 4, here, q)) = v;
                }
            }
        }
        __syncthreads();
    }
}

/* ------------------------------------------------------------------ Y + B h */

/* what was loaded, there at this place and not before or behind it */
template <class V> __device__ __forceinline__ V here(V v) {
    typedef uint32_t Words __attribute__((ext_vector_type(sizeof(V) / 4)));
    Words w = __builtin_bit_cast(Words, v);
    asm volatile("" : "+v"(w));
    return __builtin_bit_cast(V, w);
}
/* four consecutive elements of a row at any element's address, of which `left` are there; T: float or the bits of a 16-bit type; WHOLE: all four are */
template <class T> using Four = T __attribute__((ext_vector_type(4), aligned(sizeof(T))));
template <class T, bool WHOLE> __device__ __forceinline__ Four<T> load4(const void *base, size_t at, int left) {
    const T *p = static_cast<const T *>(base) + at;
    Four<T> v = {};
    if (WHOLE || left > 3) {
        v = *reinterpret_cast<const Four<T> *>(p);
    } else {
#pragma unroll
        for (int i = 0; i < 3; i++)
            if (i < left) v[i] = p[i];
    }
    return v;
}
template <class T> __device__ __forceinline__ f32x4 values(Four<T> v, bool bf16) {
    f32x4 y;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (sizeof(T) == 4) y[i] = v[i];
        else y[i] = bf16 ? to_f32(Bf16{v[i]}) : to_f32(__builtin_bit_cast(_Float16, (uint16_t)v[i]));
    }
    return y;
}
/* the one rounding of a result in 16 bits: to the nearest, ties to even */
template <class T, bool WHOLE> __device__ __forceinline__ void store4(void *base, size_t at, int left, bool bf16, f32x4 y) {
    T *p = static_cast<T *>(base) + at;
    Four<T> v;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (sizeof(T) == 4) v[i] = y[i];
        else v[i] = bf16 ? __builtin_bit_cast(uint16_t, (__bf16)y[i]) : __builtin_bit_cast(uint16_t, (_Float16)y[i]);
    }
    if (WHOLE || left > 3) {
        *reinterpret_cast<Four<T> *>(p) = v;
    } else {
#pragma unroll
        for (int i = 0; i < 3; i++)
            if (i < left) p[i] = v[i];
    }
}

/* rows of B for lane & 15 of MT groups of 16 */
template <class W, int MT> struct Rows {
    const W *b[MT];
    __device__ Rows(const Entry &e, int row0, int n_rows) {
#pragma unroll
        for (int i = 0; i < MT; i++) {
            const int row = row0 + 16 * i + (threadIdx.x & 15);
            b[i] = static_cast<const W *>(e.B) + (size_t)(row < n_rows ? row : n_rows - 1) * e.rank;
        }
    }
};

/* acc += B h over an adapter's ranks, for MT groups of 16 rows x 16 tokens; h: the lane's pieces in the workspace, 4 n of 16 bytes to 16 ranks, of
 * which the parts are added in their order */
template <class W, int MT, bool VEC>
__device__ __forceinline__ void expand_sums(const Entry &e, int row0, int n_rows, const char *h, int n, size_t part, int parts, f32x4 (&acc)[MT]) {
    const int g = (threadIdx.x & 63) >> 4;
    const Rows<W, MT> rows(e, row0, n_rows);
    for (int r = 4 * g; r < e.rank + 4 * g; r += 16, h += 64 * n) {
        Vec<W, 4> w[MT];
#pragma unroll
        for (int i = 0; i < MT; i++) w[i] = load<W, 4, VEC>(rows.b[i], r, e.rank);
        f32x4 v = *reinterpret_cast<const f32x4 *>(h);
        auto others = [&](auto most) { /* all on their way at once */
            f32x4 more[decltype(most)::value];
#pragma unroll
            for (int q = 0; q < most; q++) more[q] = *reinterpret_cast<const f32x4 *>(h + (q + 1 < parts ? q + 1 : 0) * part);
#pragma unroll
            for (int q = 0; q < most; q++) {
                const f32x4 one = here(more[q]); /* (the compiler would load where it adds, and wait for each) */
                if (q + 1 < parts) v += one;
            }
        };
        if (parts > 5) others(std::integral_constant<int, kLoraMostParts - 1>{});
        else if (parts > 3) others(std::integral_constant<int, 4>{});
        else if (parts > 1) others(std::integral_constant<int, 2>{});
        v *= e.scale;
#pragma unroll
        for (int q = 0; q < 4; q++)
#pragma unroll
            for (int i = 0; i < MT; i++) acc[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(to_f32(w[i].v[q]), v[q], acc[i], 0, 0, 0);
    }
}

/* the same where the workspace holds scale h as three numbers in bf16, whose sum it is: 12 n pieces to 32 ranks; the products are exact */
template <int MT, bool VEC>
__device__ __forceinline__ void expand_split(const Entry &e, int row0, int n_rows, const char *h, int n, f32x4 (&acc)[MT]) {
    const int g = (threadIdx.x & 63) >> 4;
    const Rows<Bf16, MT> rows(e, row0, n_rows);
    for (int r = 8 * g; r < e.rank + 8 * g; r += 32, h += 192 * n) {
        Vec<Bf16, 8> w[MT];
        bf16x8 v[3] = {};
#pragma unroll
        for (int i = 0; i < MT; i++) w[i] = load<Bf16, 8, VEC>(rows.b[i], r, e.rank);
        if (r < e.rank) { /* (what lies behind may be anything) */
#pragma unroll
            for (int k = 0; k < 3; k++) v[k] = *reinterpret_cast<const bf16x8 *>(h + 64 * k * n);
        }
#pragma unroll
        for (int k = 2; k >= 0; k--)
#pragma unroll
            for (int i = 0; i < MT; i++) acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, w[i]), v[k], acc[i], 0, 0, 0);
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
    const bool whole = row0 + kRows <= m.n_rows;
    const size_t part = (size_t)c.n_mat * c.n_tok * p.rank_pad * sizeof(float);
    const int row = 4 * (lane % kLanes), left = m.n_rows - row0 - row; /* of the run */
    const int pieces = SPLIT ? (p.rank_pad + 31) / 32 * 12 : p.rank_pad / 4;
    const char *hs = static_cast<const char *>(c.workspace) + p.h_at;
    const uint32_t *records = reinterpret_cast<const uint32_t *>(static_cast<const Group *>(c.workspace) + (size_t)tile * p.groups);
    constexpr int kWords = sizeof(Group) / 4;
    const int word = lane < kWords ? lane : 0;
    uint32_t record = slot < p.groups ? records[slot * kWords + word] : 0; /* a word to a lane, and the next group's while one is worked on */
    auto group_of = [&](auto w) {
        constexpr bool WHOLE = decltype(w)::value;
        for (int u = slot; u < p.groups;) {
            const uint32_t words = record;
            u += p.expand_slots;
            record = records[(u < p.groups ? u : slot) * kWords + word];
            const int n = __builtin_amdgcn_readlane(words, 0);
            if (n == 0) continue;
            const size_t first = (size_t)tile * kTile + __builtin_amdgcn_readlane(words, 1);
            auto token = [&](int q) { return (size_t)tile * kTile + ((uint32_t)__shfl((int)words, 2 + q / 4, 64) >> 8 * (q % 4) & 255); };
            size_t run[kSteps]; /* the tokens of the lane's runs */
#pragma unroll
            for (int s = 0; s < kSteps; s++) run[s] = token(s * kRuns + lane / kLanes);
            Four<T> raw[MATS][kSteps]; /* (on their way until the sums are there) */
#pragma unroll
            for (int s = 0; s < kSteps; s++) {
                raw[0][s] = load4<T, WHOLE>(m.Y, run[s] * m.ldy + row0 + row, left);
                if constexpr (PAIR) raw[1][s] = load4<T, WHOLE>(c.m[1].Y, run[s] * m.ldy + row0 + row, left);
            }
            f32x4 y[MATS][kSteps];
#pragma unroll
            for (int a = 0; a < MATS; a++) {
                const int at = 8 + 4 * (mat + a);
                const Entry e = {nullptr, (const void *)((uint64_t)__builtin_amdgcn_readlane(words, at + 1) << 32 | (uint32_t)__builtin_amdgcn_readlane(words, at)),
                                 (int)__builtin_amdgcn_readlane(words, at + 2), __uint_as_float(__builtin_amdgcn_readlane(words, at + 3))};
                f32x4 acc[MT] = {};
                if (e.rank != 0) {
                    const char *h = hs + piece_at((size_t)(mat + a) * c.n_tok + first, pieces, lane >> 4, n, (lane & 15) < n ? lane & 15 : 0);
                    if constexpr (SPLIT) {
                        if (e.rank % 8 == 0)
                            expand_split<MT, true>(e, row0, m.n_rows, h, n, acc);
                        else
                            expand_split<MT, false>(e, row0, m.n_rows, h, n, acc);
                    } else {
                        if (e.rank % 4 == 0)
                            expand_sums<W, MT, true>(e, row0, m.n_rows, h, n, part, p.parts, acc);
                        else
                            expand_sums<W, MT, false>(e, row0, m.n_rows, h, n, part, p.parts, acc);
                    }
                    wave_meets();
#pragma unroll
                    for (int i = 0; i < MT; i++) *reinterpret_cast<f32x4 *>(&turn[wv][(lane & 15) * kStride + 16 * i + 4 * (lane >> 4)]) = acc[i];
                    wave_meets();
                }
#pragma unroll
                for (int s = 0; s < kSteps; s++) {
                    y[a][s] = values<T>(here(raw[a][s]), y_bf16);
                    if (e.rank != 0) y[a][s] += *reinterpret_cast<const f32x4 *>(&turn[wv][(s * kRuns + lane / kLanes) * kStride + row]);
                }
            }
            if constexpr (PAIR) {
#pragma unroll
                for (int s = 0; s < kSteps; s++)
#pragma unroll
                    for (int r = 0; r < 4; r++) y[0][s][r] = mxfp4::silu_mul(y[0][s][r], y[MATS - 1][s][r]);
            }
#pragma unroll
            for (int s = 0; s < kSteps; s++)
                if (s * kRuns + lane / kLanes < n) store4<O, WHOLE>(m.out, run[s] * m.ldo + row0 + row, left, o_bf16, y[0][s]);
        }
    };
    if (whole) group_of(std::true_type{});
    else group_of(std::false_type{});
}

/* ------------------------------------------------------------------ a few tokens */

/* One launch for a few tokens: a workgroup makes 1024 results of a token, and h itself before, which costs it a look at all of A, but no second launch and no
 * search for tokens that share an adapter. A wave has NS pieces of 512 columns (8 to a lane, in registers) and its share of the ranks; the lanes'
 * sums are added in 16 lanes by moves between lanes, the rest in LDS in a fixed order. */
constexpr int kFewPiece = 512, kFewMaxRank = 64, kFewTokens = 64;
constexpr size_t kFewBytes = 384 << 10, kFewBytesAll = 40 << 20; /* of A, that a workgroup reads and all of them */
template <class W, class X, class T, class O, int NS, bool PAIR>
__global__ void __launch_bounds__(kLoraFewThreads)
lora_few_kernel(LoraCall c, LoraPlan p) {
    constexpr int MATS = PAIR ? 2 : 1, kWaves = kLoraFewThreads / 64;
    __shared__ float sums[MATS][kFewMaxRank][4 * kWaves]; /* [rank][piece's wave, 16 lanes] */
    __shared__ __attribute__((aligned(16))) float hs[MATS][kFewMaxRank];
    const int lane = threadIdx.x & 63, wv = uniform((int)(threadIdx.x >> 6));
    const size_t token = blockIdx.y;
    int block = blockIdx.x;
    LoraTensor m = c.m[0];
    if (!PAIR && block >= p.row_blocks[0]) {
        block -= p.row_blocks[0];
        m = c.m[1];
        if (block >= p.row_blocks[1]) {
            block -= p.row_blocks[1];
            m = c.m[2];
        }
    }
    const int id = uniform(c.ids[token]);
    /* the wave's columns, and which of the ranks */
    const int pieces = (c.n_cols + kFewPiece - 1) / kFewPiece, columns = NS > 1 || pieces > kWaves ? kWaves : pieces, shares = kWaves / columns;
    const int share = wv / columns, piece = wv % columns;
    const X *x0 = static_cast<const X *>(c.X) + token * c.ldx;
    int at[NS];
    float x[NS][8];
#pragma unroll
    for (int s = 0; s < NS; s++) {
        at[s] = (piece + s * kWaves) * kFewPiece + 8 * lane;
        const Vec<X, 8> v = load<X, 8, false>(x0, at[s], c.n_cols);
#pragma unroll
        for (int i = 0; i < 8; i++) x[s][i] = to_f32(v.v[i]);
    }
    const int row = block * kLoraFewThreads + threadIdx.x;
    const bool there = row < m.n_rows;
    float y[MATS];
#pragma unroll
    for (int a = 0; a < MATS; a++) {
        y[a] = 0.0f;
        if (there) {
            const size_t e = token * m.ldy + row;
            if constexpr (sizeof(T) == 4) y[a] = static_cast<const float *>(a ? c.m[1].Y : m.Y)[e];
            else {
                const uint16_t bits = static_cast<const uint16_t *>(a ? c.m[1].Y : m.Y)[e];
                y[a] = c.y_type == T_BF16 ? to_f32(Bf16{bits}) : to_f32(__builtin_bit_cast(_Float16, bits));
            }
        }
    }
    Entry e[MATS];
#pragma unroll
    for (int a = 0; a < MATS; a++) {
        e[a] = entry_of(PAIR ? c.m[a].adapters : m.adapters, id >= 0 && id < c.n_adapter ? id : -1, c.max_rank);
        e[a].A = uniform(e[a].A);
        e[a].B = uniform(e[a].B);
        e[a].rank = uniform(e[a].rank);
    }
#pragma unroll
    for (int a = 0; a < MATS; a++) {
        const W *A = static_cast<const W *>(e[a].A);
        const bool whole = c.n_cols % 8 == 0;
        for (int r0 = share; r0 < e[a].rank && share < shares; r0 += 4 * shares) {
            Vec<W, 8> w[4][NS];
            float sum[4] = {};
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const int r = r0 + q * shares < e[a].rank ? r0 + q * shares : r0;
#pragma unroll
                for (int s = 0; s < NS; s++) w[q][s] = whole ? load<W, 8, true>(A + (size_t)r * c.n_cols, at[s], c.n_cols) : load<W, 8, false>(A + (size_t)r * c.n_cols, at[s], c.n_cols);
            }
#pragma unroll
            for (int q = 0; q < 4; q++) {
#pragma unroll
                for (int s = 0; s < NS; s++)
#pragma unroll
                    for (int i = 0; i < 8; i++) sum[q] = fmaf(to_f32(w[q][s].v[i]), x[s][i], sum[q]);
                sum[q] += dpp_mov<0xB1>(sum[q]);
                sum[q] += dpp_mov<0x4E>(sum[q]);
                sum[q] += dpp_mov<0x141>(sum[q]);
                sum[q] += dpp_mov<0x140>(sum[q]); /* each of 16 lanes has their sum */
                if (lane % 16 == q && r0 + q * shares < e[a].rank) sums[a][r0 + q * shares][4 * piece + lane / 16] = sum[q];
            }
        }
    }
    __syncthreads();
#pragma unroll
    for (int a = 0; a < MATS; a++)
        for (int r = wv; r < e[a].rank; r += kWaves) { /* a wave to a rank */
            const float h = wave_sum_dpp(lane < 4 * columns ? sums[a][r][lane] : 0.0f);
            if (lane == 0) hs[a][r] = h * e[a].scale;
        }
    __syncthreads();
    if (!there) return;
#pragma unroll
    for (int a = 0; a < MATS; a++) {
        const W *B = static_cast<const W *>(e[a].B) + (size_t)row * e[a].rank;
        const bool whole = e[a].rank % 8 == 0;
        float sum = 0.0f;
        for (int r = 0; r < e[a].rank; r += 8) {
            const Vec<W, 8> w = whole ? load<W, 8, true>(B, r, e[a].rank) : load<W, 8, false>(B, r, e[a].rank);
#pragma unroll
            for (int i = 0; i < 8; i++) sum = r + i < e[a].rank ? fmaf(to_f32(w.v[i]), hs[a][r + i], sum) : sum;
        }
        y[a] += sum;
    }
    if constexpr (PAIR) y[0] = mxfp4::silu_mul(y[0], y[MATS - 1]);
    const size_t o = token * m.ldo + row;
    if constexpr (sizeof(O) == 4) static_cast<float *>(m.out)[o] = y[0];
    else static_cast<uint16_t *>(m.out)[o] = c.out_type == T_BF16 ? __builtin_bit_cast(uint16_t, (__bf16)y[0]) : __builtin_bit_cast(uint16_t, (_Float16)y[0]);
}

template <class W, class X, class T, class O, bool PAIR> void launch_few(const LoraCall &c, const LoraPlan &p) {
    const dim3 grid(p.row_blocks_all, c.n_tok), block(kLoraFewThreads);
    if (c.n_cols <= kFewPiece * kLoraFewThreads / 64)
        hipLaunchKernelGGL((lora_few_kernel<W, X, T, O, 1, PAIR>), grid, block, 0, c.stream, c, p);
    else
        hipLaunchKernelGGL((lora_few_kernel<W, X, T, O, 2, PAIR>), grid, block, 0, c.stream, c, p);
}
template <class W, class X, bool PAIR> void launch_few(const LoraCall &c, const LoraPlan &p) {
    const bool y32 = c.y_type == T_F32, o32 = c.out_type == T_F32;
    if (y32 && o32) launch_few<W, X, float, float, PAIR>(c, p);
    else if (y32) launch_few<W, X, float, uint16_t, PAIR>(c, p);
    else if (o32) launch_few<W, X, uint16_t, float, PAIR>(c, p);
    else launch_few<W, X, uint16_t, uint16_t, PAIR>(c, p);
}
template <class W, class X> void launch_few(const LoraCall &c, const LoraPlan &p) {
    if (c.pair) launch_few<W, X, true>(c, p);
    else launch_few<W, X, false>(c, p);
}

template <class W, class X, int RT> void launch_shrink(const LoraCall &c, const LoraPlan &p) {
    /* the tensors' workgroups for the same tokens a multiple of eight apart: on one die, where they share X */
    const dim3 grid((uint32_t)p.shrink_workgroups()), block(kLoraShrinkThreads);
    if constexpr (RT < 4 || native<W, X>()) {
        if (p.token_groups == 2) {
            hipLaunchKernelGGL((lora_shrink_kernel<W, X, RT, 2>), grid, block, 0, c.stream, c, p);
            return;
        }
    }
    hipLaunchKernelGGL((lora_shrink_kernel<W, X, RT, 1>), grid, block, 0, c.stream, c, p);
}
template <class W, class X> void launch_shrink(const LoraCall &c, const LoraPlan &p) {
    if (p.rank_tiles == 1) launch_shrink<W, X, 1>(c, p);
    else if (p.rank_tiles == 2) launch_shrink<W, X, 2>(c, p);
    else if constexpr (!Same<W, float>::value) launch_shrink<W, X, 4>(c, p);
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
    if (p.few) {
        if (c.x_type == T_F32) launch_few<W, float>(c, p);
        else if (c.x_type == T_F16) launch_few<W, _Float16>(c, p);
        else launch_few<W, Bf16>(c, p);
        return hipGetLastError();
    }
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

/* 16 ranks, 32 or, in 16 bits, 64 to a workgroup: the registers of 64 in fp32 do not fit, and the activations twice cost less than that (2048 tokens of 4096
 * columns, rank 64, three tensors: 50 us for the first launch, 61 with 64 ranks) */
static int lora_rank_tiles(int max_rank, uint32_t lora_type) { return max_rank <= 16 ? 1 : max_rank <= 32 || lora_type == T_F32 ? 2 : 4; }
static int lora_rank_blocks(int max_rank, uint32_t lora_type) {
    const int ranks = 16 * lora_rank_tiles(max_rank, lora_type);
    return (max_rank + ranks - 1) / ranks;
}
/* 16 tokens to a workgroup of the first launch or, where those would not all run at once, 32, which halves the reads of A (both launches, columns 4096: 2048
 * tokens, three tensors of rank 64: 50 us, 59 with 16; 1300 tokens: 37 us, 34 with 16; 1024 tokens, gate and up of rank 32: 58 us, 51 with 16) */
static int lora_token_groups(int n_mat, int max_rank, int n_tok) {
    return ((long long)n_tok + 15) / 16 * n_mat * lora_rank_blocks(max_rank, T_F16) >= 256 ? 2 : 1;
}

/* how many parts the columns are cut into at most: as far as a workgroup for each compute unit needs, and at least 64 columns for a wave; the second
 * launch reads every part of h again for each of its rows' workgroups */
static int lora_most_parts(int n_mat, int max_rank, int n_cols, int n_tok) {
    const long long tokens = 16ll * lora_token_groups(n_mat, max_rank, n_tok), groups = (n_tok + tokens - 1) / tokens * n_mat * lora_rank_blocks(max_rank, T_F16);
    const long long want = groups >= 96 ? 1 : 256 / groups, most = n_cols / (64 * kShrinkWaves);
    const long long parts = want < most ? want : most;
    return (int)(parts > kLoraMostParts ? kLoraMostParts : parts < 1 ? 1 : parts);
}

/* The groups of every tile, of which there are at most as many as tokens, or half of them twice as many; then h in fp32 for each part, or, of one part, as three
 * numbers in bf16. What fewer tokens, tensors, ranks or columns need is not more: tokens * parts is at most 256 * 16 / (n_mat * blocks of ranks) where there is more than one
 * part, and a block has up to 64 ranks. */
static size_t lora_records(int n_tok, int groups) { return ((size_t)n_tok + kTile - 1) / kTile * groups * sizeof(Group); }
size_t lora_workspace_bytes(int n_mat, int max_rank, int n_cols, int n_tok) {
    const size_t rank_pad = (max_rank + 15) / 16 * 16, tokens = n_tok, split = tokens * ((rank_pad + 31) / 32 * 192);
    const size_t columns = n_cols / (64 * kShrinkWaves), parts = columns < 1 ? 1 : columns > kLoraMostParts ? kLoraMostParts : columns;
    const size_t whole = tokens * rank_pad, cut = whole * parts, most = (rank_pad < 64 ? rank_pad : 64) * ((256 * 16 + n_mat - 1) / n_mat);
    const size_t sums = (cut < most ? cut : most > whole ? most : whole) * sizeof(float);
    return lora_records(n_tok, (n_tok < kTile ? n_tok : kTile) * lora_token_groups(n_mat, max_rank, n_tok)) + n_mat * (split > sums ? split : sums);
}

LoraPlan lora_plan(const LoraCall &c) {
    LoraPlan p;
    const size_t element = c.lora_type == T_F32 ? 4 : 2;
    const bool native = c.lora_type == c.x_type && c.lora_type != T_F32;
    p.tiles = (int)(((long long)c.n_tok + kTile - 1) / kTile);
    p.n_mat = c.n_mat;
    p.rank_pad = (c.max_rank + 15) / 16 * 16;
    p.rank_tiles = lora_rank_tiles(c.max_rank, c.lora_type);
    p.rank_blocks = lora_rank_blocks(c.max_rank, c.lora_type);
    p.token_groups = p.rank_tiles < 4 || native ? lora_token_groups(c.n_mat, c.max_rank, c.n_tok) : 1; /* (the registers) */
    /* the most groups that a tile can have */
    const int tokens = c.n_tok < kTile ? c.n_tok : kTile, size = 16 * p.token_groups;
    const long long classes = c.n_adapter + 1ll < tokens ? c.n_adapter + 1ll : tokens, bound = (tokens - classes) / size + classes, full = (tokens + size - 1) / size;
    const long long others = (long long)p.tiles * p.n_mat * p.rank_blocks;
    p.groups = (int)bound * p.token_groups;
    p.h_at = lora_records(c.n_tok, p.groups);
    const int most = lora_most_parts(c.n_mat, c.max_rank, c.n_cols, c.n_tok);
    const long long fill = 256 / (bound * others); /* a workgroup on each compute unit: two do not find room */
    p.parts = (int)(fill < 1 ? 1 : fill < most ? fill : most);
    p.split = p.parts == 1 && c.lora_type == T_BF16;
    const size_t a_bytes = (size_t)c.max_rank * c.n_cols * element * (c.pair ? 2 : 1);
    p.few = c.n_tok <= kFewTokens && c.max_rank <= kFewMaxRank && c.n_cols <= 2 * kFewPiece * kLoraFewThreads / 64 && a_bytes <= kFewBytes;
    if (p.few) {
        long long blocks = 0;
        for (int i = 0; i < (c.pair ? 1 : c.n_mat); i++) blocks += ((long long)c.m[i].n_rows + kLoraFewThreads - 1) / kLoraFewThreads;
        p.few = blocks * c.n_tok * a_bytes <= kFewBytesAll && blocks * c.n_tok * kLoraFewThreads < 1ll << 32;
    }
    /* 64 rows to a wave of the second launch, which reads h once for them, or 16 where 64 make few workgroups, and for up to 8 tokens (10 tokens of 719 rows,
     * rank 128: 7.1 us, 12.5 with 64; 16 beside Q, K and V of 6144 rows: 10.8, 15; 200 of 4096 rows, rank 32, 688 workgroups: 7.8, 6.6 with 64). Where h
     * goes as three bf16 numbers it is always 64: many tokens, and any number of them where rows are narrower than 2048 columns (both launches, 1024 columns, 4096 rows, rank 128, 8 adapters: 1
     * token 12.6 us, 12.2 with fp32 and 16 rows; 8 tokens 14.3, 14.4; 32 tokens 13.6, 14.4; 32 tokens and three tensors 18.7, 22.7). */
    auto row_blocks = [&](int rows) {
        p.row_blocks_all = 0;
        for (int i = 0; i < 3; i++) {
            p.row_blocks[i] = i < c.n_mat && (i == 0 || !c.pair) ? (int)(((long long)c.m[i].n_rows + rows - 1) / rows) : 0;
            p.row_blocks_all += p.row_blocks[i];
        }
    };
    p.row_tiles = 4;
    row_blocks(p.few ? kLoraFewThreads : 64 * kExpandWaves);
    if (!p.few && !p.split && (c.n_tok <= 8 || (long long)p.row_blocks_all * p.groups * p.tiles <= 384)) {
        p.row_tiles = 1;
        row_blocks(16 * kExpandWaves);
    }
    /* a workgroup for each group, unless that makes more than run at once: then several groups to a workgroup, in the first launch one for each that
     * a prompt of one adapter has and a quarter more (2048 tokens in runs of 64 adapters, rank 16, three tensors: 15.4 us for the first launch with 256 workgroups, 31.3 with 1024,
     * most of which have no group; 2048 tokens in runs of 6 adapters in fp32, rank 64: 36 us, 53 without the quarter more) */
    auto slots = [&](long long bound, long long least, long long others, long long many) {
        const long long want = others > 0 && many / others > least ? many / others : least;
        return (int)(want < bound ? want : bound);
    };
    p.shrink_slots = slots(bound, full + (full + 3) / 4, others * p.parts, 256);
    p.expand_slots = slots(p.groups, 1, (long long)p.tiles * p.row_blocks_all, 4096);
    return p;
}

hipError_t launch_lora(const LoraCall &c, const LoraPlan &p) {
    return c.lora_type == T_F32 ? launch_both<float>(c, p) : c.lora_type == T_F16 ? launch_both<_Float16>(c, p) : launch_both<Bf16>(c, p);
}

}  // namespace qlin
