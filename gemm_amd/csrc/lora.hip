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

namespace qlin {

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

struct Bf16 { uint16_t bits; };
__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(_Float16 v) { return (float)v; }
__device__ __forceinline__ float to_f32(Bf16 v) { return __uint_as_float((uint32_t)v.bits << 16); }

template <class T, int N> struct alignas(sizeof(T) * N < 16 ? sizeof(T) * N : 16) Vec { T v[N]; };

template <class A, class B> struct Same { static constexpr bool value = false; };
template <class A> struct Same<A, A> { static constexpr bool value = true; };

constexpr int kTile = 64; /* tokens of a tile: a lane each */
constexpr int kWaves = 4;

/* N elements p[at..], zeros from `end` on; VEC: p + at on the vector's alignment, at and end multiples of N */
template <class T, int N, bool VEC> __device__ __forceinline__ Vec<T, N> load(const T *p, int at, int end) {
    Vec<T, N> e = {};
    if constexpr (VEC) {
        if (at < end) e = *reinterpret_cast<const Vec<T, N> *>(p + at);
    } else {
#pragma unroll
        for (int i = 0; i < N; i++)
            if (at + i < end) e.v[i] = p[at + i];
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
    Entry e = {nullptr, nullptr, 0, 0.0f};
    if (id >= 0 && table) { /* (no table where a tensor has no rows) */
        const LoraEntry v = table[id];
        if (v.A && v.B && v.rank > 0 && v.rank <= max_rank) e = {v.A, v.B, v.rank, v.scale};
    }
    return e;
}

/* The classes of a tile of tokens, one after the other: which tokens share an id (a lane's bit is its token's), and which. An id
 * outside of the table counts as -1. */
struct Classes {
    int mine;
    uint64_t left;
    __device__ Classes(const int32_t *ids, int n_tok, int n_adapter, int tile) {
        const long long t = (long long)tile * kTile + (threadIdx.x & 63);
        mine = -2;
        if (t < n_tok) {
            const int v = ids[t];
            mine = v >= 0 && v < n_adapter ? v : -1;
        }
        left = __ballot(mine != -2);
    }
    __device__ uint64_t next(int &id) {
        id = __builtin_amdgcn_readlane(mine, __builtin_ctzll(left));
        const uint64_t same = __ballot(mine == id);
        left &= ~same;
        return same;
    }
};

/* lane q: the token (of the tile's 64) that is the q-th of a class; past the class some other */
__device__ __forceinline__ int packed_order(uint64_t same) {
    const int lane = threadIdx.x & 63;
    const int before = __builtin_amdgcn_mbcnt_hi((uint32_t)(same >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)same, 0));
    const int place = (same >> lane) & 1 ? before : __popcll(same) + lane - before;
    return __builtin_amdgcn_ds_permute(place * 4, lane);
}

/* ------------------------------------------------------------------ h = A x */

/* sums over steps [k0, k1) of 32 columns for RT groups of 16 ranks and NJ groups of 16 tokens; rows of A from its rank on are not looked at */
template <class W, class X, int RT, bool VEC>
__device__ __forceinline__ void shrink_sums(const W *A, int rank0, int rank, const X *const (&x)[4], int n_groups, int n_cols, int k0, int k1, f32x4 (&acc)[4][RT]) {
    const int lane = threadIdx.x & 63, g = lane >> 4;
    const W *a[RT];
#pragma unroll
    for (int i = 0; i < RT; i++) {
        const int row = rank0 + 16 * i + (lane & 15);
        a[i] = A + (size_t)(row < rank ? row : rank - 1) * n_cols;
    }
    for (int s = k0; s < k1; s++) {
        const int at = 32 * s + 8 * g;
        Vec<W, 8> w[RT];
#pragma unroll
        for (int i = 0; i < RT; i++)
            if (rank0 + 16 * i < rank) w[i] = load<W, 8, VEC>(a[i], at, n_cols);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if (j >= n_groups) break;
            const Vec<X, 8> v = load<X, 8, VEC>(x[j], at, n_cols);
#pragma unroll
            for (int i = 0; i < RT; i++) {
                if (rank0 + 16 * i >= rank) break;
                if constexpr (Same<W, Bf16>::value && Same<X, Bf16>::value) {
                    acc[j][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, w[i]), __builtin_bit_cast(bf16x8, v), acc[j][i], 0, 0, 0);
                } else if constexpr (Same<W, _Float16>::value && Same<X, _Float16>::value) {
                    acc[j][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, w[i]), __builtin_bit_cast(f16x8, v), acc[j][i], 0, 0, 0);
                } else { /* the e-th of a lane's eight columns with the e-th of the other lanes': any order of columns does, the same on both sides */
#pragma unroll
                    for (int e = 0; e < 8; e++) acc[j][i] = __builtin_amdgcn_mfma_f32_16x16x4f32(to_f32(w[i].v[e]), to_f32(v.v[e]), acc[j][i], 0, 0, 0);
                }
            }
        }
    }
}

template <class W, class X, int RT>
__global__ void __launch_bounds__(64 * kWaves)
lora_shrink_kernel(LoraCall c, LoraPlan p) {
    __shared__ f32x4 red[kWaves][RT][64];
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    uint32_t b = blockIdx.x;
    const int slot = b % p.slots; b /= p.slots;
    const int part = b % p.parts; b /= p.parts;
    const int block = b % p.rank_blocks; b /= p.rank_blocks;
    const int mat = b % c.n_mat, tile = b / c.n_mat;
    const LoraTensor *m = mat == 0 ? &c.m[0] : mat == 1 ? &c.m[1] : &c.m[2];
    const X *x0 = static_cast<const X *>(c.X);
    const int rank0 = block * 16 * RT;
    const int steps = (c.n_cols + 31) / 32, share = part * kWaves + wv, shares = p.parts * kWaves;
    const int k0 = (int)((long long)steps * share / shares), k1 = (int)((long long)steps * (share + 1) / shares);
    const bool x_vec = c.n_cols % 8 == 0 && on(c.X, 16) && (size_t)c.ldx * sizeof(X) % 16 == 0;
    float *h = c.workspace + ((size_t)part * c.n_mat + mat) * c.n_tok * p.rank_pad;
    Classes classes(c.ids, c.n_tok, c.n_adapter, tile);
    for (int k = 0; classes.left; k++) {
        int id;
        const uint64_t same = classes.next(id);
        if (k % p.slots != slot) continue;
        const Entry e = entry_of(m->adapters, id, c.max_rank);
        if (e.rank <= rank0) continue; /* no adapter, or none of its ranks here: nothing is read of h either */
        const int count = __popcll(same), groups = (count + 15) / 16;
        const int order = packed_order(same);
        const X *x[4];
        size_t token[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int q = 16 * j + (lane & 15);
            token[j] = (size_t)tile * kTile + __shfl(order, q < count ? q : 0, 64);
            x[j] = x0 + token[j] * c.ldx;
        }
        f32x4 acc[4][RT] = {};
        const W *A = static_cast<const W *>(e.A);
        if (x_vec && on(A, 16))
            shrink_sums<W, X, RT, true>(A, rank0, e.rank, x, groups, c.n_cols, k0, k1, acc);
        else
            shrink_sums<W, X, RT, false>(A, rank0, e.rank, x, groups, c.n_cols, k0, k1, acc);
        /* the waves' sums, added in the waves' order */
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if (j >= groups) break;
#pragma unroll
            for (int i = 0; i < RT; i++) red[wv][i][lane] = acc[j][i];
            __syncthreads();
            for (int i = wv; i < RT; i += kWaves) {
                f32x4 v = red[0][i][lane];
#pragma unroll
                for (int w = 1; w < kWaves; w++) v += red[w][i][lane];
                const int r = rank0 + 16 * i + 4 * (lane >> 4);
#pragma unroll
                for (int q = 0; q < 4; q++)
                    if (r + q >= e.rank) v[q] = 0.0f;
                if (16 * j + (lane & 15) < count && r < p.rank_pad) *reinterpret_cast<f32x4 *>(h + token[j] * p.rank_pad + r) = v;
            }
            __syncthreads();
        }
    }
}

/* ------------------------------------------------------------------ Y + B h */

/* four consecutive elements of a row, of which `left` are there; VEC-aligned rows in one load */
__device__ __forceinline__ f32x4 load4(const void *base, size_t at, int left, uint32_t type, bool vec) {
    f32x4 y = {};
    if (type == T_F32) {
        const float *p = static_cast<const float *>(base) + at;
        if (vec && left > 3) return *reinterpret_cast<const f32x4 *>(p);
        for (int i = 0; i < 4; i++)
            if (i < left) y[i] = p[i];
    } else {
        Vec<uint16_t, 4> v = {};
        const uint16_t *p = static_cast<const uint16_t *>(base) + at;
        if (vec && left > 3)
            v = *reinterpret_cast<const Vec<uint16_t, 4> *>(p);
        else
            for (int i = 0; i < 4; i++)
                if (i < left) v.v[i] = p[i];
#pragma unroll
        for (int i = 0; i < 4; i++) y[i] = type == T_BF16 ? to_f32(Bf16{v.v[i]}) : to_f32(__builtin_bit_cast(_Float16, v.v[i]));
    }
    return y;
}
/* the one rounding of a result in 16 bits: to the nearest, ties to even */
__device__ __forceinline__ void store4(void *base, size_t at, int left, uint32_t type, bool vec, f32x4 y) {
    if (type == T_F32) {
        float *p = static_cast<float *>(base) + at;
        if (vec && left > 3) {
            *reinterpret_cast<f32x4 *>(p) = y;
            return;
        }
        for (int i = 0; i < 4; i++)
            if (i < left) p[i] = y[i];
    } else {
        Vec<uint16_t, 4> v;
#pragma unroll
        for (int i = 0; i < 4; i++) v.v[i] = type == T_BF16 ? __builtin_bit_cast(uint16_t, (__bf16)y[i]) : __builtin_bit_cast(uint16_t, (_Float16)y[i]);
        uint16_t *p = static_cast<uint16_t *>(base) + at;
        if (vec && left > 3) {
            *reinterpret_cast<Vec<uint16_t, 4> *>(p) = v;
            return;
        }
        for (int i = 0; i < 4; i++)
            if (i < left) p[i] = v.v[i];
    }
}

/* sums over an adapter's ranks for one group of 16 rows x 16 tokens; h: the tokens' in LDS */
template <class W, bool VEC>
__device__ __forceinline__ f32x4 expand_sums(const W *row, int rank, const float *h, f32x4 acc) {
    const int g = (threadIdx.x & 63) >> 4;
    for (int r = 0; r < rank; r += 16) {
        const Vec<W, 4> w = load<W, 4, VEC>(row, r + 4 * g, rank);
        const f32x4 v = *reinterpret_cast<const f32x4 *>(h + r + 4 * g);
#pragma unroll
        for (int i = 0; i < 4; i++) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(to_f32(w.v[i]), v[i], acc, 0, 0, 0);
    }
    return acc;
}

/* a workgroup: 16 MT rows on each of its waves, of one tensor or, PAIR, of gate and up */
template <class W, int MT, bool PAIR>
__global__ void __launch_bounds__(64 * kWaves)
lora_expand_kernel(LoraCall c, LoraPlan p) {
    extern __shared__ __attribute__((aligned(16))) float hs[]; /* [PAIR ? 2 : 1][16 tokens][rank_pad + 4] */
    constexpr int MATS = PAIR ? 2 : 1;
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4;
    uint32_t b = blockIdx.x;
    const int slot = b % p.slots; b /= p.slots;
    int mat = 0, block = b % p.row_blocks_all;
    const int tile = b / p.row_blocks_all;
    if (!PAIR) {
        if (block >= p.row_blocks[0]) { block -= p.row_blocks[0]; mat = 1; }
        if (mat == 1 && block >= p.row_blocks[1]) { block -= p.row_blocks[1]; mat = 2; }
    }
    const LoraTensor *m = mat == 0 ? &c.m[0] : mat == 1 ? &c.m[1] : &c.m[2];
    const int n_rows = m->n_rows, ldy = m->ldy, ldo = m->ldo;
    const int row0 = (block * kWaves + wv) * 16 * MT;
    const int stride = p.rank_pad + 4;
    const bool y_vec = on(m->Y, c.y_type == T_F32 ? 16 : 8) && (!PAIR || on(c.m[1].Y, c.y_type == T_F32 ? 16 : 8)) && ldy % 4 == 0;
    const bool o_vec = on(m->out, c.out_type == T_F32 ? 16 : 8) && ldo % 4 == 0;
    Classes classes(c.ids, c.n_tok, c.n_adapter, tile);
    for (int k = 0; classes.left; k++) {
        int id;
        const uint64_t same = classes.next(id);
        if (k % p.slots != slot) continue;
        Entry e[MATS];
#pragma unroll
        for (int a = 0; a < MATS; a++) e[a] = entry_of(PAIR ? c.m[a].adapters : m->adapters, id, c.max_rank);
        const int count = __popcll(same);
        const int order = packed_order(same);
        for (int j = 0; 16 * j < count; j++) {
            const int q = 16 * j + (lane & 15);
            const size_t token = (size_t)tile * kTile + __shfl(order, q < count ? q : 0, 64);
            /* h of the group's tokens: the parts' sums in their order */
            __syncthreads();
#pragma unroll
            for (int a = 0; a < MATS; a++) {
                for (int v = wv; 16 * v < e[a].rank; v += kWaves) { /* lane: token lane & 15, four ranks */
                    const size_t part = (size_t)c.n_mat * c.n_tok * p.rank_pad;
                    const float *from = c.workspace + ((size_t)(mat + a) * c.n_tok + token) * p.rank_pad + 16 * v + 4 * g;
                    f32x4 sum = *reinterpret_cast<const f32x4 *>(from);
                    for (int s = 1; s < p.parts; s++) sum += *reinterpret_cast<const f32x4 *>(from + s * part);
                    *reinterpret_cast<f32x4 *>(hs + (a * 16 + (lane & 15)) * stride + 16 * v + 4 * g) = sum * e[a].scale;
                }
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < MT; i++) {
                if (row0 + 16 * i >= n_rows) break;
                f32x4 acc[MATS] = {};
#pragma unroll
                for (int a = 0; a < MATS; a++) {
                    const int row = row0 + 16 * i + (lane & 15);
                    const W *w = static_cast<const W *>(e[a].B) + (size_t)(row < n_rows ? row : n_rows - 1) * e[a].rank;
                    const float *h = hs + (a * 16 + (lane & 15)) * stride;
                    if (e[a].rank % 4 == 0 && on(e[a].B, 4 * sizeof(W)))
                        acc[a] = expand_sums<W, true>(w, e[a].rank, h, acc[a]);
                    else
                        acc[a] = expand_sums<W, false>(w, e[a].rank, h, acc[a]);
                }
                const int row = row0 + 16 * i + 4 * g, left = n_rows - row;
                if (q < count && left > 0) {
                    f32x4 y = load4(m->Y, token * ldy + row, left, c.y_type, y_vec) + acc[0];
                    if constexpr (PAIR) {
                        const f32x4 u = load4(c.m[1].Y, token * ldy + row, left, c.y_type, y_vec) + acc[1];
#pragma unroll
                        for (int r = 0; r < 4; r++) y[r] = y[r] / (1.0f + expf(-y[r])) * u[r];
                    }
                    store4(m->out, token * ldo + row, left, c.out_type, o_vec, y);
                }
            }
        }
    }
}

template <class W, class X> hipError_t launch_shrink(const LoraCall &c, const LoraPlan &p) {
    const dim3 grid((uint32_t)p.shrink_workgroups()), block(64 * kWaves);
    if (p.rank_tiles == 1)
        hipLaunchKernelGGL((lora_shrink_kernel<W, X, 1>), grid, block, 0, c.stream, c, p);
    else if (p.rank_tiles == 2)
        hipLaunchKernelGGL((lora_shrink_kernel<W, X, 2>), grid, block, 0, c.stream, c, p);
    else
        hipLaunchKernelGGL((lora_shrink_kernel<W, X, 4>), grid, block, 0, c.stream, c, p);
    return hipGetLastError();
}

template <class W> hipError_t launch_both(const LoraCall &c, const LoraPlan &p) {
    hipError_t err = c.x_type == T_F32 ? launch_shrink<W, float>(c, p) : c.x_type == T_F16 ? launch_shrink<W, _Float16>(c, p) : launch_shrink<W, Bf16>(c, p);
    if (err != hipSuccess) return err;
    const dim3 grid((uint32_t)p.expand_workgroups()), block(64 * kWaves);
    const size_t lds = (size_t)(c.pair ? 2 : 1) * 16 * (p.rank_pad + 4) * sizeof(float);
    if (c.pair) {
        if (p.row_tiles == 1)
            hipLaunchKernelGGL((lora_expand_kernel<W, 1, true>), grid, block, lds, c.stream, c, p);
        else
            hipLaunchKernelGGL((lora_expand_kernel<W, 4, true>), grid, block, lds, c.stream, c, p);
    } else {
        if (p.row_tiles == 1)
            hipLaunchKernelGGL((lora_expand_kernel<W, 1, false>), grid, block, lds, c.stream, c, p);
        else
            hipLaunchKernelGGL((lora_expand_kernel<W, 4, false>), grid, block, lds, c.stream, c, p);
    }
    return hipGetLastError();
}

}  // namespace

/* how many parts the columns are cut into: enough workgroups for the chip without the classes, whose number is not known here, and at least
 * two steps of 32 columns for a wave */
static int lora_parts(int n_mat, int max_rank, int n_cols, int n_tok) {
    const long long tiles = ((long long)n_tok + kTile - 1) / kTile, ranks = ((long long)max_rank + 63) / 64;
    const long long want = 1024 / (tiles * n_mat * ranks), most = (n_cols + 255) / 256;
    const long long parts = want < most ? want : most;
    return (int)(parts > 16 ? 16 : parts < 1 ? 1 : parts);
}

size_t lora_workspace_bytes(int n_mat, int max_rank, int n_cols, int n_tok) {
    return (size_t)lora_parts(n_mat, max_rank, n_cols, n_tok) * n_mat * n_tok * ((max_rank + 15) / 16 * 16) * sizeof(float);
}

LoraPlan lora_plan(const LoraCall &c) {
    LoraPlan p;
    p.tiles = (int)(((long long)c.n_tok + kTile - 1) / kTile);
    p.rank_pad = (c.max_rank + 15) / 16 * 16;
    p.rank_tiles = p.rank_pad <= 16 ? 1 : p.rank_pad <= 32 ? 2 : 4;
    p.rank_blocks = (p.rank_pad + 16 * p.rank_tiles - 1) / (16 * p.rank_tiles);
    p.parts = lora_parts(c.n_mat, c.max_rank, c.n_cols, c.n_tok);
    p.row_tiles = c.n_tok <= kTile ? 1 : 4;
    p.n_mat = c.n_mat;
    p.row_blocks_all = 0;
    for (int i = 0; i < 3; i++) {
        p.row_blocks[i] = i < c.n_mat && (i == 0 || !c.pair) ? (int)(((long long)c.m[i].n_rows + 16 * kWaves * p.row_tiles - 1) / (16 * kWaves * p.row_tiles)) : 0;
        p.row_blocks_all += p.row_blocks[i];
    }
    long long classes = c.n_tok < kTile ? c.n_tok : kTile;
    if (c.n_adapter + 1ll < classes) classes = c.n_adapter + 1ll;
    const long long others = (long long)p.tiles * p.n_mat * p.rank_blocks * p.parts;
    const long long want = 4096 / (others > 0 ? others : 1);
    p.slots = (int)(want < 1 ? 1 : want < classes ? want : classes);
    return p;
}

hipError_t launch_lora(uint32_t w_type, const LoraCall &c, const LoraPlan &p) {
    return w_type == T_F32 ? launch_both<float>(c, p) : w_type == T_F16 ? launch_both<_Float16>(c, p) : launch_both<Bf16>(c, p);
}

}  // namespace qlin
