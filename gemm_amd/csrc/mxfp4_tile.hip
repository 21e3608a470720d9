/*
 * mxfp4_tile.hip - products of MXFP4 operands (mxfp4.h) for many tokens: tiles of 64 MB rows x 64 NB tokens on four waves, two by two.
 *
 *   Y[t, r] = sum_k X[t, k] W[r, k]          or, of two tensors, silu(X . gate) * (X . up)
 *
 * v_mfma_scale_f32_32x32x64_f8f6f4 on 4-bit operands (from registers 9.6 PFLOP/s on constant operands and 6.45 on random ones, where the
 * part's power limits it; the 16x16x128 form 6.9 at best), fp32 sums.
 * A wave holds 32 MB rows x 32 NB tokens as sums in registers. Both operands go from memory to LDS by load-to-LDS requests of 1 KB, an
 * operand tile each, three column tiles ahead of their use in four stages; a fragment is one ds_read_b128 without bank conflicts,
 * fetched half a column tile (64 columns) ahead into the second of two register sets. The exponents of 512 columns come the same
 * way, a dword per lane, row and block, one byte for each of four column tiles. One barrier per column tile, in its middle: from there
 * on fragments come from the next stage.
 *   Of two tensors, the first MB / 2 row blocks of a wave are gate rows and the others the same rows of up: both sums of a result are in
 * one lane.
 *   What bounds it: 256 x 256 tiles take 0.80 us per column tile on random operands, 5.4 PFLOP/s over the chip, and 0.50 on zeros: the
 * power limit. Beside that the results of a round of tiles leave at its end, with nothing left to multiply: 4096 x 4096 of them 13 us
 * in fp32 and 9 in bf16, launch and first loads included. 4096 x 4096 columns x 4096 tokens 39 us in fp32 (3.5 PFLOP/s) and 35 in bf16, 4096 x 16384 x
 * 4096 113 to 115 (4.8), 14336 x 4096 x 2048 in bf16 63 to 69, gate and up of 512 tokens 35.5 to 37.
 */
#include "mxfp4.h"

#include <cmath>

#include "gemm_kq_formats.h"

namespace qlin {
using namespace mxfp4;

namespace {

using kq::dma16;

template <int VM> QLIN_INL void wait_vmcnt_lds() { /* vmcnt(VM) and lgkmcnt(0) */
    __builtin_amdgcn_s_waitcnt((VM & 15) | ((VM >> 4) << 14) | (7 << 4));
}

/* the stages are objects of their own: a fetch from one never waits for a request into another */
template <int MB, int NB, int ST> QLIN_INL uint8_t *stage_of() {
    __shared__ __attribute__((aligned(1024))) uint8_t stage[(4 * MB + 4 * NB) * kTileBytes];
    return stage;
}
template <int MB, int NB> QLIN_INL uint8_t *exponents_of() {
    __shared__ __attribute__((aligned(1024))) uint8_t exponents[(4 * MB + 4 * NB) * kScaleBytes];
    return exponents;
}

template <int MB_, int NB_, bool PAIR_> struct Ctx {
    static constexpr int MB = MB_, NB = NB_, kReq = MB + NB, kExpReq = (MB + NB + 3) / 4, kSlots = MB * NB;
    static constexpr bool PAIR = PAIR_;
    f32x16 acc[MB][NB];
    u32x4 a[2][MB], b[2][NB];     /* fragments, [half column tile] */
    int ea[2][MB], eb[2][NB];     /* exponents of these 512 columns */
    int na[2][MB], nb[2][NB];     /* and of the next */
    __amdgpu_buffer_rsrc_t w_rsrc, x_rsrc, e_rsrc[kExpReq];
    uint32_t w_off[MB], x_off[NB]; /* of this wave's row groups, in scalar registers */
    uint32_t e_off[kExpReq];
    int e_to[kExpReq];
    uint32_t lane16, a_at, b_at, ea_at, eb_at;
    int wave, tiles, quads;
    /* byte offset of row block m in a stage, for wave row 0 */
    static constexpr int block(int m) { return PAIR && m >= MB / 2 ? (2 * MB + 2 * (m - MB / 2)) : 2 * m; }
};

constexpr int first_of(int t, int n, int slots) { return t >= slots ? n : (t * n + slots - 1) / slots; }

template <int ST, int I, class C> QLIN_INL void request(C &c, int tile) { /* requests 0 .. kReq - 1 of this wave for a column tile */
    const uint32_t at = (uint32_t)min(tile, c.tiles - 1) * kTileBytes; /* past the last tile: a harmless repetition */
    uint8_t *st = stage_of<C::MB, C::NB, ST>();
    if constexpr (I < C::MB) dma16(c.w_rsrc, st + (C::MB * c.wave + I) * kTileBytes, c.lane16, c.w_off[I] + at);
    else dma16(c.x_rsrc, st + (4 * C::MB + C::NB * c.wave + I - C::MB) * kTileBytes, c.lane16, c.x_off[I - C::MB] + at);
}
template <int I, class C> QLIN_INL void request_exponents(C &c, int quad) {
    dma16(c.e_rsrc[I], exponents_of<C::MB, C::NB>() + c.e_to[I], c.e_off[I], (uint32_t)min(quad, c.quads - 1) * kScaleBytes);
}
/* fragment I of half H of stage ST: a 0, b 0 .. NB - 1, a 1 .. */
template <int ST, int H, int I, class C> QLIN_INL void fetch(C &c) {
    const uint8_t *st = stage_of<C::MB, C::NB, ST>();
    if constexpr (I >= 1 && I <= C::NB)
        c.b[H][I - 1] = *reinterpret_cast<const u32x4 *>(st + c.b_at + 2 * (I - 1) * kTileBytes + H * 512);
    else
        c.a[H][I ? I - C::NB : 0] = *reinterpret_cast<const u32x4 *>(st + c.a_at + C::block(I ? I - C::NB : 0) * kTileBytes + H * 512);
}
template <int I, class C> QLIN_INL void fetch_exponent(C &c) { /* of the next 512 columns, 0 .. 2 kReq - 1 */
    const uint8_t *e = exponents_of<C::MB, C::NB>();
    constexpr int h = I & 1, i = I >> 1;
    if constexpr (i < C::MB) c.na[h][i] = *reinterpret_cast<const int *>(e + c.ea_at + C::block(i) * kScaleBytes + h * 128);
    else c.nb[h][i - C::MB] = *reinterpret_cast<const int *>(e + c.eb_at + 2 * (i - C::MB) * kScaleBytes + h * 128);
}

template <int LO, int HI, class F> QLIN_INL void each(F fn) {
    if constexpr (LO < HI) {
        fn(std::integral_constant<int, LO>{});
        each<LO + 1, HI>(fn);
    }
}

/* slot T of half H of column tile `tile`, which is number U of its four */
template <int U, int H, int T, class C> QLIN_INL void slot(C &c, int tile) {
    constexpr int S = C::kSlots, m = T / C::NB, n = T % C::NB, g = H * S + T;
    if constexpr (H == 1 && T == 0) {
        /* The next tile's requests of this wave have landed: younger are those of the tile after it (with the exponents', which
         * tile 0 of a quad requests after this point) and those of the one behind so far. The fragments of this tile are in
         * registers, so that after the barrier its stage may be written. */
        constexpr int so_far = first_of(S, C::kReq, 2 * S);
        wait_vmcnt_lds<C::kReq + so_far + (U == 1 ? C::kExpReq : 0)>();
        __builtin_amdgcn_s_barrier();
    }
    c.acc[m][n] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(widened(c.b[H][n]), widened(c.a[H][m]), c.acc[m][n], 4, 4, U, c.eb[H][n], U, c.ea[H][m]);
    constexpr int early = S > 4 ? S * 3 / 4 : S; /* fragments are there before they are used */
    each<first_of(T, C::kReq, early), first_of(T + 1, C::kReq, early)>([&](auto i) {
        if constexpr (H == 0) fetch<U, 1, decltype(i)::value>(c);
        else fetch<(U + 1) & 3, 0, decltype(i)::value>(c);
    });
    if constexpr (U == 0 && H == 1 && T == 0) each<0, C::kExpReq>([&](auto i) { request_exponents<decltype(i)::value>(c, (tile >> 2) + 1); });
    if constexpr (U == 3) each<first_of(g, 2 * C::kReq, 2 * S), first_of(g + 1, 2 * C::kReq, 2 * S)>([&](auto i) { fetch_exponent<decltype(i)::value>(c); });
    each<first_of(g, C::kReq, 2 * S), first_of(g + 1, C::kReq, 2 * S)>([&](auto i) { request<(U + 3) & 3, decltype(i)::value>(c, tile + 3); });
    __builtin_amdgcn_sched_barrier(0);
}
template <int U, class C> QLIN_INL void run_tile(C &c, int tile) {
    each<0, C::kSlots>([&](auto t) { slot<U, 0, decltype(t)::value>(c, tile); });
    each<0, C::kSlots>([&](auto t) { slot<U, 1, decltype(t)::value>(c, tile); });
}
template <class C> QLIN_INL void take_exponents(C &c) {
#pragma unroll
    for (int h = 0; h < 2; h++) {
#pragma unroll
        for (int m = 0; m < C::MB; m++) c.ea[h][m] = c.na[h][m];
#pragma unroll
        for (int n = 0; n < C::NB; n++) c.eb[h][n] = c.nb[h][n];
    }
}

template <bool STREAM> QLIN_INL void put(float *to, float v) {
    if constexpr (STREAM) __builtin_nontemporal_store(v, to);
    else *to = v;
}
/* Two results of this lane's row, of tokens t and t + 1, of which those below `tokens` are there; to = the row's place in token t. 32 lanes
 * hold 32 consecutive rows: a store instruction writes two runs of 128 bytes of F32, or after an exchange between neighbouring lanes
 * four of 64 bytes of BF16. STREAM marks them as not read again soon: what would wait in the L2 for the end of the kernel goes to
 * memory beside the next tiles' products (14336 x 4096, 1024 tokens in 128 x 128 tiles 45.6 -> 36.8 us, 4096 tokens in 256 x 256 141 -> 137),
 * but only where rows lie on 64 bytes, so that a run is whole sectors: else they are written twice (23207 rows x 576, 1073 tokens 28 -> 58,
 * rows on 32 bytes 26 -> 45). */
template <bool STREAM> QLIN_INL void put2(float *to, size_t ldy, float a, float b, int tokens, int rows_left) {
    if (rows_left <= 0) return;
    if (tokens > 0) put<STREAM>(to, a);
    if (tokens > 1) put<STREAM>(to + ldy, b);
}
template <bool STREAM> QLIN_INL void put2(__bf16 *to, size_t ldy, float a, float b, int tokens, int rows_left) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    typedef bf16x2 anywhere __attribute__((aligned(2)));
    const bool odd = threadIdx.x & 1; /* even lanes store token t of both rows, odd ones token t + 1 */
    const float other = __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(odd ? a : b), 0xB1, 0xf, 0xf, true));
    const bf16x2 v = {(__bf16)(odd ? other : a), (__bf16)(odd ? b : other)}; /* nearest even, the one rounding of a result */
    to += odd ? (ptrdiff_t)ldy - 1 : 0;
    rows_left += odd;
    if (tokens <= (int)odd) return;
    if (rows_left > 1) {
        if constexpr (STREAM) __builtin_nontemporal_store(v, reinterpret_cast<anywhere *>(to));
        else *reinterpret_cast<anywhere *>(to) = v;
    } else if (rows_left == 1) to[0] = v[0];
}

/* The same for two row blocks, 32 rows apart and all there: after a second exchange a token's 128 bytes of both are one instruction's (in
 * 64-byte runs 58.7 MB of results were 85.4 MB of writes to memory). */
template <bool STREAM> QLIN_INL void put2x2(__bf16 *to, size_t ldy, float a0, float b0, float a1, float b1, int tokens) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    const bool odd = threadIdx.x & 1;
    auto swapped = [](uint32_t v) { return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xf, 0xf, true); };
    auto rows_of = [&](float a, float b) { /* both rows of the lane pair, token t in even lanes, t + 1 in odd ones */
        const float other = __uint_as_float(swapped(__float_as_uint(odd ? a : b)));
        const bf16x2 v = {(__bf16)(odd ? other : a), (__bf16)(odd ? b : other)};
        return __builtin_bit_cast(uint32_t, v);
    };
    const uint32_t v0 = rows_of(a0, b0), v1 = rows_of(a1, b1), other = swapped(odd ? v0 : v1);
    /* even lanes: the first block's rows of both tokens; odd ones: the second's */
    typedef uint32_t anywhere __attribute__((aligned(2)));
    __bf16 *at = to + (odd ? 31 : 0);
    const uint32_t first = odd ? other : v0, second = odd ? v1 : other;
    if (tokens > 0) {
        if constexpr (STREAM) __builtin_nontemporal_store(first, reinterpret_cast<anywhere *>(at));
        else *reinterpret_cast<anywhere *>(at) = first;
    }
    if (tokens > 1) {
        if constexpr (STREAM) __builtin_nontemporal_store(second, reinterpret_cast<anywhere *>(at + ldy));
        else *reinterpret_cast<anywhere *>(at + ldy) = second;
    }
}

/* the bytes of an operand from row group `from` of a part with `pitch` bytes per group, as a buffer descriptor counts them */
QLIN_INL uint32_t bytes_from(int groups, int from, uint32_t pitch) {
    const size_t n = (size_t)(groups - from) * pitch;
    return n > 0xFFFFFFFFu ? 0xFFFFFFFFu : (uint32_t)n;
}

template <int MB, int NB, bool PAIR, class OUT>
__global__ void __launch_bounds__(kTileThreads, MB + NB > 4 ? 1 : 2)
tile_kernel(const uint8_t *__restrict__ W, const uint8_t *__restrict__ up, const uint8_t *__restrict__ X, OUT *__restrict__ Y, int n_rows, int n_tok, Shape w,
            Shape x, size_t ldy, int row_tiles, int tok_tiles, bool stream) {
    /* Consecutive workgroups go to different dies, each with an L2 of its own: a die takes a run of the tiles, numbered through groups of
     * kGroup row tiles, in a group the row tiles of a token tile first, so that what runs at a time on a die shares its rows and tokens. */
    constexpr int kGroup = 8;
    const unsigned n_tiles = (unsigned)row_tiles * (unsigned)tok_tiles, per_die = gridDim.x >> 3;
    const unsigned id = (blockIdx.x & 7) * per_die + (blockIdx.x >> 3);
    if (id >= n_tiles) return;
    const unsigned of_group = (unsigned)kGroup * tok_tiles, first = id / of_group * kGroup, rest = id % of_group;
    const unsigned height = min((unsigned)row_tiles - first, (unsigned)kGroup);
    const int tok_tile = rest / height, row_tile = first + rest % height;
    constexpr int kRowGroups = PAIR ? 2 * MB : 4 * MB; /* row groups of a tensor per tile */
    const int lane = threadIdx.x & 63;
    Ctx<MB, NB, PAIR> c;
    using C = Ctx<MB, NB, PAIR>;
    c.wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    c.tiles = w.tiles;
    c.quads = w.quads;
    c.lane16 = lane * 16;
    const int wm = c.wave >> 1, wn = c.wave & 1;
    const uint32_t code_pitch = (uint32_t)w.tiles * kTileBytes, exp_pitch = (uint32_t)w.quads * kScaleBytes;
    const int g0 = row_tile * kRowGroups, x0 = tok_tile * 4 * NB;
    /* codes: this wave requests MB row groups of the 4 MB (of two tensors, waves 0 and 1 gate's and 2 and 3 up's) and NB token groups;
     * groups past the end repeat the last one */
    const bool of_up = PAIR && c.wave >= 2;
    c.w_rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(of_up ? up : W) + (size_t)g0 * code_pitch, 0, bytes_from(w.groups, g0, code_pitch), 0x00020000);
    c.x_rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(X) + (size_t)x0 * code_pitch, 0, bytes_from(x.groups, x0, code_pitch), 0x00020000);
#pragma unroll
    for (int i = 0; i < MB; i++) c.w_off[i] = (uint32_t)min(MB * (of_up ? c.wave - 2 : c.wave) + i, w.groups - 1 - g0) * code_pitch;
#pragma unroll
    for (int i = 0; i < NB; i++) c.x_off[i] = (uint32_t)min(NB * c.wave + i, x.groups - 1 - x0) * code_pitch;
    /* exponents: request id holds four groups' 256 bytes, ids below MB those of the rows */
#pragma unroll
    for (int i = 0; i < C::kExpReq; i++) {
        const int id = min(c.wave + 4 * i, MB + NB - 1);
        const bool rows = id < MB, second = PAIR && rows && 2 * id >= MB;
        const uint8_t *part = rows ? (second ? up : W) + w.code_bytes() + (size_t)g0 * exp_pitch : X + x.code_bytes() + (size_t)x0 * exp_pitch;
        const int last = rows ? w.groups - 1 - g0 : x.groups - 1 - x0;
        const int group = (rows ? 4 * id - (second ? 2 * MB : 0) : 4 * (id - MB)) + (lane >> 4);
        c.e_rsrc[i] = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(part), 0, bytes_from(last + 1, 0, exp_pitch), 0x00020000);
        c.e_off[i] = (uint32_t)min(group, last) * exp_pitch + (lane & 15) * 16;
        c.e_to[i] = id * 4 * kScaleBytes;
    }
    /* a lane's block of a 32-row fragment: row l % 32, that is group (l / 16) % 2, and block l / 32 of a half's two */
    const uint32_t in_pair = (lane >> 4) & 1, in_half = lane >> 5, in_group = lane & 15;
    constexpr int kWaveGroups = PAIR ? MB : 2 * MB;
    c.a_at = (wm * kWaveGroups + in_pair) * kTileBytes + in_half * 256 + in_group * 16;
    c.b_at = (4 * MB + wn * 2 * NB + in_pair) * kTileBytes + in_half * 256 + in_group * 16;
    c.ea_at = (wm * kWaveGroups + in_pair) * kScaleBytes + in_half * 64 + in_group * 4;
    c.eb_at = (4 * MB + wn * 2 * NB + in_pair) * kScaleBytes + in_half * 64 + in_group * 4;
#pragma unroll
    for (int m = 0; m < MB; m++)
#pragma unroll
        for (int n = 0; n < NB; n++)
#pragma unroll
            for (int v = 0; v < 16; v++) c.acc[m][n][v] = 0.0f;

    /* The last columns' one to three tiles of a quad: a chain of tiles behind the loop, or where its registers would spill (16 blocks) a
     * whole quad, whose missing tiles multiply repeated codes by 2^-127 twice: their exponent bytes are 0 on both sides, and 2^-254
     * times any sum of codes is 0 in fp32. */
    constexpr bool kChain = MB * NB <= 8;
    each<0, C::kExpReq>([&](auto i) { request_exponents<decltype(i)::value>(c, 0); });
    each<0, C::kReq>([&](auto i) { request<0, decltype(i)::value>(c, 0); });
    each<0, C::kReq>([&](auto i) { request<1, decltype(i)::value>(c, 1); });
    each<0, C::kReq>([&](auto i) { request<2, decltype(i)::value>(c, 2); });
    wait_vmcnt_lds<2 * C::kReq>();
    __builtin_amdgcn_s_barrier();
    each<0, 2 * C::kReq>([&](auto i) { fetch_exponent<decltype(i)::value>(c); });
    take_exponents(c);
    each<0, C::kReq>([&](auto i) { fetch<0, 0, decltype(i)::value>(c); });
#pragma unroll 1
    for (int tile = 0; tile < c.tiles - (kChain ? 3 : 0); tile += 4) {
        run_tile<0>(c, tile);
        run_tile<1>(c, tile + 1);
        run_tile<2>(c, tile + 2);
        run_tile<3>(c, tile + 3);
        take_exponents(c);
    }
    if constexpr (kChain) {
        const int full = c.tiles & ~3;
        if (c.tiles & 3) run_tile<0>(c, full);
        if (c.tiles & 2) run_tile<1>(c, full + 1);
        if ((c.tiles & 3) == 3) run_tile<2>(c, full + 2);
    }
    wait_vmcnt_lds<0>(); /* requests past the last tile are still on their way into LDS */

    /* register v of lane l: token 8 (v / 4) + 4 (l / 32) + v % 4, row l % 32 */
    constexpr int kOut = PAIR ? MB / 2 : MB;
    const int t0 = (tok_tile * 2 + wn) * 32 * NB + 4 * (lane >> 5), r0 = (row_tile * 2 + wm) * 32 * kOut + (lane & 31);
    const bool whole = n_rows - row_tile * 64 * kOut >= 64 * kOut;
    auto store = [&](auto streams) {
#pragma unroll
        for (int n = 0; n < NB; n++)
#pragma unroll
            for (int v = 0; v < 16; v += 2) {
                const int t = t0 + 32 * n + 8 * (v / 4) + v % 4;
                OUT *y = Y + (size_t)t * ldy + r0;
                auto result = [&](int m, int i) {
                    if constexpr (PAIR) return silu_mul(c.acc[m][n][i], c.acc[m + MB / 2][n][i]);
                    else return c.acc[m][n][i];
                };
                if constexpr (sizeof(OUT) == 2 && kOut % 2 == 0) {
                    if (whole) {
#pragma unroll
                        for (int m = 0; m < kOut; m += 2)
                            put2x2<decltype(streams)::value>(y + 32 * m, ldy, result(m, v), result(m, v + 1), result(m + 1, v), result(m + 1, v + 1), n_tok - t);
                        continue;
                    }
                }
#pragma unroll
                for (int m = 0; m < kOut; m++) put2<decltype(streams)::value>(y + 32 * m, ldy, result(m, v), result(m, v + 1), n_tok - t, n_rows - r0 - 32 * m);
            }
    };
    if (stream) store(std::true_type{});
    else store(std::false_type{});
}

template <int MB, int NB, bool PAIR, class OUT> hipError_t tiles(const Mxfp4Product &p) {
    const Shape w = shape_of(p.n_rows, p.n_cols), x = shape_of(p.n_tok, p.n_cols);
    constexpr int kRows = (PAIR ? 32 : 64) * MB, kTok = 64 * NB;
    const int row_tiles = (p.n_rows + kRows - 1) / kRows, tok_tiles = (p.n_tok + kTok - 1) / kTok;
    const dim3 grid((unsigned)mxfp4_launch(10 * MB + NB, p).workgroups);
    const bool stream = (reinterpret_cast<uintptr_t>(p.Y) & 63) == 0 && (size_t)p.ldy * sizeof(OUT) % 64 == 0;
    tile_kernel<MB, NB, PAIR, OUT><<<grid, kTileThreads, 0, p.stream>>>(p.W, p.up, static_cast<const uint8_t *>(p.X), static_cast<OUT *>(p.Y), p.n_rows, p.n_tok, w, x, (size_t)p.ldy, row_tiles, tok_tiles, stream);
    return hipGetLastError();
}
template <int MB, int NB> hipError_t tiles_for(const Mxfp4Product &p) {
    if (p.up) {
        if constexpr (MB % 2 == 0) return p.bf16_out ? tiles<MB, NB, true, __bf16>(p) : tiles<MB, NB, true, float>(p);
        else return hipErrorInvalidValue;
    }
    return p.bf16_out ? tiles<MB, NB, false, __bf16>(p) : tiles<MB, NB, false, float>(p);
}

}  // namespace

hipError_t launch_mxfp4_tiles(int mb, int nb, const Mxfp4Product &p) {
    switch (10 * mb + nb) {
    case 44: return tiles_for<4, 4>(p);
    case 22: return tiles_for<2, 2>(p);
    case 21: return tiles_for<2, 1>(p);
    case 11: return tiles_for<1, 1>(p);
    default: return hipErrorInvalidValue;
    }
}

namespace {

/* What a product takes, us: `start`, then the longest of the rounds that the tiles make of the chip (`resident` workgroups per compute
 * unit), one at a time (`wait` per column tile: the chain of requests, barriers and matrix instructions of a workgroup that has the unit to
 * itself, `rest` per tile) or side by side (`work`: what they take of the unit from each other); the weights from memory; and the
 * results to it, per MB. Fitted to 229 measured products of 17 to 4096 tokens, 256 to 28672 rows and 256 to 14336 columns, which
 * the smallest estimate's kernel takes 1.6 % longer than the fastest in the mean and 28 % at most (23551 rows x 6912, 169 tokens: 39 us against
 * 30 of a 128 x 256 tile, which was built with two more shapes and left out: together they gain 0.1 %). 420 others, F32 and BF16 in
 * equal parts and rows of any alignment, 2.5 % and 30 % (with costs of results by type and alignment, fitted to them, 2.1 %). */
struct TileCost { int mb, nb, resident; float start, wait, work, rest, result, weights; };
constexpr TileCost kTileCosts[] = {{1, 1, 4, 2.888f, 0.123f, 0.097f, 0.552f, 0.108f, 0.163f},
                                   {2, 1, 3, 3.019f, 0.105f, 0.149f, 1.114f, 0.114f, 0.167f},
                                   {2, 2, 2, 2.368f, 0.167f, 0.202f, 2.146f, 0.155f, 0.220f},
                                   {4, 4, 1, 0.378f, 0.493f, 0.003f, 8.793f, 0.154f, 0.326f}};
float rounds(double n, int at_a_time) { return (float)ceil(n / at_a_time); }
float tile_us(const TileCost &c, const Mxfp4Product &p, int n_cu) {
    const Shape w = shape_of(p.n_rows, p.n_cols);
    const int rows = (p.up ? 32 : 64) * c.mb, tok = 64 * c.nb;
    const double n = ceil((double)p.n_rows / rows) * ceil((double)p.n_tok / tok);
    const float alone = rounds(n, n_cu * c.resident) * (c.wait * w.tiles + c.rest), together = rounds(n, n_cu) * (c.work * w.tiles + c.rest / c.resident);
    const double mb_in = (double)w.bytes() * (p.up ? 2 : 1) * 1e-6, mb_out = (double)p.n_rows * p.n_tok * (p.bf16_out ? 2 : 4) * 1e-6;
    return c.start + fmaxf(fmaxf(alone, together), c.weights * (float)mb_in) + c.result * (float)mb_out;
}
/* the kernel of 16 rows per workgroup: what its workgroups read, or the weights from memory, or the 32-column-tile pieces of a wave in turn */
float few_us(const Mxfp4Product &p) {
    const Shape w = shape_of(p.n_rows, p.n_cols), x = shape_of(p.n_tok, p.n_cols);
    const int mats = p.up ? 2 : 1, nt = x.groups < 4 ? x.groups : 4;
    const double kb = (double)w.groups * ((x.groups + nt - 1) / nt) * w.tiles;
    const double mb_in = (double)w.bytes() * mats * 1e-6, mb_out = (double)p.n_rows * p.n_tok * (p.bf16_out ? 2 : 4) * 1e-6;
    return 3.2253f + fmaxf(fmaxf((float)(kb * 1e-3 * (0.0189 * mats + 0.0894 * nt)), 0.1766f * (float)mb_in), 1.2065f * ((w.tiles + 31) / 32)) + 0.7458f * (float)mb_out;
}

}  // namespace

int mxfp4_choice(const Mxfp4Product &p, int n_cu) {
    /* up to 16 tokens, one token group: never more than 5 % behind the tiles, and without a launch to quantise for the fewest */
    if (p.n_tok <= 16) return 0;
    int best = 0;
    float least = few_us(p);
    for (const TileCost &c : kTileCosts) {
        if (p.up && c.mb == 1) continue; /* no row block for the second tensor */
        const float t = tile_us(c, p, n_cu);
        if (t < least) least = t, best = 10 * c.mb + c.nb;
    }
    return best;
}

Mxfp4Launch mxfp4_launch(int kernel, const Mxfp4Product &p) {
    const Shape w = shape_of(p.n_rows, p.n_cols), x = shape_of(p.n_tok, p.n_cols);
    if (kernel == 0) return {(size_t)w.groups * ((x.groups + 3) / 4), kFewThreads}; /* (up to four token groups each) */
    const size_t rows = (p.up ? 32 : 64) * (kernel / 10), tok = 64 * (kernel % 10);
    const size_t tiles = (p.n_rows + rows - 1) / rows * ((p.n_tok + tok - 1) / tok);
    return {(tiles + 7) / 8 * 8, kTileThreads}; /* (as many for each die) */
}

hipError_t launch_mxfp4_product(const Mxfp4Product &p, int n_cu) {
    const int k = mxfp4_choice(p, n_cu);
    return k == 0 ? launch_mxfp4_few(p) : launch_mxfp4_tiles(k / 10, k % 10, p);
}

}  // namespace qlin
