/*
 * mxfp4_few.hip - products of MXFP4 operands (mxfp4.h), one workgroup per 16 rows of weights, its waves along K.
 *
 *   Y[t, r] = sum_k X[t, k] W[r, k]          or, of two tensors, silu(X . gate) * (X . up)
 *
 * v_mfma_scale_f32_16x16x128_f8f6f4 multiplies 16 rows by 16 tokens over 128 columns and applies both blocks' powers of two: the
 * products of codes are exact, the sums are fp32. Every load is a whole kilobyte of an operand in the instruction's own lane order,
 * from memory to registers. A wave takes 512 columns at a time (four instructions per row group and token group share one dword of
 * exponents per lane), wave w the 512-column pieces w, w + waves, ...; the waves' sums meet in LDS and are added in the waves' order.
 *   A token or a few come as floats: every wave quantises the 512 columns of its piece itself, eight elements per lane, and turns them
 * into operand order through 272 bytes of LDS per token. That repeats the work in every workgroup, but it is done while the weights
 * are on their way, and saves the launch of a kernel that would have nothing else to do.
 *   Bound by memory: one token x 14336 x 4096 8.0 us, 3.9 TB/s (a bare read of the 31 MB 5.9), 28672 x 4096 12.4 us, 5.0 TB/s (9.9),
 * 151936 x 4096 54.8 us, 6.0 TB/s (48.6); what is missing is the start of the launch and the last workgroups' sums. Four tokens
 * of an operand 58.7 us at the last size. 16 rows are the fewest of the instruction, and eight waves along K give a short
 * tensor (1000 rows: 63 workgroups) the most requests at a time.
 */
#include "mxfp4_quant.h"

namespace qlin {
using namespace mxfp4;

namespace {

/* the first `left` of four results to consecutive elements, at any element address */
__device__ __forceinline__ void store4(float *y, f32x4 a, int left) {
    typedef f32x4 anywhere __attribute__((aligned(4)));
    if (left > 3) {
        *reinterpret_cast<anywhere *>(y) = a;
    } else {
        for (int v = 0; v < 3; v++)
            if (v < left) y[v] = a[v];
    }
}
__device__ __forceinline__ void store4(__bf16 *y, f32x4 a, int left) {
    typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
    typedef bf16x4 anywhere __attribute__((aligned(2)));
    const bf16x4 b = {(__bf16)a[0], (__bf16)a[1], (__bf16)a[2], (__bf16)a[3]}; /* nearest even, the one rounding of a result */
    if (left > 3) {
        *reinterpret_cast<anywhere *>(y) = b;
    } else {
        for (int v = 0; v < 3; v++)
            if (v < left) y[v] = b[v];
    }
}

constexpr int kFewFloats = 8; /* tokens that a workgroup quantises itself, at most */

/* A wave's lanes read from LDS what others of its lanes wrote, and write it anew: one wave's requests to LDS stay in order, and this keeps the compiler from
 * changing it. No instruction. */
__device__ __forceinline__ void wave_meets() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

/* MATS 2: gate and up; NT: token groups of 16 per workgroup; XT: uint8_t for an operand, or the floats' type (FLOATS tokens at most, rows
 * that can be read in 16-byte loads) */
template <int MATS, int NT, int WAVES, int FLOATS, class XT, class OUT>
__global__ void __launch_bounds__(64 * WAVES)
few_kernel(const uint8_t *__restrict__ W, const uint8_t *__restrict__ up, const XT *__restrict__ X, OUT *__restrict__ Y, int n_rows, int n_tok, Shape w, Shape x,
           int n_cols, size_t ldx, size_t ldy) {
    constexpr bool kFloats = !std::is_same<XT, uint8_t>::value;
    static_assert(!kFloats || (NT == 1 && FLOATS <= kFewFloats), "floats come in one token group");
    __shared__ f32x4 sums[WAVES][MATS * NT][64];
    __shared__ __attribute__((aligned(16))) uint32_t packed[kFloats ? WAVES : 1][FLOATS][64 + 4]; /* of a piece: codes, exponents */
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int token_blocks = (x.groups + NT - 1) / NT;
    const int group = blockIdx.x / (unsigned)token_blocks, t0 = (blockIdx.x - group * token_blocks) * NT;
    f32x4 acc[MATS][NT] = {};
    for (int q = wave; q < w.quads; q += WAVES) {
        u32x4 a[MATS][4], b[NT][4];
        int sa[MATS], sb[NT];
        float v[FLOATS][8];
        if constexpr (kFloats) { /* ahead of the weights, so that waiting for them does not wait for those */
#pragma unroll
            for (int t = 0; t < FLOATS; t++)
                if (t < n_tok) load8<XT, true>(X + t * ldx + q * 512 + lane * 8, n_cols - q * 512 - lane * 8, v[t]);
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int tile = min(4 * q + i, w.tiles - 1);
#pragma unroll
            for (int m = 0; m < MATS; m++)
                a[m][i] = *reinterpret_cast<const u32x4 *>((m ? up : W) + ((size_t)group * w.tiles + tile) * kTileBytes + lane * 16);
            if constexpr (!kFloats)
#pragma unroll
                for (int n = 0; n < NT; n++)
                    b[n][i] = *reinterpret_cast<const u32x4 *>(X + ((size_t)min(t0 + n, x.groups - 1) * x.tiles + tile) * kTileBytes + lane * 16);
        }
#pragma unroll
        for (int m = 0; m < MATS; m++)
            sa[m] = *reinterpret_cast<const int *>((m ? up : W) + w.code_bytes() + ((size_t)group * w.quads + q) * kScaleBytes + lane * 4);
        if constexpr (kFloats) {
            wave_meets();
#pragma unroll
            for (int t = 0; t < FLOATS; t++)
                if (t < n_tok) {
                    const Packed p = pack8(v[t], lane & 3);
                    const int block = lane >> 2;
                    uint32_t *to = packed[wave][t];
                    to[block * 4 + dword_of(lane & 3)] = p.codes;
                    if ((lane & 3) == 0) reinterpret_cast<uint8_t *>(to + 64)[(block & 3) * 4 + (block >> 2)] = (uint8_t)p.exponent;
                }
            wave_meets();
            /* lane 16 g + t of the instruction: block g of token t (those past the last repeat it) */
            const uint32_t *from = packed[wave][min(lane & 15, n_tok - 1)];
#pragma unroll
            for (int i = 0; i < 4; i++) b[0][i] = *reinterpret_cast<const u32x4 *>(from + (4 * i + (lane >> 4)) * 4);
            sb[0] = (int)from[64 + (lane >> 4)];
        } else {
#pragma unroll
            for (int n = 0; n < NT; n++)
                sb[n] = *reinterpret_cast<const int *>(X + x.code_bytes() + ((size_t)min(t0 + n, x.groups - 1) * x.quads + q) * kScaleBytes + lane * 4);
        }
        const int tiles = w.tiles - 4 * q; /* of these four, those that are there */
        auto step = [&](auto at) {
            constexpr int i = decltype(at)::value;
            if (i < tiles) {
#pragma unroll
                for (int m = 0; m < MATS; m++)
#pragma unroll
                    for (int n = 0; n < NT; n++)
                        acc[m][n] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(widened(a[m][i]), widened(b[n][i]), acc[m][n], 4, 4, i, sa[m], i, sb[n]);
            }
        };
        step(std::integral_constant<int, 0>{});
        step(std::integral_constant<int, 1>{});
        step(std::integral_constant<int, 2>{});
        step(std::integral_constant<int, 3>{});
    }
#pragma unroll
    for (int m = 0; m < MATS; m++)
#pragma unroll
        for (int n = 0; n < NT; n++) sums[wave][m * NT + n][lane] = acc[m][n];
    __syncthreads();
    /* lane l of the result holds rows 4 (l / 16) .. + 3 of token l % 16 */
    for (int i = threadIdx.x; i < NT * 64; i += 64 * WAVES) {
        const int n = i >> 6, l = i & 63, t = (t0 + n) * 16 + (l & 15), r = group * 16 + (l >> 4) * 4;
        f32x4 s[MATS];
#pragma unroll
        for (int m = 0; m < MATS; m++) {
            s[m] = sums[0][m * NT + n][l];
#pragma unroll
            for (int v = 1; v < WAVES; v++) s[m] += sums[v][m * NT + n][l];
        }
        if constexpr (MATS == 2)
            for (int v = 0; v < 4; v++) s[0][v] = silu_mul(s[0][v], s[1][v]);
        if (t < n_tok && r < n_rows) store4(Y + (size_t)t * ldy + r, s[0], n_rows - r);
    }
}

template <int MATS, int NT, int FLOATS, class XT, class OUT> hipError_t few(const Mxfp4Product &p) {
    constexpr int kWaves = kFewThreads / 64;
    const Shape w = shape_of(p.n_rows, p.n_cols), x = shape_of(p.n_tok, p.n_cols);
    const dim3 grid((unsigned)mxfp4_launch(0, p).workgroups);
    few_kernel<MATS, NT, kWaves, FLOATS, XT, OUT><<<grid, kFewThreads, 0, p.stream>>>(p.W, p.up, static_cast<const XT *>(p.X), static_cast<OUT *>(p.Y), p.n_rows, p.n_tok, w, x,
                                                                             p.n_cols, (size_t)p.ldx, (size_t)p.ldy);
    return hipGetLastError();
}
template <int MATS, class XT, class OUT> hipError_t few_floats(const Mxfp4Product &p) {
    return p.n_tok <= 4 ? few<MATS, 1, 4, XT, OUT>(p) : few<MATS, 1, kFewFloats, XT, OUT>(p);
}
template <int MATS, class OUT> hipError_t few_tokens(const Mxfp4Product &p) {
    if (p.x_type == T_F32) return few_floats<MATS, float, OUT>(p);
    if (p.x_type == T_F16) return few_floats<MATS, _Float16, OUT>(p);
    if (p.x_type == T_BF16) return few_floats<MATS, Bf16, OUT>(p);
    const int groups = (p.n_tok + 15) / 16;
    if (groups == 1) return few<MATS, 1, 1, uint8_t, OUT>(p);
    if (groups == 2) return few<MATS, 2, 1, uint8_t, OUT>(p);
    if (groups == 3) return few<MATS, 3, 1, uint8_t, OUT>(p);
    return few<MATS, 4, 1, uint8_t, OUT>(p);
}

}  // namespace

hipError_t launch_mxfp4_few(const Mxfp4Product &p) {
    if (p.up) return p.bf16_out ? few_tokens<2, __bf16>(p) : few_tokens<2, float>(p);
    return p.bf16_out ? few_tokens<1, __bf16>(p) : few_tokens<1, float>(p);
}

/* A launch of its own to quantise costs about 2.7 us. Here a piece (512 columns of a token) costs each of the row groups about 0.07 us per
 * thousand: 14336 x 4096, 4 tokens (29 k pieces) 9.0 us against 10; 4096 x 14336, 4 tokens (29 k) 8.4 to 10.5 against 10.6; 151936 x 4096
 * (76 k per token) 1 token 58.4 against 57, 4 tokens 74 against 60. From five tokens on their registers cost workgroups in flight too. In a
 * graph, bf16: 4096 x 4096, 8 tokens (16 k) 6.1 against 7.0, gate and up of 6144 x 4096, 5 tokens (15 k) 8.2 against 8.45 and 6 tokens
 * (18 k) 8.9 against 8.5; one tensor of that size, 8 tokens (25 k) 7.5 against 7.7. With nine tokens and more (a third variant, left out) 512 x 2048
 * 5.7 against 5.4, 14336 x 4096 22 against 12. */
bool mxfp4_quantises_in_product(const Mxfp4Product &p) {
    const size_t kPieces = p.n_tok <= 4 ? 32768 : 16384;
    const Shape w = shape_of(p.n_rows, p.n_cols);
    if (p.x_type == T_MXFP4 || p.n_tok > kFewFloats || (size_t)w.groups * w.quads * p.n_tok > kPieces) return false;
    return p.x_type == T_F32 ? reads_wide<float>(p.X, p.n_cols, p.ldx) : reads_wide<Bf16>(p.X, p.n_cols, p.ldx);
}

}  // namespace qlin
