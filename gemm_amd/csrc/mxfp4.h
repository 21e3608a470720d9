/*
 * mxfp4.h - rows of microscaled 4-bit numbers (MXFP4: 32 e2m1 codes that share a power of two) as operands of the scaled
 * matrix instructions, and what the kernels on them share (mxfp4_pack.hip makes operands, mxfp4_few.hip and mxfp4_tile.hip
 * multiply them).
 *
 * The operand of n_rows rows of n_cols elements. Rows go in groups of 16, columns in tiles of 128; what is missing from the
 * last group and tile holds zeros.
 *   codes   [row group][column tile] 1 KB each: 16 bytes (one block of 32 codes) per lane of v_mfma_scale_f32_16x16x128_f8f6f4,
 *           lane 16 g + r the block g of row r. Inside a block the codes lie as in a GGML block, elements j and j + 16 in byte j:
 *           the products of a block are summed, so any order serves that both factors share, and laying out a GGML tensor moves
 *           blocks without touching a code.
 *   scales  behind the codes, [row group][four column tiles] 256 bytes each: byte b of lane 16 g + r's dword is the exponent of
 *           block g of row r in column tile 4 q + b. A matrix instruction takes one byte of a register as its lane's exponent, so
 *           one load serves four of them.
 * Every load of an operand is then 16 (4) consecutive bytes per lane, 1 KB (256 bytes) per wave. A lane of the 32x32x64 instruction finds
 * its block in the same tiles (two row groups, two of the four blocks): from LDS the codes come without bank conflicts, while the
 * exponents of the second row group, 256 bytes on, are in the first's banks, two cycles more a read (516096 in 14336 x 4096 x 2048 tokens,
 * all compute units together, beside 4.8 million that LDS is busy).
 */
#ifndef QLIN_MXFP4_H
#define QLIN_MXFP4_H

#include <type_traits>

#include "qlin_internal.h"

namespace qlin {
namespace mxfp4 {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kGroupRows = 16, kTileCols = 128, kTileBytes = 1024, kScaleBytes = 256;
constexpr int kBlock = 32, kBlockBytes = 17; /* of the GGML format: [exponent][16 bytes of codes] */
constexpr int kPackThreads = 256, kFewThreads = 512, kTileThreads = 256; /* of a workgroup that makes operands or blocks, of those that multiply */

/* where an operand's parts lie */
struct Shape {
    int groups, tiles, quads; /* groups of 16 rows; tiles of 128 columns; scale dwords per row and block: ceil(tiles / 4) */
    __host__ __device__ size_t code_bytes() const { return (size_t)groups * tiles * kTileBytes; }
    __host__ __device__ size_t bytes() const { return code_bytes() + (size_t)groups * quads * kScaleBytes; }
};
__host__ __device__ inline Shape shape_of(int n_rows, int n_cols) {
    const int tiles = n_cols / kTileCols + (n_cols % kTileCols != 0);
    return {n_rows / kGroupRows + (n_rows % kGroupRows != 0), tiles, tiles / 4 + (tiles % 4 != 0)};
}

/* four codes are four of the instruction's eight operand registers (format 4 = e2m1) */
__device__ __forceinline__ i32x8 widened(u32x4 v) { return i32x8{(int)v[0], (int)v[1], (int)v[2], (int)v[3], 0, 0, 0, 0}; }

/* silu(gate) * up, silu(g) = g / (1 + exp(-g)), in 13 instructions (with expf and a division 25, which is 6 us for the 64 results per
 * lane of a tile of 256 x 256). exp(-g) = 2^t (1 + lo ln 2), t = -g log2 e rounded and lo what the rounding left, so that the error of
 * t, up to 2^-18 for large |g|, does not become a relative one of the exponential; the rest is v_exp_f32 and v_rcp_f32 of one unit in
 * the last place each. Beyond +-200 the exponential is infinite or lost against 1 either way, and t stays finite. */
__device__ __forceinline__ float silu_mul(float gate, float up) {
    constexpr float kLog2e = 1.44269504088896341f, kLog2eRest = 1.92596299e-8f; /* log2 e as a sum of two floats */
    const float g = -fminf(fmaxf(gate, -200.0f), 200.0f);
    const float t = g * kLog2e;
    const float lo = fmaf(g, kLog2eRest, fmaf(g, kLog2e, -t));
    const float e = __builtin_amdgcn_exp2f(t);
    const float sum = fmaf(fminf(e, 3e38f), lo * 0.693147181f, 1.0f + e); /* (an infinite e stays the infinity) */
    return gate * __builtin_amdgcn_rcpf(sum) * up;
}

}  // namespace mxfp4

/* rows of X (F32, F16, BF16: quantised; MXFP4: GGML blocks, n_cols a multiple of 32 and ldx ignored) as an operand */
hipError_t launch_mxfp4_operand(uint32_t type, const void *X, void *op, int n_rows, int n_cols, int ldx, hipStream_t stream);
/* float rows to GGML blocks, n_cols a multiple of 32 */
hipError_t launch_mxfp4_blocks(uint32_t type, const void *X, void *W, int n_rows, int n_cols, int ldx, hipStream_t stream);

/* Y[t * ldy + r] = sum over k of X[t][k] W[r][k], or with `up` silu(X . W) * (X . up); W and up operands, X an operand (x_type MXFP4) or
 * floats where mxfp4_quantises_in_product; Y F32 or BF16 */
struct Mxfp4Product {
    const uint8_t *W, *up;
    uint32_t x_type;
    const void *X;
    void *Y;
    int n_rows, n_cols, n_tok, ldx, ldy;
    bool bf16_out;
    hipStream_t stream;
};
bool mxfp4_quantises_in_product(const Mxfp4Product &p);
hipError_t launch_mxfp4_few(const Mxfp4Product &p);
/* in tiles of 64 mb rows (32 mb of each of two tensors) x 64 nb tokens; (mb, nb) = (4, 4), (2, 2), (2, 1), (1, 1) */
hipError_t launch_mxfp4_tiles(int mb, int nb, const Mxfp4Product &p);
/* the kernel for a product: 0 = launch_mxfp4_few, 10 mb + nb = tiles */
int mxfp4_choice(const Mxfp4Product &p, int n_cu);
/* what its launch consists of */
struct Mxfp4Launch { size_t workgroups, threads; };
Mxfp4Launch mxfp4_launch(int kernel, const Mxfp4Product &p);
hipError_t launch_mxfp4_product(const Mxfp4Product &p, int n_cu);

}  // namespace qlin
#endif
