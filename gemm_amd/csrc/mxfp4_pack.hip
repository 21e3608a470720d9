/*
 * mxfp4_pack.hip - float rows to MXFP4, as GGML blocks or as an operand of the matrix instructions (mxfp4.h), and GGML blocks to
 * an operand.
 *
 * A block of 32 elements x shares the power of two 2^p that puts its largest magnitude into [4, 8): p = floor(log2 max|x|) - 2, at
 * least -127, stored as p + 127. A code is the e2m1 number (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign) nearest to x / 2^p, on a tie the
 * one with the even code, and 6 beyond 6: what v_cvt_scalef32_pk_fp4_f32 computes. Magnitudes of (6, 8) of a block's largest binade
 * so become 6; the larger power of two would halve the resolution of all others. A block that holds an infinity or a NaN gets
 * exponent 255, NaN of the E8M0 format - every product with it is NaN - and codes of magnitude 6, which the decoders of this library
 * turn into infinities.
 *
 * Four lanes share a block, 8 consecutive elements each, so that a wave reads 512 consecutive elements of a row, 16 bytes per lane
 * and load in 16-bit types. The 4 KB of codes that a workgroup makes pass LDS once: out of the lanes they would go to memory in
 * pieces of 4 bytes. Bound by memory for many rows (4096 x 14336 fp32 to blocks 48 to 59 us, 4.5 to 5.5 TB/s) and by the launch for
 * few (2048 x 4096 bf16 to an operand 6.5 us, 24 x 14336 4). Blocks of 151936 x 4096 to an operand 117 us, 5.7 TB/s (429 by single bytes).
 */
#include "mxfp4_quant.h"

namespace qlin {
using namespace mxfp4;

namespace {

/* one workgroup: a row group's 512 columns */
template <class T, bool VEC>
__global__ void __launch_bounds__(kPackThreads) operand_kernel(const T *__restrict__ X, uint8_t *__restrict__ op, int n_rows, int n_cols, size_t ldx, Shape s) {
    constexpr int kRun = 16 * 4 + 4; /* dwords from one block of a tile to the next: 16 rows, and 4 against bank conflicts */
    __shared__ __attribute__((aligned(16))) uint32_t codes[16 * kRun];
    __shared__ __attribute__((aligned(16))) uint8_t scales[kScaleBytes];
    const int group = blockIdx.x / (unsigned)s.quads, quad = blockIdx.x - group * s.quads;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int block = lane >> 2, q = lane & 3; /* of the 512 columns' 16 */
    const int col = quad * 512 + lane * 8;
    float x[4][8];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int row = group * 16 + 4 * wave + i;
        load8<T, VEC>(X + (size_t)row * ldx + col, row < n_rows ? n_cols - col : 0, x[i]);
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int r = 4 * wave + i;
        const Packed p = pack8(x[i], q);
        codes[block * kRun + r * 4 + dword_of(q)] = p.codes;
        if (q == 0) scales[((block & 3) * 16 + r) * 4 + (block >> 2)] = (uint8_t)p.exponent;
    }
    __syncthreads();
    const int tile = quad * 4 + wave;
    if (tile < s.tiles)
        *reinterpret_cast<uint4 *>(op + ((size_t)group * s.tiles + tile) * kTileBytes + lane * 16) =
            *reinterpret_cast<const uint4 *>(codes + (4 * wave + (lane >> 4)) * kRun + (lane & 15) * 4);
    if (threadIdx.x < 16)
        *reinterpret_cast<uint4 *>(op + s.code_bytes() + ((size_t)group * s.quads + quad) * kScaleBytes + threadIdx.x * 16) =
            *reinterpret_cast<const uint4 *>(scales + threadIdx.x * 16);
}

/* the same from GGML blocks: codes and exponents are moved, not changed. A lane loads a block, 16 bytes at any address: sixteen lanes read a
 * row's 272 bytes */
__global__ void __launch_bounds__(kPackThreads) operand_of_blocks_kernel(const uint8_t *__restrict__ W, uint8_t *__restrict__ op, int n_rows, int n_blocks, Shape s) {
    constexpr int kRun = 16 * 4 + 4; /* as in operand_kernel */
    __shared__ __attribute__((aligned(16))) uint32_t codes[16 * kRun];
    __shared__ __attribute__((aligned(16))) uint8_t scales[kScaleBytes];
    const int group = blockIdx.x / (unsigned)s.quads, quad = blockIdx.x - group * s.quads;
    const int r = threadIdx.x >> 4, block = threadIdx.x & 15, row = group * 16 + r, n = quad * 16 + block;
    u32x4 v = {};
    uint8_t e = 0;
    if (row < n_rows && n < n_blocks) {
        const uint8_t *b = W + ((size_t)row * n_blocks + n) * kBlockBytes;
        e = b[0];
        __builtin_memcpy(&v, b + 1, 16);
    }
    *reinterpret_cast<u32x4 *>(codes + block * kRun + r * 4) = v;
    scales[((block & 3) * 16 + r) * 4 + (block >> 2)] = e;
    __syncthreads();
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, tile = quad * 4 + wave;
    if (tile < s.tiles)
        *reinterpret_cast<uint4 *>(op + ((size_t)group * s.tiles + tile) * kTileBytes + lane * 16) =
            *reinterpret_cast<const uint4 *>(codes + (4 * wave + (lane >> 4)) * kRun + (lane & 15) * 4);
    if (threadIdx.x < 16)
        *reinterpret_cast<uint4 *>(op + s.code_bytes() + ((size_t)group * s.quads + quad) * kScaleBytes + threadIdx.x * 16) =
            *reinterpret_cast<const uint4 *>(scales + threadIdx.x * 16);
}

/* one workgroup: 256 consecutive blocks of the rows end to end, 4352 bytes of the result */
template <class T, bool VEC>
__global__ void __launch_bounds__(kPackThreads) blocks_kernel(const T *__restrict__ X, uint8_t *__restrict__ W, size_t n_blocks, int per_row, size_t ldx, bool wide) {
    constexpr int kBytes = 256 * kBlockBytes;
    __shared__ __attribute__((aligned(16))) uint8_t out[kBytes];
    const size_t first = (size_t)blockIdx.x * 256;
    const size_t row0 = first / (unsigned)per_row; /* (per_row > 0: a kernel is launched for whole blocks only) */
    const unsigned block0 = (unsigned)(first - row0 * per_row);
    const int q = threadIdx.x & 3;
    float x[4][8];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const unsigned n = block0 + 64 * i + (threadIdx.x >> 2), down = n / (unsigned)per_row;
        const size_t row = row0 + down, col = (size_t)(n - down * per_row) * kBlock + 8 * q;
        const bool there = first + 64 * i + (threadIdx.x >> 2) < n_blocks;
        load8<T, VEC>(X + (there ? row * ldx + col : 0), there ? 8 : 0, x[i]);
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        uint8_t *b = out + (64 * i + (threadIdx.x >> 2)) * kBlockBytes;
        const Packed p = pack8(x[i], q);
        if (q == 0) b[0] = (uint8_t)p.exponent;
        __builtin_memcpy(b + 1 + 4 * dword_of(q), &p.codes, 4);
    }
    __syncthreads();
    uint8_t *to = W + first * kBlockBytes;
    const int bytes = (int)min((size_t)256, n_blocks - first) * kBlockBytes;
    if (wide) {
        for (int i = threadIdx.x; i < bytes / 16; i += 256) reinterpret_cast<uint4 *>(to)[i] = reinterpret_cast<const uint4 *>(out)[i];
        const int done = bytes & ~15;
        if ((int)threadIdx.x < bytes - done) to[done + threadIdx.x] = out[done + threadIdx.x];
    } else {
        for (int i = threadIdx.x; i < bytes; i += 256) to[i] = out[i];
    }
}

template <class T> hipError_t operand_of(const void *X, void *op, int n_rows, int n_cols, int ldx, hipStream_t stream) {
    const Shape s = shape_of(n_rows, n_cols);
    const dim3 grid((unsigned)s.groups * (unsigned)s.quads);
    const T *x = static_cast<const T *>(X);
    uint8_t *o = static_cast<uint8_t *>(op);
    if (reads_wide<T>(X, n_cols, ldx)) operand_kernel<T, true><<<grid, kPackThreads, 0, stream>>>(x, o, n_rows, n_cols, (size_t)ldx, s);
    else operand_kernel<T, false><<<grid, kPackThreads, 0, stream>>>(x, o, n_rows, n_cols, (size_t)ldx, s);
    return hipGetLastError();
}

template <class T> hipError_t blocks_of(const void *X, void *W, int n_rows, int n_cols, int ldx, hipStream_t stream) {
    const int per_row = n_cols / kBlock;
    const size_t n_blocks = (size_t)n_rows * per_row;
    const dim3 grid((unsigned)((n_blocks + 255) / 256));
    const bool wide = (reinterpret_cast<uintptr_t>(W) & 15) == 0;
    const T *x = static_cast<const T *>(X);
    uint8_t *w = static_cast<uint8_t *>(W);
    if (reads_wide<T>(X, n_cols, ldx)) blocks_kernel<T, true><<<grid, kPackThreads, 0, stream>>>(x, w, n_blocks, per_row, (size_t)ldx, wide);
    else blocks_kernel<T, false><<<grid, kPackThreads, 0, stream>>>(x, w, n_blocks, per_row, (size_t)ldx, wide);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_mxfp4_operand(uint32_t type, const void *X, void *op, int n_rows, int n_cols, int ldx, hipStream_t stream) {
    if (type == T_F32) return operand_of<float>(X, op, n_rows, n_cols, ldx, stream);
    if (type == T_F16) return operand_of<_Float16>(X, op, n_rows, n_cols, ldx, stream);
    if (type == T_BF16) return operand_of<Bf16>(X, op, n_rows, n_cols, ldx, stream);
    const Shape s = shape_of(n_rows, n_cols);
    operand_of_blocks_kernel<<<dim3((unsigned)s.groups * (unsigned)s.quads), kPackThreads, 0, stream>>>(
        static_cast<const uint8_t *>(X), static_cast<uint8_t *>(op), n_rows, n_cols / kBlock, s);
    return hipGetLastError();
}

hipError_t launch_mxfp4_blocks(uint32_t type, const void *X, void *W, int n_rows, int n_cols, int ldx, hipStream_t stream) {
    if (type == T_F32) return blocks_of<float>(X, W, n_rows, n_cols, ldx, stream);
    if (type == T_F16) return blocks_of<_Float16>(X, W, n_rows, n_cols, ldx, stream);
    return blocks_of<Bf16>(X, W, n_rows, n_cols, ldx, stream);
}

}  // namespace qlin
