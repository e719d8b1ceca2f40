// Product of two microscaled 4-bit matrices, Y[M,N] = A[M,K] * W[N,K]^T, with the per-token and per-channel factors and
// the bias in the epilogue. No counterpart in the reference.
#include "fp4_common.cuh"
#include "trace_range.h"

namespace duq4 {
namespace fp4 {

struct GemmArgs {
    uint32_t M, N, K;
    const uint8_t *a, *a_scales, *w, *w_scales;
    const float *a_rows, *w_rows;   // factor per token / per channel, or null
    const void *bias;
    void *out;
    uint64_t ldo;
};

// y = acc * token factor * channel factor + bias, rounded once
template <class T>
__device__ __forceinline__ uint16_t finish(float acc, float ra, float rw, float b) {
    return (uint16_t)(Two<T>::down(__fmaf_rn(__fmul_rn(acc, ra), rw, b), 0.f) & 0xFFFFu);
}

// 64 x 64 outputs per CTA, 32 columns of K at a time as floats in shared memory.
template <int FMT, class T>
__global__ void __launch_bounds__(256) fp4_gemm_simt_kernel(const GemmArgs a) {
    __shared__ float sa[32][65], sw[32][65];
    const uint32_t m0 = blockIdx.y * 64, n0 = blockIdx.x * 64, tiles = scale_tiles(FMT, a.K);
    const uint32_t tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    float acc[4][4] = {};
    for (uint32_t k0 = 0; k0 < a.K; k0 += 32) {
        // 128 rows (64 of A, 64 of W), two threads each, 16 columns per thread
        const uint32_t r = threadIdx.x >> 1, half = threadIdx.x & 1, lr = r & 63;
        const bool is_w = r >= 64;
        const uint32_t row = (is_w ? n0 : m0) + lr, k = k0 + half * 16;
        float (*dst)[65] = is_w ? sw : sa;
        uint2 w = make_uint2(0, 0);
        float s = 0.f;
        if (row < (is_w ? a.N : a.M)) {
            w = *reinterpret_cast<const uint2 *>((is_w ? a.w : a.a) + (size_t)row * (a.K >> 1) + (k >> 1));
            const uint32_t blk = k / block_of(FMT);
            s = block_scale_to_float<FMT>((is_w ? a.w_scales : a.a_scales)[scale_offset(tiles, row, blk >> 2) + (blk & 3)]);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float2 f = __half22float2(e2m1x2_to_half2((j < 4 ? w.x : w.y) >> (8 * (j & 3)) & 0xFFu));
            dst[half * 16 + 2 * j][lr] = f.x * s;
            dst[half * 16 + 2 * j + 1][lr] = f.y * s;
        }
        __syncthreads();
#pragma unroll 8
        for (int kk = 0; kk < 32; ++kk) {
            float x[4], y[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) { x[i] = sa[kk][ty * 4 + i]; y[i] = sw[kk][tx * 4 + i]; }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(x[i], y[j], acc[i][j]);
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t m = m0 + ty * 4 + i, n = n0 + tx * 4 + j;
            if (m >= a.M || n >= a.N) continue;
            const float b = a.bias ? Two<T>::up1(reinterpret_cast<const uint16_t *>(a.bias)[n]) : 0.f;
            reinterpret_cast<uint16_t *>(a.out)[m * a.ldo + n] =
                finish<T>(acc[i][j], a.a_rows ? a.a_rows[m] : 1.f, a.w_rows ? a.w_rows[n] : 1.f, b);
        }
}

template <int FMT, class T>
static int gemm(const GemmArgs &a, cudaStream_t st) {
    const dim3 grid(cdiv(a.N, 64), cdiv(a.M, 64));
    if (grid.y > 65535) return DUQ4_ERR_SHAPE;
    fp4_gemm_simt_kernel<FMT, T><<<grid, 256, 0, st>>>(a);
    return launch_status();
}

static int check_gemm(int format, int dtype, uint32_t N, uint32_t K, uint64_t ldo) {
    if (format != kMX && format != kNV) return DUQ4_ERR_MODE;
    if (dtype != DUQ4_DTYPE_F16 && dtype != DUQ4_DTYPE_BF16) return DUQ4_ERR_MODE;
    if (K == 0 || K % 32 != 0 || ldo < N) return DUQ4_ERR_SHAPE;
    return DUQ4_OK;
}
static bool aligned(const void *p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

static int run(int format, int dtype, const GemmArgs &a, cudaStream_t st) {
    if (format == kMX) return dtype == DUQ4_DTYPE_F16 ? gemm<kMX, __half>(a, st) : gemm<kMX, __nv_bfloat16>(a, st);
    return dtype == DUQ4_DTYPE_F16 ? gemm<kNV, __half>(a, st) : gemm<kNV, __nv_bfloat16>(a, st);
}

static size_t up256(size_t v) { return (v + 255) / 256 * 256; }

}  // namespace fp4
}  // namespace duq4

using namespace duq4;
using namespace duq4::fp4;

extern "C" {

int duq4_linear_fp4(int format, const uint8_t *A, const uint8_t *A_block_scales, const float *A_row_scales, const uint8_t *W,
                    const uint8_t *W_block_scales, const float *W_row_scales, uint32_t M, uint32_t N, uint32_t K, const void *bias, int dtype,
                    void *out, uint64_t ldo, void *stream) {
    DUQ4_TRACE();
    if (ldo == 0) ldo = N;
    int rc = check_gemm(format, dtype, N, K, ldo);
    if (rc) return rc;
    if (M == 0 || N == 0) return DUQ4_OK;
    if (!A || !A_block_scales || !W || !W_block_scales || !out) return DUQ4_ERR_NULL;
    if (!aligned(A, 16) || !aligned(A_block_scales, 16) || !aligned(W, 16) || !aligned(W_block_scales, 16) || !aligned(A_row_scales, 4) ||
        !aligned(W_row_scales, 4) || !aligned(bias, 2) || !aligned(out, 2))
        return DUQ4_ERR_ALIGN;
    const GemmArgs a{M, N, K, A, A_block_scales, W, W_block_scales, A_row_scales, W_row_scales, bias, out, ldo};
    return run(format, dtype, a, (cudaStream_t)stream);
}

size_t duq4_linear_fp4_workspace_bytes(int format, uint32_t M, uint32_t K) {
    return up256((size_t)M * (K / 2)) + up256(duq4_fp4_scale_bytes(format, M, K)) + up256((size_t)M * 4);
}

int duq4_linear_fp4_from_16bit(int format, int dtype, const void *x, const uint8_t *W, const uint8_t *W_block_scales,
                               const float *W_row_scales, uint32_t M, uint32_t N, uint32_t K, const void *bias, void *out, uint64_t ldo,
                               void *workspace, size_t workspace_bytes, void *stream) {
    DUQ4_TRACE();
    if (ldo == 0) ldo = N;
    int rc = check_gemm(format, dtype, N, K, ldo);
    if (rc) return rc;
    if (M == 0 || N == 0) return DUQ4_OK;
    if (!x || !W || !W_block_scales || !out) return DUQ4_ERR_NULL;
    if (!workspace || !aligned(workspace, 256) || workspace_bytes < duq4_linear_fp4_workspace_bytes(format, M, K)) return DUQ4_ERR_WORKSPACE;
    uint8_t *codes = (uint8_t *)workspace, *scales = codes + up256((size_t)M * (K / 2));
    float *rows = format == kNV ? (float *)(scales + up256(duq4_fp4_scale_bytes(format, M, K))) : nullptr;
    rc = duq4_fp4_quantize(format, dtype, x, M, K, K, codes, scales, rows, stream);
    if (rc) return rc;
    return duq4_linear_fp4(format, codes, scales, rows, W, W_block_scales, W_row_scales, M, N, K, bias, dtype, out, ldo, stream);
}

}  // extern "C"
