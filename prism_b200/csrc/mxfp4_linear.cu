// y [M, N] = x [M, K] W [N, K]^T (+ bias) with W in microscaled 4-bit floating point (mxfp4.cuh), x in bfloat16 as it is or
// brought to 4 bits first (a block of 32 along a row at a time, as W was).
//
// CUDA cores: a CTA takes 64 rows of W and 32 of x, and walks K by blocks of 32, whose values both sides leave in shared
// memory in float32; a thread has 4 x 2 sums.
#include "mxfp4.cuh"

namespace prism {
namespace mx {

constexpr int TN = 64, TM = 32;

template <typename TO>
__global__ void __launch_bounds__(256) linear_kernel(const __nv_bfloat16* __restrict__ x_in, long long ldx, const uint8_t* __restrict__ codes,
                                                     const uint8_t* __restrict__ scales, const void* __restrict__ bias, int bias_bf16,
                                                     TO* __restrict__ y, long long ldy, int M, int N, int K, int groups, int four) {
    __shared__ float ws[TN][BLOCK + 1], xs[TM][BLOCK + 1];
    pdl_wait();
    pdl_trigger();
    const __nv_bfloat16* x = pdl_fresh(x_in);
    const int n0 = blockIdx.x * TN, m0 = blockIdx.y * TM, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int tn = threadIdx.x & 15, tm = threadIdx.x >> 4;
    float acc[4][2] = {};
    for (int b = 0; b * BLOCK < K; ++b) {
        __syncthreads();
        const int k = b * BLOCK + lane;
        for (int i = warp; i < TN; i += 8) {
            const int n = n0 + i;
            float v = 0.f;
            if (n < N) {
                const uint32_t byte = codes[(size_t)n * (groups * (GROUP / 2)) + k / 2];
                v = element(byte >> (4 * (k & 1)) & 15) * scale_value(scales[scale_at(n, b, groups)]);
            }
            ws[i][lane] = v;
        }
        for (int i = warp; i < TM; i += 8) {
            float v = m0 + i < M && k < K ? __bfloat162float(x[(long long)(m0 + i) * ldx + k]) : 0.f;
            if (four) {
                const int byte = scale_byte(__reduce_max_sync(0xffffffffu, __float_as_uint(v) & 0x7fffffffu));
                v = byte == 255 ? scale_value(255) : element(pack2(v * scale_inverse(byte), 0.f)) * scale_value(byte);
            } else if (!isfinite(v)) {
                v = scale_value(255);
            }
            xs[i][lane] = v;
        }
        __syncthreads();
#pragma unroll 8
        for (int j = 0; j < BLOCK; ++j) {
            const float a0 = xs[tm][j], a1 = xs[tm + 16][j];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float w = ws[tn + 16 * i][j];
                acc[i][0] = fmaf(a0, w, acc[i][0]);
                acc[i][1] = fmaf(a1, w, acc[i][1]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int n = n0 + tn + 16 * i, m = m0 + tm + 16 * h;
            if (n < N && m < M) y[(long long)m * ldy + n] = from_float<TO>(acc[i][h] + (bias != nullptr ? load_param(bias, bias_bf16, n) : 0.f));
        }
}

}  // namespace mx
}  // namespace prism

// x [M, K] bfloat16 (row stride ldx); codes, scales: W [N, K]; y [M, N] of `out_dtype` (row stride ldy); act_bits 16 or 4
PRISM_EXPORT int prism_mxfp4_linear(const void* x, long long ldx, const void* codes, const void* scales, const void* bias, int bias_dtype,
                                    void* y, int out_dtype, long long ldy, int M, int N, int K, int act_bits, cudaStream_t stream) {
    using namespace prism;
    if (M <= 0 || N <= 0) return 0;
    if (K <= 0 || (act_bits != 16 && act_bits != 4) || ((uintptr_t)codes & 31)) return (int)cudaErrorInvalidValue;
    const dim3 grid((N + mx::TN - 1) / mx::TN, (M + mx::TM - 1) / mx::TM), block(256);
    const uint8_t *c = static_cast<const uint8_t*>(codes), *s = static_cast<const uint8_t*>(scales);
    const __nv_bfloat16* xb = static_cast<const __nv_bfloat16*>(x);
    const int groups = mx::groups_of(K), bb = bias_dtype == PRISM_DTYPE_BF16, four = act_bits == 4;
    if (out_dtype == PRISM_DTYPE_BF16)
        return (int)launch_kernel(mx::linear_kernel<__nv_bfloat16>, grid, block, 0, stream, xb, ldx, c, s, bias, bb,
                                  static_cast<__nv_bfloat16*>(y), ldy, M, N, K, groups, four);
    return (int)launch_kernel(mx::linear_kernel<float>, grid, block, 0, stream, xb, ldx, c, s, bias, bb, static_cast<float*>(y), ldy, M, N, K,
                              groups, four);
}
