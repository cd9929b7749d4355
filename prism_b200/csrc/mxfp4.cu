// Rows to microscaled 4-bit floating point and back (mxfp4.cuh has the format).
//
// Bound by memory: 2 or 4 bytes read and 17/32 written an element, and back.  Four neighbouring threads share a block of 32:
// each takes 8 values in one or two wide loads, the largest magnitude goes round by two shuffles, and each stores its 8 codes
// as one word; a warp reads 512 consecutive bytes of a bfloat16 row and writes 128.
#include "mxfp4.cuh"
#include "vec.cuh"

namespace prism {
namespace mx {

// x [rows, K] (row stride ld); rows_each: rows of one matrix of a stack, whose scales start at a tile of their own
template <typename T>
__global__ void quantise_kernel(const T* __restrict__ x_in, long long ld, int rows, int rows_each, int K, int groups, int wide,
                                uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
    pdl_wait();
    pdl_trigger();
    const T* x = pdl_fresh(x_in);
    const int per_row = groups * (GROUP / 8);
    const long long total = (long long)rows * per_row;
    const size_t tiles_each = (size_t)((rows_each + TILE_ROWS - 1) / TILE_ROWS) * groups * TILE_BYTES;
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (long long)gridDim.x * blockDim.x) {
        // total is a multiple of 16 and threads of a block's four are neighbours: all four are here or none
        const int r = (int)(i / per_row), c = (int)(i - (long long)r * per_row) * 8;
        const T* p = x + (long long)r * ld + c;
        float v[8];
        if (wide && c + 8 <= K) {
            load8(p, v);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = c + j < K ? to_float(p[j]) : 0.f;
        }
        uint32_t most = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) most = max(most, __float_as_uint(v[j]) & 0x7fffffffu);
        const uint32_t four = 0xfu << (threadIdx.x & 28);
        most = max(most, __shfl_xor_sync(four, most, 1));
        most = max(most, __shfl_xor_sync(four, most, 2));
        const int byte = scale_byte(most);
        const float inv = byte == 255 ? 0.f : scale_inverse(byte);
        uint32_t word = 0;
        if (byte != 255)
#pragma unroll
            for (int j = 0; j < 4; ++j) word |= pack2(v[2 * j] * inv, v[2 * j + 1] * inv) << (8 * j);
        *reinterpret_cast<uint32_t*>(codes + (size_t)r * (groups * (GROUP / 2)) + c / 2) = word;
        if ((threadIdx.x & 3) == 0) {
            const int m = r / rows_each;
            scales[m * tiles_each + scale_at(r - m * rows_each, c / BLOCK, groups)] = (uint8_t)byte;
        }
    }
}

template <typename T>
__global__ void dequantise_kernel(const uint8_t* __restrict__ codes_in, const uint8_t* __restrict__ scales_in, int rows, int rows_each,
                                  int K, int groups, T* __restrict__ out) {
    pdl_wait();
    pdl_trigger();
    const uint8_t *codes = pdl_fresh(codes_in), *scales = pdl_fresh(scales_in);
    const int per_row = (K + 7) / 8;
    const long long total = (long long)rows * per_row;
    const size_t tiles_each = (size_t)((rows_each + TILE_ROWS - 1) / TILE_ROWS) * groups * TILE_BYTES;
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (long long)gridDim.x * blockDim.x) {
        const int r = (int)(i / per_row), c = (int)(i - (long long)r * per_row) * 8;
        const uint32_t word = *reinterpret_cast<const uint32_t*>(codes + (size_t)r * (groups * (GROUP / 2)) + c / 2);
        const int m = r / rows_each;
        const float s = scale_value(scales[m * tiles_each + scale_at(r - m * rows_each, c / BLOCK, groups)]);
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = element(word >> (4 * j) & 15) * s;
        T* o = out + (long long)r * K + c;
        if (K % 8 == 0) {
            store8(o, v);
        } else {
            for (int j = 0; j < 8 && c + j < K; ++j) o[j] = from_float<T>(v[j]);
        }
    }
}

inline int blocks_for(long long threads) {
    const long long b = (threads + 255) / 256;
    return (int)(b < 148 * 8 ? b : 148 * 8);
}

}  // namespace mx
}  // namespace prism

// x [rows, K] of `dtype` (row stride ldx elements) -> codes [rows, Kp / 2], scales; rows: a stack of matrices of rows_each rows
PRISM_EXPORT int prism_mxfp4_quantize(const void* x, int dtype, long long ldx, int rows, int rows_each, int K, void* codes, void* scales,
                                      cudaStream_t stream) {
    using namespace prism;
    if (rows <= 0 || K <= 0) return 0;
    if (rows_each <= 0 || rows % rows_each || ((uintptr_t)codes & 15)) return (int)cudaErrorInvalidValue;
    const int groups = mx::groups_of(K), bf = dtype == PRISM_DTYPE_BF16;
    const int wide = ((uintptr_t)x & 15) == 0 && ldx % (bf ? 8 : 4) == 0;
    const dim3 grid(mx::blocks_for((long long)rows * groups * 16)), block(256);
    uint8_t *c = static_cast<uint8_t*>(codes), *s = static_cast<uint8_t*>(scales);
    if (bf)
        return (int)launch_kernel(mx::quantise_kernel<__nv_bfloat16>, grid, block, 0, stream, static_cast<const __nv_bfloat16*>(x), ldx, rows,
                                  rows_each, K, groups, wide, c, s);
    return (int)launch_kernel(mx::quantise_kernel<float>, grid, block, 0, stream, static_cast<const float*>(x), ldx, rows, rows_each, K, groups,
                              wide, c, s);
}

// the values: out [rows, K] of `dtype`, contiguous, 16-byte aligned
PRISM_EXPORT int prism_mxfp4_dequantize(const void* codes, const void* scales, int rows, int rows_each, int K, void* out, int dtype,
                                        cudaStream_t stream) {
    using namespace prism;
    if (rows <= 0 || K <= 0) return 0;
    if (rows_each <= 0 || rows % rows_each || ((uintptr_t)codes & 15) || ((uintptr_t)out & 15)) return (int)cudaErrorInvalidValue;
    const int groups = mx::groups_of(K);
    const dim3 grid(mx::blocks_for((long long)rows * ((K + 7) / 8))), block(256);
    const uint8_t *c = static_cast<const uint8_t*>(codes), *s = static_cast<const uint8_t*>(scales);
    if (dtype == PRISM_DTYPE_BF16)
        return (int)launch_kernel(mx::dequantise_kernel<__nv_bfloat16>, grid, block, 0, stream, c, s, rows, rows_each, K, groups,
                                  static_cast<__nv_bfloat16*>(out));
    return (int)launch_kernel(mx::dequantise_kernel<float>, grid, block, 0, stream, c, s, rows, rows_each, K, groups, static_cast<float*>(out));
}
