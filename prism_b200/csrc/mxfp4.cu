// Rows to microscaled 4-bit floating point and back (mxfp4.cuh has the format).
//
// Bound by memory: 2 or 4 bytes read and 17/32 written an element, and back.  A CTA has one tile of scales, 128 rows by 128
// columns: 16 threads share a row's 256 bytes (bfloat16), each with 8 values in one or two wide loads; all of a thread's rows
// are asked for before the first is worked on.  Four neighbours share a block of 32: its largest magnitude goes round by two
// shuffles, each stores its 8 codes as one word, and the tile's 512 scale bytes leave together through shared memory.
// 37,888 x 3,584 in bfloat16: to 4 bits in 61 us (5.6 TB/s), back in 54 (6.3 TB/s), 0.86 and 0.97 of the rate at which the device
// copies; a row at a time a thread, each load waited for, both took 190 us together.  Rows whose length is no multiple of eight are
// put side by side in shared memory before they are stored: 20,000 x 1,003 back 59 -> 17 us.
#include "mxfp4.cuh"
#include "vec.cuh"

namespace prism {
namespace mx {

constexpr int THREADS = 256, AT_ONCE = 8, ROWS = THREADS / 16;      // rows of a round of the CTA

__device__ __forceinline__ int scale_place(int r) { return (r & 31) * 16 + r / 32 * 4; }       // of row r of a tile, block 0

template <typename T> struct alignas(16) Eight { T v[8]; };

// x: a stack of matrices [rows, K] (row stride ld); grid (groups, tiles of rows, matrices)
template <typename T>
__global__ void __launch_bounds__(THREADS) quantise_kernel(const T* __restrict__ x_in, long long ld, int rows, int K, int groups, int wide,
                                                           uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
    __shared__ __align__(16) uint8_t sc[TILE_BYTES];
    pdl_wait();
    pdl_trigger();
    const int g = blockIdx.x, r0 = blockIdx.y * TILE_ROWS, c = (threadIdx.x & 15) * 8, k = g * GROUP + c, first = threadIdx.x >> 4;
    const size_t row0 = (size_t)blockIdx.z * rows + r0;
    const T* x = pdl_fresh(x_in) + (long long)row0 * ld + k;
    uint8_t* code = codes + row0 * (groups * (size_t)(GROUP / 2)) + k / 2;
    const int here = min(TILE_ROWS, rows - r0);
    auto finish = [&](const float (&v)[8], int r) {
        uint32_t most = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) most = max(most, __float_as_uint(v[j]) & 0x7fffffffu);
        most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
        const int byte = scale_byte(most);
        const float inv = scale_inverse(byte);
        uint32_t word = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) word |= pack2(v[2 * j] * inv, v[2 * j + 1] * inv) << (8 * j);
        if (r < here) {
            *reinterpret_cast<uint32_t*>(code + (size_t)r * (groups * (GROUP / 2))) = byte == 255 ? 0 : word;
            if ((threadIdx.x & 3) == 0) sc[scale_place(r) + c / BLOCK] = (uint8_t)byte;
        }
    };
    if (wide && here == TILE_ROWS && (g + 1) * GROUP <= K) {               // a whole tile: all of a thread's loads, then its work
        Eight<T> raw[AT_ONCE];
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) raw[i] = *reinterpret_cast<const Eight<T>*>(x + (long long)(i * ROWS + first) * ld);
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
            float v[8];
            load8(reinterpret_cast<const T*>(&raw[i]), v);
            finish(v, i * ROWS + first);
        }
    } else {
#pragma unroll 1
        for (int r = first; r < ROWS * ((here + ROWS - 1) / ROWS); r += ROWS) {          // whole warps go round together
            const T* p = x + (long long)r * ld;
            float v[8];
            if (wide && r < here && k + 8 <= K) {
                load8(p, v);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = r < here && k + j < K ? to_float(p[j]) : 0.f;
            }
            finish(v, r);
        }
    }
    __syncthreads();
    if (threadIdx.x < 32)
        reinterpret_cast<uint4*>(scales + (((size_t)blockIdx.z * gridDim.y + blockIdx.y) * groups + g) * TILE_BYTES)[threadIdx.x] =
            reinterpret_cast<const uint4*>(sc)[threadIdx.x];
}

template <typename T>
__global__ void __launch_bounds__(THREADS) dequantise_kernel(const uint8_t* __restrict__ codes_in, const uint8_t* __restrict__ scales_in, int rows,
                                                             int K, int groups, T* __restrict__ out, long long ldm) {
    __shared__ __align__(16) uint8_t sc[TILE_BYTES];
    pdl_wait();
    pdl_trigger();
    const int g = blockIdx.x, r0 = blockIdx.y * TILE_ROWS, c = (threadIdx.x & 15) * 8, k = g * GROUP + c, first = threadIdx.x >> 4;
    const size_t row0 = (size_t)blockIdx.z * rows + r0;
    const uint8_t* code = pdl_fresh(codes_in) + row0 * (groups * (size_t)(GROUP / 2)) + k / 2;
    out += blockIdx.z * ldm + (long long)r0 * K;
    const int here = min(TILE_ROWS, rows - r0);
    uint32_t word[AT_ONCE];
    static_assert(ROWS * AT_ONCE == TILE_ROWS, "one round");
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) {
        const int r = i * ROWS + first;
        word[i] = r < here ? *reinterpret_cast<const uint32_t*>(code + (size_t)r * (groups * (GROUP / 2))) : 0;
    }
    if (threadIdx.x < 32)
        reinterpret_cast<uint4*>(sc)[threadIdx.x] =
            reinterpret_cast<const uint4*>(pdl_fresh(scales_in) + (((size_t)blockIdx.z * gridDim.y + blockIdx.y) * groups + g) * TILE_BYTES)[threadIdx.x];
    __syncthreads();
    __shared__ T line[THREADS / 32][2][GROUP];                           // rows that no wide store fits go out element by element, side by side
    T(*mine)[GROUP] = line[threadIdx.x / 32];
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) {
        const int r = i * ROWS + first;
        if (i * ROWS >= here) break;
        const float s = r < here ? scale_value(sc[scale_place(r) + c / BLOCK]) : 0.f;
        float v[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 e = elements2(word[i] >> (8 * j));
            v[2 * j] = e.x * s;
            v[2 * j + 1] = e.y * s;
        }
        if (K % 8 == 0) {
            if (r < here && k < K) store8(out + (size_t)r * K + k, v);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) mine[lane / 16][c + j] = from_float<T>(v[j]);
            __syncwarp();
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int at = lane + 32 * (j & 3), row = r - lane / 16 + j / 4;
                if (row < here && g * GROUP + at < K) out[(size_t)row * K + g * GROUP + at] = mine[j / 4][at];
            }
            __syncwarp();
        }
    }
}

}  // namespace mx
}  // namespace prism

// x: a stack of `matrices` [rows, K] of `dtype` (row stride ldx elements) -> codes [..., rows, Kp / 2], scales
PRISM_EXPORT int prism_mxfp4_quantize(const void* x, int dtype, long long ldx, int matrices, int rows, int K, void* codes, void* scales,
                                      cudaStream_t stream) {
    using namespace prism;
    if (matrices <= 0 || rows <= 0 || K <= 0) return 0;
    const int groups = mx::groups_of(K), bf = dtype == PRISM_DTYPE_BF16, tiles = (rows + mx::TILE_ROWS - 1) / mx::TILE_ROWS;
    if (matrices > 65535 || tiles > 65535 || (((uintptr_t)codes | (uintptr_t)scales) & 15)) return (int)cudaErrorInvalidValue;
    const int wide = ((uintptr_t)x & 15) == 0 && ldx % (bf ? 8 : 4) == 0;
    const dim3 grid(groups, tiles, matrices), block(mx::THREADS);
    uint8_t *c = static_cast<uint8_t*>(codes), *s = static_cast<uint8_t*>(scales);
    if (bf)
        return (int)launch_kernel(mx::quantise_kernel<__nv_bfloat16>, grid, block, 0, stream, static_cast<const __nv_bfloat16*>(x), ldx, rows, K,
                                  groups, wide, c, s);
    return (int)launch_kernel(mx::quantise_kernel<float>, grid, block, 0, stream, static_cast<const float*>(x), ldx, rows, K, groups, wide, c, s);
}

// the values: out, a matrix [rows, K] of `dtype` every ldm elements
PRISM_EXPORT int prism_mxfp4_dequantize(const void* codes, const void* scales, int matrices, int rows, int K, void* out, long long ldm, int dtype,
                                        cudaStream_t stream) {
    using namespace prism;
    if (matrices <= 0 || rows <= 0 || K <= 0) return 0;
    const int groups = mx::groups_of(K), tiles = (rows + mx::TILE_ROWS - 1) / mx::TILE_ROWS;
    if (matrices > 65535 || tiles > 65535 || (((uintptr_t)codes | (uintptr_t)scales) & 15)) return (int)cudaErrorInvalidValue;
    if (K % 8 == 0 && ((uintptr_t)out & 15 || (matrices > 1 && ldm % 8))) return (int)cudaErrorInvalidValue;
    const dim3 grid(groups, tiles, matrices), block(mx::THREADS);
    const uint8_t *c = static_cast<const uint8_t*>(codes), *s = static_cast<const uint8_t*>(scales);
    if (dtype == PRISM_DTYPE_BF16)
        return (int)launch_kernel(mx::dequantise_kernel<__nv_bfloat16>, grid, block, 0, stream, c, s, rows, K, groups, static_cast<__nv_bfloat16*>(out),
                                  ldm);
    return (int)launch_kernel(mx::dequantise_kernel<float>, grid, block, 0, stream, c, s, rows, K, groups, static_cast<float*>(out), ldm);
}
