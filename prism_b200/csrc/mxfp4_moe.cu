// A whole mixture-of-experts layer for a few tokens, its experts' weights in microscaled 4-bit floating point (mxfp4.cuh):
//   z = x Wr^T (+ br);  scores, choice and weights as in moe_route.cuh;  h = act(g) u with g = Wg[e] a, u = Wu[e] a
//   (a = x, times the weight with scale_in);  y[t] = sum over the token's choices of Wd[e] h (times the weight without)
//
// CUDA cores, a warp per sum: the router and the choice, a CTA a token; the hidden values; the outputs.
#include "moe_route.cuh"
#include "mxfp4.cuh"

namespace prism {
namespace mx {

__device__ __forceinline__ float dot_row(const uint8_t* codes, const uint8_t* scales, int r, int K, int groups, int lane, const float* xf,
                                         const __nv_bfloat16* xb) {
    float sum = 0.f;
    for (int k = lane; k < K; k += 32) {
        const uint32_t byte = codes[(size_t)r * (groups * (GROUP / 2)) + k / 2];
        const float w = element(byte >> (4 * (k & 1)) & 15) * scale_value(scales[scale_at(r, k / BLOCK, groups)]);
        sum = fmaf(w, xb != nullptr ? __bfloat162float(xb[k]) : xf[k], sum);
    }
    return warp_sum(sum);
}

__global__ void moe_choose_kernel(const __nv_bfloat16* __restrict__ x_in, long long ldx, const void* __restrict__ router, int router_bf16,
                                  const void* __restrict__ rbias, int rbias_bf16, int H, int E, int top, int softmax, int renorm,
                                  const void* __restrict__ corr, int corr_bf16, int groups, int keep, float wscale, float sum_eps,
                                  int* __restrict__ sel_e, float* __restrict__ sel_w) {
    extern __shared__ float sh[];
    float *z = sh, *s = z + E, *c = s + E, *gs = c + E;
    int* counts = reinterpret_cast<int*>(gs + 2 * groups);
    int* rank = counts + E;
    pdl_wait();
    pdl_trigger();
    const __nv_bfloat16* x = pdl_fresh(x_in) + (long long)blockIdx.x * ldx;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int e = warp; e < E; e += blockDim.x / 32) {
        float sum = 0.f;
        for (int k = lane; k < H; k += 32) sum = fmaf(__bfloat162float(x[k]), load_param(router, router_bf16, (size_t)e * H + k), sum);
        sum = warp_sum(sum);
        if (lane == 0) {
            z[e] = sum + (rbias != nullptr ? load_param(rbias, rbias_bf16, e) : 0.f);
            counts[e] = 0;
        }
    }
    __syncthreads();
    if (warp == 0)
        moe_route_token(z, s, c, gs, E, top, softmax, renorm, lane, counts, sel_e + blockIdx.x * top, sel_w + blockIdx.x * top, rank, corr,
                        corr_bf16, groups, keep, wscale, sum_eps);
}

// hid [T top, F] float32: a warp per value
__global__ void moe_hidden_kernel(const __nv_bfloat16* __restrict__ x_in, long long ldx, const int* __restrict__ sel_e_in,
                                  const float* __restrict__ sel_w_in, const uint8_t* __restrict__ gc, const uint8_t* __restrict__ gs,
                                  const uint8_t* __restrict__ uc, const uint8_t* __restrict__ us, int F, int H, int E, int top, int scale_in,
                                  int act, float limit, float* __restrict__ hid) {
    pdl_wait();
    pdl_trigger();
    const __nv_bfloat16* x = pdl_fresh(x_in);
    const int *sel_e = pdl_fresh(sel_e_in), p = blockIdx.y, lane = threadIdx.x & 31, f = blockIdx.x * 8 + (threadIdx.x >> 5);
    if (f >= F) return;
    const float w = pdl_fresh(sel_w_in)[p];
    const int e = sel_e[p], groups = groups_of(H);
    const size_t cb = (size_t)e * F * groups * (GROUP / 2), sb = (size_t)e * ((F + 127) / 128) * groups * TILE_BYTES;
    const __nv_bfloat16* row = x + (long long)(p / top) * ldx;
    float g = dot_row(gc + cb, gs + sb, f, H, groups, lane, nullptr, row), u = dot_row(uc + cb, us + sb, f, H, groups, lane, nullptr, row);
    if (scale_in) { g *= w; u *= w; }
    const float h = moe_glu(g, u, act, limit);
    if (lane == 0) hid[(size_t)p * F + f] = scale_in ? h : h * w;
}

template <typename TO>
__global__ void moe_down_kernel(const float* __restrict__ hid_in, const int* __restrict__ sel_e_in, const uint8_t* __restrict__ dc,
                                const uint8_t* __restrict__ ds, int F, int H, int top, TO* __restrict__ y, long long ldy) {
    pdl_wait();
    pdl_trigger();
    const float* hid = pdl_fresh(hid_in);
    const int *sel_e = pdl_fresh(sel_e_in), t = blockIdx.y, lane = threadIdx.x & 31, n = blockIdx.x * 8 + (threadIdx.x >> 5);
    if (n >= H) return;
    const int groups = groups_of(F);
    float sum = 0.f;
    for (int j = 0; j < top; ++j) {
        const int e = sel_e[t * top + j];
        sum += dot_row(dc + (size_t)e * H * groups * (GROUP / 2), ds + (size_t)e * ((H + 127) / 128) * groups * TILE_BYTES, n, F, groups, lane,
                       hid + (size_t)(t * top + j) * F, nullptr);
    }
    if (lane == 0) y[(long long)t * ldy + n] = from_float<TO>(sum);
}

}  // namespace mx
}  // namespace prism

// x [T, H] bfloat16; router [E, H] (+ rbias [E]); gate, up [E, F, H] and down [E, H, F] in 4 bits; corr [E] or null.
// Scratch: sel_e int [T top], sel_w float [T top], hid float [T top, F].  y [T, H] of `out_dtype` (row stride ldy).
PRISM_EXPORT int prism_mxfp4_moe(const void* x, long long ldx, const void* router, int router_dtype, const void* rbias, int rbias_dtype,
                                 const void* gate_codes, const void* gate_scales, const void* up_codes, const void* up_scales,
                                 const void* down_codes, const void* down_scales, int T, int H, int F, int E, int top, int softmax, int renorm,
                                 int scale_in, int act, float limit, const void* corr, int corr_dtype, int groups, int keep, float wscale,
                                 float sum_eps, void* y, int out_dtype, long long ldy, int* sel_e, float* sel_w, float* hid,
                                 cudaStream_t stream) {
    using namespace prism;
    if (T <= 0) return 0;
    if (H <= 0 || F <= 0 || E <= 0 || top < 1 || top > E || (long long)T * top > 65535) return (int)cudaErrorInvalidValue;
    const __nv_bfloat16* xb = static_cast<const __nv_bfloat16*>(x);
    const size_t smem = (3 * E + 2 * groups) * 4 + (E + top) * 4;
    if (smem > 48 * 1024) return (int)cudaErrorInvalidValue;
    auto u8 = [](const void* p) { return static_cast<const uint8_t*>(p); };
    cudaError_t rc = launch_kernel(mx::moe_choose_kernel, dim3(T), dim3(256), smem, stream, xb, ldx, router, router_dtype == PRISM_DTYPE_BF16, rbias,
                                   rbias_dtype == PRISM_DTYPE_BF16, H, E, top, softmax, renorm, corr, corr_dtype == PRISM_DTYPE_BF16, groups, keep,
                                   wscale, sum_eps, sel_e, sel_w);
    if (rc != cudaSuccess) return (int)rc;
    rc = launch_kernel(mx::moe_hidden_kernel, dim3((F + 7) / 8, T * top), dim3(256), 0, stream, xb, ldx, sel_e, sel_w, u8(gate_codes),
                       u8(gate_scales), u8(up_codes), u8(up_scales), F, H, E, top, scale_in, act, limit, hid);
    if (rc != cudaSuccess) return (int)rc;
    const dim3 grid((H + 7) / 8, T);
    if (out_dtype == PRISM_DTYPE_BF16)
        return (int)launch_kernel(mx::moe_down_kernel<__nv_bfloat16>, grid, dim3(256), 0, stream, hid, sel_e, u8(down_codes), u8(down_scales), F, H,
                                  top, static_cast<__nv_bfloat16*>(y), ldy);
    return (int)launch_kernel(mx::moe_down_kernel<float>, grid, dim3(256), 0, stream, hid, sel_e, u8(down_codes), u8(down_scales), F, H, top,
                              static_cast<float*>(y), ldy);
}
