// Low-rank adapters of many requests beside a projection that they share:  out[t] = base[t] + s_l (x[t] A_l^T) B_l^T  with l = ids[t] the
// adapter of token t's request, or out[t] = base[t] where it has none (ids[t] < 0).
//
// A projection that runs as one product over stacked matrices (q, k, v; gate, up) has its adapters' A and B per matrix: "slices", groups of
// neighbouring result columns.  a [L, G, r, Kp]: r rows of a slice's A, zeros beyond K; b [L, N, r]: the rows of all slices' B.  r is a
// multiple of 16, Kp of 8 (rows start on 16 bytes), zeros beyond an adapter's own rank.  Sums in float32, one rounding where a result is stored.
#include "vec.cuh"

namespace prism {
namespace lowrank {

constexpr int THREADS = 256;
constexpr int MOST_RANK = 128, MOST_SLICES = 8;

struct Slices {
    int n, first[MOST_SLICES + 1];            // slice g has the result columns first[g] .. first[g + 1] - 1
};

// the adapter of a token, -1 for none; an id outside the stack is reported and taken as none
__device__ __forceinline__ int adapter_of(const int* ids, int t, int L, int* err) {
    const int l = ids[t];
    if (l >= L) {
        report_error(err, PRISM_ERR_ADAPTER_RANGE);
        return -1;
    }
    return l < 0 ? -1 : l;
}

template <typename T, typename O>
__global__ void __launch_bounds__(THREADS)
low_rank_token_kernel(const T* __restrict__ x_, long long ldx, const T* __restrict__ a, const T* __restrict__ b, const float* __restrict__ scale,
                      const int* __restrict__ ids_, const O* __restrict__ base_, long long ldb, O* __restrict__ out, long long ldo, int K, int Kp,
                      int r, int L, Slices slices, int* err) {
    __shared__ float h[MOST_RANK];
    pdl_trigger();
    pdl_wait();
    const int t = blockIdx.x, g = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, N = slices.first[slices.n];
    const int n0 = slices.first[g], n1 = slices.first[g + 1];
    const T* x = pdl_fresh(x_) + t * ldx;
    const O* base = base_ ? pdl_fresh(base_) + t * ldb : nullptr;
    const int l = adapter_of(pdl_fresh(ids_), t, L, err);
    if (l >= 0)
        for (int j = warp; j < r; j += THREADS / 32) {
            const T* row = a + (((size_t)l * slices.n + g) * r + j) * Kp;
            float s = 0.f;
            for (int k = lane; k < K; k += 32) s += to_float(x[k]) * to_float(row[k]);
            s = warp_sum(s);
            if (lane == 0) h[j] = s * scale[l];
        }
    __syncthreads();
    for (int n = n0 + threadIdx.x; n < n1; n += THREADS) {
        float s = 0.f;
        if (l >= 0) {
            const T* row = b + ((size_t)l * N + n) * r;
            for (int j = 0; j < r; ++j) s += h[j] * to_float(row[j]);
        }
        out[t * ldo + n] = from_float<O>(base ? to_float(base[n]) + s : s);
    }
}

}  // namespace lowrank
}  // namespace prism

// first: G + 1 column borders (host memory).  base may be null (nothing to add to), or out itself.
PRISM_EXPORT int prism_low_rank(const void* x, long long ldx, int dtype, const void* a, const void* b, const float* scale, const int* ids,
                                const void* base, long long ldb, void* out, long long ldo, int out_dtype, int T, int K, int Kp, int r, int L, int G,
                                const int* first, int singles, int* err, cudaStream_t stream) {
    using namespace prism::lowrank;
    typedef __nv_bfloat16 bf16;
    if (T <= 0) return 0;
    if (G < 1 || G > MOST_SLICES || r < 16 || r % 16 || r > MOST_RANK || K < 1 || Kp < K || Kp % 8 || L < 1) return (int)cudaErrorInvalidValue;
    Slices s;
    s.n = G;
    for (int g = 0; g <= G; ++g) s.first[g] = first[g];
    for (int g = 0; g < G; ++g)
        if (s.first[g] >= s.first[g + 1]) return (int)cudaErrorInvalidValue;
    const dim3 grid(T, G), block(THREADS);
#define PRISM_LOW_RANK(TX, TO)                                                                                                                    \
    (int)prism::launch_kernel(low_rank_token_kernel<TX, TO>, grid, block, 0, stream, (const TX*)x, ldx, (const TX*)a, (const TX*)b, scale, ids, \
                              (const TO*)base, ldb, (TO*)out, ldo, K, Kp, r, L, s, err)
    if (dtype == PRISM_DTYPE_F32) return out_dtype == PRISM_DTYPE_F32 ? PRISM_LOW_RANK(float, float) : PRISM_LOW_RANK(float, bf16);
    return out_dtype == PRISM_DTYPE_F32 ? PRISM_LOW_RANK(bf16, float) : PRISM_LOW_RANK(bf16, bf16);
#undef PRISM_LOW_RANK
}
