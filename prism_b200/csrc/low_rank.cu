// Low-rank adapters of many requests beside a projection that they share:  out[t] = base[t] + s_l (x[t] A_l^T) B_l^T  with l = ids[t] the
// adapter of token t's request, or out[t] = base[t] where it has none (ids[t] < 0).
//
// A projection that runs as one product over stacked matrices (q, k, v; gate, up) has its adapters' A and B per matrix: "slices", groups of
// neighbouring result columns.  a [L, G, r, Kp]: r rows of a slice's A, zeros beyond K; b [L, N, r]: the rows of all slices' B.  r is a
// multiple of 16, Kp of 8 (rows start on 16 bytes), zeros beyond an adapter's own rank.  Sums in float32, one rounding where a result is stored.
//
// Here: a few tokens at a time on CUDA cores - decoding requests, each with an adapter of its own, where every byte of A and B is used once and
// the kernel is bound by reading them, and 32-bit floats.  low_rank_tile.cu has the portions of prompts.
//
// A cluster of eight CTAs takes one token (or eight neighbours) and a range of one slice's columns: each computes an eighth of the hidden values
// over the whole K and writes them into all CTAs' shared memory, then all have the hidden vector and share the columns.  So it is one launch, no
// sum crosses CTAs, and B's first 32 KB a CTA are asked for before the hidden values are waited for.
#include "vec.cuh"

namespace prism {
namespace lowrank {

constexpr int THREADS = 256, WARPS = THREADS / 32;
constexpr int CTAS = 8;                       // of a cluster
constexpr int AHEAD = 8;                      // 16-byte loads of B in flight a thread
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

// 16 bytes of a row: E values
template <typename T> struct Chunk;
template <> struct Chunk<float> {
    static constexpr int E = 4;
    static __device__ __forceinline__ void unpack(const uint4& r, float (&v)[4]) {
        v[0] = __uint_as_float(r.x), v[1] = __uint_as_float(r.y), v[2] = __uint_as_float(r.z), v[3] = __uint_as_float(r.w);
    }
};
template <> struct Chunk<__nv_bfloat16> {
    static constexpr int E = 8;
    static __device__ __forceinline__ void unpack(const uint4& r, float (&v)[8]) {
        const uint32_t u[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) v[2 * i] = __uint_as_float(u[i] << 16), v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
};

// TT: tokens a cluster takes.  Tokens of several adapters among them are taken one adapter after the other.
template <typename T, typename O, int TT>
__global__ void __launch_bounds__(THREADS)
low_rank_kernel(const T* __restrict__ x_, long long ldx, int x_whole, const T* __restrict__ a, const T* __restrict__ b, const float* __restrict__ scale,
                const int* __restrict__ ids_, const O* __restrict__ base_, long long ldb, O* out_, long long ldo, int first_token, int tokens, int K, int Kp,
                int r, int L, Slices slices, int parts, int* err) {
    constexpr int E = Chunk<T>::E;
    __shared__ float hidden[TT][MOST_RANK];
    __shared__ float partial[WARPS][TT];
    asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");              // here: peers may write into this CTA's memory
    pdl_trigger();
    pdl_wait();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    uint32_t me;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(me));
    const int g = blockIdx.y / parts, part = blockIdx.y % parts, N = slices.first[slices.n];
    const int t0 = first_token + blockIdx.z * TT, here = min(TT, first_token + tokens - t0);
    // this CTA's columns: an eighth of its cluster's share of the slice
    const int wide = slices.first[g + 1] - slices.first[g], shares = parts * CTAS, each = (wide + shares - 1) / shares;
    const int n0 = slices.first[g] + min(wide, (part * CTAS + (int)me) * each), n1 = min(slices.first[g + 1], n0 + each);
    const T* x = pdl_fresh(x_) + (size_t)t0 * ldx;
    const O* base = base_ ? pdl_fresh(base_) + (size_t)t0 * ldb : nullptr;
    O* out = out_ + (size_t)t0 * ldo;

    int id[TT];
#pragma unroll
    for (int i = 0; i < TT; ++i) id[i] = i < here ? adapter_of(pdl_fresh(ids_), t0 + i, L, err) : -1;
#pragma unroll
    for (int i = 0; i < TT; ++i)
        if (i < here && id[i] < 0 && out_ != base_)
            for (int n = n0 + tid; n < n1; n += THREADS) out[(size_t)i * ldo + n] = base ? base[(size_t)i * ldb + n] : from_float<O>(0.f);
    bool all_here = false;

    // B's chunks: `lanes` neighbours share a row, each with the same part of every row that it meets
    const int chunks = r / E;
    int lanes = 1;
    while (lanes < chunks) lanes *= 2;
    const int chunk = lane % lanes, rows_at_once = THREADS / lanes, row0 = tid / lanes;
    const bool holds = chunk < chunks;

#pragma unroll 1
    for (int p = 0; p < TT; ++p) {
        int l = -1;
        bool mine[TT];
        {
            bool again = false;
#pragma unroll
            for (int i = 0; i < TT; ++i) {
                if (i == p) l = id[i];
            }
#pragma unroll
            for (int i = 0; i < TT; ++i) {
                mine[i] = id[i] == l;
                again |= i < p && mine[i];
            }
            if (l < 0 || again) continue;                          // the same for the whole cluster
        }
        const T* B = b + ((size_t)l * N + n0) * r + chunk * E;
        uint4 ahead[AHEAD];
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            const int n = row0 + j * rows_at_once;
            ahead[j] = holds && n < n1 - n0 ? __ldg(reinterpret_cast<const uint4*>(B + (size_t)n * r)) : make_uint4(0, 0, 0, 0);
        }
        // an eighth of the hidden values, several warps a row where there are fewer rows than warps
        const int rows = r / CTAS;
        int split = 1;
        while (split * 2 * rows <= WARPS) split *= 2;
        const int sub = warp % split;
        const T* A = a + (((size_t)l * slices.n + g) * r + me * rows) * Kp;
        for (int j0 = 0; j0 < rows; j0 += WARPS / split) {
            const int j = j0 + warp / split;
            float s[TT];
#pragma unroll
            for (int i = 0; i < TT; ++i) s[i] = 0.f;
            if (j < rows) {
                const T* row = A + (size_t)j * Kp;
#pragma unroll TT == 1 ? 8 : 2
                for (int k = (sub * 32 + lane) * E; k < K; k += split * 32 * E) {
                    float w[E];
                    Chunk<T>::unpack(__ldg(reinterpret_cast<const uint4*>(row + k)), w);
#pragma unroll
                    for (int i = 0; i < TT; ++i) {
                        if (TT > 1 && !mine[i]) continue;
                        float v[E];
                        const T* xi = x + (size_t)i * ldx + k;
                        if (x_whole && k + E <= K) {
                            Chunk<T>::unpack(*reinterpret_cast<const uint4*>(xi), v);
                        } else {
#pragma unroll
                            for (int e = 0; e < E; ++e) v[e] = k + e < K ? to_float(xi[e]) : 0.f;
                        }
#pragma unroll
                        for (int e = 0; e < E; ++e) s[i] = fmaf(v[e], w[e], s[i]);
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < TT; ++i) {
                s[i] = warp_sum(s[i]);
                if (lane == 0) partial[warp][i] = s[i];
            }
            __syncthreads();
            if (!all_here) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
            all_here = true;
            for (int task = tid; task < TT * (WARPS / split) * CTAS; task += THREADS) {          // a hidden value, for one of the CTAs
                const int c = task % CTAS, i = task / CTAS % TT, q = task / CTAS / TT;
                if (j0 + q < rows) {
                    float h = 0.f;
                    for (int w = 0; w < split; ++w) h += partial[q * split + w][i];
                    uint32_t at;
                    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;"
                                 : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(&hidden[i][me * rows + j0 + q])), "r"(c));
                    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(at), "f"(h * scale[l]) : "memory");
                }
            }
            __syncthreads();
        }
        asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
        float h[TT][E];
#pragma unroll
        for (int i = 0; i < TT; ++i)
#pragma unroll
            for (int e = 0; e < E; ++e) h[i][e] = holds ? hidden[i][chunk * E + e] : 0.f;
        for (int m = 0; m < n1 - n0; m += AHEAD * rows_at_once) {
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) {
                const int n = m + j * rows_at_once + row0;
                if (m + j * rows_at_once >= n1 - n0) break;
                float w[E];
                Chunk<T>::unpack(ahead[j], w);
                const int next = n + AHEAD * rows_at_once;
                if (holds && next < n1 - n0) ahead[j] = __ldg(reinterpret_cast<const uint4*>(B + (size_t)next * r));
#pragma unroll
                for (int i = 0; i < TT; ++i) {
                    if (TT > 1 && !mine[i]) continue;
                    float s = 0.f;
#pragma unroll
                    for (int e = 0; e < E; ++e) s = fmaf(h[i][e], w[e], s);
                    for (int o = 1; o < lanes; o <<= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
                    if (chunk == 0 && n < n1 - n0)
                        out[(size_t)i * ldo + n0 + n] = from_float<O>(base ? to_float(base[(size_t)i * ldb + n0 + n]) + s : s);
                }
            }
        }
        if (TT > 1) asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");      // `hidden` is written again
    }
    if (!all_here) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
}

template <typename T, typename O, int TT>
int launch(const void* x, long long ldx, const void* a, const void* b, const float* scale, const int* ids, const void* base, long long ldb, void* out,
           long long ldo, int first_token, int tokens, int K, int Kp, int r, int L, const Slices& s, int* err, int sms, cudaStream_t stream) {
    if (tokens <= 0) return 0;
    const int groups = (tokens + TT - 1) / TT;
    if (groups > 65535) return (int)cudaErrorInvalidValue;
    // clusters that share a slice's columns: as many as keep B's part of a CTA within what it asks for ahead, while all CTAs together are no
    // more than four an SM
    int widest = 0;
    for (int g = 0; g < s.n; ++g) widest = max(widest, s.first[g + 1] - s.first[g]);
    const long long bytes = (long long)widest * r * (int)sizeof(T), ahead = (long long)CTAS * THREADS * AHEAD * 16;
    const int parts = (int)max(1ll, min((bytes + ahead - 1) / ahead, 4ll * sms / ((long long)CTAS * s.n * groups)));
    const int whole = (reinterpret_cast<uintptr_t>(x) % 16 == 0) && (ldx * (long long)sizeof(T) % 16 == 0 || tokens + first_token == 1);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(CTAS, s.n * parts, groups);
    cfg.blockDim = dim3(THREADS);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = CTAS, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = prism::pdl_enabled() ? 2 : 1;
    return (int)cudaLaunchKernelEx(&cfg, low_rank_kernel<T, O, TT>, (const T*)x, ldx, whole, (const T*)a, (const T*)b, scale, ids, (const O*)base, ldb, (O*)out,
                                   ldo, first_token, tokens, K, Kp, r, L, s, parts, err);
}

}  // namespace lowrank
}  // namespace prism

// first: G + 1 column borders (host memory).  base may be null (nothing to add to), or out itself.  The first `singles` tokens one by one, the
// others eight at a time.
PRISM_EXPORT int prism_low_rank(const void* x, long long ldx, int dtype, const void* a, const void* b, const float* scale, const int* ids,
                                const void* base, long long ldb, void* out, long long ldo, int out_dtype, int T, int K, int Kp, int r, int L, int G,
                                const int* first, int singles, int sms, int* err, cudaStream_t stream) {
    using namespace prism::lowrank;
    typedef __nv_bfloat16 bf16;
    if (T <= 0) return 0;
    if (G < 1 || G > MOST_SLICES || r < 16 || r % 16 || r > MOST_RANK || K < 1 || Kp < K || Kp % 8 || L < 1 || singles < 0 || singles > T || sms < 1)
        return (int)cudaErrorInvalidValue;
    Slices s;
    s.n = G;
    for (int g = 0; g <= G; ++g) s.first[g] = first[g];
    for (int g = 0; g < G; ++g)
        if (s.first[g] >= s.first[g + 1]) return (int)cudaErrorInvalidValue;
#define PRISM_LOW_RANK(TX, TO, TT, at, n) launch<TX, TO, TT>(x, ldx, a, b, scale, ids, base, ldb, out, ldo, at, n, K, Kp, r, L, s, err, sms, stream)
#define PRISM_LOW_RANK_TYPES(TT, at, n)                                                                                          \
    (dtype == PRISM_DTYPE_F32 ? (out_dtype == PRISM_DTYPE_F32 ? PRISM_LOW_RANK(float, float, TT, at, n) : PRISM_LOW_RANK(float, bf16, TT, at, n)) \
                              : (out_dtype == PRISM_DTYPE_F32 ? PRISM_LOW_RANK(bf16, float, TT, at, n) : PRISM_LOW_RANK(bf16, bf16, TT, at, n)))
    const int code = PRISM_LOW_RANK_TYPES(1, 0, singles);
    return code != 0 ? code : PRISM_LOW_RANK_TYPES(8, singles, T - singles);
#undef PRISM_LOW_RANK_TYPES
#undef PRISM_LOW_RANK
}
