// Low-rank adapters of many requests beside a projection that they share:  out[t] = base[t] + s_l (x[t] A_l^T) B_l^T  with l = ids[t] the
// adapter of token t's request, or out[t] = base[t] where it has none (ids[t] < 0).
//
// A projection that runs as one product over stacked matrices (q, k, v; gate, up) has its adapters' A and B per matrix: "slices", groups of
// neighbouring result columns.  a [L, G, r, Kp]: r rows of a slice's A, zeros beyond K; b [L, N, r]: the rows of all slices' B.  r is a
// multiple of 16, Kp of 8 (rows start on 16 bytes).  ranks [L, G]: so many rows of a slice's A, and columns of its B, are the adapter's own, the others
// zeros; a hidden value beyond them is 0 whatever x is (infinity times a zero that only fills up room would be NaN).  Sums in float32, one
// rounding where a result is stored.
//
// Here, on CUDA cores: decoding requests, each with an adapter of its own, where every byte of A and B is used once and the kernel is bound by
// reading them; and portions of prompts in 32-bit floats, or of sizes that TMA does not take.  low_rank_tile.cu has the portions on tensor cores.
//
// Decoding: a cluster of up to eight CTAs takes one token and a range of one slice's columns; each computes its share of the hidden values over the whole K
// and writes them into all CTAs' shared memory, then all have the hidden vector and share the columns.  So it is one launch, no sum crosses
// CTAs, and B's first 16 or 32 KB a CTA and the results that they are added to are asked for before the hidden values are waited for.  A thread has two
// 16-byte chunks of a row of B: with one each, and four rows ahead, registers were spilled and an instruction in two was not arithmetic (64 tokens, gate and up
// of the 7B shape, rank 16: 40 us, so 32; without registers in memory 23, 4.1 TB/s).  One token there takes 4.3 us, four of them launch, first loads and two barriers of the cluster.
//
// Portions: 32 tokens at a time, hidden values (a cluster shares K, its sums meet through distributed shared memory) and results in a launch
// each.  A tile's tokens may have several adapters: it is gone through once for each of them.  512 tokens of one adapter, gate and up of the 7B shape, rank 16, in
// float32: 173 us, of two 176; one by one 207.  Reading and writing the shared result takes 24 of them, the rest are loads of single values from shared memory.
#include "vec.cuh"

namespace prism {
namespace lowrank {

constexpr int CTAS = 8;                       // of a cluster that shares K, and of one token's at most
constexpr int AHEAD = 2, EACH = 2;            // rows of B in flight a thread, and its 16-byte chunks of each
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

// four bytes of memory into shared memory, through no register
__device__ __forceinline__ void async_word(void* to, const void* from) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from) : "memory");
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

__device__ __forceinline__ void cluster_barrier() { asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t peer(const void* p, int cta) {
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(cta));
    return at;
}
__device__ __forceinline__ uint32_t rank_in_cluster() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}

// ---- one token ----------------------------------------------------------------------------------------------

// Forms of it, by the clusters of a launch, as a cluster's CTAs are neighbours and so many run at a time.  512 threads and an SM's registers, eight loads of A in
// flight a thread: 15 clusters on 148 SMs.  512 threads and half of them, where a CTA has much of A: 33.  Else 256 threads, three or four CTAs an SM, in clusters of eight,
// four and two: the fewest CTAs an SM that run at a time.  With four an SM registers are short: of a thread's 44 bytes go through memory, 56 with float32 results, 20
// with float32 adapters (36 to 68 and 12 in the second form, 8 to 12 and none with three an SM).  Microseconds (bfloat16, the 7B shape,
// an adapter a token): down projection of rank 64, by the first two forms and the third of eight, 4 tokens 8.4, 10.8, 15.2; 24 tokens 19.9, 17.8, 22.9; q, k and v of
// rank 16, 12 tokens three an SM 4.8, four 5.9; 64 tokens in clusters of eight, four and two 18.4, 14.0, 8.1 (the first two as they were with registers in
// memory); gate and up, 64 tokens four an SM 23.0, three 27.5, 96 tokens 35.9 and 26.5.
// The parameters take 160 bytes, ordered so that nothing lies between them: with 168 a launch costs the host 0.35 us more.
template <typename T, typename O, int THREADS, int PER_SM, int TEAM>
__global__ void __launch_bounds__(THREADS, PER_SM)
low_rank_token_kernel(const T* __restrict__ x_, long long ldx, const T* __restrict__ a, const T* __restrict__ b,
                      const float* __restrict__ scale, const int* __restrict__ ranks, const int* __restrict__ ids_, const O* __restrict__ base_, long long ldb,
                      O* out_, long long ldo, int K, int Kp, int r, int L, const __grid_constant__ Slices slices, int parts, int x_whole, int* err) {
    constexpr int E = Chunk<T>::E, WARPS = THREADS / 32;
    __shared__ float hidden[MOST_RANK];
    __shared__ float partial[MOST_RANK / TEAM][WARPS];             // a hidden value's share of a warp
    __shared__ float scale_l;                                      // the adapter's, and its rank: asked for here, needed behind the sums
    __shared__ int own;
    asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");              // here: peers may write into this CTA's memory
    pdl_trigger();
    pdl_wait();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, me = (int)rank_in_cluster();
    const int g = blockIdx.y / parts, part = blockIdx.y % parts, N = slices.first[slices.n], t = blockIdx.z;
    // this CTA's columns: its part of its cluster's share of the slice
    const int wide = slices.first[g + 1] - slices.first[g], shares = parts * TEAM, each = (wide + shares - 1) / shares;
    const int n0 = slices.first[g] + min(wide, (part * TEAM + me) * each), mine = min(slices.first[g + 1], n0 + each) - n0;
    const T* x = pdl_fresh(x_) + (size_t)t * ldx;
    const O* base = base_ ? pdl_fresh(base_) + (size_t)t * ldb + n0 : nullptr;
    O* out = out_ + (size_t)t * ldo + n0;
    const int l = adapter_of(pdl_fresh(ids_), t, L, err);
    if (l < 0) {                                                   // the same for the whole cluster
        if (out_ != base_)
            for (int n = tid; n < mine; n += THREADS) out[n] = base ? base[n] : from_float<O>(0.f);
        asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
        return;
    }
    // Before B's loads, or in 32 bits behind them: there registers are short the other way about (microseconds before and behind them: 64 tokens, gate and up
    // of rank 16 in bfloat16 24.1, 24.7; 200 tokens of it in float32 107.8, 99.9)
    auto ask = [&]() {
        if (tid != 0) return;
        async_word(&scale_l, scale + l);
        if (ranks) async_word(&own, ranks + l * slices.n + g);
        else own = r;
    };
    if (sizeof(T) == 2) ask();
    // B's chunks: `lanes` neighbours share a row, each with the same two parts of every row that it meets
    const int chunks = r / E;
    int lanes = 1;
    while (lanes * EACH < chunks) lanes *= 2;
    const int chunk = lane % lanes, rows_at_once = THREADS / lanes, row0 = tid / lanes;
    // a part that is not there: the last one, with hidden values of zero
    int part_at[EACH];
#pragma unroll
    for (int c = 0; c < EACH; ++c) part_at[c] = min(chunk + c * lanes, chunks - 1) * E;
    const T* B = b + ((size_t)l * N + n0) * r;
    uint4 ahead[AHEAD][EACH];
    O old[AHEAD];                                                  // as they lie in memory: to change their type is to wait for them
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
        const int n = row0 + j * rows_at_once;
#pragma unroll
        for (int c = 0; c < EACH; ++c)
            ahead[j][c] = n < mine ? __ldg(reinterpret_cast<const uint4*>(B + (size_t)n * r + part_at[c])) : make_uint4(0, 0, 0, 0);
        old[j] = chunk == 0 && n < mine && base ? base[n] : from_float<O>(0.f);
    }
    if (sizeof(T) == 4) ask();
    // this CTA's part of the hidden values, several warps a row where there are fewer rows than warps
    const int rows = r / TEAM;
    int split = 1;
    while (split * 2 * rows <= WARPS) split *= 2;
    const int sub = warp % split;
    for (int j = warp / split; j < rows; j += WARPS / split) {
        const T* row = a + (((size_t)l * slices.n + g) * r + me * rows + j) * Kp;
        float s = 0.f;
        int k = (sub * 32 + lane) * E;
        if (x_whole) {
            // several chunks of A and x on their way at a time, without a branch between them
            constexpr int U = PER_SM == 1 ? 8 : PER_SM == 2 ? 4 : 2;
            const int stride = split * 32 * E;
            for (; k + (U - 1) * stride + E <= K; k += U * stride) {
                uint4 w[U], v[U];
#pragma unroll
                for (int i = 0; i < U; ++i) w[i] = __ldg(reinterpret_cast<const uint4*>(row + k + i * stride));
#pragma unroll
                for (int i = 0; i < U; ++i) v[i] = *reinterpret_cast<const uint4*>(x + k + i * stride);
#pragma unroll
                for (int i = 0; i < U; ++i) {
                    float wf[E], vf[E];
                    Chunk<T>::unpack(w[i], wf), Chunk<T>::unpack(v[i], vf);
#pragma unroll
                    for (int e = 0; e < E; ++e) s = fmaf(vf[e], wf[e], s);
                }
            }
        }
#pragma unroll 2
        for (; k < K; k += split * 32 * E) {
            float w[E], v[E];
            Chunk<T>::unpack(__ldg(reinterpret_cast<const uint4*>(row + k)), w);
            if (x_whole && k + E <= K) {
                Chunk<T>::unpack(*reinterpret_cast<const uint4*>(x + k), v);
            } else {
#pragma unroll
                for (int e = 0; e < E; ++e) v[e] = k + e < K ? to_float(x[k + e]) : 0.f;
            }
#pragma unroll
            for (int e = 0; e < E; ++e) s = fmaf(v[e], w[e], s);
        }
        s = warp_sum(s);
        if (lane == 0) partial[j][sub] = s;
    }
    if (tid == 0) asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    if (tid < rows * TEAM) {                                       // a hidden value, for one of the CTAs
        const int c = tid % TEAM, q = tid / TEAM;
        float h = 0.f;
        for (int w = 0; w < split; ++w) h += partial[q][w];
        h = me * rows + q < own ? h * scale_l : 0.f;
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(peer(&hidden[me * rows + q], c)), "f"(h) : "memory");
    }
    __syncwarp();
    cluster_barrier();
    float h[EACH][E];
#pragma unroll
    for (int c = 0; c < EACH; ++c)
#pragma unroll
        for (int e = 0; e < E; ++e) h[c][e] = chunk + c * lanes < chunks ? hidden[part_at[c] + e] : 0.f;
    const int pass = AHEAD * rows_at_once;
    const size_t step = (size_t)rows_at_once * r;
    const T* next = B + (size_t)(row0 + pass) * r;
    int n = row0;
    for (int m = 0; m < mine; m += pass) {
#pragma unroll
        for (int i = 0; i < AHEAD; ++i, n += rows_at_once, next += step) {
            if (m + i * rows_at_once >= mine) break;
            float w[EACH][E], sum = to_float(old[i]);
#pragma unroll
            for (int c = 0; c < EACH; ++c) Chunk<T>::unpack(ahead[i][c], w[c]);
            if (n + pass < mine) {
#pragma unroll
                for (int c = 0; c < EACH; ++c)
                    ahead[i][c] = __ldg(reinterpret_cast<const uint4*>(next + part_at[c]));
                if (chunk == 0 && base) old[i] = base[n + pass];
            }
#pragma unroll
            for (int c = 0; c < EACH; ++c)
#pragma unroll
                for (int e = 0; e < E; ++e) sum = fmaf(h[c][e], w[c][e], sum);
            for (int o = 1; o < lanes; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (chunk == 0 && n < mine) out[n] = from_float<O>(sum);
        }
    }
}

template <typename T, typename O>
int launch_tokens(const void* x, long long ldx, const void* a, const void* b, const float* scale, const int* ranks, const int* ids, const void* base,
                  long long ldb, void* out, long long ldo, int tokens, int K, int Kp, int r, int L, const Slices& s, int* err, int sms, cudaStream_t stream) {
    constexpr int MOST = 65535;                // tokens of a launch: its grid's third size
    int code = 0;
    for (; tokens > MOST && code == 0; tokens -= MOST) {
        code = launch_tokens<T, O>(x, ldx, a, b, scale, ranks, ids, base, ldb, out, ldo, MOST, K, Kp, r, L, s, err, sms, stream);
        x = (const T*)x + MOST * ldx, ids += MOST, base = base ? (const O*)base + MOST * ldb : nullptr, out = (O*)out + MOST * ldo;
    }
    if (tokens <= 0 || code != 0) return code;
    // Clusters at a time with an SM a CTA, with half of one, a third and a quarter.  Where a CTA has much of A, up to 18 are launched in the first form all the same:
    // rows without an adapter (of a captured step that has fewer requests than rows, say) are over at once.  16 tokens, down projection, 303 KB of A a CTA, eight
    // adapters: 17.3 us if all 16 have one, in the second form 16.0; if one of them has none 10.9 and 16.3.
    const bool much = (long long)r / CTAS * Kp * (int)sizeof(T) >= 128 * 1024;
    const int wholes = sms / CTAS * 5 / 6, halves = much ? sms * 9 / (CTAS * 5) : 0, thirds = sms * 9 / 25, quarters = sms * 12 / 25;
    const int first_form = much ? sms / CTAS : wholes;
    // clusters that share a slice's columns, each with hidden values of its own: as many as keep B's part of a CTA within what it asks for ahead, while
    // all run at a time
    int widest = 0;
    for (int g = 0; g < s.n; ++g) widest = max(widest, s.first[g + 1] - s.first[g]);
    const long long bytes = (long long)widest * r * (int)sizeof(T), ahead = (long long)CTAS * 512 * AHEAD * EACH * 16;
    const int parts = (int)max(1ll, min((bytes + ahead - 1) / ahead, (long long)wholes / ((long long)s.n * tokens)));
    const int whole = (reinterpret_cast<uintptr_t>(x) % 16 == 0) && (ldx * (long long)sizeof(T) % 16 == 0 || tokens == 1);
    cudaLaunchConfig_t cfg = {};
    // the form: kernel, its threads and its clusters' size together
    const int clusters = s.n * parts * tokens;
    auto kernel = low_rank_token_kernel<T, O, 256, 4, 2>;
    int threads = 256, ctas = 2;
    if (clusters <= first_form) kernel = low_rank_token_kernel<T, O, 512, 1, 8>, threads = 512, ctas = 8;
    else if (clusters <= halves) kernel = low_rank_token_kernel<T, O, 512, 2, 8>, threads = 512, ctas = 8;
    else if (clusters <= thirds) kernel = low_rank_token_kernel<T, O, 256, 3, 8>, ctas = 8;
    else if (clusters <= quarters) kernel = low_rank_token_kernel<T, O, 256, 4, 8>, ctas = 8;
    else if (clusters <= 2 * thirds) kernel = low_rank_token_kernel<T, O, 256, 3, 4>, ctas = 4;
    else if (clusters <= 2 * quarters) kernel = low_rank_token_kernel<T, O, 256, 4, 4>, ctas = 4;
    else if (clusters <= 4 * thirds) kernel = low_rank_token_kernel<T, O, 256, 3, 2>, ctas = 2;
    cfg.gridDim = dim3(ctas, s.n * parts, tokens);
    cfg.blockDim = dim3(threads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ctas, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = prism::pdl_enabled() ? 2 : 1;
    return (int)cudaLaunchKernelEx(&cfg, kernel, (const T*)x, ldx, (const T*)a, (const T*)b, scale, ranks, ids, (const O*)base, ldb, (O*)out,
                                   ldo, K, Kp, r, L, s, parts, whole, err);
}

// ---- portions -----------------------------------------------------------------------------------------------

constexpr int TOKENS = 32;                    // of a tile
constexpr int DEEP = 64;                      // of K at a time
constexpr int HT = 512, PT = 256;             // threads of either launch
constexpr int COLUMNS = 128;                  // results of a tile

// The tokens' adapters (-1: none, or beyond the end) and the different ones among them, in order.  By the first warp.
__device__ __forceinline__ void list_adapters(const int* ids, int t0, int tokens, int L, int* own, int* list, int* count, int* err) {
    const int lane = threadIdx.x;
    const int id = t0 + lane < tokens ? adapter_of(ids, t0 + lane, L, err) : -1;
    own[lane] = id;
    const uint32_t same = __match_any_sync(0xffffffffu, id);
    const bool first = id >= 0 && __ffs(same) - 1 == lane;
    const uint32_t found = __ballot_sync(0xffffffffu, first);
    if (first) list[__popc(found & ((1u << lane) - 1))] = id;
    if (lane == 0) *count = __popc(found);
}

// hidden [tokens, G r] float32.  A thread: two tokens by up to four of a slice's hidden values.
template <typename T>
__global__ void __launch_bounds__(HT)
low_rank_plain_hidden_kernel(const T* __restrict__ x_, long long ldx, const T* __restrict__ a, const float* __restrict__ scale,
                             const int* __restrict__ ranks, const int* __restrict__ ids_, float* __restrict__ hidden, int tokens, int K, int Kp, int r, int G, int L, int* err) {
    __shared__ float xs[TOKENS][DEEP + 1];
    __shared__ float as[MOST_RANK][DEEP + 1];                      // behind the last block, this CTA's sums
    float* sums = &as[0][0];                                       // [TOKENS][r]
    __shared__ int own[TOKENS], list[TOKENS], count;
    pdl_trigger();
    pdl_wait();
    const int tid = threadIdx.x, lane = tid & 31, q = tid >> 5, me = (int)rank_in_cluster(), t0 = blockIdx.y * TOKENS, g = blockIdx.z;
    if (q == 0) list_adapters(pdl_fresh(ids_), t0, tokens, L, own, list, &count, me == 0 && g == 0 ? err : nullptr);
    __syncthreads();
    const T* x = pdl_fresh(x_) + (size_t)t0 * ldx;
    constexpr int XN = TOKENS * DEEP / HT, AN = MOST_RANK * DEEP / HT;         // values a thread brings of a block
    for (int p = 0; p < count; ++p) {
        const int l = list[p];
        const T* A = a + ((size_t)l * G + g) * r * Kp;
        float acc[2][4] = {};
        float xv[XN];
        T av[AN];
        auto bring = [&](int k0) {
#pragma unroll
            for (int i = 0; i < XN; ++i) {
                const int row = (tid + i * HT) / DEEP, k = k0 + (tid + i * HT) % DEEP;
                xv[i] = t0 + row < tokens && k < K ? to_float(x[(size_t)row * ldx + k]) : 0.f;
            }
#pragma unroll
            for (int i = 0; i < AN; ++i) {
                const int row = (tid + i * HT) / DEEP, k = k0 + (tid + i * HT) % DEEP;
                if (row < r) av[i] = k < K ? A[(size_t)row * Kp + k] : from_float<T>(0.f);
            }
        };
        bring(me * DEEP);
        for (int k0 = me * DEEP; k0 < K; k0 += CTAS * DEEP) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < XN; ++i) xs[(tid + i * HT) / DEEP][(tid + i * HT) % DEEP] = xv[i];
#pragma unroll
            for (int i = 0; i < AN; ++i)
                if ((tid + i * HT) / DEEP < r) as[(tid + i * HT) / DEEP][(tid + i * HT) % DEEP] = to_float(av[i]);
            __syncthreads();
            if (k0 + CTAS * DEEP < K) bring(k0 + CTAS * DEEP);     // the next block's, while this one's are used
#pragma unroll 4
            for (int k = 0; k < DEEP; ++k) {
                float u[2], w[4];
#pragma unroll
                for (int i = 0; i < 2; ++i) u[i] = xs[q * 2 + i][k];
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = lane + 32 * i < r ? as[lane + 32 * i][k] : 0.f;
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int c = 0; c < 4; ++c) acc[i][c] = fmaf(u[i], w[c], acc[i][c]);
            }
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int c = 0; c < 4; ++c)
                if (lane + 32 * c < r) sums[(q * 2 + i) * r + lane + 32 * c] = acc[i][c];
        cluster_barrier();
        // a CTA adds up four tokens' sums
        for (int v = tid; v < TOKENS / CTAS * r; v += HT) {
            const int row = me * (TOKENS / CTAS) + v / r, c = v % r;
            if (own[row] != l) continue;
            float part[CTAS], s = 0.f;
#pragma unroll
            for (int i = 0; i < CTAS; ++i) asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(part[i]) : "r"(peer(sums + row * r + c, i)) : "memory");
#pragma unroll
            for (int i = 0; i < CTAS; ++i) s += part[i];
            hidden[((size_t)(t0 + row) * G + g) * r + c] = ranks == nullptr || c < ranks[l * G + g] ? s * scale[l] : 0.f;
        }
        __syncwarp();
        cluster_barrier();
    }
}

// A thread: four tokens by four columns
template <typename T, typename O>
__global__ void __launch_bounds__(PT)
low_rank_plain_result_kernel(const float* __restrict__ hidden_, const T* __restrict__ b, const int* __restrict__ ids_, const O* base, long long ldb, O* out,
                             long long ldo, int tokens, int r, int L, Slices slices) {
    extern __shared__ float plain_smem[];
    __shared__ int own[TOKENS], list[TOKENS], count;
    const int pitch = r + 1;
    float* hs = plain_smem;                                        // [TOKENS][r]
    float* bs = plain_smem + TOKENS * r;                           // [COLUMNS][pitch]
    pdl_trigger();
    pdl_wait();
    const int tid = threadIdx.x, lane = tid & 31, q = tid >> 5, t0 = blockIdx.y * TOKENS, N = slices.first[slices.n];
    int g = 0, tile = blockIdx.x;
    while (g + 1 < slices.n && tile >= (slices.first[g + 1] - slices.first[g] + COLUMNS - 1) / COLUMNS)
        tile -= (slices.first[g + 1] - slices.first[g] + COLUMNS - 1) / COLUMNS, ++g;
    const int n0 = slices.first[g] + tile * COLUMNS, wide = min(COLUMNS, slices.first[g + 1] - n0);
    if (q == 0) list_adapters(pdl_fresh(ids_), t0, tokens, L, own, list, &count, nullptr);
    float old[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c)
            old[i][c] = base && t0 + q * 4 + i < tokens && lane + 32 * c < wide ? to_float(base[(size_t)(t0 + q * 4 + i) * ldb + n0 + lane + 32 * c]) : 0.f;
    __syncthreads();
    const float* hidden = pdl_fresh(hidden_) + ((size_t)t0 * slices.n + g) * r;
    for (int p = 0; p < count; ++p) {
        const int l = list[p];
        __syncthreads();
        for (int i = tid; i < TOKENS * r; i += PT) hs[i] = own[i / r] == l ? hidden[(size_t)(i / r) * slices.n * r + i % r] : 0.f;
        const T* B = b + ((size_t)l * N + n0) * r;
#pragma unroll 8
        for (int i = tid; i < wide * r; i += PT) bs[i / r * pitch + i % r] = to_float(B[i]);
        __syncthreads();
        float acc[4][4] = {};
#pragma unroll 4
        for (int k = 0; k < r; ++k) {
            float u[4], w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) u[i] = hs[(q * 4 + i) * r + k];
#pragma unroll
            for (int c = 0; c < 4; ++c) w[c] = bs[(lane + 32 * c) * pitch + k];
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int c = 0; c < 4; ++c) acc[i][c] = fmaf(u[i], w[c], acc[i][c]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (own[q * 4 + i] == l)
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    if (lane + 32 * c < wide) out[(size_t)(t0 + q * 4 + i) * ldo + n0 + lane + 32 * c] = from_float<O>(old[i][c] + acc[i][c]);
    }
    if ((const O*)out != base)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (own[q * 4 + i] < 0 && t0 + q * 4 + i < tokens)
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    if (lane + 32 * c < wide) out[(size_t)(t0 + q * 4 + i) * ldo + n0 + lane + 32 * c] = from_float<O>(old[i][c]);
}

template <typename T, typename O>
int launch_portions(const void* x, long long ldx, const void* a, const void* b, const float* scale, const int* ranks, const int* ids, const void* base,
                    long long ldb, void* out, long long ldo, int tokens, int K, int Kp, int r, int L, const Slices& s, void* hidden, int* err, cudaStream_t stream) {
    constexpr int MOST = 65535 * TOKENS;       // tokens of a launch; the next one's hidden values take the place of its own
    int code = 0;
    for (; tokens > MOST && code == 0; tokens -= MOST) {
        code = launch_portions<T, O>(x, ldx, a, b, scale, ranks, ids, base, ldb, out, ldo, MOST, K, Kp, r, L, s, hidden, err, stream);
        x = (const T*)x + MOST * ldx, ids += MOST, base = base ? (const O*)base + MOST * ldb : nullptr, out = (O*)out + MOST * ldo;
    }
    if (tokens <= 0 || code != 0) return code;
    const int tiles = (tokens + TOKENS - 1) / TOKENS;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(CTAS, tiles, s.n);
    cfg.blockDim = dim3(HT);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = CTAS, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = prism::pdl_enabled() ? 2 : 1;
    code = (int)cudaLaunchKernelEx(&cfg, low_rank_plain_hidden_kernel<T>, (const T*)x, ldx, (const T*)a, scale, ranks, ids, (float*)hidden, tokens, K, Kp, r, s.n, L,
                                       err);
    if (code != 0) return code;
    int columns = 0;
    for (int g = 0; g < s.n; ++g) columns += (s.first[g + 1] - s.first[g] + COLUMNS - 1) / COLUMNS;
    const size_t smem = ((size_t)TOKENS * r + (size_t)COLUMNS * (r + 1)) * 4;
    prism::open_smem(low_rank_plain_result_kernel<T, O>, smem);
    return (int)prism::launch_kernel(low_rank_plain_result_kernel<T, O>, dim3(columns, tiles), dim3(PT), smem, stream, (const float*)hidden, (const T*)b, ids,
                                     (const O*)base, ldb, (O*)out, ldo, tokens, r, L, s);
}

}  // namespace lowrank
}  // namespace prism

namespace prism {
namespace lowrank {

int run(const void* x, long long ldx, int dtype, const void* a, const void* b, const float* scale, const int* ranks, const int* ids, const void* base,
        long long ldb, void* out, long long ldo, int out_dtype, int T, int K, int Kp, int r, int L, int G, const int* first, void* hidden, int sms,
        int* err, cudaStream_t stream) {
    typedef __nv_bfloat16 bf16;
    if (T <= 0) return 0;
    if (G < 1 || G > MOST_SLICES || r < 16 || r % 16 || r > MOST_RANK || K < 1 || Kp < K || Kp % 8 || L < 1 || sms < 1) return (int)cudaErrorInvalidValue;
    Slices s;
    s.n = G;
    for (int g = 0; g <= G; ++g) s.first[g] = first[g];
    for (int g = 0; g < G; ++g)
        if (s.first[g] >= s.first[g + 1]) return (int)cudaErrorInvalidValue;
#define PRISM_LOW_RANK(TX, TO)                                                                                                              \
    (hidden ? launch_portions<TX, TO>(x, ldx, a, b, scale, ranks, ids, base, ldb, out, ldo, T, K, Kp, r, L, s, hidden, err, stream)          \
            : launch_tokens<TX, TO>(x, ldx, a, b, scale, ranks, ids, base, ldb, out, ldo, T, K, Kp, r, L, s, err, sms, stream))
    if (dtype == PRISM_DTYPE_F32) return out_dtype == PRISM_DTYPE_F32 ? PRISM_LOW_RANK(float, float) : PRISM_LOW_RANK(float, bf16);
    return out_dtype == PRISM_DTYPE_F32 ? PRISM_LOW_RANK(bf16, float) : PRISM_LOW_RANK(bf16, bf16);
#undef PRISM_LOW_RANK
}

}  // namespace lowrank
}  // namespace prism

// first: G + 1 column borders (host memory).  base may be null (nothing to add to), or out itself.  hidden null: all T tokens one by one; else in
// tiles, with T G r floats of workspace there.  All r rows of every A count.
PRISM_EXPORT int prism_low_rank(const void* x, long long ldx, int dtype, const void* a, const void* b, const float* scale, const int* ids,
                                const void* base, long long ldb, void* out, long long ldo, int out_dtype, int T, int K, int Kp, int r, int L, int G,
                                const int* first, void* hidden, int sms, int* err, cudaStream_t stream) {
    return prism::lowrank::run(x, ldx, dtype, a, b, scale, nullptr, ids, base, ldb, out, ldo, out_dtype, T, K, Kp, r, L, G, first, hidden, sms, err, stream);
}

// The same with ranks [L, G]: how many rows of A each adapter has in each slice; null: all r.
PRISM_EXPORT int prism_low_rank_ranked(const void* x, long long ldx, int dtype, const void* a, const void* b, const float* scale, const int* ranks,
                                       const int* ids, const void* base, long long ldb, void* out, long long ldo, int out_dtype, int T, int K, int Kp,
                                       int r, int L, int G, const int* first, void* hidden, int sms, int* err, cudaStream_t stream) {
    return prism::lowrank::run(x, ldx, dtype, a, b, scale, ranks, ids, base, ldb, out, ldo, out_dtype, T, K, Kp, r, L, G, first, hidden, sms, err, stream);
}
