// A token from each row of float32 logits by temperature, top-k, top-p and min-p, at a uniform number u that the host supplies.
//
// With m the row's largest logit and w_i = exp((x_i - m) / T), tokens stand in the order (logit down, index up).  Kept are
// the first top_k of them; of these the shortest prefix whose weight reaches top_p of theirs; of these the ones with w_i >= min_p.
// Each filter keeps a prefix of that order, so together they keep the shortest of the three.  The draw is the inverse CDF in the
// order of the indices, as in sample.cu: the first kept index whose running weight exceeds u times the weight of all kept.
// T <= 0: the largest, lowest index on ties.  NaN counts as -infinity, which is never kept; a row with nothing else gives token 0.
//
// Weights come from 64-bit arithmetic (relative error below 2^-50).  The draw adds them up as whole numbers, w_i * 2^46 rounded: such sums are exact, so neither
// the order of additions nor the number of CTAs that share a row can change them, and every thread sees the same running weight; a draw is decided
// to about 1e-12 of the weight (in float32 one row in thirty over 150,000 tokens would be decided by rounding).  top_p = 0.9999999 ends a
// prefix among weights that such steps do not resolve: its sums are 64-bit floats, added in an order that V alone fixes.
//
// One cluster of CTAs a row: each keeps its slice of the logits in shared memory, so that the row is read once, and the CTAs' sums meet
// through distributed shared memory.
#include "common.cuh"

namespace prism {
namespace draw {

typedef unsigned long long u64;
constexpr int THREADS = 512;
constexpr int WARPS = THREADS / 32;
constexpr int MOST_CTAS = 8;
constexpr int MOST_SLICE = 40 * 1024;          // values of a slice that stay in shared memory; of a larger one every pass reads memory

__device__ __forceinline__ uint32_t rank_in_cluster() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}
__device__ __forceinline__ u64 read_peer(const u64* p, int cta) {
    uint32_t at;
    u64 v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(cta));
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(at) : "memory");
    return v;
}
template <typename W> __device__ __forceinline__ W warp_sum64(W v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ u64 warp_max64(u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const u64 t = __shfl_xor_sync(0xffffffffu, v, o);
        v = t > v ? t : v;
    }
    return v;
}

// A token's place in the order as one number, larger is better: the logit's bits so that they compare as whole numbers, then the index
__device__ __forceinline__ u64 place_of(float x, int i) {
    const uint32_t b = __float_as_uint(x);
    return ((u64)(b ^ ((uint32_t)((int)b >> 31) | 0x80000000u)) << 32) | (uint32_t)~i;
}
__device__ __forceinline__ float value_at(u64 place) {
    const uint32_t k = (uint32_t)(place >> 32);
    return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
__device__ __forceinline__ float clean(float x) { return x != x ? -INFINITY : x + 0.f; }       // -0 becomes 0: they are one value

struct Row {
    double top, per;             // largest logit; log2(e) / T
    double one;                  // a weight of 1 as a whole number: 2^46, or less where V of them would not fit
    const double* table;         // 2^(-j / 64)
};

// -log2 of a token's weight, 0 for the largest itself
__device__ __forceinline__ double depth(const Row& r, float x) {
    const double v = (double)x;
    return v == r.top ? 0.0 : (r.top - v) * r.per;
}
// 2^-d = 2^-(n / 64) 2^-f with |f| <= 1/128: the second factor by the series of exp(-f ln 2) to the fifth power (the next term is below
// 2^-54), the first from a table of 64 and the exponent
__device__ __forceinline__ double weight(const Row& r, double d) {
    if (!(d < 1000.0)) return 0.0;
    const double shift = 6755399441055744.0;                     // 1.5 * 2^52: rounds to a whole number, which the low bits then hold
    const double t = fma(d, 64.0, shift);
    const int n = __double2loint(t);
    const double f = fma(t - shift, -1.0 / 64, d);
    constexpr double L = 0.69314718055994530942;
    double q = fma(f, -L * L * L * L * L / 120, L * L * L * L / 24);
    q = fma(f, q, -L * L * L / 6);
    q = fma(f, q, L * L / 2);
    q = fma(f, q, -L);
    q = fma(f, q, 1.0);
    q *= r.table[n & 63];
    return __hiloint2double(__double2hiint(q) - ((n >> 6) << 20), __double2loint(q));
}
// A weight of up to 1 as a whole number: 2^52 + w 2^bits has its whole part in the low 52 bits
__device__ __forceinline__ u64 whole(const Row& r, double w) {
    return (u64)__double_as_longlong(fma(w, r.one, 4503599627370496.0)) & 0xfffffffffffffull;
}

struct Shared {
    double table[64];
    u64 slot[2][WARPS];          // per-warp results of a reduction; [..][0] then holds the CTA's, for its peers
    u64 part[2];
};

struct Team {
    Shared* s;
    int ctas, me, turn;
    // Over the cluster, for every thread.  Slots are used in turn: a CTA that is one reduction ahead writes others than its peers still read.
    __device__ __forceinline__ u64 sum(u64 v) { return reduce<u64>(v, [](u64 t) { return warp_sum64(t); }); }
    __device__ __forceinline__ u64 max(u64 v) { return reduce<u64>(v, [](u64 t) { return warp_max64(t); }); }
    __device__ __forceinline__ double sum(double v) { return reduce<double>(v, [](double t) { return warp_sum64(t); }); }
    static __device__ __forceinline__ u64 bits_of(u64 v) { return v; }
    static __device__ __forceinline__ u64 bits_of(double v) { return (u64)__double_as_longlong(v); }
    static __device__ __forceinline__ void of_bits(u64 b, u64& v) { v = b; }
    static __device__ __forceinline__ void of_bits(u64 b, double& v) { v = __longlong_as_double((long long)b); }
    template <typename W, typename F> __device__ __forceinline__ W reduce(W v, F warp_all) {
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        turn ^= 1;
        v = warp_all(v);
        if (lane == 0) s->slot[turn][warp] = bits_of(v);
        __syncthreads();
        of_bits(lane < WARPS ? s->slot[turn][lane] : 0, v);
        v = warp_all(v);
        if (ctas == 1) return v;
        if (threadIdx.x == 0) s->part[turn] = bits_of(v);
        cluster_barrier();
        of_bits(lane < ctas ? read_peer(&s->part[turn], lane) : 0, v);
        return warp_all(v);
    }
};

__global__ void __launch_bounds__(THREADS)
sample_filtered_kernel(const float* __restrict__ logits_, long long ld, int R, int V, int per_cta, int resident, const float* __restrict__ temperature_,
                       const float* __restrict__ u_, const int* __restrict__ top_k_, const float* __restrict__ top_p_,
                       const float* __restrict__ min_p_, const int* __restrict__ rows_, int* __restrict__ out, int* __restrict__ kept_out,
                       float* __restrict__ logprob_out, int* err) {
    extern __shared__ float slice[];
    __shared__ Shared sh;
    const int tid = threadIdx.x;
    Team team;
    team.s = &sh;
    team.ctas = gridDim.x;
    team.me = team.ctas > 1 ? (int)rank_in_cluster() : 0;
    team.turn = 0;
    if (tid < 64) sh.table[tid] = exp2(-tid / 64.0);
    pdl_trigger();
    pdl_wait();
    const int row = rows_ ? pdl_fresh(rows_)[blockIdx.y] : blockIdx.y;
    if (row < 0 || row >= R) {                                     // the same for the whole cluster: nobody waits for anybody
        if (tid == 0) report_error(err, PRISM_ERR_ROW_RANGE);
        return;
    }
    const float* x = pdl_fresh(logits_) + (size_t)row * ld;
    const int c0 = min(team.me * per_cta, V), n = min(per_cta, V - c0);
    x += c0;
    const float T = temperature_ ? pdl_fresh(temperature_)[row] : 0.f;

    u64 best = 0;
    for (int i = tid; i < n; i += THREADS) {
        const float v = clean(x[i]);
        if (resident) slice[i] = v;
        const u64 p = place_of(v, c0 + i);
        best = p > best ? p : best;
    }
    best = team.max(best);
    const float top = value_at(best);
    if (!(T > 0.f) || top == -INFINITY) {
        const bool none = top == -INFINITY;
        if (team.me == 0 && tid == 0) {
            out[row] = none ? 0 : (int)~(uint32_t)best;
            if (kept_out) kept_out[row] = none ? 0 : 1;
            if (logprob_out) logprob_out[row] = none ? -INFINITY : 0.f;
        }
        if (team.ctas > 1) cluster_barrier();                      // peers may still read this CTA's part
        return;
    }
    auto value = [&](int i) { return resident ? slice[i] : clean(x[i]); };
    Row r;
    r.top = (double)top;
    r.per = 1.44269504088896340736 / (double)T;
    const int bits = min(46, 63 - (31 - __clz(V)));                // V weights of 1 stay below 2^64
    r.one = (double)(1ull << bits);
    r.table = sh.table;

    const int k = top_k_ ? pdl_fresh(top_k_)[row] : 0;
    const float p = top_p_ ? pdl_fresh(top_p_)[row] : 1.f, mp = min_p_ ? fminf(pdl_fresh(min_p_)[row], 1.f) : 0.f;
    const double deepest = mp > 0.f ? -log2((double)mp) : INFINITY;

    // The largest place whose measure, over the tokens from it on upwards, reaches the target: one bit after the other
    u64 cut = 0;
    if (k > 0 && k < V) {
        u64 at = 0;
        for (int bit = 63; bit >= 0; --bit) {
            const u64 trial = at | (1ull << bit);
            u64 m = 0;
            for (int i = tid; i < n; i += THREADS) m += place_of(value(i), c0 + i) >= trial;
            if (team.sum(m) >= (u64)k) at = trial;
        }
        cut = at;
    }
    if (p < 1.f) {
        double all = 0;
        for (int i = tid; i < n; i += THREADS)
            if (place_of(value(i), c0 + i) >= cut) all += weight(r, depth(r, value(i)));
        const double target = fmax((double)p, 0.0) * team.sum(all);
        u64 at = 0;
        for (int bit = 63; bit >= 0; --bit) {
            const u64 trial = at | (1ull << bit), from = trial > cut ? trial : cut;
            double m = 0;
            for (int i = tid; i < n; i += THREADS)
                if (place_of(value(i), c0 + i) >= from) m += weight(r, depth(r, value(i)));
            m = team.sum(m);
            if (m > 0 && m >= target) at = trial;
        }
        cut = at > cut ? at : cut;
    }

    // The draw: every thread a run of neighbours, its weight after those of the runs before it
    const int run = ((n + THREADS - 1) / THREADS) | 1;             // odd: neighbours' places lie in different banks
    const int i0 = min(tid * run, n), i1 = min(i0 + run, n);
    u64 own = 0, count = 0;
    for (int i = i0; i < i1; ++i) {
        const float v = value(i);
        const double d = depth(r, v);
        if (place_of(v, c0 + i) >= cut && d <= deepest && d < INFINITY) own += whole(r, weight(r, d)), ++count;
    }
    const int lane = tid & 31, warp = tid >> 5;
    u64 upto = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 t = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += t;
    }
    count = team.sum(count);                                       // its barriers also end the use of the slots below
    team.turn ^= 1;
    if (lane == 31) sh.slot[team.turn][warp] = upto;
    __syncthreads();
    u64 mine = 0;
    for (int w = 0; w < WARPS; ++w) {
        if (w < warp) upto += sh.slot[team.turn][w];
        mine += sh.slot[team.turn][w];
    }
    u64 total = mine;
    if (team.ctas > 1) {
        if (tid == 0) sh.part[team.turn] = mine;
        cluster_barrier();
        total = 0;
        for (int c = 0; c < team.ctas; ++c) {
            const u64 t = read_peer(&sh.part[team.turn], c);
            if (c < team.me) upto += t;
            total += t;
        }
    }
    const float u = pdl_fresh(u_)[row];
    const double goal = u < 1.f ? fmax((double)u, 0.0) * (double)total : (double)(total - 1);
    if ((double)upto > goal && !((double)(upto - own) > goal)) {   // one thread of the cluster: the running weight passes the goal in its run
        u64 run_to = upto - own;
        for (int i = i0; i < i1; ++i) {
            const float v = value(i);
            const double d = depth(r, v);
            if (place_of(v, c0 + i) >= cut && d <= deepest && d < INFINITY) {
                run_to += whole(r, weight(r, d));
                if ((double)run_to > goal) {
                    out[row] = c0 + i;
                    if (kept_out) kept_out[row] = (int)count;
                    if (logprob_out) logprob_out[row] = (float)(-0.69314718055994530942 * (d + (log2((double)total) - bits)));
                    break;
                }
            }
        }
    }
    if (team.ctas > 1) cluster_barrier();
}

}  // namespace draw
}  // namespace prism

// One token a row of logits [.., V] (pitch ld), for the rows in `rows` (null: the first n).  temperature, u, top_k, top_p, min_p and the
// results are by row of logits, of which there are R; n of them are wanted.  top_k, top_p, min_p, temperature, kept, logprob may be null.
PRISM_EXPORT int prism_sample_filtered(const float* logits, long long ld, int n, int R, int V, const float* temperature, const float* u, const int* top_k,
                                       const float* top_p, const float* min_p, const int* rows, int* out, int* kept, float* logprob,
                                       int* err, cudaStream_t stream) {
    using namespace prism::draw;
    if (n <= 0) return 0;
    if (V < 1 || n > 65535 || n > R || u == nullptr || out == nullptr) return (int)cudaErrorInvalidValue;
    int ctas = 1;
    while (ctas < MOST_CTAS && V > 4096 * ctas) ctas *= 2;
    const int per_cta = ((V + ctas - 1) / ctas + 3) & ~3;
    const int resident = per_cta <= MOST_SLICE;
    const size_t smem = resident ? (size_t)per_cta * 4 : 0;
    prism::open_smem(sample_filtered_kernel, smem);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas, n);
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ctas, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = prism::pdl_enabled() ? 2 : 1;
    return (int)cudaLaunchKernelEx(&cfg, sample_filtered_kernel, logits, ld, R, V, per_cta, resident, temperature, u, top_k, top_p, min_p, rows, out,
                                   kept, logprob, err);
}
