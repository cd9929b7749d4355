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
// through distributed shared memory.  A cut is found without sorting the row: tokens are counted (for top_p: weighed) in 512 bins of
// 1/32 of a power of two down to 2^-16 of the largest, each CTA's in shared memory; after one barrier every thread adds up one bin of all CTAs, and a scan
// shows the bin that holds the cut.  If the tokens down to there are 512 or fewer (a top_k or a nucleus as they are in use), one CTA collects and
// sorts them, one a thread, and draws from them; the other CTAs are done.  Else the bin's own tokens are collected and sorted, if it has
// 512 at most, or divided into 512 bins by the bits of their place in the order (their number there: exact, ties and all), until it has; the
// draw is then a pass over the row.
#include "common.cuh"

#include <type_traits>

namespace prism {
namespace draw {

typedef unsigned long long u64;
constexpr int THREADS = 512;
constexpr int WARPS = THREADS / 32;
constexpr int MOST_CTAS = 8;
constexpr int MOST_SLICE = 48 * 1024;          // values of a slice that stay in shared memory; of a larger one every pass reads memory
constexpr int MOST_V = MOST_CTAS * 65000;      // a CTA's bins are sums of 16-bit numbers in 32 bits
constexpr int BINS = THREADS;                  // one a thread
constexpr int LIST = THREADS;                  // tokens that are sorted, one a thread
constexpr int STEPS = 32;                      // bins of a power of two
constexpr int FINE = 128;                      // steps of a power of two that weights are tabled for
constexpr float LEAST = -3.402823466e38f;      // the lowest value that counts: below is -infinity only

__device__ __forceinline__ uint32_t rank_in_cluster() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t peer(const void* p, int cta) {
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(cta));
    return at;
}
__device__ __forceinline__ u64 read_peer(const u64* p, int cta) {
    u64 v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(peer(p, cta)) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t read_peer(const uint32_t* p, int cta) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(peer(p, cta)) : "memory");
    return v;
}
__device__ __forceinline__ void write_peer(double* p, int cta, double v) {
    asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(peer(p, cta)), "d"(v) : "memory");
}
__device__ __forceinline__ void write_peer(uint32_t* p, int cta, uint32_t v) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(peer(p, cta)), "r"(v) : "memory");
}
template <typename W> __device__ __forceinline__ W warp_sum64(W v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// A token's place in the order as one number, larger is better: the logit's bits so that they compare as whole numbers, then the index
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x);
    return b ^ ((uint32_t)((int)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }
__device__ __forceinline__ u64 place_of(float x, int i) { return ((u64)key_of(x) << 32) | (uint32_t)~i; }
__device__ __forceinline__ float value_at(u64 place) { return value_of((uint32_t)(place >> 32)); }
__device__ __forceinline__ float clean(float x) { return x != x ? -INFINITY : x + 0.f; }       // -0 becomes 0: they are one value

__device__ __forceinline__ double power_of_two(int e) { return __hiloint2double((1023 + e) << 20, 0); }

struct Row {
    double top, per;             // largest logit; log2(e) / T
    float floor;                 // tokens below have no weight: it would be less than 2^-1000
    double one;                  // a weight of 1 as a whole number: 2^46, or less where V of them would not fit
    const double* table;         // 2^(-j / FINE)
};

// -log2 of a token's weight, 0 for the largest itself
__device__ __forceinline__ double depth(const Row& r, float x) { return (r.top - (double)x) * r.per; }
// 2^-d with d = depth(x) = n / 128 + f / 128, |f| <= 1/2: the second factor by the series of exp(-f ln 2 / 128) to the fourth power (the next term is
// below 2^-49), the first from a table of 128 and the exponent.  n: also says which bin the token is in.  Free of branches, so
// that several tokens' chains of 64-bit operations overlap.
__device__ __forceinline__ double weight(const Row& r, float x, int& n) {
    const bool counts = x >= r.floor;
    const double v = r.top - (double)(counts ? x : (float)r.top);
    const double shift = 6755399441055744.0;                     // 1.5 * 2^52: rounds to a whole number, which the low bits then hold
    const double t = fma(v, r.per * FINE, shift);
    n = __double2loint(t);
    const double f = fma(v, r.per * FINE, shift - t);
    constexpr double L = 0.69314718055994530942 / FINE;
    double q = fma(f, L * L * L * L / 24, -L * L * L / 6);
    q = fma(f, q, L * L / 2);
    q = fma(f, q, -L);
    q = fma(f, q, 1.0);
    q *= r.table[n & (FINE - 1)];
    q = __hiloint2double(__double2hiint(q) - ((n / FINE) << 20), __double2loint(q));
    n = counts ? n : 1 << 30;
    return counts ? q : 0.0;
}
__device__ __forceinline__ double weight(const Row& r, float x) {
    int n;
    return weight(r, x, n);
}
// A weight of up to 1 as a whole number: 2^52 + w 2^bits has its whole part in the low 52 bits
__device__ __forceinline__ u64 whole(const Row& r, double w) {
    return (u64)__double_as_longlong(fma(w, r.one, 4503599627370496.0)) & 0xfffffffffffffull;
}

struct Shared {
    double table[FINE];
    u64 slot[2][WARPS];          // per-warp results of a reduction
    uint32_t slot32[2][WARPS];
    u64 scanned[WARPS];          // and of a scan
    uint32_t counted[WARPS];
    u64 part[2][2];              // the CTA's, for its peers
    uint32_t part32[2];
    uint32_t bins[4][BINS];      // counts, and the sums of the weights' low, middle and high 16 bits
    double all_w[BINS];          // of all CTAs
    uint32_t all_n[BINS];
    u64 listed[LIST];            // this CTA's tokens of those that are collected
    u64 exchange[LIST];          // of a sort
    uint32_t listed_n;
    int crossing;
    uint32_t before_n, in_n;     // of the bin that holds a cut: tokens before it, and in it
    double before_w;
    u64 cut;
    double per, deepest;
};

__device__ __forceinline__ u64 bits_of(u64 v) { return v; }
__device__ __forceinline__ u64 bits_of(double v) { return (u64)__double_as_longlong(v); }
__device__ __forceinline__ void of_bits(u64 b, u64& v) { v = b; }
__device__ __forceinline__ void of_bits(u64 b, double& v) { v = __longlong_as_double((long long)b); }

// Results over the cluster, for every thread.  Slots are used in turn: a CTA that is one reduction ahead writes others than its peers still read.
struct Team {
    Shared* s;
    int ctas, me, turn;
    __device__ __forceinline__ void barrier() const {
        if (ctas > 1) cluster_arrive(), cluster_wait();
        else __syncthreads();
    }
    template <typename F> __device__ __forceinline__ uint32_t reduce32(uint32_t v, F warp_all) {
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        turn ^= 1;
        v = warp_all(v);
        if (lane == 0) s->slot32[turn][warp] = v;
        __syncthreads();
        v = warp_all(lane < WARPS ? s->slot32[turn][lane] : 0);
        if (ctas == 1) return v;
        if (threadIdx.x == 0) s->part32[turn] = v;
        barrier();
        return warp_all(lane < ctas ? read_peer(&s->part32[turn], lane) : 0);
    }
    __device__ __forceinline__ uint32_t max(uint32_t v) { return reduce32(v, [](uint32_t t) { return __reduce_max_sync(0xffffffffu, t); }); }
    __device__ __forceinline__ uint32_t sum(uint32_t v) { return reduce32(v, [](uint32_t t) { return __reduce_add_sync(0xffffffffu, t); }); }
    // Two sums under one barrier
    template <typename W> __device__ __forceinline__ void sum(W& a, uint32_t& b) {
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        turn ^= 1;
        a = warp_sum64(a), b = __reduce_add_sync(0xffffffffu, b);
        if (lane == 0) s->slot[turn][warp] = bits_of(a), s->slot32[turn][warp] = b;
        __syncthreads();
        of_bits(lane < WARPS ? s->slot[turn][lane] : 0, a);
        a = warp_sum64(a), b = __reduce_add_sync(0xffffffffu, lane < WARPS ? s->slot32[turn][lane] : 0);
        if (ctas == 1) return;
        if (threadIdx.x == 0) s->part[turn][0] = bits_of(a), s->part32[turn] = b;
        barrier();
        of_bits(lane < ctas ? read_peer(&s->part[turn][0], lane) : 0, a);
        a = warp_sum64(a), b = __reduce_add_sync(0xffffffffu, lane < ctas ? read_peer(&s->part32[turn], lane) : 0);
    }
};

// Sums over the threads up to this one, of whole numbers or floats; `all`: over all of them.  Every thread passes two barriers.
template <typename W> __device__ __forceinline__ W scan_cta(W v, u64* slots, W& all) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const W t = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += t;
    }
    __syncthreads();
    if (lane == 31) slots[warp] = bits_of(v);
    __syncthreads();
    W before = 0, t;
    all = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
        of_bits(slots[w], t);
        if (w == warp) before = all;
        all += t;
    }
    return before + v;
}

// One number a thread, the largest first.  Only the first `n` threads hold any; the others hold 0 and get 0.
__device__ __forceinline__ u64 sort_cta(u64 v, int n, u64* exchange) {
    const int tid = threadIdx.x;
    int most = 32;
    while (most < n) most *= 2;
    for (int size = 2; size <= most; size *= 2)
        for (int stride = size / 2; stride > 0; stride /= 2) {
            u64 t;
            if (stride < 32) {
                t = __shfl_xor_sync(0xffffffffu, v, stride);
            } else {
                __syncthreads();
                exchange[tid] = v;
                __syncthreads();
                t = exchange[tid ^ stride];
            }
            const bool larger = ((tid & size) == 0) == ((tid & stride) == 0);       // which of the two this thread keeps
            v = (v > t) == larger ? v : t;
        }
    return v;
}

// A CTA's slice, four values at a time; beyond its end -infinity.  Kept in shared memory, or read from memory and made clean again every time.
template <bool RESIDENT> struct Slice {
    const float* x;
    float4* kept;
    int n;
    bool endless;                // the largest is +infinity: such logits share the probability, as if they were 0 and the others masked
    __device__ __forceinline__ float4 load(int i4) const {
        const int i = 4 * i4;
        return make_float4(clean(x[i]), i + 1 < n ? clean(x[i + 1]) : -INFINITY, i + 2 < n ? clean(x[i + 2]) : -INFINITY,
                           i + 3 < n ? clean(x[i + 3]) : -INFINITY);
    }
    __device__ __forceinline__ void get(int i4, float (&v)[4]) const {
        const float4 t = RESIDENT ? kept[i4] : load(i4);
        v[0] = t.x, v[1] = t.y, v[2] = t.z, v[3] = t.w;
        if (endless)
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = v[j] == INFINITY ? 0.f : -INFINITY;
    }
};

template <bool RESIDENT>
__global__ void __launch_bounds__(THREADS, 2)
sample_filtered_kernel(const float* __restrict__ logits_, long long ld, int R, int V, int per_cta, const float* __restrict__ temperature_,
                       const float* __restrict__ u_, const int* __restrict__ top_k_, const float* __restrict__ top_p_,
                       const float* __restrict__ min_p_, const int* __restrict__ rows_, int* __restrict__ out, int* __restrict__ kept_out,
                       float* __restrict__ logprob_out, int* err) {
    extern __shared__ __align__(16) float slice_memory[];
    __shared__ Shared sh;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    Team team;
    team.s = &sh;
    team.ctas = gridDim.x;
    team.me = team.ctas > 1 ? (int)rank_in_cluster() : 0;
    team.turn = 0;
    if (tid < FINE) sh.table[tid] = exp2(-tid / (double)FINE);
    pdl_trigger();
    pdl_wait();
    const int row = rows_ ? pdl_fresh(rows_)[blockIdx.y] : blockIdx.y;
    if (row < 0 || row >= R) {                                     // the same for the whole cluster: nobody waits for anybody
        if (tid == 0) report_error(err, PRISM_ERR_ROW_RANGE);
        return;
    }
    const int c0 = min(team.me * per_cta, V), n = min(per_cta, V - c0), nv = (n + 3) / 4;
    Slice<RESIDENT> slice;
    slice.x = pdl_fresh(logits_) + (size_t)row * ld + c0;
    slice.kept = reinterpret_cast<float4*>(slice_memory);
    slice.n = n;
    slice.endless = false;
    const float T = temperature_ ? pdl_fresh(temperature_)[row] : 0.f;
    const int k = top_k_ ? pdl_fresh(top_k_)[row] : 0;
    const float p = top_p_ ? pdl_fresh(top_p_)[row] : 1.f, mp = min_p_ ? fminf(pdl_fresh(min_p_)[row], 1.f) : 0.f;
    const float u = pdl_fresh(u_)[row];

    float top = -INFINITY;
    if (RESIDENT && (reinterpret_cast<uintptr_t>(slice.x) & 15) == 0) {
        constexpr int AHEAD = 10;                                  // loads in flight: 80 KB a CTA
        const float4* x4 = reinterpret_cast<const float4*>(slice.x);
        const int n4 = n / 4;
        for (int i0 = tid; i0 < n4; i0 += AHEAD * THREADS) {
            float4 v[AHEAD];
#pragma unroll
            for (int j = 0; j < AHEAD; ++j)
                if (i0 + j * THREADS < n4) v[j] = __ldcs(x4 + i0 + j * THREADS);
#pragma unroll
            for (int j = 0; j < AHEAD; ++j)
                if (i0 + j * THREADS < n4) {
                    v[j] = make_float4(clean(v[j].x), clean(v[j].y), clean(v[j].z), clean(v[j].w));
                    top = fmaxf(fmaxf(top, fmaxf(v[j].x, v[j].y)), fmaxf(v[j].z, v[j].w));
                    slice.kept[i0 + j * THREADS] = v[j];
                }
        }
        if (n4 < nv && tid == 0) {
            const float4 v = slice.kept[n4] = slice.load(n4);
            top = fmaxf(fmaxf(top, fmaxf(v.x, v.y)), fmaxf(v.z, v.w));
        }
    } else {
#pragma unroll 4
        for (int i = tid; i < nv; i += THREADS) {
            const float4 v = slice.load(i);
            if (RESIDENT) slice.kept[i] = v;
            top = fmaxf(fmaxf(top, fmaxf(v.x, v.y)), fmaxf(v.z, v.w));
        }
    }
    if (tid == THREADS - 1) {                                      // for all, behind the barrier of the largest logit
        sh.per = 1.44269504088896340736 / (double)T;
        sh.deepest = mp > 0.f ? -log2((double)mp) : INFINITY;
    }
    top = value_of(team.max(key_of(top)));
    if (!(T > 0.f) || top == -INFINITY) {
        uint32_t best = 0;                                         // complement of the lowest index
        if (top > -INFINITY)
            for (int i = tid; i < nv; i += THREADS) {
                float v[4];
                slice.get(i, v);
#pragma unroll
                for (int j = 3; j >= 0; --j)
                    if (v[j] == top) best = max(best, ~(uint32_t)(c0 + 4 * i + j));
            }
        best = team.max(best);
        const bool none = top == -INFINITY;
        if (team.me == 0 && tid == 0) {
            out[row] = none ? 0 : (int)~best;
            if (kept_out) kept_out[row] = none ? 0 : 1;
            if (logprob_out) logprob_out[row] = none ? -INFINITY : 0.f;
        }
        team.barrier();                                            // peers may still read this CTA's part
        return;
    }
    if (top == INFINITY) slice.endless = true, top = 0.f;
    Row r;
    r.top = (double)top;
    r.per = sh.per;
    r.floor = __double2float_ru(r.top - 1000.0 / r.per);
    const int bits = min(46, 63 - (31 - __clz(V)));                // V weights of 1 stay below 2^64
    r.one = (double)(1ull << bits);
    r.table = sh.table;
    // min_p as the lowest value that it keeps
    float lowest = LEAST;
    if (mp > 0.f) {
        lowest = fmaxf(LEAST, __double2float_rd(r.top - sh.deepest / r.per));
        for (int i = 0; i < 4 && lowest < top && depth(r, lowest) > sh.deepest; ++i) lowest = nextafterf(lowest, INFINITY);
    }

    u64 cut = 0;                 // kept are the tokens from this place on upwards ...
    u64 most = ~0ull;            // ... and as many at most
    double target = -1;          // weight of the prefix that top_p asks for, once known
    bool few = false;            // the kept tokens are among the collected ones, one a thread of CTA 0
    u64 mine = 0;                // the collected token of this thread
    int few_n = 0;
    auto weight_at = [&](u64 place) { return weight(r, value_at(place)); };

    // The tokens with `which(value, index)` from `low` up to `high`, at most LIST of them in all: one a thread, for CTA 0 or (`for_all`) every CTA.
    // Returns their number.
    auto collect = [&](float low, float high, auto which, bool for_all) {
        if (tid == 0) sh.listed_n = 0;
        __syncthreads();
#pragma unroll 2
        for (int i = tid; i < nv; i += THREADS) {
            float v[4];
            slice.get(i, v);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (v[j] >= low && v[j] <= high && which(v[j], c0 + 4 * i + j)) {
                    const uint32_t at = atomicAdd(&sh.listed_n, 1u);
                    if (at < LIST) sh.listed[at] = place_of(v[j], c0 + 4 * i + j);
                }
        }
        team.barrier();
        mine = 0;
        if (team.ctas == 1) {
            const int have = min((int)sh.listed_n, LIST);
            if (tid < have) mine = sh.listed[tid];
            return have;
        }
        if (!for_all && team.me != 0) return 0;
        const int m = lane < team.ctas ? min((int)read_peer(&sh.listed_n, lane), LIST) : 0;
        int upto = m;
#pragma unroll
        for (int o = 1; o < MOST_CTAS; o <<= 1) {
            const int t = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += t;
        }
        int from = 0, at = tid;
#pragma unroll
        for (int c = 0; c < MOST_CTAS; ++c) {
            const int end = __shfl_sync(0xffffffffu, upto, c), count = __shfl_sync(0xffffffffu, m, c);
            if (tid >= end - count && tid < end) from = c, at = tid - (end - count);
        }
        const int have = min(__shfl_sync(0xffffffffu, upto, MOST_CTAS - 1), LIST);
        if (tid < have) mine = read_peer(&sh.listed[at], from);
        return have;
    };

    // Finds where the first k tokens end (by_weight false) or the shortest prefix of weight p of what `cut` leaves (true): in `cut`, or among
    // the collected tokens (`few`)
    auto search = [&](auto kind) {
        constexpr bool by_weight = decltype(kind)::value;
        // Bins by depth, from `octave` on (tokens are counted by their depth at temperature 1), or (`placed`) by place, from `high` down in steps
        // of 2^shift.  All that counts at a level lies between the values lo_v and hi_v.
        bool placed = false;
        u64 high = 0;
        int shift = 0, octave = 0;
        float lo_v = cut ? value_at(cut) : LEAST, hi_v = top;
        uint32_t base_n = 0;
        double base_w = 0;
        const float per32 = 1.44269504f * STEPS;
        // A token's bin; BINS: behind them all, -1: before them (by depth, what is before them is above hi_v and has 0).  fine: its weight's steps
        auto bin_of = [&](float v, int i, int fine) {
            if (placed) {
                const u64 at = place_of(v, i);
                return at > high ? -1 : (int)min((high - at) >> shift, (u64)BINS);
            }
            if (by_weight) return min(max(0, fine / (FINE / STEPS) - octave * STEPS), BINS);
            const float at = (top - v) * per32 - (float)(octave * STEPS);
            return at < (float)BINS ? (int)fmaxf(at, 0.f) : BINS;
        };
        auto fine_of = [&](float v) {
            int n = 0;
            if (by_weight && !placed) weight(r, v, n);
            return n;
        };
        // A value below all of the bins up to b: a border with room for rounding, for a first look
        auto below = [&](int b) {
            if (placed) return fmaxf(LEAST, value_at(high - min(high, (u64)(b + 1) << shift)));
            const double d = octave + (b + 1.0) / STEPS;
            const double v = (double)top - (by_weight ? d / r.per : d * 0.69314718055994530942);
            return fmaxf(LEAST, (float)(v - 1e-6 * (fabs(v) + fabs((double)top))));
        };
        for (int level = 0; level < 16; ++level) {
#pragma unroll
            for (int j = 0; j < (by_weight ? 4 : 1); ++j) sh.bins[j][tid] = 0;
            if (tid == 0) sh.crossing = BINS;
            __syncthreads();
            double tail = 0;                                       // beyond the bins: weight, at level 0 only, and number of tokens
            uint32_t tail_n = 0;
#pragma unroll 2
            for (int i = tid; i < nv; i += THREADS) {
                float v[4];
                slice.get(i, v);
                bool on[4], any = false;
#pragma unroll
                for (int j = 0; j < 4; ++j) any |= on[j] = v[j] >= lo_v && v[j] <= hi_v;
                if (!any) continue;
                double w[4];
                int fine[4];
                if (by_weight)
#pragma unroll
                    for (int j = 0; j < 4; ++j) w[j] = weight(r, v[j], fine[j]);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (!on[j] || (cut && place_of(v[j], c0 + 4 * i + j) < cut)) continue;
                    const int b = bin_of(v[j], c0 + 4 * i + j, by_weight ? fine[j] : 0);
                    if (b < 0) continue;
                    if (b == BINS) {
                        ++tail_n;
                        if (by_weight && level == 0) tail += w[j];
                        continue;
                    }
                    atomicAdd(&sh.bins[0][b], 1u);
                    if (by_weight) {                               // of about 2^47: 16 bits of it at a time, so that 65,535 fit in 32
                        const int oct = placed ? octave : octave + b / STEPS;
                        const u64 m = (u64)__double_as_longlong(fma(w[j], power_of_two(47 + oct), 4503599627370496.0)) & 0xfffffffffffffull;
                        atomicAdd(&sh.bins[1][b], (uint32_t)m & 0xffffu);
                        atomicAdd(&sh.bins[2][b], (uint32_t)(m >> 16) & 0xffffu);
                        atomicAdd(&sh.bins[3][b], (uint32_t)(m >> 32));
                    }
                }
            }
            // the barriers of these sums are those of the bins
            if (by_weight) team.sum(tail, tail_n);
            else tail_n = team.sum(tail_n);
            uint32_t in = 0, n_all;
            double w_in = 0, w_all = 0, w_upto = 0;
            if (by_weight) {
                // each CTA adds up its share of the bins, a lane a CTA's, and tells all
                const int ctas = team.ctas, b = team.me * (BINS / ctas) + tid / ctas, c = tid % ctas;
                if (ctas > 1) {
                    u64 n_l0 = (u64)read_peer(&sh.bins[0][b], c) << 40;           // the low limbs' sum of 8 CTAs has 35 bits
                    n_l0 += read_peer(&sh.bins[1][b], c);
                    u64 l1 = read_peer(&sh.bins[2][b], c), l2 = read_peer(&sh.bins[3][b], c);
                    for (int o = 1; o < ctas; o <<= 1) {
                        n_l0 += __shfl_xor_sync(0xffffffffu, n_l0, o);
                        l1 += __shfl_xor_sync(0xffffffffu, l1, o);
                        l2 += __shfl_xor_sync(0xffffffffu, l2, o);
                    }
                    const double l0 = (double)(n_l0 & 0xffffffffffull);
                    write_peer(&sh.all_w[b], c, fma((double)l2, 4294967296.0, fma((double)l1, 65536.0, l0)));
                    write_peer(&sh.all_n[b], c, (uint32_t)(n_l0 >> 40));
                    team.barrier();
                    in = sh.all_n[tid], w_in = sh.all_w[tid];
                } else {
                    in = sh.bins[0][tid];
                    w_in = fma((double)sh.bins[3][tid], 4294967296.0, fma((double)sh.bins[2][tid], 65536.0, (double)sh.bins[1][tid]));
                }
                w_in *= power_of_two(-47 - (placed ? octave : octave + tid / STEPS));
                w_upto = base_w + scan_cta<double>(w_in, sh.scanned, w_all);
            } else {
                uint32_t part[MOST_CTAS];
#pragma unroll
                for (int c = 0; c < MOST_CTAS; ++c)
                    part[c] = c >= team.ctas ? 0 : team.ctas > 1 ? read_peer(&sh.bins[0][tid], c) : sh.bins[0][tid];
#pragma unroll
                for (int c = 0; c < MOST_CTAS; ++c) in += part[c];
            }
            u64 n_all64;
            const uint32_t upto = base_n + (uint32_t)scan_cta<u64>(in, sh.scanned, n_all64);
            n_all = (uint32_t)n_all64;
            if (level == 0) {
                if (by_weight) {
                    target = fmax((double)p, 0.0) * (w_all + tail);
                } else if (n_all + tail_n <= (uint32_t)k) {        // fewer tokens than top_k asks for
                    team.barrier();                                // the bins may be cleared again
                    return;
                }
            }
            const bool last_resort = tail_n == 0;                  // by rounding a weight may end just below the target
            if (in > 0 && (by_weight ? w_upto >= target && w_upto > 0 : upto >= (uint32_t)k)) atomicMin(&sh.crossing, tid);
            __syncthreads();
            if (sh.crossing == BINS && last_resort) {
                __syncthreads();
                if (in > 0 && upto == base_n + n_all) atomicMin(&sh.crossing, tid);
                __syncthreads();
            }
            const int b = sh.crossing;
            if (tid == b) sh.before_n = upto - in, sh.in_n = in, sh.before_w = w_upto - w_in;
            __syncthreads();
            auto of_bin = [&](float v, int i) { return bin_of(v, i, fine_of(v)) == b && (!cut || place_of(v, i) >= cut); };
            if (b < BINS) {
                const uint32_t before_n = sh.before_n, in_n = sh.in_n;
                const double before_w = sh.before_w;
                lo_v = fmaxf(lo_v, below(b));
                if (before_n + in_n <= LIST) {
                    few_n = collect(lo_v, top, [&](float v, int i) { return bin_of(v, i, fine_of(v)) <= b && (!cut || place_of(v, i) >= cut); }, false);
                    few = true;
                    return;
                }
                if (in_n <= LIST) {
                    const int got = collect(lo_v, hi_v, of_bin, true);
                    mine = sort_cta(mine, got, sh.exchange);
                    // the first of them that reaches the target, else the last
                    double run = 0, rest;
                    if (by_weight) run = before_w + scan_cta<double>(tid < got ? weight_at(mine) : 0, sh.scanned, rest);
                    if (tid == 0) sh.crossing = got - 1;
                    __syncthreads();
                    if (tid < got && (by_weight ? run >= target : before_n + tid + 1 >= (uint32_t)k)) atomicMin(&sh.crossing, tid);
                    __syncthreads();
                    if (tid == sh.crossing) sh.cut = mine;
                    __syncthreads();
                    cut = sh.cut;
                    __syncthreads();
                    return;
                }
                base_n = before_n, base_w = before_w;
            } else {
                base_n += n_all, base_w += w_all;                  // the cut is among the tail
            }
            // the places of the bin's tokens, or of the tail's: their range is what is divided next
            u64 lo = 0, hi = 0;                                    // complement of the lowest, and the highest
#pragma unroll 2
            for (int i = tid; i < nv; i += THREADS) {
                float v[4];
                slice.get(i, v);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (v[j] >= lo_v && v[j] <= hi_v && of_bin(v[j], c0 + 4 * i + j)) {
                        const u64 at = place_of(v[j], c0 + 4 * i + j);
                        hi = at > hi ? at : hi;
                        lo = ~at > lo ? ~at : lo;
                    }
            }
            // each in two steps: the value, then the index among those that have it
            auto most64 = [&](u64 t) {
                const uint32_t h = team.max((uint32_t)(t >> 32));
                return ((u64)h << 32) | team.max((uint32_t)(t >> 32) == h ? (uint32_t)t : 0);
            };
            hi = most64(hi);
            lo = ~most64(lo);
            hi_v = value_at(hi), lo_v = value_at(lo);
            if (!by_weight && hi_v < r.floor) {                    // what lies there weighs nothing: which of it is kept makes no difference
                most = (u64)k;
                return;
            }
            const double next = by_weight ? depth(r, hi_v) : (double)(top - hi_v) * 1.4426950408889634;
            if (!placed && b == BINS && level < 4 && next < 500.0) {
                octave = max((int)next, octave);
            } else {
                placed = true;
                high = hi;
                shift = max(0, 64 - __clzll((long long)(hi - lo)) - 9);
                octave = (int)fmin(depth(r, hi_v), 900.0);
            }
        }
    };
    if (k > 0 && k < V) search(std::integral_constant<bool, false>());
    if (!few && p < 1.f) search(std::integral_constant<bool, true>());

    if (few) {
        if (team.ctas > 1) cluster_arrive();
        if (team.me == 0) {
            // CTA 0 has all that can be kept: in order, cut, then by index
            mine = sort_cta(mine, few_n, sh.exchange);
            int len = k > 0 ? min(k, few_n) : few_n;
            float v = value_at(mine);
            if (p < 1.f) {
                double all;
                const double run = scan_cta<double>(tid < len ? weight(r, v) : 0, sh.scanned, all);
                if (target < 0) target = fmax((double)p, 0.0) * all;
                if (tid == 0) sh.crossing = len - 1;
                __syncthreads();
                if (tid < len && run >= target) atomicMin(&sh.crossing, tid);
                __syncthreads();
                len = sh.crossing + 1;
            }
            const bool keep = tid < len && v >= lowest;
            const int count = __syncthreads_count(keep);
            const uint32_t index = ~(uint32_t)mine;
            mine = sort_cta(keep ? ((u64)~index << 32) | (mine >> 32) : 0, count, sh.exchange);
            v = value_of((uint32_t)mine);
            const u64 own = tid < count ? whole(r, weight(r, v)) : 0;
            u64 total;
            const u64 upto = scan_cta<u64>(own, sh.scanned, total);
            const double goal = u < 1.f ? fmax((double)u, 0.0) * (double)total : (double)(total - 1);
            if ((double)upto > goal && !((double)(upto - own) > goal)) {
                out[row] = (int)~(uint32_t)(mine >> 32);
                if (kept_out) kept_out[row] = count;
                if (logprob_out) logprob_out[row] = (float)(-0.69314718055994530942 * (depth(r, v) + (log2((double)total) - bits)));
            }
        }
        __syncwarp();
        if (team.ctas > 1) cluster_wait();
        return;
    }
    // The draw over the row: every warp a run of neighbours, its weight after those of the runs before it
    const int run = ((nv + WARPS - 1) / WARPS + 31) & ~31;         // in fours
    const int i0 = min(warp * run, nv), i1 = min(i0 + run, nv);
    const float cut_v = cut ? value_at(cut) : LEAST;
    lowest = fmaxf(lowest, cut_v);
    auto kept_weights = [&](int i, u64 (&w)[4], float (&v)[4], uint32_t& count) {
        slice.get(i, v);
        bool on[4], any = false;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            any |= on[j] = v[j] >= lowest && !(cut && v[j] == cut_v && place_of(v[j], c0 + 4 * i + j) < cut);
            w[j] = 0;
        }
        if (any)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const u64 t = whole(r, weight(r, v[j]));
                if (on[j]) w[j] = t, ++count;
            }
        return w[0] + w[1] + w[2] + w[3];
    };
    u64 own = 0, w[4];
    float v[4];
    uint32_t count = 0;
#pragma unroll 2
    for (int i = i0 + lane; i < i1; i += 32) own += kept_weights(i, w, v, count);
    own = warp_sum64(own);
    count = __reduce_add_sync(0xffffffffu, count);
    if (lane == 0) sh.scanned[warp] = own, sh.counted[warp] = count;
    __syncthreads();
    u64 before = 0, total = 0;
    count = 0;
#pragma unroll
    for (int c = 0; c < WARPS; ++c) {
        if (c == warp) before = total;
        total += sh.scanned[c];
        count += sh.counted[c];
    }
    if (team.ctas > 1) {
        if (tid == 0) sh.part[0][0] = total, sh.part[0][1] = count;
        team.barrier();
        const u64 t = lane < team.ctas ? read_peer(&sh.part[0][0], lane) : 0;
        before += warp_sum64(lane < team.me ? t : 0);
        total = warp_sum64(t);
        count = __reduce_add_sync(0xffffffffu, lane < team.ctas ? (uint32_t)read_peer(&sh.part[0][1], lane) : 0);
        cluster_arrive();                                          // nothing of the peers is read any more
    }
    if ((u64)count > most) count = (uint32_t)most;
    const double goal = u < 1.f ? fmax((double)u, 0.0) * (double)total : (double)(total - 1);
    if ((double)(before + own) > goal && !((double)before > goal)) {              // one warp of the cluster: the running weight passes the goal in its run
        uint32_t unused = 0;
        for (int i = i0; i < i1; i += 32) {
            u64 s = i + lane < i1 ? kept_weights(i + lane, w, v, unused) : 0;
            const u64 mine4 = s;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const u64 t = __shfl_up_sync(0xffffffffu, s, o);
                if (lane >= o) s += t;
            }
            const uint32_t passed = __ballot_sync(0xffffffffu, (double)(before + s) > goal);
            if (passed) {
                if (lane == __ffs(passed) - 1) {
                    before += s - mine4;
                    int at = -1;
                    float x = 0;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        before += w[j];
                        if (at < 0 && (double)before > goal) at = c0 + 4 * (i + lane) + j, x = v[j];
                    }
                    out[row] = at;
                    if (kept_out) kept_out[row] = (int)count;
                    if (logprob_out) logprob_out[row] = (float)(-0.69314718055994530942 * (depth(r, x) + (log2((double)total) - bits)));
                }
                break;
            }
            before += __shfl_sync(0xffffffffu, s, 31);
        }
    }
    __syncwarp();
    if (team.ctas > 1) cluster_wait();
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
    if (V < 1 || V > MOST_V || n > 65535 || n > R || u == nullptr || out == nullptr) return (int)cudaErrorInvalidValue;
    int ctas = 1;
    while (ctas < MOST_CTAS && V > 4096 * ctas) ctas *= 2;
    const int per_cta = ((V + ctas - 1) / ctas + 3) & ~3;
    const bool resident = per_cta <= MOST_SLICE;
    const auto kernel = resident ? sample_filtered_kernel<true> : sample_filtered_kernel<false>;
    const size_t smem = resident ? (size_t)per_cta * 4 : 0;
    if (smem > 16 * 1024) prism::open_smem(kernel, MOST_SLICE * 4);              // beside 24 KB of its own
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
    return (int)cudaLaunchKernelEx(&cfg, kernel, logits, ld, R, V, per_cta, temperature, u, top_k, top_p, min_p, rows, out,
                                   kept, logprob, err);
}
