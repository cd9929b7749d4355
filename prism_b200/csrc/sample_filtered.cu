// A token from each row of float32 logits by temperature, top-k, top-p and min-p, at a uniform number u that the host supplies.
//
// With m the row's largest logit and w_i = exp((x_i - m) / T), tokens stand in the order (logit down, index up).  Kept are
// the first top_k of them; of these the shortest prefix whose weight reaches top_p of theirs; of these the ones with w_i >= min_p.
// Each filter keeps a prefix of that order, so together they keep the shortest of the three.  The draw is the inverse CDF in the
// order of the indices, as in sample.cu: the first kept index whose running weight exceeds u times the weight of all kept (u below 0 counts as 0,
// 1 and more and NaN as the largest float32 below 1).
// T <= 0: the largest, lowest index on ties.  NaN counts as -infinity, which is never kept; a row with nothing else gives token 0.
//
// Weights come from 64-bit arithmetic (relative error below 2^-48 + 2^-51 |x_i - m| / T: the series and the rounded 1 / T).  The draw adds them up as whole numbers, w_i * 2^46 rounded: such sums are exact, so neither
// the order of additions nor the number of CTAs that share a row can change them, and every thread sees the same running weight; a draw is decided
// to about 1e-12 of the weight (in float32 one row in thirty over 150,000 tokens would be decided by rounding), and a token of less than 2^-47 is never drawn.  top_p = 0.9999999 ends a
// prefix among weights that such steps do not resolve: its sums are 64-bit floats, added in an order that V alone fixes.
//
// One cluster of CTAs a row: each keeps its slice of the logits in shared memory, so that the row is read once, and the CTAs' sums meet
// through distributed shared memory.  A cut is found without sorting the row: tokens are counted (for top_p: weighed) in 512 bins of
// 1/32 of a power of two down to 2^-16 of the largest, each CTA's in shared memory; after one barrier every thread adds up one bin of all CTAs, and a scan
// shows the bin that holds the cut.   If the tokens down to there are 512 or fewer (a top_k or a nucleus as they are in use), one CTA collects and
// sorts them, one a thread, and draws from them; the other CTAs are done.  Else the bin's own tokens are collected and sorted, if it has
// 512 at most, or divided into 512 bins by the bits of their place in the order (their number there: exact, ties and all), until it has; the
// draw is then a pass over the row.
//
// Measured on a B200, rows of 152,064, microseconds for 1, 16, 64 and 256 of them: top-k with or without top-p 11.6, 15.7, 46, 143; top-p alone 36, 66, 104, 328;
// min-p 10, 13, 26, 108; none 14, 21, 42, 158.  Reading 256 rows takes 24: a few rows are bound by the chain of steps (a barrier of the cluster costs half a
// microsecond with what is read behind it, weighing a CTA's 19,000 tokens 8 us, half of it instructions around the 64-bit ones), many by the turns that
// 33 clusters at a time take, about 15 us each.
#include "common.cuh"

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
constexpr int COPIES = 16;                     // of the table of weights: neighbouring threads read banks of their own
constexpr float LEAST = -3.402823466e38f;      // the lowest value that counts: below is -infinity only
constexpr float PER_LOGIT = 1.44269504f * STEPS;                   // bins of a unit of logits, where tokens are counted

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
__device__ __forceinline__ u64 bits_of(u64 v) { return v; }
__device__ __forceinline__ u64 bits_of(double v) { return (u64)__double_as_longlong(v); }
__device__ __forceinline__ void of_bits(u64 b, u64& v) { v = b; }
__device__ __forceinline__ void of_bits(u64 b, double& v) { v = __longlong_as_double((long long)b); }

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

// What a CTA knows and shares.  The parts of this kernel that a row passes once are functions that are not inlined, and find their operands here:
// inlined everywhere they made 184 KB of code, and a CTA spent more time on fetching it than on its slice.
struct Shared {
    double table[STEPS * COPIES];              // 2^(-j / STEPS)
    u64 slot[2][WARPS];                        // per-warp results of a reduction; slots are used in turn, as a CTA may be one reduction ahead
    uint32_t slot32[2][WARPS];
    u64 scanned[WARPS];                        // and of a scan
    uint32_t counted[WARPS];
    u64 part[2][2];                            // the CTA's, for its peers
    uint32_t part32[2];
    uint32_t bins[4][BINS];                    // counts, and the sums of the weights' low, middle and high 16 bits
    double all_w[BINS];                        // of all CTAs
    uint32_t all_n[BINS];
    u64 listed[LIST];                          // this CTA's tokens of those that are collected
    u64 exchange[LIST];                        // of a sort
    uint32_t listed_n;
    int crossing;
    uint32_t border;
    uint32_t before_n, in_n;                   // of the bin that holds a cut: tokens before it, and in it
    double before_w;
    u64 cut;
    // the row
    const float* x;                            // the CTA's slice
    double top, per, deepest, one;             // largest logit; log2(e) / T; depth of min_p; a weight of 1 as a whole number: 2^46, or less where V of them would not fit
    float floor;                               // tokens below have no weight: it would be less than 2^-999
    float p, u;
    int n, c0, ctas, me, k, bits, row;
    bool endless;                              // the largest is +infinity: such logits share the probability, as if they were 0 and the others masked
};
__shared__ Shared sh;
extern __shared__ __align__(16) float4 kept_slice[];

__device__ __forceinline__ void team_barrier() {
    if (sh.ctas > 1) cluster_arrive(), cluster_wait();
    else __syncthreads();
}
__device__ __forceinline__ uint32_t warp_all(uint32_t v, bool max) {
    return max ? __reduce_max_sync(0xffffffffu, v) : __reduce_add_sync(0xffffffffu, v);
}
// Over the cluster, for every thread
__device__ __noinline__ uint32_t team_reduce(uint32_t v, bool max, int turn) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    v = warp_all(v, max);
    if (lane == 0) sh.slot32[turn][warp] = v;
    __syncthreads();
    v = warp_all(lane < WARPS ? sh.slot32[turn][lane] : 0, max);
    if (sh.ctas == 1) return v;
    if (threadIdx.x == 0) sh.part32[turn] = v;
    team_barrier();
    return warp_all(lane < sh.ctas ? read_peer(&sh.part32[turn], lane) : 0, max);
}
// A weight and a number at once
__device__ __forceinline__ void team_sum(double& v, uint32_t& n, int turn) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    v = warp_sum64(v), n = warp_all(n, false);
    if (lane == 0) sh.slot[turn][warp] = bits_of(v), sh.slot32[turn][warp] = n;
    __syncthreads();
    of_bits(lane < WARPS ? sh.slot[turn][lane] : 0, v);
    v = warp_sum64(v), n = warp_all(lane < WARPS ? sh.slot32[turn][lane] : 0, false);
    if (sh.ctas == 1) return;
    if (threadIdx.x == 0) sh.part[turn][0] = bits_of(v), sh.part32[turn] = n;
    team_barrier();
    of_bits(lane < sh.ctas ? read_peer(&sh.part[turn][0], lane) : 0, v);
    n = lane < sh.ctas ? read_peer(&sh.part32[turn], lane) : 0;
    v = warp_sum64(v), n = warp_all(n, false);
}
// Sums over the threads up to this one; `all`: over all of them.  Every thread passes two barriers.
__device__ __forceinline__ uint32_t scan32(uint32_t v, uint32_t& all) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t t = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += t;
    }
    __syncthreads();
    if (lane == 31) sh.counted[warp] = v;
    __syncthreads();
    const uint32_t t = lane < WARPS ? sh.counted[lane] : 0;
    all = __reduce_add_sync(0xffffffffu, t);
    return v + __reduce_add_sync(0xffffffffu, lane < warp ? t : 0);
}
template <typename W> __device__ __noinline__ W scan64(W v) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const W t = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += t;
    }
    __syncthreads();
    if (lane == 31) sh.scanned[warp] = bits_of(v);
    __syncthreads();
    W t;
    of_bits(lane < warp ? sh.scanned[lane] : 0, t);                // 0 is zero of either kind
    return warp_sum64(t) + v;
}
// after a scan64: what it is for the last thread
template <typename W> __device__ __forceinline__ W scanned_all() {
    const int lane = threadIdx.x & 31;
    W t;
    of_bits(lane < WARPS ? sh.scanned[lane] : 0, t);
    return warp_sum64(t);
}

// One number a thread, the largest first.  Only the first `n` threads hold any; the others hold 0 and get 0.
__device__ __noinline__ u64 sort_cta(u64 v, int n) {
    const int tid = threadIdx.x;
#pragma unroll 1
    for (int size = 2; size / 2 < n; size *= 2)
#pragma unroll 1
        for (int stride = size / 2; stride > 0; stride /= 2) {
            u64 t;
            if (stride < 32) {
                t = __shfl_xor_sync(0xffffffffu, v, stride);
            } else {
                __syncthreads();
                sh.exchange[tid] = v;
                __syncthreads();
                t = sh.exchange[tid ^ stride];
            }
            const bool larger = ((tid & size) == 0) == ((tid & stride) == 0);       // which of the two this thread keeps
            v = (v > t) == larger ? v : t;
        }
    return v;
}

// -log2 of a token's weight, 0 for the largest itself
__device__ __forceinline__ double depth(float x) { return (sh.top - (double)x) * sh.per; }
// 2^-d with d = depth(x) = n / 32 + f / 32, |f| <= 1/2: the second factor by the series of exp(-f ln 2 / 32) to the fifth power (the next term is
// below 2^-48), the first from a table of 32 and the exponent.  n: its step, by which tokens are sorted into bins.  Free of branches, so
// that several tokens' chains of 64-bit operations overlap.
struct Weigher {
    double top, per;
    float floor;
    __device__ __forceinline__ Weigher() : top(sh.top), per(sh.per * STEPS), floor(sh.floor) {}
    // the weight times 2^(n / 32 rounded down): half to one, roundings aside.  n is huge for tokens below the floor.
    __device__ __forceinline__ double scaled(float x, int& n) const {
        const bool counts = x >= floor;
        const double v = top - (double)(counts ? x : (float)top);
        const double shift = 6755399441055744.0;                   // 1.5 * 2^52: rounds to a whole number, which the low bits then hold
        const double t = fma(v, per, shift);
        n = __double2loint(t);
        const double f = fma(v, per, shift - t);
        constexpr double L = 0.69314718055994530942 / STEPS;
        double q = fma(f, -L * L * L * L * L / 120, L * L * L * L / 24);
        q = fma(f, q, -L * L * L / 6);
        q = fma(f, q, L * L / 2);
        q = fma(f, q, -L);
        q = fma(f, q, 1.0);
        q *= sh.table[(n & (STEPS - 1)) * COPIES + threadIdx.x % COPIES];
        n = counts ? n : 1 << 30;
        return q;
    }
    static __device__ __forceinline__ double unscaled(double q, int n) {
        return n < 1 << 30 ? __hiloint2double(__double2hiint(q) - ((n / STEPS) << 20), __double2loint(q)) : 0.0;
    }
    __device__ __forceinline__ double operator()(float x, int& n) const {
        const double q = scaled(x, n);
        return unscaled(q, n);
    }
};
__device__ __noinline__ double weight(float x) {
    int n;
    return Weigher()(x, n);
}
__device__ __noinline__ int step_of(float x) {
    int n;
    Weigher()(x, n);
    return n;
}
// A weight of up to 1 as a whole number: 2^52 + w 2^bits has its whole part in the low 52 bits, above which OFFSET stands
constexpr u64 OFFSET = 0x4330000000000000ull;
__device__ __forceinline__ u64 offset_whole(double w, double one) { return (u64)__double_as_longlong(fma(w, one, 4503599627370496.0)); }
__device__ __forceinline__ u64 whole(double w, double one) { return offset_whole(w, one) - OFFSET; }

// The slice, four values at a time; beyond its end -infinity.  Kept in shared memory, or read from memory and made clean again every time.
__device__ __forceinline__ float4 load_four(const float* x, int n, int i4) {
    const int i = 4 * i4;
    return make_float4(clean(x[i]), i + 1 < n ? clean(x[i + 1]) : -INFINITY, i + 2 < n ? clean(x[i + 2]) : -INFINITY,
                       i + 3 < n ? clean(x[i + 3]) : -INFINITY);
}
template <bool RESIDENT> __device__ __forceinline__ void get(int i4, float (&v)[4], bool endless) {
    const float4 t = RESIDENT ? kept_slice[i4] : load_four(sh.x, sh.n, i4);
    v[0] = t.x, v[1] = t.y, v[2] = t.z, v[3] = t.w;
    if (!RESIDENT && endless)                                      // a slice that is kept has been changed
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = v[j] == INFINITY ? 0.f : -INFINITY;
}

// Lists this CTA's tokens whose values are from low_v up to high_v and whose places are from low_p up to high_p, LIST of them at most.  The caller's
// barrier follows.
template <bool RESIDENT> __device__ __noinline__ void list(float low_v, float high_v, u64 low_p, u64 high_p) {
    if (threadIdx.x == 0) sh.listed_n = 0;
    __syncthreads();
    const bool endless = sh.endless;
    const int nv = (sh.n + 3) / 4, c0 = sh.c0;
#pragma unroll 2
    for (int i = threadIdx.x; i < nv; i += THREADS) {
        float v[4];
        get<RESIDENT>(i, v, endless);
        if (!(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])) >= low_v)) continue;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (v[j] >= low_v && v[j] <= high_v) {
                const u64 at = place_of(v[j], c0 + 4 * i + j);
                if (at < low_p || at > high_p) continue;
                const uint32_t slot = atomicAdd(&sh.listed_n, 1u);
                if (slot < LIST) sh.listed[slot] = at;
            }
    }
}
// Behind the barrier: how many all CTAs have listed
__device__ __forceinline__ int listed() {
    const int lane = threadIdx.x & 31;
    return (int)__reduce_add_sync(0xffffffffu, sh.ctas == 1 ? (lane == 0 ? sh.listed_n : 0) : lane < sh.ctas ? read_peer(&sh.listed_n, lane) : 0);
}
// If these are at most LIST: one a thread, 0 for the threads behind them
__device__ __noinline__ u64 take() {
    const int tid = threadIdx.x, lane = tid & 31;
    if (sh.ctas == 1) return tid < (int)sh.listed_n ? sh.listed[tid] : 0;
    const int m = lane < sh.ctas ? (int)read_peer(&sh.listed_n, lane) : 0;
    int upto = m;
#pragma unroll
    for (int o = 1; o < MOST_CTAS; o <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += t;
    }
    int from = -1, at = 0;
#pragma unroll
    for (int c = 0; c < MOST_CTAS; ++c) {
        const int end = __shfl_sync(0xffffffffu, upto, c), count = __shfl_sync(0xffffffffu, m, c);
        if (tid >= end - count && tid < end) from = c, at = tid - (end - count);
    }
    return from >= 0 ? read_peer(&sh.listed[at], from) : 0;
}

// A thread's bin of all CTAs' counts
__device__ __forceinline__ uint32_t counted_in() {
    if (sh.ctas == 1) return sh.bins[0][threadIdx.x];
    uint32_t part[MOST_CTAS], in = 0;
#pragma unroll
    for (int c = 0; c < MOST_CTAS; ++c) part[c] = c < sh.ctas ? read_peer(&sh.bins[0][threadIdx.x], c) : 0;
#pragma unroll
    for (int c = 0; c < MOST_CTAS; ++c) in += part[c];
    return in;
}

// A first try, for a small top_k: the threads' largest values (`first`) are counted in bins, and down to the bin of the k-th of them there are at least k
// tokens, seldom many more: these hold all that can be kept.  Returns their number if they are few: then the first CTA's threads have one each in
// `mine`; else -1.
template <bool RESIDENT> __device__ __noinline__ int attempt(float first, u64& mine) {
    const int tid = threadIdx.x, k = sh.k;
    const float top = (float)sh.top;
    sh.bins[0][tid] = 0;
    if (tid == 0) sh.crossing = BINS;
    __syncthreads();
    if (first > -INFINITY) atomicAdd(&sh.bins[0][(int)fminf((top - first) * PER_LOGIT, BINS - 1.f)], 1u);
    team_barrier();
    uint32_t all;
    const uint32_t in = counted_in(), upto = scan32(in, all);
    if (upto >= (uint32_t)k && upto - in < (uint32_t)k) sh.crossing = tid;
    __syncthreads();
    const int b = sh.crossing;
    int n = LIST + 1;
    if (b != BINS - 1) {
        float low = LEAST;                                         // fewer than k threads have any token: all tokens, if they are few
        if (b < BINS) {
            const float d = (float)(b + 1) / PER_LOGIT;
            low = fmaxf(LEAST, top - d - 1e-6f * (d + fabsf(top)));
        }
        list<RESIDENT>(low, top, 0, ~0ull);
        team_barrier();
        n = listed();
    }
    if (n <= LIST) {
        if (sh.me == 0) mine = take();
        return n;
    }
    team_barrier();                                                // peers may still read bins and lengths
    return -1;
}

// What a search goes by: bins by depth, from `octave` on (tokens are counted by their depth at temperature 1), or (`placed`) by place, from `high` down in
// steps of 2^shift.  All that counts lies between the values lo_v and hi_v and the places low and high.
struct Range {
    bool by_weight, placed;
    int shift, octave;
    u64 low, high;
    float lo_v, hi_v;
};
// A token's bin by depth, BINS: behind them all; step: its weight's
__device__ __forceinline__ int bin_of(bool by_weight, int octave, float v, int step) {
    if (by_weight) return min(max(0, step - octave * STEPS), BINS);
    const float at = ((float)sh.top - v) * PER_LOGIT - (float)(octave * STEPS);
    return at < (float)BINS ? (int)fmaxf(at, 0.f) : BINS;
}
// The lowest value whose bin by depth is b or before it.  A value's bin is what bin_of() says, roundings and all, so the border is searched for by it: THREADS
// values at once, from a border by arithmetic with room for rounding on either side.
__device__ __noinline__ float border(bool by_weight, int octave, int b) {
    const double d = octave + (b + (by_weight ? 0.5 : 1.0)) / STEPS;
    const double v = sh.top - (by_weight ? d / sh.per : d * 0.69314718055994530942), room = 1e-6 * (fabs(v) + fabs(sh.top));
    // rounded outwards: among the smallest numbers a float's step is wider than the room
    uint32_t out = key_of(fmaxf(LEAST, __double2float_rd(v - room))), in = key_of(fminf((float)sh.top, fmaxf(LEAST, __double2float_ru(v + room))));
    if (out > in) out = in;
    // `in` has a bin up to b; the border is not below `out`
#pragma unroll 1
    while (out < in) {                                             // at most four rounds
        const uint32_t stride = (in - out) / THREADS + 1;
        const u64 at = (u64)out + (u64)stride * threadIdx.x;
        if (threadIdx.x == 0) sh.border = in;
        __syncthreads();
        if (at < in) {
            const float x = value_of((uint32_t)at);
            if (bin_of(by_weight, octave, x, by_weight ? step_of(x) : 0) <= b) atomicMin(&sh.border, (uint32_t)at);
        }
        __syncthreads();
        const uint32_t found = sh.border;
        __syncthreads();
        const uint32_t steps = (found - out + stride - 1) / stride;            // values tried that are outside: the border lies behind the last of them
        out = steps == 0 ? found : out + (steps - 1) * stride + 1;
        in = found;
    }
    return value_of(in);
}

// A token into its bin; false: it is behind them all.  Weights: of about 2^47, 16 bits at a time, so that 65,000 of them fit in 32.
__device__ __forceinline__ bool put(const Range& r, u64 at, float v, double w, int step) {
    const int b = r.placed ? (int)((r.high - at) >> r.shift) : bin_of(r.by_weight, r.octave, v, step);
    if (b >= BINS) return false;
    atomicAdd(&sh.bins[0][b], 1u);
    if (r.by_weight) {
        const int oct = r.placed ? r.octave : r.octave + b / STEPS;
        const u64 m = (u64)__double_as_longlong(fma(w, power_of_two(47 + oct), 4503599627370496.0)) - OFFSET;
        atomicAdd(&sh.bins[1][b], (uint32_t)m & 0xffffu);
        atomicAdd(&sh.bins[2][b], (uint32_t)(m >> 16) & 0xffffu);
        atomicAdd(&sh.bins[3][b], (uint32_t)(m >> 32));
    }
    return true;
}
// The first time for all of the slice's tokens, as the most of the time goes here: bins by depth from 0 on, four tokens side by side.  `tail`, `tail_n`: weight
// and number of those behind the bins.
template <bool RESIDENT, bool BY_WEIGHT> __device__ __noinline__ void fill_first(double& tail_out, uint32_t& tail_n_out) {
    const Weigher weigh;
    const bool endless = sh.endless;
    const int nv = (sh.n + 3) / 4;
    double tail = 0;
    uint32_t tail_n = 0;
#pragma unroll 1
    for (int i = threadIdx.x; i < nv; i += THREADS) {
        float v[4];
        get<RESIDENT>(i, v, endless);
        if (BY_WEIGHT) {
            double q[4];
            int step[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) q[j] = weigh.scaled(v[j], step[j]);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (step[j] < BINS) {
                    const u64 m = offset_whole(q[j], 140737488355328.0);          // 2^47
                    atomicAdd(&sh.bins[0][step[j]], 1u);
                    atomicAdd(&sh.bins[1][step[j]], (uint32_t)m & 0xffffu);
                    atomicAdd(&sh.bins[2][step[j]], (uint32_t)m >> 16);
                    atomicAdd(&sh.bins[3][step[j]], (uint32_t)(m >> 32) & 0xfffffu);
                } else if (v[j] >= LEAST) {
                    tail += Weigher::unscaled(q[j], step[j]);
                    ++tail_n;
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int b = bin_of(false, 0, v[j], 0);
                if (b < BINS) atomicAdd(&sh.bins[0][b], 1u);
                else tail_n += v[j] >= LEAST;
            }
        }
    }
    tail_out = tail, tail_n_out = tail_n;
}
// Later the slice's tokens of a range
template <bool RESIDENT> __device__ __noinline__ void fill(const Range& range, double& tail_out, uint32_t& tail_n_out) {
    const Range r = range;
    const Weigher weigh;
    const bool endless = sh.endless;
    const int nv = (sh.n + 3) / 4, c0 = sh.c0;
    double tail = 0;
    uint32_t tail_n = 0;
#pragma unroll 1
    for (int i = threadIdx.x; i < nv; i += THREADS) {
        float v[4];
        get<RESIDENT>(i, v, endless);
        if (!(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])) >= r.lo_v)) continue;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const u64 at = place_of(v[j], c0 + 4 * i + j);
            if (v[j] < r.lo_v || v[j] > r.hi_v || at < r.low || at > r.high) continue;
            int step = 0;
            const double w = r.by_weight ? weigh(v[j], step) : 0.0;
            if (!put(r, at, v[j], w, step)) tail += w, ++tail_n;
        }
    }
    tail_out = tail, tail_n_out = tail_n;
}

// Finds where the first k tokens end (by_weight false) or the shortest prefix of weight p of the tokens from the place `cut` on (true).  Returns the place
// of its last token; or, if the tokens down to its bin are few, their number in few_n, and each of the first CTA's threads has one in `mine`.  target:
// the weight that is asked for.
template <bool RESIDENT> __device__ __noinline__ u64 search(bool by_weight, u64 cut, int& turn, int& few_n, u64& mine, double& target) {
    const int tid = threadIdx.x;
    Range r;
    r.by_weight = by_weight, r.placed = false, r.shift = r.octave = 0, r.low = cut, r.high = ~0ull, r.lo_v = LEAST, r.hi_v = (float)sh.top;
    uint32_t base_n = 0, in_n = ~0u;
    double base_w = 0;
#pragma unroll 1
    for (int level = 0; level < 16; ++level) {
#pragma unroll
        for (int j = 0; j < 4; ++j) sh.bins[j][tid] = 0;
        if (tid == 0) sh.crossing = BINS;
        double tail = 0;
        uint32_t tail_n = 0;
        bool from_list = false;
        if (in_n <= MOST_CTAS * LIST) {                            // few of the slice's tokens are in the range: listed, one a thread, if they fit
            list<RESIDENT>(r.lo_v, r.hi_v, r.low, r.high);
            __syncthreads();
            from_list = sh.listed_n <= LIST;
        } else {
            __syncthreads();
        }
        if (from_list) {
            if (tid < (int)sh.listed_n) {
                const u64 at = sh.listed[tid];
                put(r, at, value_at(at), by_weight ? weight(value_at(at)) : 0, 0);
            }
        } else if (level > 0 || cut) {
            fill<RESIDENT>(r, tail, tail_n);
        } else if (by_weight) {
            fill_first<RESIDENT, true>(tail, tail_n);
        } else {
            fill_first<RESIDENT, false>(tail, tail_n);
        }
        // the barrier of these sums is that of the bins
        if (by_weight && level == 0) team_sum(tail, tail_n, turn ^= 1);
        else tail_n = team_reduce(tail_n, false, turn ^= 1);
        uint32_t in, n_all;
        double w_in = 0, w_all = 0, w_upto = 0;
        if (by_weight) {
            // each CTA adds up its share of the bins, a lane a CTA's, and tells all
            const int ctas = sh.ctas, b = sh.me * (BINS / ctas) + tid / ctas, c = tid % ctas;
            if (ctas > 1) {
                u64 n_l0 = (u64)read_peer(&sh.bins[0][b], c) << 40;               // the low limbs' sum of 8 CTAs has 35 bits
                n_l0 += read_peer(&sh.bins[1][b], c);
                u64 l1 = read_peer(&sh.bins[2][b], c), l2 = read_peer(&sh.bins[3][b], c);
#pragma unroll 1
                for (int o = 1; o < ctas; o <<= 1) {
                    n_l0 += __shfl_xor_sync(0xffffffffu, n_l0, o);
                    l1 += __shfl_xor_sync(0xffffffffu, l1, o);
                    l2 += __shfl_xor_sync(0xffffffffu, l2, o);
                }
                const double l0 = (double)(n_l0 & 0xffffffffffull);
                write_peer(&sh.all_w[b], c, fma((double)l2, 4294967296.0, fma((double)l1, 65536.0, l0)));
                write_peer(&sh.all_n[b], c, (uint32_t)(n_l0 >> 40));
                team_barrier();
                in = sh.all_n[tid], w_in = sh.all_w[tid];
            } else {
                in = sh.bins[0][tid];
                w_in = fma((double)sh.bins[3][tid], 4294967296.0, fma((double)sh.bins[2][tid], 65536.0, (double)sh.bins[1][tid]));
            }
            w_in *= power_of_two(-47 - (r.placed ? r.octave : r.octave + tid / STEPS));
            w_upto = base_w + scan64<double>(w_in);
            w_all = scanned_all<double>();
        } else {
            in = counted_in();
        }
        const uint32_t upto = base_n + scan32(in, n_all);
        if (level == 0) {
            if (by_weight) {
                target = fmax((double)sh.p, 0.0) * (w_all + tail);
            } else if (n_all + tail_n <= (uint32_t)sh.k) {         // fewer tokens than top_k asks for
                team_barrier();                                    // the bins may be cleared again
                return cut;
            }
        }
        if (in > 0 && (by_weight ? w_upto >= target && w_upto > 0 : upto >= (uint32_t)sh.k)) atomicMin(&sh.crossing, tid);
        __syncthreads();
        if (sh.crossing == BINS && tail_n == 0) {                  // by rounding a weight may end just below the target
            __syncthreads();
            if (in > 0 && upto == base_n + n_all) atomicMin(&sh.crossing, tid);
            __syncthreads();
        }
        const int b = sh.crossing;
        if (tid == b) sh.before_n = upto - in, sh.in_n = in, sh.before_w = w_upto - w_in;
        __syncthreads();
        in_n = ~0u;
        if (b == BINS && r.placed) {                               // not reached: the range has what is searched for
            team_barrier();
            return cut;
        }
        if (b < BINS) {
            base_n = sh.before_n, base_w = sh.before_w, in_n = sh.in_n;
            if (!r.placed) {
                const float to = b > 0 ? border(by_weight, r.octave, b - 1) : 0.f;
                r.lo_v = fmaxf(r.lo_v, border(by_weight, r.octave, b));
                if (b > 0) r.hi_v = value_of(key_of(to) - 1);
            } else {
                r.high -= min(r.high, (u64)b << r.shift);
                r.low = max(r.low, r.high - min(r.high, (1ull << r.shift) - 1));
                r.hi_v = fminf(r.hi_v, value_at(r.high)), r.lo_v = fmaxf(r.lo_v, value_at(r.low));
            }
        } else {
            base_n += n_all, base_w += w_all;                      // the cut is among the tail
            r.hi_v = value_of(key_of(border(by_weight, r.octave, BINS - 1)) - 1);
        }
        const bool few = in_n <= LIST && base_n + in_n <= LIST;
        if (in_n <= LIST) {
            list<RESIDENT>(r.lo_v, few ? (float)sh.top : r.hi_v, r.low, few ? ~0ull : r.high);
            team_barrier();
            const int got = min(listed(), LIST);
            if (few) {
                few_n = got;
                if (sh.me == 0) mine = take();
                return cut;
            }
            // the bin's tokens in order, and the first of them that reaches the target, else the last
            mine = sort_cta(take(), got);
            double run = 0;
            if (by_weight) run = base_w + scan64<double>(tid < got ? weight(value_at(mine)) : 0);
            if (tid == 0) sh.crossing = got - 1;
            __syncthreads();
            if (tid < got && (by_weight ? run >= target : base_n + tid + 1 >= (uint32_t)sh.k)) atomicMin(&sh.crossing, tid);
            __syncthreads();
            if (tid == sh.crossing) sh.cut = mine;
            __syncthreads();
            return sh.cut;
        }
        if (b == BINS && by_weight && level < 3) {
            r.octave += BINS / STEPS;
        } else if (!r.placed) {
            r.high = ((u64)key_of(r.hi_v) << 32) | 0xffffffffu;
            r.low = max(r.low, (u64)key_of(r.lo_v) << 32);
            r.shift = max(0, 64 - __clzll((long long)(r.high - r.low)) - 9);
            r.placed = true;
            r.octave = (int)fmin(fmax(depth(r.hi_v), 0.0), 900.0);
        } else {
            r.shift = max(0, r.shift - 9);
        }
        if (!by_weight) team_barrier();                            // the bins are cleared again
    }
    return cut;
}

__device__ __noinline__ void tell(int row, int token, float v, u64 total, int kept, int* out, int* kept_out, float* logprob_out) {
    out[row] = token;
    if (kept_out) kept_out[row] = kept;
    if (logprob_out) logprob_out[row] = (float)(-0.69314718055994530942 * (depth(v) + (log2((double)total) - sh.bits)));
}
// The running weight that the drawn token passes: less than all of it by 2^-24, so that one does.  (All but one whole unit would not do: of a total of more than
// 2^53 a 64-bit float does not tell it.)
__device__ __forceinline__ double goal_of(u64 total) { return (double)sh.u * (double)total; }

// CTA 0 has all that can be kept, one token a thread.  Up to 128 are compared each with each, four threads a token or more; of more the order is
// sorted out, cut, then sorted by index.
__device__ __noinline__ void draw_of_few(u64 mine, int n, double target, float lowest, int* out, int* kept_out, float* logprob_out) {
    const int tid = threadIdx.x, k = sh.k;
    const double share = fmax((double)sh.p, 0.0);
    const bool by_weight = sh.p < 1.f;
    int count;
    u64 own, upto, total;
    float v;
    uint32_t index;
    bool keep;
    if (n <= LIST / 4) {
        u64* places = sh.exchange;
        u64* weights = sh.listed;                                  // read by take() and by nobody else
        int lanes = 32;
        while (lanes > 4 && THREADS / lanes < n) lanes /= 2;
        __syncthreads();
        if (tid < n) places[tid] = mine, weights[tid] = whole(weight(value_at(mine)), sh.one);
        __syncthreads();
        const int e = tid / lanes;
        const bool here = e < n;
        const u64 place = here ? places[e] : 0;
        own = here ? weights[e] : 0;
        v = value_at(place), index = ~(uint32_t)place;
        int rank = 0;
        upto = 0;
#pragma unroll 4
        for (int j = tid % lanes; j < n; j += lanes)
            if (places[j] >= place) ++rank, upto += weights[j];
#pragma unroll 1
        for (int o = 1; o < lanes; o <<= 1) {
            rank += __shfl_xor_sync(0xffffffffu, rank, o);
            upto += __shfl_xor_sync(0xffffffffu, upto, o);
        }
        keep = here && v >= lowest;
        if (k > 0) keep = keep && rank <= k;
        if (by_weight) {
            if (target < 0) {
                if (here && rank == min(k, n)) sh.cut = upto;
                __syncthreads();
                target = share * (double)sh.cut;
            } else {
                target *= sh.one;
            }
            keep = keep && (rank == 1 || (double)(upto - own) < target);
        }
        __syncthreads();
        if (here && !keep && tid % lanes == 0) weights[e] = 0;
        keep = keep && tid % lanes == 0;
        count = __syncthreads_count(keep);
        upto = total = 0;
#pragma unroll 4
        for (int j = tid % lanes; j < n; j += lanes) {
            const u64 t = weights[j];
            total += t;
            if (~(uint32_t)places[j] <= index) upto += t;
        }
#pragma unroll 1
        for (int o = 1; o < lanes; o <<= 1) {
            total += __shfl_xor_sync(0xffffffffu, total, o);
            upto += __shfl_xor_sync(0xffffffffu, upto, o);
        }
    } else {
        mine = sort_cta(mine, n);
        int len = k > 0 ? min(k, n) : n;
        v = value_at(mine);
        if (by_weight) {
            const double run = scan64<double>(tid < len ? weight(v) : 0);
            if (target < 0) target = share * scanned_all<double>();
            if (tid == 0) sh.crossing = len - 1;
            __syncthreads();
            if (tid < len && run >= target) atomicMin(&sh.crossing, tid);
            __syncthreads();
            len = sh.crossing + 1;
        }
        keep = tid < len && v >= lowest;
        count = __syncthreads_count(keep);
        index = ~(uint32_t)mine;
        mine = sort_cta(keep ? ((u64)~index << 32) | (mine >> 32) : 0, count);
        v = value_of((uint32_t)mine), index = ~(uint32_t)(mine >> 32);
        keep = tid < count;
        own = keep ? whole(weight(v), sh.one) : 0;
        upto = scan64<u64>(own);
        total = scanned_all<u64>();
    }
    const double goal = goal_of(total);
    if (keep && (double)upto > goal && !((double)(upto - own) > goal)) tell(sh.row, (int)index, v, total, count, out, kept_out, logprob_out);
}

// Of four tokens the weights of those that are kept, as whole numbers with an OFFSET each; `count`: how many
template <bool RESIDENT>
__device__ __forceinline__ u64 kept_weights(const Weigher& weigh, double one, float lowest, float cut_v, int cut_i, bool endless, int at, int i, u64 (&w)[4],
                                            float (&v)[4], uint32_t& count) {
    get<RESIDENT>(i, v, endless);
    bool on[4];
    u64 sum = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) on[j] = v[j] >= lowest && (v[j] != cut_v || at + j <= cut_i), w[j] = 0;
    if (on[0] || on[1] || on[2] || on[3])
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            int step;
            const double q = weigh(v[j], step);
            if (on[j]) sum += w[j] = offset_whole(q, one), ++count;
        }
    return sum;
}
// The draw over the row, from the tokens from the place `cut` and the value `lowest` on: every warp has a run of neighbours, its weight after those of the
// runs before it
template <bool RESIDENT> __device__ __noinline__ void draw_of_row(u64 cut, float lowest, int* out, int* kept_out, float* logprob_out) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, c0 = sh.c0, nv = (sh.n + 3) / 4, ctas = sh.ctas;
    const int run = ((nv + WARPS - 1) / WARPS + 31) & ~31;         // in fours
    const int i0 = min(warp * run, nv), i1 = min(i0 + run, nv);
    const bool endless = sh.endless;
    const double one = sh.one;
    const Weigher weigh;
    const float cut_v = cut ? value_at(cut) : -INFINITY;
    const int cut_i = (int)~(uint32_t)cut;
    lowest = fmaxf(lowest, cut_v);
    u64 own = 0, w[4];
    float v[4];
    uint32_t count = 0;
#pragma unroll 1
    for (int i = i0 + lane; i < i1; i += 32) own += kept_weights<RESIDENT>(weigh, one, lowest, cut_v, cut_i, endless, c0 + 4 * i, i, w, v, count);
    own = warp_sum64(own - count * OFFSET);
    count = __reduce_add_sync(0xffffffffu, count);
    __syncthreads();
    if (lane == 0) sh.scanned[warp] = own, sh.counted[warp] = count;
    __syncthreads();
    u64 t = lane < WARPS ? sh.scanned[lane] : 0;
    u64 before = warp_sum64(lane < warp ? t : 0), total = warp_sum64(t);
    count = __reduce_add_sync(0xffffffffu, lane < WARPS ? sh.counted[lane] : 0);
    if (ctas > 1) {
        if (tid == 0) sh.part[0][0] = total, sh.part[0][1] = count;
        team_barrier();
        t = lane < ctas ? read_peer(&sh.part[0][0], lane) : 0;
        count = __reduce_add_sync(0xffffffffu, lane < ctas ? (uint32_t)read_peer(&sh.part[0][1], lane) : 0);
        before += warp_sum64(lane < sh.me ? t : 0);
        total = warp_sum64(t);
        cluster_arrive();                                          // nothing of the peers is read any more
    }
    const double goal = goal_of(total);
    if ((double)(before + own) > goal && !((double)before > goal)) {              // one warp of the cluster: the running weight passes the goal in its run
#pragma unroll 1
        for (int i = i0; i < i1; i += 32) {
            uint32_t have = 0;
            u64 s = i + lane < i1 ? kept_weights<RESIDENT>(weigh, one, lowest, cut_v, cut_i, endless, c0 + 4 * (i + lane), i + lane, w, v, have) : 0;
            const u64 mine4 = s -= have * OFFSET;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const u64 up = __shfl_up_sync(0xffffffffu, s, o);
                if (lane >= o) s += up;
            }
            const uint32_t passed = __ballot_sync(0xffffffffu, (double)(before + s) > goal);
            if (passed) {
                if (lane == __ffs(passed) - 1) {
                    before += s - mine4;
                    int at = -1;
                    float x = 0;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        before += w[j] ? w[j] - OFFSET : 0;
                        if (at < 0 && (double)before > goal) at = c0 + 4 * (i + lane) + j, x = v[j];
                    }
                    tell(sh.row, at, x, total, (int)count, out, kept_out, logprob_out);
                }
                break;
            }
            before += __shfl_sync(0xffffffffu, s, 31);
        }
    }
    __syncwarp();
    if (ctas > 1) cluster_wait();
}

template <bool RESIDENT>
__global__ void __launch_bounds__(THREADS, 2)
sample_filtered_kernel(const float* __restrict__ logits_, long long ld, int R, int V, int per_cta, const float* __restrict__ temperature_,
                       const float* __restrict__ u_, const int* __restrict__ top_k_, const float* __restrict__ top_p_,
                       const float* __restrict__ min_p_, const int* __restrict__ rows_, int* __restrict__ out, int* __restrict__ kept_out,
                       float* __restrict__ logprob_out, int* err) {
    const int tid = threadIdx.x;
    sh.table[tid] = exp2(-(tid / COPIES) / (double)STEPS);
    static_assert(STEPS * COPIES == THREADS, "one entry a thread");
    pdl_trigger();
    pdl_wait();
    const int row = rows_ ? pdl_fresh(rows_)[blockIdx.y] : blockIdx.y;
    if (row < 0 || row >= R) {                                     // the same for the whole cluster: nobody waits for anybody
        if (tid == 0) report_error(err, PRISM_ERR_ROW_RANGE);
        return;
    }
    const int ctas = gridDim.x, me = ctas > 1 ? (int)rank_in_cluster() : 0, c0 = min(me * per_cta, V), n = min(per_cta, V - c0), nv = (n + 3) / 4;
    const float* x = pdl_fresh(logits_) + (size_t)row * ld + c0;
    const float T = temperature_ ? pdl_fresh(temperature_)[row] : 0.f;
    const int k = top_k_ ? pdl_fresh(top_k_)[row] : 0;
    const float p = top_p_ ? pdl_fresh(top_p_)[row] : 1.f, min_p = min_p_ ? pdl_fresh(min_p_)[row] : 0.f, mp = min_p > 0.f ? fminf(min_p, 1.f) : 0.f;
    const float u = pdl_fresh(u_)[row];

    float top = -INFINITY;
    if (RESIDENT && (reinterpret_cast<uintptr_t>(x) & 15) == 0) {
        constexpr int AHEAD = 10;                                  // loads in flight: 80 KB a CTA
        const float4* x4 = reinterpret_cast<const float4*>(x);
        const int n4 = n / 4;
#pragma unroll 1
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
                    kept_slice[i0 + j * THREADS] = v[j];
                }
        }
        if (n4 < nv && tid == 0) {
            const float4 v = kept_slice[n4] = load_four(x, n, n4);
            top = fmaxf(fmaxf(top, fmaxf(v.x, v.y)), fmaxf(v.z, v.w));
        }
    } else {
#pragma unroll 4
        for (int i = tid; i < nv; i += THREADS) {
            const float4 v = load_four(x, n, i);
            if (RESIDENT) kept_slice[i] = v;
            top = fmaxf(fmaxf(top, fmaxf(v.x, v.y)), fmaxf(v.z, v.w));
        }
    }
    if (tid == THREADS - 1) {                                      // for all, behind the barrier of the largest logit
        sh.x = x, sh.n = n, sh.c0 = c0, sh.ctas = ctas, sh.me = me, sh.row = row;
        sh.k = k < V ? k : 0, sh.p = p;
        sh.u = u < 1.f ? fmaxf(u, 0.f) : 1.f - 0x1p-24f;             // what is not in [0, 1), NaN too, as its nearer end there
        sh.per = 1.44269504088896340736 / (double)T;
        sh.deepest = mp > 0.f ? -log2((double)mp) : INFINITY;
        sh.bits = min(46, 63 - (31 - __clz(V)));                   // V weights of 1 stay below 2^64
        sh.one = (double)(1ull << sh.bits);
        sh.endless = false;
    }
    __syncthreads();
    int turn = 1;
    float first = top;                                             // this thread's largest
    top = value_of(team_reduce(key_of(top), true, turn));
    if (!(T > 0.f) || top == -INFINITY) {
        uint32_t best = 0;                                         // complement of the lowest index
        if (top > -INFINITY)
#pragma unroll 1
            for (int i = tid; i < nv; i += THREADS) {
                float v[4];
                get<RESIDENT>(i, v, false);
#pragma unroll
                for (int j = 3; j >= 0; --j)
                    if (v[j] == top) best = max(best, ~(uint32_t)(c0 + 4 * i + j));
            }
        best = team_reduce(best, true, turn ^= 1);
        const bool none = top == -INFINITY;
        if (me == 0 && tid == 0) {
            out[row] = none ? 0 : (int)~best;
            if (kept_out) kept_out[row] = none ? 0 : 1;
            if (logprob_out) logprob_out[row] = none ? -INFINITY : 0.f;
        }
        team_barrier();                                            // peers may still read this CTA's part
        return;
    }
    if (top == INFINITY) {
        if (RESIDENT)
#pragma unroll 1
            for (int i = tid; i < 4 * nv; i += THREADS) {
                float* kept = reinterpret_cast<float*>(kept_slice);
                kept[i] = kept[i] == INFINITY ? 0.f : -INFINITY;
            }
        top = 0.f, first = first == INFINITY ? 0.f : -INFINITY;
        if (tid == 0) sh.endless = true;
    }
    if (tid == 0) {
        sh.top = (double)top;
        sh.floor = fmaxf(LEAST, __double2float_ru((double)top - 693.0 * (double)T));           // at an infinite temperature all but -infinity count
    }
    __syncthreads();
    // min_p as the lowest value that it keeps
    float lowest = LEAST;
    if (mp > 0.f) {
        lowest = fmaxf(LEAST, __double2float_rd(sh.top - sh.deepest / sh.per));
#pragma unroll 1
        for (int i = 0; i < 4 && lowest < top && depth(lowest) > sh.deepest; ++i) lowest = value_of(key_of(lowest) + 1);
    }
    u64 cut = 0;                                                   // kept are the tokens from this place on upwards,
    u64 mine = 0;                                                  // or they are among few_n tokens that CTA 0 has, one a thread
    int few_n = -1;
    double target = -1;                                            // weight of the prefix that top_p asks for, once known
    if (sh.k > 0) {
        if (sh.k <= LIST / 2) few_n = attempt<RESIDENT>(first, mine);
        if (few_n < 0) cut = search<RESIDENT>(false, 0, turn, few_n, mine, target);
    }
    if (few_n < 0 && p < 1.f) cut = search<RESIDENT>(true, cut, turn, few_n, mine, target);
    if (few_n >= 0) {
        if (ctas > 1) cluster_arrive();
        if (me == 0) draw_of_few(mine, few_n, target, lowest, out, kept_out, logprob_out);
        __syncwarp();
        if (ctas > 1) cluster_wait();
    } else {
        draw_of_row<RESIDENT>(cut, lowest, out, kept_out, logprob_out);
    }
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
    // Eight CTAs for a large row: with four 152,064 tokens took by top-p 87 us (16 rows; eight: 68), by top-k 13.8 (15.6), 64 rows 55 (46); with sixteen 64 and 26,
    // 64 rows 174 (108) and 74.  Slices in shared memory: read again from L2 instead, 16 rows took 18.7 us by top-k and 82 by top-p.
    int ctas = 1;
    while (ctas < MOST_CTAS && V > 4096 * ctas) ctas *= 2;
    const int per_cta = ((V + ctas - 1) / ctas + 3) & ~3;
    const bool resident = per_cta <= MOST_SLICE;
    const auto kernel = resident ? sample_filtered_kernel<true> : sample_filtered_kernel<false>;
    const size_t smem = resident ? (size_t)per_cta * 4 : 0;
    if (smem > 16 * 1024) prism::open_smem(kernel, MOST_SLICE * 4);              // beside 27 KB of its own
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
