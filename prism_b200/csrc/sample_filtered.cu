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

namespace prism {
namespace draw {

typedef unsigned long long u64;
constexpr int THREADS = 512;
constexpr int WARPS = THREADS / 32;
constexpr int MOST_CTAS = 8;
constexpr int MOST_SLICE = 40 * 1024;          // values of a slice that stay in shared memory; of a larger one every pass reads memory
constexpr int MOST_V = MOST_CTAS * 65535;      // a CTA's bins are sums of 16-bit numbers in 32 bits
constexpr int BINS = THREADS;                  // one a thread
constexpr int LIST = THREADS;                  // tokens that are sorted, one a thread
constexpr int STEPS = 32;                      // bins of a power of two

__device__ __forceinline__ uint32_t rank_in_cluster() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}
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
__device__ __forceinline__ uint4 read_peer(const uint4* p, int cta) {
    uint4 v;
    asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(peer(p, cta)) : "memory");
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

__device__ __forceinline__ double power_of_two(int e) { return __hiloint2double((1023 + e) << 20, 0); }

struct Shared {
    double table[64];
    u64 slot[2][WARPS];          // per-warp results of a reduction
    u64 scanned[WARPS];          // and of a scan
    u64 part[2][2];              // the CTA's, for its peers
    uint4 bins[BINS];            // count, and the sum of the weights' low, middle and high 16 bits; a sort's exchange
    u64 listed[LIST];            // this CTA's tokens of those that are collected
    uint32_t listed_n;
    int crossing;
    uint32_t before_n, in_n;     // of the bin that holds a cut: tokens before it, and in it
    double before_w;
    u64 cut;
};

struct Team {
    Shared* s;
    int ctas, me, turn;
    __device__ __forceinline__ void barrier() const {
        if (ctas > 1) cluster_barrier();
        else __syncthreads();
    }
    // Over the cluster, for every thread.  Slots are used in turn: a CTA that is one reduction ahead writes others than its peers still read.
    __device__ __forceinline__ u64 sum(u64 v) { return reduce<u64>(v, [](u64 t) { return warp_sum64(t); }); }
    __device__ __forceinline__ u64 max(u64 v) { return reduce<u64>(v, [](u64 t) { return warp_max64(t); }); }
    static __device__ __forceinline__ u64 bits_of(u64 v) { return v; }
    static __device__ __forceinline__ u64 bits_of(double v) { return (u64)__double_as_longlong(v); }
    static __device__ __forceinline__ void of_bits(u64 b, u64& v) { v = b; }
    static __device__ __forceinline__ void of_bits(u64 b, double& v) { v = __longlong_as_double((long long)b); }
    // of the CTA; its result is left for the peers in part[turn][0]
    template <typename W, typename F> __device__ __forceinline__ W reduce_cta(W v, F warp_all) {
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        turn ^= 1;
        v = warp_all(v);
        if (lane == 0) s->slot[turn][warp] = bits_of(v);
        __syncthreads();
        of_bits(lane < WARPS ? s->slot[turn][lane] : 0, v);
        v = warp_all(v);
        if (threadIdx.x == 0) s->part[turn][0] = bits_of(v);
        return v;
    }
    template <typename W, typename F> __device__ __forceinline__ W gather_parts(F warp_all) {
        W v;
        const int lane = threadIdx.x & 31;
        of_bits(lane < ctas ? read_peer(&s->part[turn][0], lane) : 0, v);
        return warp_all(v);
    }
    template <typename W, typename F> __device__ __forceinline__ W reduce(W v, F warp_all) {
        v = reduce_cta<W>(v, warp_all);
        if (ctas == 1) return v;
        cluster_barrier();
        return gather_parts<W>(warp_all);
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
    if (lane == 31) slots[warp] = Team::bits_of(v);
    __syncthreads();
    W before = 0, t;
    all = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
        Team::of_bits(slots[w], t);
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

__global__ void __launch_bounds__(THREADS, 2)
sample_filtered_kernel(const float* __restrict__ logits_, long long ld, int R, int V, int per_cta, int resident, const float* __restrict__ temperature_,
                       const float* __restrict__ u_, const int* __restrict__ top_k_, const float* __restrict__ top_p_,
                       const float* __restrict__ min_p_, const int* __restrict__ rows_, int* __restrict__ out, int* __restrict__ kept_out,
                       float* __restrict__ logprob_out, int* err) {
    extern __shared__ __align__(16) float slice[];
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
    const int k = top_k_ ? pdl_fresh(top_k_)[row] : 0;
    const float p = top_p_ ? pdl_fresh(top_p_)[row] : 1.f, mp = min_p_ ? fminf(pdl_fresh(min_p_)[row], 1.f) : 0.f;
    const float u = pdl_fresh(u_)[row];

    float top = -INFINITY;
    if (resident && (reinterpret_cast<uintptr_t>(x) & 15) == 0) {
        constexpr int AHEAD = 5;                                   // loads in flight: 40 KB a CTA
        const float4* x4 = reinterpret_cast<const float4*>(x);
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
                    reinterpret_cast<float4*>(slice)[i0 + j * THREADS] = v[j];
                }
        }
        for (int i = n4 * 4 + tid; i < n; i += THREADS) top = fmaxf(top, slice[i] = clean(x[i]));
    } else {
        for (int i = tid; i < n; i += THREADS) {
            const float v = clean(x[i]);
            if (resident) slice[i] = v;
            top = fmaxf(top, v);
        }
    }
    top = value_at(team.max(place_of(top, 0)));
    auto raw = [&](int i) { return resident ? slice[i] : clean(x[i]); };
    if (!(T > 0.f) || top == -INFINITY) {
        u64 best = 0;
        if (top > -INFINITY)
            for (int i = tid; i < n; i += THREADS)
                if (raw(i) == top) {
                    best = place_of(top, c0 + i);
                    break;
                }
        best = team.max(best);
        const bool none = top == -INFINITY;
        if (team.me == 0 && tid == 0) {
            out[row] = none ? 0 : (int)~(uint32_t)best;
            if (kept_out) kept_out[row] = none ? 0 : 1;
            if (logprob_out) logprob_out[row] = none ? -INFINITY : 0.f;
        }
        team.barrier();                                            // peers may still read this CTA's part
        return;
    }
    // infinities share the probability: as if they were 0 and the others masked
    const bool endless = top == INFINITY;
    if (endless) top = 0.f;
    auto value = [&](int i) {
        const float v = raw(i);
        return endless ? (v == INFINITY ? 0.f : -INFINITY) : v;
    };
    Row r;
    r.top = (double)top;
    r.per = 1.44269504088896340736 / (double)T;
    const int bits = min(46, 63 - (31 - __clz(V)));                // V weights of 1 stay below 2^64
    r.one = (double)(1ull << bits);
    r.table = sh.table;
    const double deepest = mp > 0.f ? -log2((double)mp) : INFINITY;

    u64 cut = 0;                 // kept are the tokens from this place on upwards ...
    u64 most = ~0ull;            // ... and as many at most
    double target = -1;          // weight of the prefix that top_p asks for, once known
    bool few = false;            // the kept tokens are among the collected ones, one a thread of CTA 0
    u64 mine = 0;                // the collected token of this thread
    int few_n = 0;
    auto weight_at = [&](u64 place) { return weight(r, depth(r, value_at(place))); };

    // The tokens with `which(place)`, at most LIST of them in all: one a thread, for CTA 0 or (`for_all`) every CTA.  Returns their number.
    auto collect = [&](auto which, bool for_all) {
        if (tid == 0) sh.listed_n = 0;
        __syncthreads();
        for (int i = tid; i < n; i += THREADS) {
            const float v = value(i);
            if (v > -INFINITY && which(v, c0 + i)) {
                const uint32_t at = atomicAdd(&sh.listed_n, 1u);
                if (at < LIST) sh.listed[at] = place_of(v, c0 + i);
            }
        }
        team.barrier();
        int have = 0;
        mine = 0;
        if (for_all || team.me == 0)
            for (int c = 0; c < team.ctas; ++c) {
                const int m = min((int)(team.ctas > 1 ? read_peer(&sh.listed_n, c) : sh.listed_n), LIST);
                const int at = tid - have;
                if (at >= 0 && at < m) mine = team.ctas > 1 ? read_peer(&sh.listed[at], c) : sh.listed[at];
                have += m;
            }
        return min(have, LIST);
    };

    // Finds where the first k tokens end (by_weight false) or the shortest prefix of weight p of what `cut` leaves (true): in `cut`, or among
    // the collected tokens (`few`)
    auto search = [&](bool by_weight) {
        bool placed = false;                                       // level 0: bins by depth; then by place, from `high` down in steps of 2^shift
        u64 high = 0;
        int shift = 0, octave = 0;
        uint32_t base_n = 0;
        double base_w = 0;
        const float per32 = 1.44269504f * STEPS;                   // tokens are counted by depth at temperature 1
        for (int level = 0; level < 9; ++level) {
            sh.bins[tid] = make_uint4(0, 0, 0, 0);
            if (tid == 0) sh.crossing = BINS;
            __syncthreads();
            double tail = 0;                                       // beyond the bins: weight, or number of tokens
            u64 tail_n = 0;
            for (int i = tid; i < n; i += THREADS) {
                const float v = value(i);
                if (!(v > -INFINITY)) continue;
                int b;
                double w = 0;
                if (!placed) {
                    if (!by_weight) {
                        const float at = (top - v) * per32;
                        if (!(at < (float)BINS)) {
                            ++tail_n;
                            continue;
                        }
                        b = (int)at;
                    } else {
                        if (cut && place_of(v, c0 + i) < cut) continue;
                        const double d = depth(r, v);
                        w = weight(r, d);
                        if (!(d < (BINS - 1.0) / STEPS)) {
                            tail += w, ++tail_n;
                            continue;
                        }
                        b = __double2int_rn(d * STEPS);
                        octave = b / STEPS;
                    }
                } else {
                    const u64 at = place_of(v, c0 + i);
                    if (at > high || (cut && at < cut)) continue;
                    const u64 down = (high - at) >> shift;
                    if (down >= BINS) continue;
                    b = (int)down;
                    if (by_weight) w = weight(r, depth(r, v));
                }
                atomicAdd(&sh.bins[b].x, 1u);
                if (by_weight) {                                   // of about 2^47: 16 bits of it at a time, so that 65,535 fit in 32
                    const u64 m = (u64)__double_as_longlong(fma(w, power_of_two(47 + octave), 4503599627370496.0)) & 0xfffffffffffffull;
                    atomicAdd(&sh.bins[b].y, (uint32_t)m & 0xffffu);
                    atomicAdd(&sh.bins[b].z, (uint32_t)(m >> 16) & 0xffffu);
                    atomicAdd(&sh.bins[b].w, (uint32_t)(m >> 32));
                }
            }
            if (!placed) {                                         // its barriers are those of the bins
                if (by_weight) tail = team.reduce<double>(tail, [](double t) { return warp_sum64(t); });
                tail_n = team.sum(tail_n);
            } else {
                team.barrier();
            }
            u64 l0 = 0, l1 = 0, l2 = 0;
            uint32_t in = 0;
            for (int c = 0; c < team.ctas; ++c) {
                const uint4 t = team.ctas > 1 ? read_peer(&sh.bins[tid], c) : sh.bins[tid];
                in += t.x, l0 += t.y, l1 += t.z, l2 += t.w;
            }
            const int oct = placed ? octave : tid / STEPS;
            double w_in = 0, w_all = 0, w_upto = 0;
            uint32_t n_all;
            if (by_weight) {
                w_in = fma((double)l2, 4294967296.0, fma((double)l1, 65536.0, (double)l0)) * power_of_two(-47 - oct);
                w_upto = base_w + scan_cta<double>(w_in, sh.scanned, w_all);
            }
            const uint32_t upto = base_n + (uint32_t)scan_cta<u64>(in, sh.scanned, mine);
            n_all = (uint32_t)mine;
            if (!placed) {
                if (by_weight) target = fmax((double)p, 0.0) * (w_all + tail);
                else if ((u64)n_all + tail_n <= (u64)k) {          // fewer tokens than top_k asks for
                    team.barrier();                                // the bins may be cleared again
                    return;
                }
            }
            const bool last_resort = by_weight && (placed || tail_n == 0);         // by rounding the sum may end just below the target
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
            if (b < BINS) {
                const uint32_t before_n = sh.before_n, in_n = sh.in_n;
                const double before_w = sh.before_w;
                auto bin_of = [&](float v, int i) {                // as above
                    if (placed) {
                        const u64 at = place_of(v, i);
                        return at > high ? -1 : (int)min((high - at) >> shift, (u64)BINS);
                    }
                    if (!by_weight) {
                        const float at = (top - v) * per32;
                        return at < (float)BINS ? (int)at : BINS;
                    }
                    const double d = depth(r, v);
                    return d < (BINS - 1.0) / STEPS ? __double2int_rn(d * STEPS) : BINS;
                };
                if (before_n + in_n <= LIST) {
                    few_n = collect([&](float v, int i) { return bin_of(v, i) <= b && (!cut || place_of(v, i) >= cut); }, false);
                    few = true;
                    return;
                }
                if (in_n <= LIST) {
                    const int got = collect([&](float v, int i) { return bin_of(v, i) == b && (!cut || place_of(v, i) >= cut); }, true);
                    mine = sort_cta(mine, got, reinterpret_cast<u64*>(sh.bins));
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
            // the places of the bin's tokens, or of the tail's: their range is divided next
            u64 lo = 0, hi = 0;                                    // complement of the lowest, and the highest
            for (int i = tid; i < n; i += THREADS) {
                const float v = value(i);
                if (!(v > -INFINITY)) continue;
                const u64 at = place_of(v, c0 + i);
                if (cut && at < cut) continue;
                bool in_range;
                if (placed) {
                    in_range = at <= high && (int)min((high - at) >> shift, (u64)BINS) == b;
                } else if (!by_weight) {
                    const float f = (top - v) * per32;
                    in_range = (f < (float)BINS ? (int)f : BINS) == b;
                } else {
                    const double d = depth(r, v);
                    in_range = (d < (BINS - 1.0) / STEPS ? __double2int_rn(d * STEPS) : BINS) == b;
                }
                if (in_range) {
                    hi = at > hi ? at : hi;
                    lo = ~at > lo ? ~at : lo;
                }
            }
            hi = team.max(hi);
            lo = ~team.max(lo);
            if (!by_weight && depth(r, value_at(hi)) >= 1000.0) {  // what lies there weighs nothing: which of it is kept makes no difference
                most = (u64)k;
                return;
            }
            placed = true;
            high = hi;
            shift = max(0, 64 - __clzll((long long)(hi - lo)) - 9);
            octave = (int)fmin(depth(r, value_at(hi)), 900.0);
        }
    };
    if (k > 0 && k < V) search(false);
    if (!few && p < 1.f) search(true);

    u64 own = 0, upto, total, count;
    double d_own = 0;
    if (few) {
        if (team.ctas > 1) asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");
        if (team.me == 0) {
            // CTA 0 has all that can be kept: in order, cut, then by index
            mine = sort_cta(mine, few_n, reinterpret_cast<u64*>(sh.bins));
            int len = k > 0 ? min(k, few_n) : few_n;
            const double d = tid < len ? depth(r, value_at(mine)) : INFINITY, w = tid < len ? weight(r, d) : 0;
            if (p < 1.f) {
                double all;
                const double run = scan_cta<double>(w, sh.scanned, all);
                if (target < 0) target = fmax((double)p, 0.0) * all;
                if (tid == 0) sh.crossing = len - 1;
                __syncthreads();
                if (tid < len && run >= target) atomicMin(&sh.crossing, tid);
                __syncthreads();
                len = sh.crossing + 1;
            }
            const bool keep = tid < len && d <= deepest;
            count = (u64)__syncthreads_count(keep);
            const uint32_t index = ~(uint32_t)mine;
            mine = sort_cta(keep ? ((u64)~index << 32) | (mine >> 32) : 0, (int)count, reinterpret_cast<u64*>(sh.bins));
            const bool have = tid < (int)count;
            d_own = have ? depth(r, value_at(mine << 32)) : INFINITY;
            own = have ? whole(r, weight(r, d_own)) : 0;
            upto = scan_cta<u64>(own, sh.scanned, total);
            const double goal = u < 1.f ? fmax((double)u, 0.0) * (double)total : (double)(total - 1);
            if ((double)upto > goal && !((double)(upto - own) > goal)) {
                out[row] = (int)~(uint32_t)(mine >> 32);
                if (kept_out) kept_out[row] = (int)count;
                if (logprob_out) logprob_out[row] = (float)(-0.69314718055994530942 * (d_own + (log2((double)total) - bits)));
            }
        }
        if (team.ctas > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
        return;
    }
    // The draw: every thread a run of neighbours, its weight after those of the runs before it
    const int run = ((n + THREADS - 1) / THREADS) | 1;             // odd: neighbours' places lie in different banks
    const int i0 = min(tid * run, n), i1 = min(i0 + run, n);
    const float lowest = cut ? value_at(cut) : -INFINITY;
    count = 0;
    for (int i = i0; i < i1; ++i) {
        const float v = value(i);
        if (!(v >= lowest) || v == -INFINITY || (v == lowest && place_of(v, c0 + i) < cut)) continue;
        const double d = depth(r, v);
        if (d <= deepest) own += whole(r, weight(r, d)), ++count;
    }
    u64 cta_total;
    upto = scan_cta<u64>(own, sh.scanned, cta_total);
    count = team.reduce_cta<u64>(count, [](u64 t) { return warp_sum64(t); });
    total = cta_total;
    if (team.ctas > 1) {
        if (tid == 0) sh.part[team.turn][1] = cta_total;
        cluster_barrier();
        count = team.gather_parts<u64>([](u64 t) { return warp_sum64(t); });
        total = 0;
        for (int c = 0; c < team.ctas; ++c) {
            const u64 t = read_peer(&sh.part[team.turn][1], c);
            if (c < team.me) upto += t;
            total += t;
        }
    }
    count = count < most ? count : most;
    const double goal = u < 1.f ? fmax((double)u, 0.0) * (double)total : (double)(total - 1);
    if ((double)upto > goal && !((double)(upto - own) > goal)) {   // one thread of the cluster: the running weight passes the goal in its run
        u64 run_to = upto - own;
        for (int i = i0; i < i1; ++i) {
            const float v = value(i);
            if (!(v >= lowest) || v == -INFINITY || (v == lowest && place_of(v, c0 + i) < cut)) continue;
            const double d = depth(r, v);
            if (d <= deepest) {
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
    team.barrier();
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
