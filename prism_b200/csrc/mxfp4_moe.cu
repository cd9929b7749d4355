// A whole mixture-of-experts layer for up to 64 tokens, its experts' weights in microscaled 4-bit floating point (mxfp4.cuh),
// in one launch:
//   z = x Wr^T (+ br);  scores, choice and weights as in moe_route.cuh;  h = act(g) u with g = Wg[e] a, u = Wu[e] a
//   (a = x, times the weight with scale_in);  y[t] = sum over the token's choices of Wd[e] h (times the weight without)
//
// Bound by the chosen experts' bytes where they are many and by the chain of dependent steps where they are few.  One
// cooperative kernel, a CTA an SM, so that the steps cost a barrier each instead of a launch, and the weights of the second
// product are on their way while the first one's sums are still being taken out:
//   1. router logits (a warp per token and few experts; the warp that finishes a token's last ones makes its choice) and x as
//      two 8-bit terms (mxfp4_mma.cuh); barrier over the grid
//   2. every CTA reads the choices and lists the experts that have tokens
//   3. gate and up: 128 rows of either and all tokens (high terms, low terms) as columns of one tcgen05.mma each; the sums of
//      an expert's tokens become h, as three terms (a warp's 32 lanes are one block): h is not of bfloat16's 8 significant bits as x
//      is, and two terms would round it to about those; three hold it to 2^-14 of itself and 2^-27 of its block's largest.  With two
//      a whole layer's result was off by 0.0018 of its scale instead of 0.0017, bfloat16's own rounding; the third costs nothing at 1
//      token, 1 % at 16 and 5 % at 64 (below: 84.9 us with two)
//   4. down: 256 rows, the expert's own tokens as columns, once all of its h is there (a counter per expert)
//   5. barrier over the grid; y is the sum of a token's choices in their order
// In 3 and 4 the blocks (expert, rows, 128 of K) are dealt to the CTAs evenly as one line; a tile that several CTAs have part of
// is added up by the last to come, in the CTAs' order: results do not depend on timing.
//
// 1 token through 2 of 8 experts of 3 x 672 x 2,048: 22.7 us, of which (taken at 21.4) routing and its barrier 5.7, lists 2, the
// first weights 3, two hand-overs of a tile's shares some 4 each, the last barrier and sums 1.5.  16 tokens through 8 of 3 x 1,184 x
// 4,096: 40.5 us.  64 tokens through 64 of 3 x 1,024 x 2,048, 8 a token: 89.4 us for 214 MB, of which 28 until the first products
// (routing over 64 experts, lists, x laid out), 29 gate and up at 4.9 TB/s, and, taken before h had its third term, which added 4.5
// to them, 12 until an expert's h is whole and 15 down.
//
// Warp 0 streams weights and their scales, warp 2 x and h, warp 1 issues the products, warps 4-11 take the sums out.  Every
// wait is bounded; on expiry all CTAs learn of it and leave without a result: the error word is set, tensor memory is freed, the
// control block is cleared and the kernel returns.
#include "moe_route.cuh"
#include "mxfp4_mma.cuh"
#include "vec.cuh"

#include <algorithm>
#include <climits>

namespace prism {
namespace mx {

constexpr int MOE_THREADS = 384, MOE_WARPS = 12, MOE_MOST_EXPERTS = 256, MOE_MOST_ENTRIES = 1024;

// TT: tokens there is room for.  COMPACT: the columns of gate and up are an expert's own tokens, whose rows of x are laid out anew for
// it; otherwise all tokens (there are few).
template <int TT_> struct MoeCfg {
    static constexpr int TT = TT_, NCOL = 2 * TT;
    static constexpr bool COMPACT = TT > 16;
    // of x two terms a token, of h three: up to 192 rows, whose scales are two tiles
    static constexpr int W_BYTES = 2 * 16384, X_BYTES = 3 * TT * 128, STAGE = W_BYTES + X_BYTES, SF = 4 * TILE_BYTES, SF_COLS = 16;
    static constexpr int FIT = 200 * 1024 / (STAGE + SF), STAGES = FIT > 8 ? 8 : FIT;
    static constexpr int USED = 6 * TT + STAGES * SF_COLS, BOTH = 12 * TT + STAGES * SF_COLS;       // columns with one set of sums, with two
    static constexpr int COLS = BOTH <= 128 ? 128 : BOTH <= 256 ? 256 : 512;
    static constexpr size_t SMEM = (size_t)STAGES * (STAGE + SF) + 1024 + 512;
    static_assert(USED <= 512 && STAGES >= 3, "tensor memory or shared memory");
};

struct Moe {
    const __nv_bfloat16* x;
    const void *router, *rbias, *corr;
    const uint8_t *gate_s, *up_s, *down_s;
    // x's terms [2 TT][Hp] and scales [groups][512] (compact: [rows][Hp] and [live][groups][512]), h's [rows][Fp] and [live][groups][2][512]
    uint8_t *xt, *xs, *h, *hs;
    float *z, *sel_w, *part1, *part2, *planes;
    int *sel_e, *counters, *ready, *control, *err;      // ready: h, then x (compact); control: see Control
    void* y;
    long long ldx, ldy;
    int T, H, F, E, top, softmax, renorm, scale_in, act, groups_of_experts, keep, dots, most_live, ncounters;
    int router_bf16, rbias_bf16, corr_bf16, out_bf16, wide;
    float limit, wscale, sum_eps;
};

// Words of the control block.  A barrier's word counts its own arrivals only, and a CTA that gave up arrives nowhere any more but
// raises GAVE_UP, which whoever waits in memory reads too: so nobody passes a barrier before all that it stands for is there.
enum Control { FIRST, SECOND, GAVE_UP, LEAVERS, TOKEN, CONTROL_WORDS = TOKEN + 64 };     // TOKEN: logits that are there, a word each

struct Lists {                             // of the experts that have tokens, in their order
    unsigned long long mask[MOE_MOST_EXPERTS];
    short slot[MOE_MOST_EXPERTS], expert[MOE_MOST_EXPERTS], count[MOE_MOST_EXPERTS], hrow8[MOE_MOST_EXPERTS], first[MOE_MOST_EXPERTS];
    // an expert's tokens from first[] on, ascending
    float weight[MOE_MOST_ENTRIES];
    short plane[MOE_MOST_ENTRIES], owner[MOE_MOST_ENTRIES];
    // by choice, token after token
    short expert_of[MOE_MOST_ENTRIES], first_plane[MOE_MOST_ENTRIES];
    unsigned char token[MOE_MOST_ENTRIES];
    int live, entries, most;               // experts with tokens, their tokens in all, the most of one
};

// until *p >= want, within the limit of every wait here and as long as no CTA has given up
__device__ __forceinline__ int load_acquire(const int* p) {
    int v;
    asm volatile("ld.acquire.gpu.global.b32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
    return v;
}
__device__ __forceinline__ bool wait_count(const int* p, int want, const int* control, volatile int* abortp) {
    unsigned long long t0 = 0;
    for (int i = 0;; ++i) {
        if (load_acquire(p) >= want) return true;
        if (i % 64 == 63) {
            const unsigned long long now = tc::globaltimer();
            if (t0 == 0) t0 = now;
            if (*abortp) return false;
            if (now - t0 > tc::WAIT_LIMIT_NS || load_acquire(control + GAVE_UP)) {
                *abortp = 1;
                return false;
            }
        }
    }
}
__device__ __forceinline__ void grid_barrier(int* control, int which, volatile int* abortp) {
    __syncthreads();
    if (threadIdx.x == 0) {
        if (!*abortp) {
            add_release(control + which, 1);                   // for all that this CTA's threads wrote before they met here
            wait_count(control + which, gridDim.x, control, abortp);
        }
        if (*abortp) add_release(control + GAVE_UP, 1);
    }
    __syncthreads();
}
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async;" ::: "memory"); }

__device__ __forceinline__ void tmem_one(uint32_t& v, uint32_t taddr) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(v) : "r"(taddr));
}

// Terms of eight values of a row (neighbouring threads have a block's others) to the rows `hi`, `lo` of a matrix of rows of
// `pitch` bytes and to its scales; su, sl: the rows' numbers there.
__device__ __forceinline__ void row_terms(const uint4& raw, int c, uint8_t* hi_row, uint8_t* lo_row, uint8_t* scales, int su, int sl) {
    const uint32_t four = 0xfu << (threadIdx.x & 28);
    uint32_t most = magnitude(raw);
    most = __vmaxu2(most, __shfl_xor_sync(four, most, 1));
    most = __vmaxu2(most, __shfl_xor_sync(four, most, 2));
    const int byte = term_byte(max(most << 16, most & 0xffff0000u));
    uint32_t hi[2], lo[2];
    terms_of_bf16(raw, byte, hi, lo);
    *reinterpret_cast<uint2*>(hi_row + c) = make_uint2(hi[0], hi[1]);
    *reinterpret_cast<uint2*>(lo_row + c) = make_uint2(lo[0], lo[1]);
    if ((threadIdx.x & 3) == 0) {
        uint8_t* s = scales + (size_t)(c / GROUP) * TILE_BYTES + c % GROUP / BLOCK;
        s[(su & 31) * 16 + su / 32 * 4] = (uint8_t)byte;
        s[(sl & 31) * 16 + sl / 32 * 4] = low_byte(byte);
    }
}

// A token's choice by one warp whose lanes keep its scores (lane, lane + 32, ...): as moe_route_token, without groups.
__device__ __forceinline__ void choose(const Moe& p, int t, const float* z) {       // z: shared memory
    constexpr int EACH = MOE_MOST_EXPERTS / 32;
    const int lane = threadIdx.x & 31;
    float s[EACH], mx = -INFINITY, den = 0.f;
    int key[EACH];
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        s[i] = lane + 32 * i < p.E ? z[lane + 32 * i] : -INFINITY;
        mx = fmaxf(mx, s[i]);
    }
    mx = warp_max(mx);
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        if (32 * i >= p.E) break;
        if (lane + 32 * i >= p.E) continue;
        s[i] = p.softmax ? expf(s[i] - mx) : moe_sigmoid(s[i]);
        den += s[i];
    }
    den = p.softmax ? warp_sum(den) : 1.f;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        const int e = lane + 32 * i;
        key[i] = INT_MIN;                                      // what cannot be chosen: no expert, no number, minus infinity
        if (e >= p.E) continue;
        if (p.softmax) s[i] = s[i] / den;
        const float c = p.corr != nullptr ? s[i] + load_param(p.corr, p.corr_bf16, e) : s[i];
        const int bits = __float_as_int(c);
        if (c > -INFINITY) key[i] = bits ^ (bits >> 31 & 0x7fffffff);          // ordered as the numbers are
        if (c == 0.f) key[i] = 0;
    }
    float chosen = 0.f, mine = 0.f;
#pragma unroll 1
    for (int j = 0; j < p.top; ++j) {
        int best = INT_MIN, at = p.E;
#pragma unroll
        for (int i = EACH - 1; i >= 0; --i)
            if (key[i] >= best && key[i] != INT_MIN) { best = key[i]; at = lane + 32 * i; }
        const int most = __reduce_max_sync(0xffffffffu, best);
        at = __reduce_min_sync(0xffffffffu, best == most && most != INT_MIN ? at : INT_MAX);
        if (at == INT_MAX) at = 0;                             // every score NaN: keep the indices legal
        float w = 0.f;
#pragma unroll
        for (int i = 0; i < EACH; ++i)
            if (lane + 32 * i == at) { w = s[i]; key[i] = INT_MIN; }
        w = __shfl_sync(0xffffffffu, w, at & 31);
        chosen += w;
        if (lane == j) mine = w;
        if (lane == 0) p.sel_e[t * p.top + j] = at;
    }
    if (lane < p.top) p.sel_w[t * p.top + lane] = (p.renorm ? mine / (chosen + p.sum_eps) : mine) * p.wscale;
}

// 1: logits, choices, x's terms.  A CTA has all logits of a token, or, where a router's rows are too many for that, `dots`
// neighbouring ones (no more than E: of one token or two), and the CTA that finishes a token's makes its choice.  Several warps
// share a row where there are few.
template <typename C> __device__ __forceinline__ void moe_route_and_terms(const Moe& p, float* scratch) {
    __shared__ int finished[2];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, back = gridDim.x - 1 - blockIdx.x;
    const int gtid = back * MOE_THREADS + threadIdx.x, threads = gridDim.x * MOE_THREADS;       // the last CTAs, which have no logits, first
    for (int i = gtid; i < p.ncounters; i += threads) p.ready[i] = 0;             // and the tiles' counters behind them
    if (!C::COMPACT) {
        const int groups = groups_of(p.H), per_row = groups * (GROUP / 8);
        const size_t pitch = (size_t)groups * GROUP;
#pragma unroll 1
        for (int i = gtid; i < p.T * per_row; i += threads) {
            const int r = i / per_row, c = (i - r * per_row) * 8;
            row_terms(row8(p.x + (long long)r * p.ldx, c, p.H, p.wide), c, p.xt + r * pitch, p.xt + (r + C::TT) * pitch, p.xs, r, r + C::TT);
        }
        fence_async();                                         // the terms are read by TMA, of all CTAs
    }
    const int parts = p.dots >= MOE_WARPS ? 1 : MOE_WARPS / p.dots, at_once = MOE_WARPS / parts, part = warp % parts;
    const int len = ((p.H + parts - 1) / parts + 7) / 8 * 8, k0 = part * len, k1 = min(p.H, k0 + len);
    const bool wide = p.wide && p.H % 8 == 0, whole = p.dots == p.E;
    // once for most CTAs; where there are more tokens than CTAs, several times
#pragma unroll 1
    for (int first = blockIdx.x * p.dots; first < p.T * p.E; first += gridDim.x * p.dots) {
        const int count = min(p.dots, p.T * p.E - first);
        if (first != blockIdx.x * p.dots) __syncthreads();     // the scratch has been read
#pragma unroll 1
        for (int i = warp / parts; i < count; i += at_once) {
            const int t = (first + i) / p.E, e = first + i - t * p.E;
            const __nv_bfloat16* row = p.x + (long long)t * p.ldx;
            float sum = 0.f;
            if (wide && p.router_bf16) {
                const __nv_bfloat16* r = static_cast<const __nv_bfloat16*>(p.router) + (size_t)e * p.H;
#pragma unroll 1
                for (int k = k0 + lane * 8; k < k1; k += 8 * 256) {              // eight pieces of either row on their way at once
                    uint4 a[8], w[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const int at = k + j * 256;
                        a[j] = at < k1 ? *reinterpret_cast<const uint4*>(row + at) : make_uint4(0, 0, 0, 0);
                        w[j] = at < k1 ? *reinterpret_cast<const uint4*>(r + at) : make_uint4(0, 0, 0, 0);
                    }
#pragma unroll
                    for (int j = 0; j < 8; ++j)
#pragma unroll
                        for (int l = 0; l < 4; ++l) {
                            const float2 f = __bfloat1622float2(reinterpret_cast<const __nv_bfloat162*>(&a[j])[l]);
                            const float2 g = __bfloat1622float2(reinterpret_cast<const __nv_bfloat162*>(&w[j])[l]);
                            sum = fmaf(f.x, g.x, sum);
                            sum = fmaf(f.y, g.y, sum);
                        }
                }
            } else {
#pragma unroll 8
                for (int k = k0 + lane; k < k1; k += 32) sum = fmaf(to_float(row[k]), load_param(p.router, p.router_bf16, (size_t)e * p.H + k), sum);
            }
            sum = warp_sum(sum);
            if (lane == 0) scratch[i * parts + part] = sum;
        }
        __syncthreads();
        float* zs = scratch + p.dots * parts;                      // the logits, of a token or (then for two warps) of two
        for (int i = threadIdx.x; i < count; i += MOE_THREADS) {
            const int t = (first + i) / p.E, e = first + i - t * p.E;
            float sum = p.rbias != nullptr ? load_param(p.rbias, p.rbias_bf16, e) : 0.f;
            for (int j = 0; j < parts; ++j) sum += scratch[i * parts + j];
            if (whole) zs[i] = sum;
            else p.z[first + i] = sum;
        }
        __syncthreads();
        const int t0 = first / p.E, t1 = (first + count - 1) / p.E;             // no more than E logits: two tokens at most
        if (!whole) {
            if (threadIdx.x < 2) {
                const int t = t0 + threadIdx.x;
                finished[threadIdx.x] = 0;
                if (t <= t1) {
                    const int here = min(first + count, (t + 1) * p.E) - max(first, t * p.E);
                    finished[threadIdx.x] = add_acq_rel(&p.control[TOKEN + t], here) == p.E - here;
                }
            }
            __syncthreads();
        }
        if (warp < 2 && (whole ? warp == 0 : finished[warp] != 0)) {
            const int t = t0 + warp;
            float* s = zs + warp * (4 * p.E + 2 * p.groups_of_experts + 16);
            if (!whole) {
                for (int e = lane; e < p.E; e += 32) s[e] = __ldcg(p.z + t * p.E + e);
                __syncwarp();
            }
            if (p.groups_of_experts > 1 && p.keep < p.groups_of_experts) {
                int* counts = reinterpret_cast<int*>(s + 3 * p.E + 2 * p.groups_of_experts);
                for (int e = lane; e < p.E; e += 32) counts[e] = 0;
                __syncwarp();
                moe_route_token(s, s + p.E, s + 2 * p.E, s + 3 * p.E, p.E, p.top, p.softmax, p.renorm, lane, counts, p.sel_e + t * p.top,
                                p.sel_w + t * p.top, counts + p.E, p.corr, p.corr_bf16, p.groups_of_experts, p.keep, p.wscale, p.sum_eps);
            } else {
                choose(p, t, s);
            }
        }
    }
}

// 2: who has tokens (the masks are zero).  False, for all threads: what was read are not choices.
__device__ __forceinline__ bool moe_lists(const Moe& p, Lists& q) {
    const int n = p.T * p.top;
    constexpr int EACH = (MOE_MOST_ENTRIES + MOE_THREADS - 1) / MOE_THREADS;
    int expert[EACH], wrong = 0;
    float weight[EACH];
#pragma unroll
    for (int h = 0; h < EACH; ++h) {
        const int i = threadIdx.x + h * MOE_THREADS;
        if (i >= n) break;
        expert[h] = __ldcg(p.sel_e + i), weight[h] = __ldcg(p.sel_w + i);
    }
#pragma unroll
    for (int h = 0; h < EACH; ++h) {
        const int i = threadIdx.x + h * MOE_THREADS, t = i / p.top;
        if (i >= n) break;
        if ((unsigned)expert[h] >= (unsigned)p.E) {              // (numbers index shared memory from here on)
            wrong = 1;
            continue;
        }
        q.expert_of[i] = (short)expert[h];
        q.weight[i] = weight[h];
        atomicOr(reinterpret_cast<unsigned int*>(&q.mask[expert[h]]) + t / 32, 1u << (t & 31));
    }
    if (__syncthreads_or(wrong)) return false;
    if (threadIdx.x < 32) {
        const int lane = threadIdx.x;
        int live = 0, first = 0, row8 = 0, most = 0;
#pragma unroll 1
        for (int e0 = 0; e0 < p.E; e0 += 32) {
            const int e = e0 + lane, c = e < p.E ? __popcll(q.mask[e]) : 0;
            const unsigned any = __ballot_sync(0xffffffffu, c > 0);
            int v = c | (c + 7) / 8 * 3 << 16;                    // inclusive sums over the lanes: tokens, rows of h / 8
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int a = __shfl_up_sync(0xffffffffu, v, o);
                if (lane >= o) v += a;
            }
            if (c > 0) {
                const int at = live + __popc(any & ((1u << lane) - 1));
                q.slot[e] = (short)at;
                q.expert[at] = (short)e;
                q.count[at] = (short)c;
                q.first[at] = (short)(first + (v & 0xffff) - c);
                q.hrow8[at] = (short)(row8 + (v >> 16) - (c + 7) / 8 * 3);
            }
            v = __shfl_sync(0xffffffffu, v, 31);
            live += __popc(any);
            first += v & 0xffff;
            row8 += v >> 16;
            most = max(most, __reduce_max_sync(0xffffffffu, c));
        }
        if (lane == 0) { q.live = live; q.entries = first; q.most = most; }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += MOE_THREADS) {
        const int t = i / p.top, j = i - t * p.top, e = q.expert_of[i];
        int same = j;                                            // scores that are not numbers can choose an expert twice
        for (int o = j - 1; o >= 0; --o)
            if (q.expert_of[t * p.top + o] == e) same = o;
        q.first_plane[i] = (short)(t * p.top + same);
        if (same != j) continue;
        const int at = q.first[q.slot[e]] + __popcll(q.mask[e] & ((1ull << t) - 1));
        q.token[at] = (unsigned char)t;
        q.plane[at] = (short)i;
        q.owner[at] = q.slot[e];
    }
    __syncthreads();
    return true;
}

// (compact) rows of x, as terms, laid out for the experts that read them; an expert's counter says how many of its rows are there
__device__ __forceinline__ void moe_compact(const Moe& p, const Lists& q) {
    const int groups = groups_of(p.H);
    const size_t pitch = (size_t)groups * GROUP;
    const int chunks = groups * (GROUP / 8), mine = (q.entries - (int)blockIdx.x + (int)gridDim.x - 1) / (int)gridDim.x;
    for (int w = threadIdx.x - 128; w < mine * chunks; w += 256) {
        const int j = w / chunks, c = (w - j * chunks) * 8, i = blockIdx.x + j * gridDim.x, l = q.owner[i];
        const int r = i - q.first[l], nt = (q.count[l] + 7) / 8 * 8;
        uint8_t* to = p.xt + (size_t)(q.hrow8[l] * 8 + r) * pitch;
        row_terms(row8(p.x + (long long)q.token[i] * p.ldx, c, p.H, p.wide), c, to, to + nt * pitch, p.xs + (size_t)l * groups * TILE_BYTES, r, nt + r);
    }
    fence_async();
    asm volatile("bar.sync 1, 256;" ::: "memory");
    for (int j = threadIdx.x - 128; j < mine; j += 256) {
        add_release(&p.ready[p.most_live + q.owner[blockIdx.x + j * gridDim.x]], 1);
    }
}

// a walk over a CTA's blocks: live expert l, tile, stage k; n blocks left
struct Walk {
    int l, tile, k, n, tiles, kb;
    __device__ __forceinline__ Walk(const Split& s, int cta, int tiles_, int kb_) : tiles(tiles_), kb(kb_) {
        const int b0 = cta < s.P ? s.start(cta) : 0, b1 = cta < s.P ? s.start(cta + 1) : 0, u = b0 / kb;
        l = u / tiles, tile = u - l * tiles, k = b0 - u * kb, n = b1 - b0;
    }
    __device__ __forceinline__ void next() { step(1); }
    __device__ __forceinline__ void step(int blocks) {           // within a unit
        n -= blocks;
        if ((k += blocks) == kb) {
            k = 0;
            if (++tile == tiles) { tile = 0; ++l; }
        }
    }
};

template <typename C>
__global__ void __launch_bounds__(MOE_THREADS, 1)
moe_kernel(const __grid_constant__ CUtensorMap map_gate, const __grid_constant__ CUtensorMap map_up, const __grid_constant__ CUtensorMap map_down,
           const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_h, const __grid_constant__ Moe p) {
    constexpr int TT = C::TT, STAGES = C::STAGES, NCOL = C::NCOL;
    extern __shared__ unsigned char smem_raw[];
    __shared__ Lists q;
    __shared__ int abort_flag, is_last, gone;
    unsigned char* tiles = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    unsigned char* sf = tiles + (size_t)STAGES * C::STAGE;
    uint64_t* full = reinterpret_cast<uint64_t*>(sf + STAGES * C::SF);
    uint64_t *empty = full + STAGES, *acc_full = empty + STAGES, *acc_empty = acc_full + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, cta = blockIdx.x, P = gridDim.x;
    volatile int* abortp = &abort_flag;
    if (threadIdx.x == 0) {
        abort_flag = 0;
        for (int s = 0; s < STAGES; ++s) { mbar_init(&full[s], 2); mbar_init(&empty[s], 1); }
        for (int s = 0; s < 2; ++s) { mbar_init(&acc_full[s], 1); mbar_init(&acc_empty[s], 8); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 2 && lane < 5) {
        const CUtensorMap* m = lane == 0 ? &map_gate : lane == 1 ? &map_up : lane == 2 ? &map_down : lane == 3 ? &map_x : &map_h;
        asm volatile("prefetch.tensormap [%0];" ::"l"(m) : "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_slot)), "r"(C::COLS));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
    }
    for (int e = threadIdx.x; e < p.E; e += MOE_THREADS) q.mask[e] = 0;
    moe_route_and_terms<C>(p, reinterpret_cast<float*>(tiles));
    fence_async();                          // the scratch becomes stages
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    grid_barrier(p.control, FIRST, abortp);
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = *tmem_slot, tmem_sf = tmem + C::COLS - STAGES * C::SF_COLS;
    if (threadIdx.x == 0) gone = *abortp;
    __syncthreads();

    if (gone || !moe_lists(p, q)) {
        if (threadIdx.x == 0) abort_flag = 1;
    } else {
        const int g1 = groups_of(p.H), g2 = groups_of(p.F), tiles1 = g2, tiles_h = (p.H + 127) / 128, tiles2 = (tiles_h + 1) / 2;
        const int total1 = q.live * tiles1 * g1, total2 = q.live * tiles2 * g2;
        // no more than about eight CTAs share a tile: joining more costs more than their blocks
        const Split s1(total1, min(min(P, total1), q.live * tiles1 * 7), g1), s2(total2, min(min(P, total2), q.live * tiles2 * 7), g2);
        Walk a(s1, cta, tiles1, g1), b(s2, cta, tiles2, g2);
        const int n1 = a.n, n = a.n + b.n;
        int* units2 = p.counters + q.live * tiles1;
        // columns of a tile's sums; two sets of them where they fit
        const int cols = max((q.most + 7) / 8 * 24, C::COMPACT ? 0 : NCOL), bufs = 4 * cols + STAGES * C::SF_COLS <= C::COLS ? 2 : 1;

        if (warp == 0) {
            uint32_t parity = 1;                                 // the first round passes at once
            int i = 0;
            for (int s = 0; i < n; ++i) {
                if (!warp_wait(&empty[s], parity, abortp)) break;
                unsigned char *st = tiles + s * C::STAGE, *ss = sf + s * C::SF;
                if (i < n1) {
                    const int e = q.expert[a.l], row = e * p.F + a.tile * 128;
                    const size_t at = ((size_t)(e * tiles1 + a.tile) * g1 + a.k) * TILE_BYTES;
                    if (elect_one()) {
                        mbar_expect_tx(&full[s], 2 * 8192 + 2 * TILE_BYTES);     // spread codes count as they are in memory
                        tma_load_2d(st, &map_gate, &full[s], a.k * 128, row);
                        tma_load_2d(st + 16384, &map_up, &full[s], a.k * 128, row);
                        bulk_load(ss, p.gate_s + at, TILE_BYTES, &full[s]);
                        bulk_load(ss + TILE_BYTES, p.up_s + at, TILE_BYTES, &full[s]);
                    }
                    a.next();
                } else {
                    const int e = q.expert[b.l], t0 = b.tile * 2, row = e * p.H + t0 * 128;
                    if (elect_one()) {
                        mbar_expect_tx(&full[s], 2 * 8192 + 2 * TILE_BYTES);
                        tma_load_2d(st, &map_down, &full[s], b.k * 128, row);
                        tma_load_2d(st + 16384, &map_down, &full[s], b.k * 128, row + 128);
                        bulk_load(ss, p.down_s + ((size_t)(e * tiles_h + t0) * g2 + b.k) * TILE_BYTES, TILE_BYTES, &full[s]);
                        // the last tile may have no partner: its scales again, never stored
                        bulk_load(ss + TILE_BYTES, p.down_s + ((size_t)(e * tiles_h + min(t0 + 1, tiles_h - 1)) * g2 + b.k) * TILE_BYTES, TILE_BYTES,
                                  &full[s]);
                    }
                    b.next();
                }
                __syncwarp();
                if (++s == STAGES) { s = 0; parity ^= 1; }
            }
            if (*abortp)
                for (int j = max(0, i - STAGES); j < i; ++j) mbar_wait(&full[j % STAGES], (j / STAGES) & 1, abortp);
        } else if (warp == 2) {
            int seen = -1;
            uint32_t parity = 1;
            fence_async();
            for (int i = 0, s = 0; i < n; ++i) {
                if (!warp_wait(&empty[s], parity, abortp)) break;
                unsigned char *st = tiles + s * C::STAGE + C::W_BYTES, *ss = sf + s * C::SF + 2 * TILE_BYTES;
                const bool one = i < n1;
                const int l = one ? a.l : b.l, k = one ? a.k : b.k;
                if (one && !C::COMPACT) {
                    if (elect_one()) {
                        mbar_expect_tx(&full[s], NCOL * 128 + TILE_BYTES);
                        tma_load_2d(st, &map_x, &full[s], k * 128, 0);
                        bulk_load(ss, p.xs + (size_t)k * TILE_BYTES, TILE_BYTES, &full[s]);
                    }
                } else {
                    if (i == n1) seen = -1;
                    if (l != seen) {                             // all of this expert's rows are there
                        if (!__all_sync(0xffffffffu, wait_count(one ? &p.ready[p.most_live + l] : &p.ready[l], one ? q.count[l] : tiles1, p.control, abortp))) break;
                        fence_async();
                        seen = l;
                    }
                    const int boxes = (q.count[l] + 7) / 8 * (one ? 2 : 3), row0 = q.hrow8[l] * 8, scales = boxes * 8 > 128 && !one ? 2 * TILE_BYTES : TILE_BYTES;
                    if (elect_one()) {
                        mbar_expect_tx(&full[s], boxes * 1024 + scales);
                        bulk_load(ss, one ? p.xs + ((size_t)l * g1 + k) * TILE_BYTES : p.hs + ((size_t)l * g2 + k) * (2 * TILE_BYTES), scales, &full[s]);
                        for (int j = 0; j < boxes; ++j) tma_load_2d(st + j * 1024, one ? &map_x : &map_h, &full[s], k * 128, row0 + j * 8);
                    }
                }
                if (one) a.next();
                else b.next();
                __syncwarp();
                if (++s == STAGES) { s = 0; parity ^= 1; }
            }
        } else if (warp == 1) {
            const uint64_t desc0 = umma_desc(smem_addr(tiles));
            const uint32_t sf0 = smem_addr(sf);
            int s = 0, buf = 0;
            uint32_t parity = 0, acc_parity = 1;                 // the first wait for each accumulator passes at once
            bool fresh = true;
            for (int i = 0; i < n; ++i) {
                if (fresh && !warp_wait(&acc_empty[buf], acc_parity, abortp)) break;
                if (!warp_wait(&full[s], parity, abortp)) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint32_t ss = sf0 + s * C::SF, tsf = tmem_sf + s * C::SF_COLS;
                const int n_cols = i < n1 ? (C::COMPACT ? (q.count[a.l] + 7) / 8 * 16 : NCOL) : (q.count[b.l] + 7) / 8 * 24;
                const uint32_t idesc = 5u << 7 | (uint32_t)(n_cols >> 3) << 17 | 1u << 23 | 1u << 27;           // E2M1 by E4M3, scales E8M0
                const uint64_t da = desc0 + (uint32_t)(s * (C::STAGE >> 4)), db = da + (C::W_BYTES >> 4);
                const uint32_t d = tmem + buf * 2 * cols;
                const bool done = i == n1 - 1 || i == n - 1 || (i < n1 ? a.k == g1 - 1 : b.k == g2 - 1);
                if (elect_one()) {
#pragma unroll
                    for (int c = 0; c < 3; ++c) scales_to_tmem(tsf + c * 4, ss + c * TILE_BYTES);
                    if (n_cols > 128) scales_to_tmem(tsf + 12, ss + 3 * TILE_BYTES);
#pragma unroll
                    for (uint32_t j = 0; j < 4; ++j)
#pragma unroll
                        for (int w = 0; w < 2; ++w)
                            umma_scaled<true>(d + w * cols, da + w * 1024 + 2 * j, db + 2 * j, idesc | j << 4 | j << 29, tsf + w * 4, tsf + 8, j > 0 || !fresh);
                    umma_commit(&empty[s]);
                    if (done) umma_commit(&acc_full[buf]);
                }
                __syncwarp();
                if (i < n1) a.next();
                else b.next();
                fresh = done;
                if (done && ++buf == bufs) { buf = 0; acc_parity ^= 1; }
                if (++s == STAGES) { s = 0; parity ^= 1; }
            }
        } else if (warp >= 4) {
            const int half = (warp - 4) / 4, quarter = warp & 3, row = quarter * 32 + lane;
            const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
            constexpr int SHARES = 8;
            int seg = 0;
            bool out = false;
            auto begin = [&]() {                                  // the sums of a segment are there; false: a wait ran out
                mbar_wait(&acc_full[seg % bufs], (seg / bufs) & 1, abortp);
                asm volatile("bar.sync 1, 256;" ::: "memory");
                if (threadIdx.x == 128) gone = *abortp;
                asm volatile("bar.sync 1, 256;" ::: "memory");
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                return gone == 0;
            };
            auto release = [&]() {
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(&acc_empty[seg % bufs]);
            };
            if (C::COMPACT) moe_compact(p, q);
            auto last_of = [&](int* counter, int others) {        // of the CTAs that share a tile
                asm volatile("bar.sync 1, 256;" ::: "memory");
                if (threadIdx.x == 128) is_last = add_acq_rel(counter, 1) == others;
                asm volatile("bar.sync 1, 256;" ::: "memory");
                return is_last != 0;
            };
            // ---- gate and up: the halves take the expert's tokens in turn
            while (a.n > 0) {
                const int l = a.l, tile = a.tile, unit = l * tiles1 + tile, take = min(a.n, g1 - a.k);
                const bool whole = take == g1;
                a.step(take);
                if (!begin()) { out = true; break; }
                const int count = q.count[l], first = q.first[l], nt = (count + 7) / 8 * 8, f = tile * 128 + row;
                const uint32_t dg = tmem + lanes + (seg % bufs) * 2 * cols, du = dg + cols;
                auto hidden = [&](int r, float g, float u) {      // all lanes of a warp: a block of 32 of row r of the expert's h
                    const float w = q.weight[q.plane[first + r]];
                    if (p.scale_in) { g *= w; u *= w; }
                    const float h = f < p.F ? moe_glu(g, u, p.act, p.limit) * (p.scale_in ? 1.f : w) : 0.f;
                    const int byte = three_term_byte(__reduce_max_sync(0xffffffffu, __float_as_uint(h) & 0x7fffffffu));
                    uint32_t term[3];
                    three_terms(h, byte, term);
                    uint8_t* to = p.h + (size_t)(q.hrow8[l] * 8 + r) * ((size_t)g2 * GROUP) + f;
                    const size_t next = (size_t)nt * g2 * GROUP;
                    to[0] = (uint8_t)term[0], to[next] = (uint8_t)term[1], to[2 * next] = (uint8_t)term[2];
                    if (lane < 3) {                               // a term's scale each
                        const int v = lane * nt + r;
                        p.hs[((size_t)l * g2 + tile) * (2 * TILE_BYTES) + quarter + v / 128 * TILE_BYTES + (v & 31) * 16 + (v & 127) / 32 * 4] =
                            byte == 255 ? 255 : (uint8_t)(byte - 5 * lane);
                    }
                };
                float* mine = p.part1 + (size_t)(cta * 2 + s1.place(cta, unit)) * (2 * TT * 128) + row;
#pragma unroll 1
                for (int r0 = half * 4; r0 < count; r0 += 8) {
                    uint32_t g[4][2], u[4][2];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int t = C::COMPACT ? min(r0 + j, nt - 1) : r0 + j < count ? q.token[first + r0 + j] : 0, lo = C::COMPACT ? nt : TT;
                        tmem_one(g[j][0], dg + t), tmem_one(g[j][1], dg + lo + t);
                        tmem_one(u[j][0], du + t), tmem_one(u[j][1], du + lo + t);
                    }
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                    for (int j = 0; j < 4; ++j) asm volatile("" : "+r"(g[j][0]), "+r"(g[j][1]), "+r"(u[j][0]), "+r"(u[j][1]));   // not before the wait
#pragma unroll 1
                    for (int j = 0; j < 4 && r0 + j < count; ++j) {
                        const float gs = __uint_as_float(g[0][0]) + __uint_as_float(g[0][1]), us = __uint_as_float(u[0][0]) + __uint_as_float(u[0][1]);
#pragma unroll
                        for (int k = 0; k < 3; ++k) g[k][0] = g[k + 1][0], g[k][1] = g[k + 1][1], u[k][0] = u[k + 1][0], u[k][1] = u[k + 1][1];
                        if (whole) hidden(r0 + j, gs, us);
                        else mine[(r0 + j) * 128] = gs, mine[(TT + r0 + j) * 128] = us;
                    }
                }
                release();
                ++seg;
                if (!whole) {
                    const int c0 = s1.owner(unit * g1), c1 = s1.owner((unit + 1) * g1 - 1);
                    if (!last_of(&p.counters[unit], c1 - c0)) continue;
                    // one CTA's share after another's, the loads of eight at once
#pragma unroll 1
                    for (int r = half * 2; r < count; r += 4) {
                        float g[2] = {}, u[2] = {};
#pragma unroll 1
                        for (int c = c0; c <= c1; c += SHARES) {
                            float gp[SHARES][2], up[SHARES][2];
#pragma unroll
                            for (int k = 0; k < SHARES; ++k) {
                                const bool there = c + k <= c1;
                                const float* from = p.part1 + (size_t)((c + k) * 2 + s1.place(c + k, unit)) * (2 * TT * 128) + r * 128 + row;
                                gp[k][0] = there ? __ldcg(from) : 0.f, gp[k][1] = there ? __ldcg(from + 128) : 0.f;
                                up[k][0] = there ? __ldcg(from + TT * 128) : 0.f, up[k][1] = there ? __ldcg(from + TT * 128 + 128) : 0.f;
                            }
#pragma unroll
                            for (int k = 0; k < SHARES; ++k)
                                g[0] += gp[k][0], g[1] += gp[k][1], u[0] += up[k][0], u[1] += up[k][1];
                        }
#pragma unroll 1
                        for (int j = 0; j < 2 && r + j < count; ++j) {
                            hidden(r + j, g[0], u[0]);
                            g[0] = g[1], u[0] = u[1];
                        }
                    }
                }
                fence_async();
                asm volatile("bar.sync 1, 256;" ::: "memory");
                if (threadIdx.x == 128) add_release(&p.ready[l], 1);
            }
            // ---- down: a half has 128 of the 256 rows
            while (!out && b.n > 0) {
                const int l = b.l, tile = b.tile, unit = l * tiles2 + tile, take = min(b.n, g2 - b.k);
                const bool whole = take == g2;
                b.step(take);
                if (!begin()) break;
                const int count = q.count[l], first = q.first[l], nt = (count + 7) / 8 * 8, f = (tile * 2 + half) * 128 + row;
                const uint32_t d = tmem + lanes + ((seg % bufs) * 2 + half) * cols;
                float* mine = p.part2 + ((size_t)(cta * 2 + s2.place(cta, unit)) * 2 + half) * (TT * 128) + row;
                auto store = [&](int r, float v) {
                    if (f < p.H) p.planes[(size_t)q.plane[first + r] * p.H + f] = v;
                };
                for (int r0 = 0; r0 < count; r0 += 8) {
                    uint32_t r[3][8];
#pragma unroll
                    for (int i = 0; i < 3; ++i)
                        asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                                     : "=r"(r[i][0]), "=r"(r[i][1]), "=r"(r[i][2]), "=r"(r[i][3]), "=r"(r[i][4]), "=r"(r[i][5]), "=r"(r[i][6]), "=r"(r[i][7])
                                     : "r"(d + i * nt + r0));
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        asm volatile("" : "+r"(r[0][j]), "+r"(r[1][j]), "+r"(r[2][j]));
                        if (r0 + j >= count) break;
                        const float v = __uint_as_float(r[0][j]) + (__uint_as_float(r[1][j]) + __uint_as_float(r[2][j]));
                        if (whole) store(r0 + j, v);
                        else mine[(r0 + j) * 128] = v;
                    }
                }
                release();
                ++seg;
                if (whole) continue;
                const int c0 = s2.owner(unit * g2), c1 = s2.owner((unit + 1) * g2 - 1);
                if (!last_of(&units2[unit], c1 - c0)) continue;
#pragma unroll 1
                for (int r = 0; r < count; r += 4) {
                    float v[4] = {};
#pragma unroll 1
                    for (int c = c0; c <= c1; c += SHARES) {
                        float part[SHARES][4];
#pragma unroll
                        for (int k = 0; k < SHARES; ++k) {
                            const bool there = c + k <= c1;
                            const float* from = p.part2 + ((size_t)((c + k) * 2 + s2.place(c + k, unit)) * 2 + half) * (TT * 128) + r * 128 + row;
#pragma unroll
                            for (int j = 0; j < 4; ++j) part[k][j] = there ? __ldcg(from + j * 128) : 0.f;
                        }
#pragma unroll
                        for (int k = 0; k < SHARES; ++k)
#pragma unroll
                            for (int j = 0; j < 4; ++j)
                                v[j] += part[k][j];
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (r + j < count) store(r + j, v[j]);
                }
            }
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    grid_barrier(p.control, SECOND, abortp);
    if (threadIdx.x == 0) gone = *abortp;
    __syncthreads();
    if (!gone) {
        for (int i = cta * MOE_THREADS + threadIdx.x; i < p.T * p.H; i += P * MOE_THREADS) {
            const int t = i / p.H, f = i - t * p.H;
            float v = 0.f;
            for (int j = 0; j < p.top; ++j) v += __ldcg(p.planes + (size_t)q.first_plane[t * p.top + j] * p.H + f);
            if (p.out_bf16) reinterpret_cast<__nv_bfloat16*>(p.y)[t * p.ldy + f] = __float2bfloat16_rn(v);
            else reinterpret_cast<float*>(p.y)[t * p.ldy + f] = v;
        }
    }
    if (threadIdx.x == 0) {
        if (gone) report_error(p.err, PRISM_ERR_WAIT_TIMEOUT);
        __threadfence();
        if (atomicAdd(&p.control[LEAVERS], 1) == P - 1)           // the last to leave clears the control block for the next launch
            for (int i = 0; i < TOKEN + p.T; ++i) p.control[i] = 0;
    }
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::COLS));
    }
}

// ---- host side ------------------------------------------------------------------------------------------------------------

struct MoePlan {
    int tt, P, most_live, most_rows, ncounters;
    bool compact;
    long long xt, xs, h, hs, z, sel_e, sel_w, part1, part2, planes, counters, bytes;
};
// ctas: at most so many (0: one an SM)
inline MoePlan moe_plan(int T, int H, int F, int E, int top, int ctas) {
    MoePlan q;
    q.tt = T <= 8 ? 8 : T <= 16 ? 16 : T <= 32 ? 32 : 64;
    q.P = ctas > 0 && ctas < sm_count() ? ctas : sm_count();
    q.most_live = E < T * top ? E : T * top;
    q.most_rows = 3 * (T * top + 7 * q.most_live);
    const long long g1 = groups_of(H), g2 = groups_of(F), tiles2 = ((H + 127) / 128 + 1) / 2;
    q.ncounters = (int)(q.most_live * (g2 + tiles2) + 2 * q.most_live);
    long long at = 0;
    auto take = [&](long long bytes) { const long long o = at; at += (bytes + 1023) / 1024 * 1024; return o; };
    q.compact = q.tt > 16;
    q.xt = take((q.compact ? (long long)q.most_rows : 2LL * q.tt) * g1 * GROUP);
    q.xs = take((q.compact ? q.most_live : 1) * g1 * TILE_BYTES);
    q.h = take((long long)q.most_rows * g2 * GROUP);
    q.hs = take(q.most_live * g2 * (2 * TILE_BYTES));
    q.z = take(4LL * T * E);
    q.sel_e = take(4LL * T * top);
    q.sel_w = take(4LL * T * top);
    q.part1 = take(4LL * q.P * 2 * 2 * q.tt * 128);
    q.part2 = take(4LL * q.P * 2 * 2 * q.tt * 128);
    q.planes = take(4LL * T * top * H);
    q.counters = take(4LL * q.ncounters);
    q.bytes = at;
    return q;
}
inline bool moe_sizes_ok(int T, int H, int F, int E, int top) {
    return T >= 1 && T <= 64 && H >= 1 && F >= 1 && E >= 1 && E <= MOE_MOST_EXPERTS && top >= 1 && top <= 16 && top <= E &&
           (long long)E * F < (1LL << 31) - 256 && (long long)E * H < (1LL << 31) - 256 && (long long)T * H < (1LL << 31) &&
           (long long)E * groups_of(F) * groups_of(H) < (1LL << 31);
}

template <typename C> int run_moe(const CUtensorMap (&m)[5], const Moe& p, int P, cudaStream_t stream) {
    auto kern = moe_kernel<C>;
    static unsigned char done[64] = {};
    open_once(kern, C::SMEM, done);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(P);
    cfg.blockDim = dim3(MOE_THREADS);
    cfg.dynamicSmemBytes = C::SMEM;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeCooperative;
    attr[0].val.cooperative = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return (int)cudaLaunchKernelEx(&cfg, kern, m[0], m[1], m[2], m[3], m[4], p);
}

}  // namespace mx
}  // namespace prism

// what prism_mxfp4_moe needs for these sizes: bytes of workspace, into need[0], and words of control, into need[1]
PRISM_EXPORT int prism_mxfp4_moe_workspace(int T, int H, int F, int E, int top, int ctas, long long* need) {
    if (!prism::mx::moe_sizes_ok(T, H, F, E, top)) return (int)cudaErrorInvalidValue;
    need[0] = prism::mx::moe_plan(T, H, F, E, top, ctas).bytes;
    need[1] = prism::mx::CONTROL_WORDS;
    return 0;
}

// x [T, H] bfloat16; router [E, H] (+ rbias [E]); gate, up [E, F, H] and down [E, H, F] in 4 bits; corr [E] or null.
// ws: workspace of the call; nothing is launched and -1 returned where its ws_bytes are too few; control: 68 ints, zero before the
// first launch (the kernel leaves them zero), of one stream's launches at a time.  y [T, H] of `out_dtype` (row stride ldy).  ctas: at most so many share the work (0: one an SM).
PRISM_EXPORT int prism_mxfp4_moe(void* ws, long long ws_bytes, int* control, const void* x, long long ldx, const void* router, int router_dtype,
                                 const void* rbias, int rbias_dtype,
                                 const void* gate_codes, const void* gate_scales, const void* up_codes, const void* up_scales,
                                 const void* down_codes, const void* down_scales, int T, int H, int F, int E, int top, int softmax, int renorm,
                                 int scale_in, int act, float limit, const void* corr, int corr_dtype, int groups, int keep, float wscale,
                                 float sum_eps, void* y, int out_dtype, long long ldy, int ctas, int* err, cudaStream_t stream) {
    using namespace prism;
    using namespace prism::mx;
    if (T <= 0) return 0;
    if (!moe_sizes_ok(T, H, F, E, top) || groups < 1 || groups > E || (((uintptr_t)gate_codes | (uintptr_t)up_codes | (uintptr_t)down_codes) & 31) ||
        (((uintptr_t)gate_scales | (uintptr_t)up_scales | (uintptr_t)down_scales) & 15) || ((uintptr_t)ws & 255))
        return (int)cudaErrorInvalidValue;
    const MoePlan q = moe_plan(T, H, F, E, top, ctas);
    if (ws_bytes < q.bytes) return WORKSPACE_TOO_SMALL;
    const int g1 = groups_of(H), g2 = groups_of(F);
    uint8_t* base = static_cast<uint8_t*>(ws);
    CUtensorMap m[5];
    int rc = byte_map(&m[0], gate_codes, (long long)E * F, (long long)g1 * 64, 128, true);
    if (!rc) rc = byte_map(&m[1], up_codes, (long long)E * F, (long long)g1 * 64, 128, true);
    if (!rc) rc = byte_map(&m[2], down_codes, (long long)E * H, (long long)g2 * 64, 128, true);
    if (!rc) rc = byte_map(&m[3], base + q.xt, q.compact ? q.most_rows : 2 * q.tt, (long long)g1 * GROUP, q.compact ? 8 : 2 * q.tt, false);
    if (!rc) rc = byte_map(&m[4], base + q.h, q.most_rows, (long long)g2 * GROUP, 8, false);
    if (rc) return rc;
    Moe p;
    p.x = static_cast<const __nv_bfloat16*>(x);
    p.router = router, p.rbias = rbias, p.corr = corr;
    p.gate_s = static_cast<const uint8_t*>(gate_scales);
    p.up_s = static_cast<const uint8_t*>(up_scales);
    p.down_s = static_cast<const uint8_t*>(down_scales);
    p.xt = base + q.xt, p.xs = base + q.xs, p.h = base + q.h, p.hs = base + q.hs;
    p.z = reinterpret_cast<float*>(base + q.z);
    p.sel_e = reinterpret_cast<int*>(base + q.sel_e);
    p.sel_w = reinterpret_cast<float*>(base + q.sel_w);
    p.part1 = reinterpret_cast<float*>(base + q.part1);
    p.part2 = reinterpret_cast<float*>(base + q.part2);
    p.planes = reinterpret_cast<float*>(base + q.planes);
    p.ready = reinterpret_cast<int*>(base + q.counters);
    p.counters = p.ready + 2 * q.most_live;
    p.control = control, p.err = err;
    p.y = y;
    p.ldx = ldx, p.ldy = ldy;
    p.T = T, p.H = H, p.F = F, p.E = E, p.top = top, p.softmax = softmax, p.renorm = renorm, p.scale_in = scale_in, p.act = act;
    p.groups_of_experts = groups, p.keep = keep;
    // a token's logits in one CTA save a pass through memory (1 token, 8 experts of 2,048: 1.1 us) while there is a warp for each of
    // them and their rows are not long for one SM (64 experts: 9.7 us over all SMs, 11.6 a token an SM)
    p.dots = E <= MOE_WARPS && (long long)E * H <= (1 << 18) && T <= q.P ? E : std::min(E, (T * E + q.P - 1) / q.P);
    p.most_live = q.most_live;
    p.ncounters = q.ncounters;
    p.router_bf16 = router_dtype == PRISM_DTYPE_BF16, p.rbias_bf16 = rbias_dtype == PRISM_DTYPE_BF16, p.corr_bf16 = corr_dtype == PRISM_DTYPE_BF16;
    p.out_bf16 = out_dtype == PRISM_DTYPE_BF16;
    p.wide = (((uintptr_t)x | (uintptr_t)router) & 15) == 0 && ldx % 8 == 0;
    p.limit = limit, p.wscale = wscale, p.sum_eps = sum_eps;
    switch (q.tt) {
        case 8: return run_moe<MoeCfg<8>>(m, p, q.P, stream);
        case 16: return run_moe<MoeCfg<16>>(m, p, q.P, stream);
        case 32: return run_moe<MoeCfg<32>>(m, p, q.P, stream);
        default: return run_moe<MoeCfg<64>>(m, p, q.P, stream);
    }
}
