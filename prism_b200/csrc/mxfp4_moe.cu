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
//      an expert's tokens become h, again as two terms (a warp's 32 lanes are one block)
//   4. down: 256 rows, the expert's own tokens as columns, once all of its h is there (a counter per expert)
//   5. barrier over the grid; y is the sum of a token's choices in their order
// In 3 and 4 the blocks (expert, rows, 128 of K) are dealt to the CTAs evenly as one line; a tile that several CTAs have part of
// is added up by the last to come, in the CTAs' order: results do not depend on timing.
//
// Warp 0 streams weights and their scales, warp 2 x and h, warp 1 issues the products, warps 4-11 take the sums out.  Every
// wait is bounded; on expiry the error word is set, tensor memory is freed, the control block is cleared and the kernel returns.
#include "moe_route.cuh"
#include "mxfp4_mma.cuh"
#include "vec.cuh"

namespace prism {
namespace mx {

constexpr int MOE_THREADS = 384, MOE_WARPS = 12, MOE_MOST_EXPERTS = 256, MOE_MOST_ENTRIES = 1024;

template <int TT_> struct MoeCfg {
    static constexpr int TT = TT_, NCOL = 2 * TT;
    static constexpr int W_BYTES = 2 * 16384, X_BYTES = NCOL * 128, STAGE = W_BYTES + X_BYTES, SF = 3 * TILE_BYTES, SF_COLS = 12;
    static constexpr int FIT = 200 * 1024 / (STAGE + SF), STAGES = FIT > 8 ? 8 : FIT;
    static constexpr int BUFS = 4 * NCOL + STAGES * SF_COLS <= 512 ? 2 : 1;
    static constexpr int USED = BUFS * 2 * NCOL + STAGES * SF_COLS;
    static constexpr int COLS = USED <= 128 ? 128 : USED <= 256 ? 256 : 512;
    static constexpr size_t SMEM = (size_t)STAGES * (STAGE + SF) + 1024 + 512;
    static_assert(USED <= 512 && STAGES >= 3, "tensor memory or shared memory");
};

struct Moe {
    const __nv_bfloat16* x;
    const void *router, *rbias, *corr;
    const uint8_t *gate_s, *up_s, *down_s;
    uint8_t *xt, *xs, *h, *hs;             // x's terms [2 TT][Hp] and scales, h's [rows][Fp] and scales [live][groups][512]
    float *z, *sel_w, *part1, *part2, *planes;
    int *sel_e, *counters, *ready, *control, *err;      // control: barrier, leavers, a counter per token
    void* y;
    long long ldx, ldy;
    int T, H, F, E, top, softmax, renorm, scale_in, act, groups_of_experts, keep, experts_a_warp, ncounters;
    int router_bf16, rbias_bf16, corr_bf16, out_bf16, wide;
    float limit, wscale, sum_eps;
};

struct Lists {                             // of the experts that have tokens, in their order
    unsigned long long mask[MOE_MOST_EXPERTS];
    short slot[MOE_MOST_EXPERTS], expert[MOE_MOST_EXPERTS], count[MOE_MOST_EXPERTS], hrow8[MOE_MOST_EXPERTS], first[MOE_MOST_EXPERTS];
    // an expert's tokens from first[] on, ascending
    float weight[MOE_MOST_ENTRIES];
    short plane[MOE_MOST_ENTRIES], first_plane[MOE_MOST_ENTRIES];
    unsigned char token[MOE_MOST_ENTRIES];
    int live;
};

// until *p >= want, within the limit of every wait here
__device__ __forceinline__ bool wait_count(const int* p, int want, volatile int* abortp) {
    unsigned long long t0 = 0;
    for (int i = 0;; ++i) {
        int v;
        asm volatile("ld.acquire.gpu.global.b32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
        if (v >= want) return true;
        if (i % 64 == 63) {
            const unsigned long long now = tc::globaltimer();
            if (t0 == 0) t0 = now;
            if (*abortp) return false;
            if (now - t0 > tc::WAIT_LIMIT_NS) {
                *abortp = 1;
                return false;
            }
        }
    }
}
__device__ __forceinline__ void grid_barrier(int* bar, int want, volatile int* abortp) {
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) {
        atomicAdd(bar, 1);
        wait_count(bar, want, abortp);
    }
    __syncthreads();
}
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async;" ::: "memory"); }

__device__ __forceinline__ float tmem_one(uint32_t taddr) {
    uint32_t r;
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(r) : "r"(taddr));
    return __uint_as_float(r);
}

// 1: logits, choices, x's terms
__device__ __forceinline__ void moe_route_and_terms(const Moe& p, float* scratch, int tt) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, gw = blockIdx.x * MOE_WARPS + warp, warps = gridDim.x * MOE_WARPS;
    const int groups = groups_of(p.H), per_row = groups * (GROUP / 8);
    const int gtid = blockIdx.x * MOE_THREADS + threadIdx.x, threads = gridDim.x * MOE_THREADS;
    for (int i = gtid; i < p.ncounters; i += threads) p.ready[i] = 0;             // and the tiles' counters behind them
    for (int i = gtid; i < p.T * per_row; i += threads) {
        const int r = i / per_row, c = (i - r * per_row) * 8;
        const __nv_bfloat16* at = p.x + (long long)r * p.ldx + c;
        float v[8];
        if (p.wide && c + 8 <= p.H) {
            load8(at, v);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = c + j < p.H ? to_float(at[j]) : 0.f;
        }
        uint32_t most = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) most = max(most, __float_as_uint(v[j]) & 0x7fffffffu);
        const uint32_t four = 0xfu << (threadIdx.x & 28);
        most = max(most, __shfl_xor_sync(four, most, 1));
        most = max(most, __shfl_xor_sync(four, most, 2));
        const int byte = term_byte(most);
        uint32_t hi[2], lo[2];
        terms_of<8>(v, byte, hi, lo);
        uint8_t* to = p.xt + (size_t)r * groups * GROUP + c;
        *reinterpret_cast<uint2*>(to) = make_uint2(hi[0], hi[1]);
        *reinterpret_cast<uint2*>(to + (size_t)tt * groups * GROUP) = make_uint2(lo[0], lo[1]);
        if ((threadIdx.x & 3) == 0) {
            uint8_t* s = p.xs + (size_t)(c / GROUP) * TILE_BYTES + c % GROUP / BLOCK;
            const int u = r + tt;
            s[(r & 31) * 16 + r / 32 * 4] = (uint8_t)byte;
            s[(u & 31) * 16 + u / 32 * 4] = low_byte(byte);
        }
    }
    fence_async();                                             // the terms are read by TMA, of all CTAs
    constexpr int MOST = 4;
    const int chunks = (p.E + p.experts_a_warp - 1) / p.experts_a_warp, items = p.T * chunks;
    for (int i = gw; i < items; i += warps) {
        const int t = i / chunks, e0 = (i - t * chunks) * p.experts_a_warp, ne = min(p.experts_a_warp, p.E - e0);
        const __nv_bfloat16* row = p.x + (long long)t * p.ldx;
        float sum[MOST] = {};
        if (p.wide && p.H % 8 == 0) {
#pragma unroll 2
            for (int k = lane * 8; k < p.H; k += 256) {
                float a[8], w[8];
                load8(row + k, a);
#pragma unroll
                for (int j = 0; j < MOST; ++j)
                    if (j < ne) {
                        load_param8(p.router, p.router_bf16, (size_t)(e0 + j) * p.H + k, w);
#pragma unroll
                        for (int l = 0; l < 8; ++l) sum[j] = fmaf(a[l], w[l], sum[j]);
                    }
            }
        } else {
            for (int k = lane; k < p.H; k += 32) {
                const float a = to_float(row[k]);
#pragma unroll
                for (int j = 0; j < MOST; ++j)
                    if (j < ne) sum[j] = fmaf(a, load_param(p.router, p.router_bf16, (size_t)(e0 + j) * p.H + k), sum[j]);
            }
        }
#pragma unroll
        for (int j = 0; j < MOST; ++j) {
            if (j >= ne) break;
            const float s = warp_sum(sum[j]);
            if (lane == 0) p.z[t * p.E + e0 + j] = s + (p.rbias != nullptr ? load_param(p.rbias, p.rbias_bf16, e0 + j) : 0.f);
        }
        int last = 0;
        if (lane == 0) {
            __threadfence();
            last = atomicAdd(&p.control[2 + t], 1) == chunks - 1;
            __threadfence();
        }
        if (!__shfl_sync(0xffffffffu, last, 0)) continue;
        __threadfence();
        float* zs = scratch + (size_t)warp * (4 * p.E + 2 * p.groups_of_experts + 16);
        int* counts = reinterpret_cast<int*>(zs + 3 * p.E + 2 * p.groups_of_experts);
        for (int e = lane; e < p.E; e += 32) {
            zs[e] = __ldcg(p.z + t * p.E + e);
            counts[e] = 0;
        }
        __syncwarp();
        moe_route_token(zs, zs + p.E, zs + 2 * p.E, zs + 3 * p.E, p.E, p.top, p.softmax, p.renorm, lane, counts, p.sel_e + t * p.top,
                        p.sel_w + t * p.top, counts + p.E, p.corr, p.corr_bf16, p.groups_of_experts, p.keep, p.wscale, p.sum_eps);
        __syncwarp();
    }
}

// 2: who has tokens
__device__ __forceinline__ void moe_lists(const Moe& p, Lists& q) {
    const int n = p.T * p.top;
    for (int e = threadIdx.x; e < p.E; e += MOE_THREADS) q.mask[e] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += MOE_THREADS) {
        const int t = i / p.top;
        atomicOr(reinterpret_cast<unsigned int*>(&q.mask[__ldcg(p.sel_e + i)]) + t / 32, 1u << (t & 31));
    }
    __syncthreads();
    if (threadIdx.x < 32) {
        const int lane = threadIdx.x;
        int live = 0, first = 0, row8 = 0;
        for (int e0 = 0; e0 < p.E; e0 += 32) {
            const int e = e0 + lane, c = e < p.E ? __popcll(q.mask[e]) : 0;
            int l = c > 0, f = c, r = (c + 7) / 8 * 2;            // inclusive sums over the lanes: experts, tokens, rows of h / 8
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int a = __shfl_up_sync(0xffffffffu, l, o), b = __shfl_up_sync(0xffffffffu, f, o), d = __shfl_up_sync(0xffffffffu, r, o);
                if (lane >= o) { l += a; f += b; r += d; }
            }
            if (c > 0) {
                const int at = live + l - 1;
                q.slot[e] = (short)at;
                q.expert[at] = (short)e;
                q.count[at] = (short)c;
                q.first[at] = (short)(first + f - c);
                q.hrow8[at] = (short)(row8 + r - (c + 7) / 8 * 2);
            }
            live += __shfl_sync(0xffffffffu, l, 31);
            first += __shfl_sync(0xffffffffu, f, 31);
            row8 += __shfl_sync(0xffffffffu, r, 31);
        }
        if (lane == 0) q.live = live;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += MOE_THREADS) {
        const int t = i / p.top, j = i - t * p.top, e = __ldcg(p.sel_e + i);
        int same = j;                                            // scores that are not numbers can choose an expert twice
        for (int o = 0; o < j; ++o)
            if (__ldcg(p.sel_e + t * p.top + o) == e) { same = o; break; }
        q.first_plane[i] = (short)(t * p.top + same);
        if (same != j) continue;
        const int at = q.first[q.slot[e]] + __popcll(q.mask[e] & ((1ull << t) - 1));
        q.token[at] = (unsigned char)t;
        q.weight[at] = __ldcg(p.sel_w + i);
        q.plane[at] = (short)i;
    }
    __syncthreads();
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
    uint64_t *empty = full + STAGES, *acc_full = empty + STAGES, *acc_empty = acc_full + C::BUFS;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + C::BUFS);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, cta = blockIdx.x, P = gridDim.x;
    volatile int* abortp = &abort_flag;
    if (threadIdx.x == 0) {
        abort_flag = 0;
        for (int s = 0; s < STAGES; ++s) { mbar_init(&full[s], 2); mbar_init(&empty[s], 1); }
        for (int s = 0; s < C::BUFS; ++s) { mbar_init(&acc_full[s], 1); mbar_init(&acc_empty[s], 8); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_slot)), "r"(C::COLS));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
    }
    moe_route_and_terms(p, reinterpret_cast<float*>(tiles), TT);
    fence_async();                          // the scratch becomes stages
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    grid_barrier(p.control, P, abortp);
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = *tmem_slot, tmem_sf = tmem + C::BUFS * 2 * NCOL;
    if (threadIdx.x == 0) gone = *abortp;
    __syncthreads();

    if (!gone) {
        moe_lists(p, q);
        const int g1 = groups_of(p.H), g2 = groups_of(p.F), tiles1 = g2, tiles_h = (p.H + 127) / 128, tiles2 = (tiles_h + 1) / 2;
        const int total1 = q.live * tiles1 * g1, total2 = q.live * tiles2 * g2;
        const Split s1(total1, min(P, total1), g1), s2(total2, min(P, total2), g2);
        Walk a(s1, cta, tiles1, g1), b(s2, cta, tiles2, g2);
        const int n1 = a.n, n = a.n + b.n;
        int* units2 = p.counters + q.live * tiles1;

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
                if (i < n1) {
                    if (elect_one()) {
                        mbar_expect_tx(&full[s], C::X_BYTES + TILE_BYTES);
                        tma_load_2d(st, &map_x, &full[s], a.k * 128, 0);
                        bulk_load(ss, p.xs + (size_t)a.k * TILE_BYTES, TILE_BYTES, &full[s]);
                    }
                    a.next();
                } else {
                    if (b.l != seen) {                           // all of this expert's h is there
                        if (!__all_sync(0xffffffffu, wait_count(&p.ready[b.l], tiles1, abortp))) break;
                        fence_async();
                        seen = b.l;
                    }
                    const int boxes = (q.count[b.l] + 7) / 8 * 2;
                    if (elect_one()) {
                        mbar_expect_tx(&full[s], boxes * 1024 + TILE_BYTES);
                        bulk_load(ss, p.hs + ((size_t)b.l * g2 + b.k) * TILE_BYTES, TILE_BYTES, &full[s]);
                        for (int j = 0; j < boxes; ++j) tma_load_2d(st + j * 1024, &map_h, &full[s], b.k * 128, (q.hrow8[b.l] + j) * 8);
                    }
                    b.next();
                }
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
                const int cols = i < n1 ? NCOL : (q.count[b.l] + 7) / 8 * 16;
                const uint32_t idesc = 5u << 7 | (uint32_t)(cols >> 3) << 17 | 1u << 23 | 1u << 27;           // E2M1 by E4M3, scales E8M0
                const uint64_t da = desc0 + (uint32_t)(s * (C::STAGE >> 4)), db = da + (C::W_BYTES >> 4);
                const uint32_t d = tmem + buf * 2 * NCOL;
                const bool done = i == n1 - 1 || i == n - 1 || (i < n1 ? a.k == g1 - 1 : b.k == g2 - 1);
                if (elect_one()) {
#pragma unroll
                    for (int c = 0; c < 3; ++c) scales_to_tmem(tsf + c * 4, ss + c * TILE_BYTES);
#pragma unroll
                    for (uint32_t j = 0; j < 4; ++j)
#pragma unroll
                        for (int w = 0; w < 2; ++w)
                            umma_scaled<true>(d + w * NCOL, da + w * 1024 + 2 * j, db + 2 * j, idesc | j << 4 | j << 29, tsf + w * 4, tsf + 8, j > 0 || !fresh);
                    umma_commit(&empty[s]);
                    if (done) umma_commit(&acc_full[buf]);
                }
                __syncwarp();
                if (i < n1) a.next();
                else b.next();
                fresh = done;
                if (done && ++buf == C::BUFS) { buf = 0; acc_parity ^= 1; }
                if (++s == STAGES) { s = 0; parity ^= 1; }
            }
        } else if (warp >= 4) {
            const int half = (warp - 4) / 4, quarter = warp & 3, row = quarter * 32 + lane;
            const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
            int seg = 0;
            bool out = false;
            auto begin = [&]() {                                  // the sums of a segment are there; false: a wait ran out
                mbar_wait(&acc_full[seg % C::BUFS], (seg / C::BUFS) & 1, abortp);
                asm volatile("bar.sync 1, 256;" ::: "memory");
                if (threadIdx.x == 128) gone = *abortp;
                asm volatile("bar.sync 1, 256;" ::: "memory");
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                return gone == 0;
            };
            auto release = [&]() {
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(&acc_empty[seg % C::BUFS]);
            };
            auto last_of = [&](int* counter, int others) {        // of the CTAs that share a tile
                __threadfence();
                asm volatile("bar.sync 1, 256;" ::: "memory");
                if (threadIdx.x == 128) is_last = atomicAdd(counter, 1) == others;
                asm volatile("bar.sync 1, 256;" ::: "memory");
                __threadfence();
                return is_last != 0;
            };
            // ---- gate and up: the halves take four of the expert's tokens in turn
            while (a.n > 0) {
                const int l = a.l, tile = a.tile, unit = l * tiles1 + tile, take = min(a.n, g1 - a.k);
                const bool whole = take == g1;
                a.step(take);
                if (!begin()) { out = true; break; }
                const int count = q.count[l], first = q.first[l], nt = (count + 7) / 8 * 8, f = tile * 128 + row;
                const uint32_t dg = tmem + lanes + (seg % C::BUFS) * 2 * NCOL, du = dg + NCOL;
                auto hidden = [&](int r, float g, float u) {      // all lanes of a warp: a block of 32 of row r of the expert's h
                    const float w = q.weight[first + r];
                    if (p.scale_in) { g *= w; u *= w; }
                    float h[4] = {f < p.F ? moe_glu(g, u, p.act, p.limit) * (p.scale_in ? 1.f : w) : 0.f, 0.f, 0.f, 0.f};
                    const int byte = term_byte(__reduce_max_sync(0xffffffffu, __float_as_uint(h[0]) & 0x7fffffffu));
                    uint32_t hi[1], lo[1];
                    terms_of<4>(h, byte, hi, lo);
                    uint8_t* to = p.h + (size_t)(q.hrow8[l] * 8 + r) * ((size_t)g2 * GROUP) + f;
                    to[0] = (uint8_t)hi[0];
                    to[(size_t)nt * g2 * GROUP] = (uint8_t)lo[0];
                    if (lane == 0) {
                        uint8_t* s = p.hs + ((size_t)l * g2 + tile) * TILE_BYTES + quarter;
                        const int v = nt + r;
                        s[(r & 31) * 16 + r / 32 * 4] = (uint8_t)byte;
                        s[(v & 31) * 16 + v / 32 * 4] = low_byte(byte);
                    }
                };
                float* mine = p.part1 + (size_t)(cta * 2 + s1.place(cta, unit)) * (2 * TT * 128) + row;
                for (int r0 = half * 4; r0 < count; r0 += 8) {
                    float g[4][2], u[4][2];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int t = r0 + j < count ? q.token[first + r0 + j] : 0;
                        g[j][0] = tmem_one(dg + t), g[j][1] = tmem_one(dg + TT + t);
                        u[j][0] = tmem_one(du + t), u[j][1] = tmem_one(du + TT + t);
                    }
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        asm volatile("" : "+f"(g[j][0]), "+f"(g[j][1]), "+f"(u[j][0]), "+f"(u[j][1]));       // not before the wait
                        if (r0 + j >= count) break;
                        const float gs = g[j][0] + g[j][1], us = u[j][0] + u[j][1];
                        if (whole) hidden(r0 + j, gs, us);
                        else mine[(r0 + j) * 128] = gs, mine[(TT + r0 + j) * 128] = us;
                    }
                }
                release();
                ++seg;
                if (!whole) {
                    const int c0 = s1.owner(unit * g1), c1 = s1.owner((unit + 1) * g1 - 1);
                    if (!last_of(&p.counters[unit], c1 - c0)) continue;
                    for (int r = half; r < count; r += 2) {
                        float g = 0.f, u = 0.f;
#pragma unroll 8
                        for (int c = c0; c <= c1; ++c) {
                            const float* from = p.part1 + (size_t)(c * 2 + s1.place(c, unit)) * (2 * TT * 128) + r * 128 + row;
                            g += __ldcg(from), u += __ldcg(from + TT * 128);
                        }
                        hidden(r, g, u);
                    }
                }
                fence_async();
                __threadfence();
                asm volatile("bar.sync 1, 256;" ::: "memory");
                if (threadIdx.x == 128) {
                    __threadfence();
                    atomicAdd(&p.ready[l], 1);
                }
            }
            // ---- down: a half has 128 of the 256 rows
            while (!out && b.n > 0) {
                const int l = b.l, tile = b.tile, unit = l * tiles2 + tile, take = min(b.n, g2 - b.k);
                const bool whole = take == g2;
                b.step(take);
                if (!begin()) break;
                const int count = q.count[l], first = q.first[l], nt = (count + 7) / 8 * 8, f = (tile * 2 + half) * 128 + row;
                const uint32_t d = tmem + lanes + ((seg % C::BUFS) * 2 + half) * NCOL;
                float* mine = p.part2 + ((size_t)(cta * 2 + s2.place(cta, unit)) * 2 + half) * (TT * 128) + row;
                auto store = [&](int r, float v) {
                    if (f < p.H) p.planes[(size_t)q.plane[first + r] * p.H + f] = v;
                };
                for (int r0 = 0; r0 < count; r0 += 8) {
                    uint32_t r[8], o[8];
                    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "r"(d + r0));
                    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                                 : "=r"(o[0]), "=r"(o[1]), "=r"(o[2]), "=r"(o[3]), "=r"(o[4]), "=r"(o[5]), "=r"(o[6]), "=r"(o[7]) : "r"(d + nt + r0));
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        asm volatile("" : "+r"(r[j]), "+r"(o[j]));
                        if (r0 + j >= count) break;
                        const float v = __uint_as_float(r[j]) + __uint_as_float(o[j]);
                        if (whole) store(r0 + j, v);
                        else mine[(r0 + j) * 128] = v;
                    }
                }
                release();
                ++seg;
                if (whole) continue;
                const int c0 = s2.owner(unit * g2), c1 = s2.owner((unit + 1) * g2 - 1);
                if (!last_of(&units2[unit], c1 - c0)) continue;
                for (int r = 0; r < count; ++r) {
                    float v = 0.f;
#pragma unroll 8
                    for (int c = c0; c <= c1; ++c)
                        v += __ldcg(p.part2 + ((size_t)(c * 2 + s2.place(c, unit)) * 2 + half) * (TT * 128) + r * 128 + row);
                    store(r, v);
                }
            }
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    grid_barrier(p.control, 2 * P, abortp);
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
        if (atomicAdd(&p.control[1], 1) == P - 1) {               // the last to leave clears the control block for the next launch
            for (int t = 0; t < p.T; ++t) p.control[2 + t] = 0;
            p.control[0] = p.control[1] = 0;
        }
    }
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::COLS));
    }
}

// ---- host side ------------------------------------------------------------------------------------------------------------

struct MoePlan {
    int tt, P, most_live, most_rows, ncounters;
    long long xt, xs, h, hs, z, sel_e, sel_w, part1, part2, planes, counters, bytes;
};
inline MoePlan moe_plan(int T, int H, int F, int E, int top) {
    MoePlan q;
    q.tt = T <= 8 ? 8 : T <= 16 ? 16 : T <= 32 ? 32 : 64;
    q.P = sm_count();
    q.most_live = E < T * top ? E : T * top;
    q.most_rows = 2 * (T * top + 7 * q.most_live);
    const long long g1 = groups_of(H), g2 = groups_of(F), tiles2 = ((H + 127) / 128 + 1) / 2;
    q.ncounters = (int)(q.most_live * (g2 + tiles2) + q.most_live);
    long long at = 0;
    auto take = [&](long long bytes) { const long long o = at; at += (bytes + 1023) / 1024 * 1024; return o; };
    q.xt = take(2LL * q.tt * g1 * GROUP);
    q.xs = take(g1 * TILE_BYTES);
    q.h = take((long long)q.most_rows * g2 * GROUP);
    q.hs = take(q.most_live * g2 * TILE_BYTES);
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
    cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::SMEM);
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

// bytes of workspace that prism_mxfp4_moe needs for these sizes, into *bytes
PRISM_EXPORT int prism_mxfp4_moe_workspace(int T, int H, int F, int E, int top, long long* bytes) {
    if (!prism::mx::moe_sizes_ok(T, H, F, E, top)) return (int)cudaErrorInvalidValue;
    *bytes = prism::mx::moe_plan(T, H, F, E, top).bytes;
    return 0;
}

// x [T, H] bfloat16; router [E, H] (+ rbias [E]); gate, up [E, F, H] and down [E, H, F] in 4 bits; corr [E] or null.
// ws: workspace of the call; control: 66 ints, zero before the first launch (the kernel leaves them zero), of one stream's
// launches at a time.  y [T, H] of `out_dtype` (row stride ldy).
PRISM_EXPORT int prism_mxfp4_moe(const void* x, long long ldx, const void* router, int router_dtype, const void* rbias, int rbias_dtype,
                                 const void* gate_codes, const void* gate_scales, const void* up_codes, const void* up_scales,
                                 const void* down_codes, const void* down_scales, int T, int H, int F, int E, int top, int softmax, int renorm,
                                 int scale_in, int act, float limit, const void* corr, int corr_dtype, int groups, int keep, float wscale,
                                 float sum_eps, void* y, int out_dtype, long long ldy, void* ws, int* control, int* err, cudaStream_t stream) {
    using namespace prism;
    using namespace prism::mx;
    if (T <= 0) return 0;
    if (!moe_sizes_ok(T, H, F, E, top) || groups < 1 || groups > E || (((uintptr_t)gate_codes | (uintptr_t)up_codes | (uintptr_t)down_codes) & 31) ||
        (((uintptr_t)gate_scales | (uintptr_t)up_scales | (uintptr_t)down_scales) & 15) || ((uintptr_t)ws & 255))
        return (int)cudaErrorInvalidValue;
    const MoePlan q = moe_plan(T, H, F, E, top);
    const int g1 = groups_of(H), g2 = groups_of(F);
    uint8_t* base = static_cast<uint8_t*>(ws);
    CUtensorMap m[5];
    int rc = byte_map(&m[0], gate_codes, (long long)E * F, (long long)g1 * 64, 128, true);
    if (!rc) rc = byte_map(&m[1], up_codes, (long long)E * F, (long long)g1 * 64, 128, true);
    if (!rc) rc = byte_map(&m[2], down_codes, (long long)E * H, (long long)g2 * 64, 128, true);
    if (!rc) rc = byte_map(&m[3], base + q.xt, 2 * q.tt, (long long)g1 * GROUP, 2 * q.tt, false);
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
    p.counters = p.ready + q.most_live;
    p.control = control, p.err = err;
    p.y = y;
    p.ldx = ldx, p.ldy = ldy;
    p.T = T, p.H = H, p.F = F, p.E = E, p.top = top, p.softmax = softmax, p.renorm = renorm, p.scale_in = scale_in, p.act = act;
    p.groups_of_experts = groups, p.keep = keep;
    const int warps = q.P * MOE_WARPS, each = (T * E + warps - 1) / warps;
    p.experts_a_warp = each < 4 ? each : 4;
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
