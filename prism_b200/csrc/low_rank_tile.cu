// Low-rank adapters (low_rank.cu has the formula) for portions of prompts: tiles of 128 tokens on the 5th-generation tensor cores, bfloat16 adapters.
//
// Two launches.  The first forms the hidden values: a cluster of eight CTAs has a tile of tokens, each CTA every eighth block of 64 k of x and of all
// slices' A (TMA, 128-byte swizzle, tcgen05.mma with the tokens as M); their sums meet through distributed shared memory, are scaled and leave as
// two bfloat16 terms, high and low (2^-16 of a hidden value is lost; one term alone would lose 2^-8, as much as rounding the result does).  The
// second multiplies them with B, 128 columns at a time, and adds the shared result: it is bound by reading and writing that - the 7B shape's gate
// and up for 2,048 tokens are 310 MB against 28 MB of everything else.  So the shared result comes and goes by TMA, boxes of 128 rows by 128 bytes, eight
// of them on their way or at work, and a thread adds its row's sums where they lie in shared memory.
//
// Measured for that, rank 64, one adapter: 17 us for the hidden values and 70 for the results on their own, 77 together (the floor is 52; torch copies the shared
// result in 48): 4.4 TB/s.  A launch that only passes boxes through takes 59: what bounds it is how fast an SM's share comes and goes.  Beside it a tile
// of 128 x 128 moves 208 KB through shared memory, 1,600 cycles at 128 bytes a cycle of some 3,600.
//
// A tile's tokens may have several adapters, or some of them none.  Up to four adapters' products lie side by side in tensor memory (in the first launch as many
// as have 256 hidden values together, and it goes through the tile again for the next).  With more than four, or where base and out are no place for TMA, it goes through the tile
// once for each adapter, and the threads store that adapter's rows: 2,048 tokens, rank 16, with 1, 2, 4, 5, 8 and 16 adapters in each tile take for gate and up 77, 94, 152, 444,
// 662 and 1,264 us (one by one 446 whatever they are), for q, k and v 24, 30, 46, 92, 132 and 247 (163 to 197).
#include "tcgen05.cuh"
#include "vec.cuh"

namespace prism {
namespace lowrank_tile {

using namespace prism::tc;
constexpr int TILE = 128;                     // tokens of a tile, and columns of one of B
constexpr int BLOCK_BYTES = TILE * TILE_K * 2;
constexpr int CTAS = 8;                       // that share a tile's K
constexpr int EPI_WARPS = 8, EPI_THREADS = EPI_WARPS * 32, ALL_THREADS = EPI_THREADS + 64;
constexpr int MOST_RANK = 128, MOST_SLICES = 8, MOST_HIDDEN = 512;
constexpr int HIDDEN_STAGES = 6;
constexpr int CHUNK = 64, CHUNK_LD = CHUNK + 4;                   // columns of sums on their way through shared memory, and their pitch
constexpr int WIDE = 128, WIDE_LD = WIDE + 4;                     // the same of hidden values

struct Tiles {
    int n, first[MOST_SLICES + 1];            // slice g has the result columns first[g] .. first[g + 1] - 1
    // of the second launch: slice g has the CTAs units[g] .. units[g + 1] - 1 of a tile of tokens, and before[g] tiles of columns lie before it
    int units[MOST_SLICES + 1], before[MOST_SLICES + 1];
};

// The tokens' adapters (-1: none, or beyond the end) and the different ones among them, in order.  By one warp.
__device__ __forceinline__ void list_adapters(const int* ids, int t0, int tokens, int L, int* own, int* list, int* count, int* err) {
    const int lane = threadIdx.x & 31;
    int n = 0, all[TILE / 32];
#pragma unroll
    for (int q = 0; q < TILE / 32; ++q) all[q] = t0 + q * 32 + lane < tokens ? ids[t0 + q * 32 + lane] : -1;
#pragma unroll
    for (int q = 0; q < TILE / 32; ++q) {
        int id = all[q];
        if (id >= L) {
            report_error(err, PRISM_ERR_ADAPTER_RANGE);
            id = -1;
        }
        id = max(id, -1);
        own[q * 32 + lane] = id;
        const uint32_t same = __match_any_sync(0xffffffffu, id);
        bool first = id >= 0 && __ffs(same) - 1 == lane;
        for (int i = 0; i < n; ++i) first = first && list[i] != id;
        const uint32_t found = __ballot_sync(0xffffffffu, first);
        if (first) list[n + __popc(found & ((1u << lane) - 1))] = id;
        n += __popc(found);
        __syncwarp();
    }
    if (lane == 0) *count = n;
}

__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) { asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory"); }
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory");
}
// After a wait that ran out: whether a copy that is on its way has landed, with a limit of its own (the flag that ends the others is set).  The CTA's
// shared memory is another one's when it leaves.
__device__ __forceinline__ void drain(uint64_t* bar, uint32_t parity) {
    const unsigned long long t0 = globaltimer();
    while (!mbar_try_wait(bar, parity) && (long long)(globaltimer() - t0) < 200000000ll) {}
}
__device__ __forceinline__ uint32_t instruction(int n) {
    return (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(TILE >> 4) << 24);
}
__device__ __forceinline__ void epilogue_barrier() { asm volatile("bar.sync 1, %0;" ::"n"(EPI_THREADS) : "memory"); }

// ---- hidden values ------------------------------------------------------------------------------------------

// hidden: [tokens][2][G r], high terms and low ones; adapters: how many a tile has
__global__ void __launch_bounds__(ALL_THREADS)
low_rank_hidden_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_a, const float* __restrict__ scale,
                       const int* __restrict__ ranks, const int* __restrict__ ids_, __nv_bfloat16* __restrict__ hidden, int* __restrict__ adapters, int tokens, int K, int r, int G, int L, int ring_bytes,
                       int most_adapters, int tmem_cols, int* err) {
    extern __shared__ unsigned char raw[];
    unsigned char* ring = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
    const int H = G * r;
    float* sums = reinterpret_cast<float*>(ring);                  // behind a pass's last product, its sums; there is memory for as many at least
    __shared__ uint64_t full[HIDDEN_STAGES], empty[HIDDEN_STAGES], done;
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_flag, own[TILE], list[TILE], count;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, me = blockIdx.x, t0 = blockIdx.y * TILE;
    const int blocks = (K + TILE_K - 1) / TILE_K, mine = blocks > me ? (blocks - me + CTAS - 1) / CTAS : 0;
    volatile int* abortp = &abort_flag;

    if (threadIdx.x == 0) {
        prefetch_map(&map_x), prefetch_map(&map_a);
        abort_flag = 0;
        for (int s = 0; s < HIDDEN_STAGES; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
        mbar_init(&done, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    pdl_wait();                               // before tensor memory is taken: a kernel that this one waits for may still want it
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_slot)), "r"(tmem_cols));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
    }
    if (warp == 2) list_adapters(pdl_fresh(ids_), t0, tokens, L, own, list, &count, me == 0 ? err : nullptr);
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = tmem_slot;
    const int passes = count;
    if (me == 0 && threadIdx.x == 0) adapters[blockIdx.y] = passes;
    pdl_trigger();                            // not before this CTA has its tensor memory: the next kernel may take the rest and wait

    // Up to most_adapters at a time: their products with a block of x lie side by side in tensor memory, a row has its own.
    const int side = min(passes, most_adapters), stage_bytes = BLOCK_BYTES + side * H * TILE_K * 2, stages = side > 0 ? min(HIDDEN_STAGES, ring_bytes / stage_bytes) : 1;
    int it = 0;                               // blocks so far, over all passes
    bool go = true;                           // no wait of this warp has run out
    for (int first = 0, p = 0; first < passes; first += side, ++p) {
        const int adapters_now = min(side, passes - first);
        if (warp == 0) {
            if (lane == 0 && !*abortp) {
                int issued = 0;
                for (int i = 0; i < mine; ++i) {
                    const int s = (it + i) % stages, round = (it + i) / stages;
                    if (round > 0 && !mbar_wait(&empty[s], (round - 1) & 1, abortp)) break;
                    unsigned char* st = ring + (size_t)s * stage_bytes;
                    mbar_expect_tx(&full[s], BLOCK_BYTES + adapters_now * H * TILE_K * 2);
                    const int k = (me + i * CTAS) * TILE_K;
                    tma_load_2d(st, &map_x, &full[s], k, t0);
                    for (int b = 0; b < adapters_now; ++b)
                        for (int g = 0; g < G; ++g)
                            tma_load_2d(st + BLOCK_BYTES + (b * H + g * r) * TILE_K * 2, &map_a, &full[s], k, (list[first + b] * G + g) * r);
                    issued = i + 1;
                }
                if (*abortp)
                    for (int i = max(0, issued - stages); i < issued; ++i) drain(&full[(it + i) % stages], ((it + i) / stages) & 1);
            }
        } else if (warp == 1) {
            if (lane == 0) {
                const uint32_t idesc = instruction(r);
                bool ok = !*abortp;
                for (int i = 0; i < mine && ok; ++i) {
                    const int s = (it + i) % stages;
                    ok = mbar_wait(&full[s], ((it + i) / stages) & 1, abortp);
                    if (!ok) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint32_t st = smem_addr(ring + (size_t)s * stage_bytes);
                    const uint64_t dx = umma_desc(st);
                    for (int row = 0; row < adapters_now * H; row += r) {          // a slice's rows start on 8 rows of 128 bytes, as r is a multiple of 16
                        const uint64_t da = umma_desc(st + BLOCK_BYTES + row * TILE_K * 2);
#pragma unroll
                        for (int k = 0; k < TILE_K / UMMA_K; ++k)
                            umma_bf16(tmem + row, dx + (uint64_t)(k * UMMA_K * 2 >> 4), da + (uint64_t)(k * UMMA_K * 2 >> 4), idesc, (i > 0 || k > 0) ? 1u : 0u);
                    }
                    umma_commit(&empty[s]);
                }
                if (mine > 0) {
                    umma_commit(&done);
                    if (*abortp) drain(&done, p & 1);          // products on their way read shared memory and write tensor memory
                }
            }
        }
        __syncwarp();
        const int q = warp & 3, half = (warp - 2) >> 2, tid = threadIdx.x - 64;        // of the epilogue's warps
        if (warp >= 2) {
            if (mine > 0) go = __all_sync(0xffffffffu, mbar_wait(&done, p & 1, abortp)) && go;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        }
        int which = -1;                       // this row's adapter among these
        if (warp >= 2)
            for (int b = 0; b < adapters_now; ++b)
                if (own[q * 32 + lane] == list[first + b]) which = b;
        const uint32_t present = __reduce_or_sync(0xffffffffu, which < 0 ? 0u : 1u << which);
        for (int c0 = 0; c0 < H; c0 += WIDE) {
            if (warp >= 2) {
                // this CTA's sums: a thread's row is its tensor memory lane
#pragma unroll
                for (int m = 0; m < WIDE / 64; ++m) {
                    const int at = m * 64 + half * 32;
                    if (c0 + at >= H) break;
                    float v[32];
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[i] = 0.f;
                    if (mine > 0 && go)
#pragma unroll 1
                        for (int b = 0; b < adapters_now; ++b) {
                            if (!(present >> b & 1)) continue;
                            float w[32];
                            tmem_load<32>(tmem + ((uint32_t)(q * 32) << 16) + b * H + c0 + at, w);         // columns beyond H are allocated, and not used
#pragma unroll
                            for (int i = 0; i < 32; ++i) v[i] = which == b ? w[i] : v[i];
                        }
                    float* row = sums + (q * 32 + lane) * WIDE_LD + at;
#pragma unroll
                    for (int i = 0; i < 32; i += 4) *reinterpret_cast<float4*>(row + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
                }
            }
            asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
            if (warp >= 2) {
                // sixteen rows of all CTAs' sums: four columns a thread at a time
                const int wide = min(WIDE, H - c0) / 4;
                for (int e = tid; e < TILE / CTAS * wide; e += EPI_THREADS) {
                    const int row = me * (TILE / CTAS) + e / wide, c = e % wide * 4, t = t0 + row;
                    int l = -1;
                    for (int b = 0; b < adapters_now; ++b)
                        if (own[row] == list[first + b]) l = own[row];
                    if (l < 0 || !go) continue;
                    const float s = scale[l];
                    int mine = 4;                                  // of these columns, the adapter's own (low_rank.cu)
                    if (ranks) {
                        const int g = (c0 + c) / r;
                        mine = ranks[l * G + g] - (c0 + c - g * r);
                    }
                    const uint32_t at = smem_addr(sums + row * WIDE_LD + c);
                    float4 part[CTAS];
#pragma unroll
                    for (int j = 0; j < CTAS; ++j) {
                        uint32_t peer;
                        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(peer) : "r"(at), "r"(j));
                        asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                                     : "=f"(part[j].x), "=f"(part[j].y), "=f"(part[j].z), "=f"(part[j].w) : "r"(peer) : "memory");
                    }
                    float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int j = 0; j < CTAS; ++j) v[0] += part[j].x, v[1] += part[j].y, v[2] += part[j].z, v[3] += part[j].w;
                    __nv_bfloat16 hi[4], lo[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float h = i < mine ? v[i] * s : 0.f;
                        hi[i] = __float2bfloat16_rn(h);
                        const float rest = h - __bfloat162float(hi[i]);
                        lo[i] = __float2bfloat16_rn(fabsf(rest) < INFINITY ? rest : 0.f);        // an infinity's rest is none
                    }
                    __nv_bfloat16* to = hidden + (size_t)t * 2 * H + c0 + c;
                    *reinterpret_cast<uint2*>(to) = *reinterpret_cast<uint2*>(hi);
                    *reinterpret_cast<uint2*>(to + H) = *reinterpret_cast<uint2*>(lo);
                }
            }
            __syncwarp();
            asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
        }
        it += mine;
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncthreads();                      // the sums have been read: the next pass's copies may come
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    }
    if (threadIdx.x == 0 && abort_flag) report_error(err, PRISM_ERR_WAIT_TIMEOUT);
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(tmem_cols));
}

// ---- results ------------------------------------------------------------------------------------------------

template <typename O> struct Eight;           // eight neighbouring results, 16 or 32 bytes
template <> struct Eight<__nv_bfloat16> {
    uint4 raw;
    __device__ __forceinline__ void load(const __nv_bfloat16* p) { raw = *reinterpret_cast<const uint4*>(p); }
    __device__ __forceinline__ void zero() { raw = make_uint4(0, 0, 0, 0); }
    __device__ __forceinline__ void get(float (&v)[8]) const { load8(reinterpret_cast<const __nv_bfloat16*>(&raw), v); }
};
template <> struct Eight<float> {
    float4 a, b;
    __device__ __forceinline__ void load(const float* p) { a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1]; }
    __device__ __forceinline__ void zero() { a = b = make_float4(0, 0, 0, 0); }
    __device__ __forceinline__ void get(float (&v)[8]) const {
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    }
};

struct Boxes { CUtensorMap base[MOST_SLICES], out[MOST_SLICES]; };         // a slice's columns each

__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, const void* src, int c0, int c1) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(map), "r"(smem_addr(src)), "r"(c0), "r"(c1) : "memory");
}

constexpr int MOST_STAGES = 3, ACCS = 4;                          // ACCS: accumulators, all of tensor memory
constexpr int PARTS = 4;                                          // groups of four warps that each have a box; with two of them 2,048 tokens took 112 us, with four 104
// A wait knows a barrier's phase by one bit, so who waits on a barrier has to wait for each of its phases.  Parts take boxes in turn and tiles of
// columns in turn: a box's memory is always the same part's (the boxes there is memory for are a multiple of the parts), and a product's barrier
// is its tile's of the next four (one that a tile later comes back to has been seen: it takes ACCS products more at least).  With six boxes a
// part met a box's third use while the second, another part's, was still on its way, and took it for its own.
constexpr int MOST_BOXES = 8, TILE_TURNS = 4;
constexpr int MOST_EVEN = 64;                                      // tiles of tokens that CTAs share evenly, by what they cost
static_assert(MOST_BOXES == 8 && PARTS == 4 && TILE_TURNS % PARTS == 0 && TILE_TURNS >= ACCS, "see above");
constexpr int RESULT_THREADS = 64 + PARTS * 128 + 64;             // and two more warps: one asks for boxes, one sends them off

// 32 columns of a warp's lanes in one load
__device__ __forceinline__ void tmem_load_wide(uint32_t at, float (&v)[32]) {
    uint32_t r[32];
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,"
                 "%28,%29,%30,%31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
                   "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
                   "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]),
                   "=r"(r[31])
                 : "r"(at));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_load_wide(uint32_t at, float (&v)[16]) { tmem_load<16>(at, v); }

// 16 bytes of results, plus sums
__device__ __forceinline__ uint4 plus(const uint4& old, const float* v, __nv_bfloat16) {
    const uint32_t u[4] = {old.x, old.y, old.z, old.w};
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 t = __floats2bfloat162_rn(__uint_as_float(u[i] << 16) + v[2 * i], __uint_as_float(u[i] & 0xffff0000u) + v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&t);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ uint4 plus(const uint4& old, const float* v, float) {
    return make_uint4(__float_as_uint(__uint_as_float(old.x) + v[0]), __float_as_uint(__uint_as_float(old.y) + v[1]),
                      __float_as_uint(__uint_as_float(old.z) + v[2]), __float_as_uint(__uint_as_float(old.w) + v[3]));
}

struct Shared {
    uint64_t full[MOST_STAGES], empty[MOST_STAGES], acc_full[TILE_TURNS * ACCS], acc_empty[ACCS], h_full, last, box_full[MOST_BOXES], box_done[MOST_BOXES],
        box_empty[MOST_BOXES];
    uint32_t tmem_slot;
    int abort_flag, own[TILE], list[TILE], count, start[MOST_EVEN + 1], several;
};
constexpr int BARRIERS = 2 * MOST_STAGES + (TILE_TURNS + 1) * ACCS + 2 + 3 * MOST_BOXES;           // the first members, one after the other
template <int PER_TILE> __device__ __forceinline__ void init_barriers(Shared& sh) {
    for (int s = 0; s < MOST_STAGES; ++s) mbar_init(&sh.full[s], 1), mbar_init(&sh.empty[s], 1);
    for (int s = 0; s < ACCS; ++s) mbar_init(&sh.acc_empty[s], 4 * min(PARTS, PER_TILE));
    for (int s = 0; s < TILE_TURNS * ACCS; ++s) mbar_init(&sh.acc_full[s], 1);
    for (int s = 0; s < MOST_BOXES; ++s) mbar_init(&sh.box_full[s], 1), mbar_init(&sh.box_done[s], 4), mbar_init(&sh.box_empty[s], 1);
    mbar_init(&sh.h_full, 1), mbar_init(&sh.last, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
}

// A part of the results: tokens from t0 on, slice g, tiles j0 to j1 - 1 of its columns.
// by_box: a bit a slice, whether its columns of base and out can go by TMA; buffers: of 16 KB there is memory for, beside the hidden values
template <typename O>
__device__ __forceinline__ void result_part(Shared& sh, const CUtensorMap& map_h, const CUtensorMap& map_b, const Boxes& boxes, const int* ids, const O* base,
                                            long long ldb, O* out, long long ldo, int by_box, int buffers, int aligned, int tokens, int r, int N, int L,
                                            const Tiles& tiles, int t0, int g, int j0, int j1, bool first) {
    constexpr int BOX_COLS = 128 / (int)sizeof(O), PER_TILE = TILE / BOX_COLS;         // columns of a box of 128 bytes a row
    extern __shared__ unsigned char raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
    const int kblocks = (r + TILE_K - 1) / TILE_K;
    unsigned char* h_hi = smem;                                                        // high terms, then low ones
    unsigned char* ring = smem + 2 * kblocks * BLOCK_BYTES;
    auto &full = sh.full, &empty = sh.empty;
    auto& acc_full = sh.acc_full;
    auto& acc_empty = sh.acc_empty;
    auto &h_full = sh.h_full, &last = sh.last;
    auto &box_full = sh.box_full, &box_done = sh.box_done, &box_empty = sh.box_empty;
    auto &own = sh.own, &list = sh.list;
    int& count = sh.count;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    volatile int* abortp = &sh.abort_flag;
    const int n_first = tiles.first[g], n_end = tiles.first[g + 1];
    if (warp == 2) list_adapters(ids, t0, tokens, L, own, list, &count, nullptr);
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = sh.tmem_slot;
    const int passes = count;
    // Up to ACCS adapters: their products with a tile of columns lie side by side in tensor memory, a thread takes its row's, and the results go by
    // boxes.  Else one adapter after the other.
    // The memory: eight boxes, and three tiles of B, or four and two of twice the size (four boxes and seven tiles, where a tile has two adapters
    // and uses up B faster, took 2,048 tokens of such tiles from 119 to 124 us)
    const int depth_log = kblocks == 1 ? 3 : 2, depth = 1 << depth_log, stages = (buffers - depth) / kblocks;
    unsigned char* box = ring + stages * kblocks * BLOCK_BYTES;
    float* sums = reinterpret_cast<float*>(box);                                       // where no boxes are used
    const bool nothing = passes == 0 && (const O*)out == base, by_boxes = !nothing && passes <= ACCS && (by_box >> g & 1);
    if (first) pdl_trigger();                            // not before this CTA has its tensor memory: the next kernel may take the rest and wait
    // products are numbered: tile by tile and in it adapter by adapter, or adapter by adapter
    const int products = passes * (j1 - j0);
    struct Turn {                             // of a product: its tile and its adapter's number among the tile's
        int tile = 0, adapter = 0;
        __device__ __forceinline__ void next(bool by_boxes, int tiles, int adapters) {
            if (by_boxes) {
                if (++adapter == adapters) adapter = 0, ++tile;
            } else if (++tile == tiles) {
                tile = 0, ++adapter;
            }
        }
    };

    if (warp == 0) {
        if (lane == 0 && products > 0) {
            // a token's hidden values are its own adapter's, whichever B they are multiplied with: other rows of a product are not used
            mbar_expect_tx(&h_full, 2 * kblocks * BLOCK_BYTES);
            for (int term = 0; term < 2; ++term)
                for (int k = 0; k < kblocks; ++k)
                    tma_load_2d(h_hi + (term * kblocks + k) * BLOCK_BYTES, &map_h, &h_full, (term * tiles.n + g) * r + k * TILE_K, t0);
            Turn turn;
            int i = 0, s = 0, round = 0;
            for (; i < products; ++i) {
                if (round > 0 && !mbar_wait(&empty[s], (round - 1) & 1, abortp)) break;
                mbar_expect_tx(&full[s], kblocks * BLOCK_BYTES);
                for (int k = 0; k < kblocks; ++k)
                    tma_load_2d(ring + (s * kblocks + k) * BLOCK_BYTES, &map_b, &full[s], k * TILE_K, list[turn.adapter] * N + n_first + (j0 + turn.tile) * TILE);
                turn.next(by_boxes, j1 - j0, passes);
                if (++s == stages) s = 0, ++round;
            }
            // the last products have read their tiles of B: nothing is on its way to a barrier when the part ends
            for (int k = max(0, i - stages); k < i && !*abortp; ++k) mbar_wait(&empty[k % stages], (k / stages) & 1, abortp);
            if (*abortp) {
                drain(&h_full, 0);
                for (int k = max(0, i - stages); k < i; ++k) drain(&full[k % stages], (k / stages) & 1);
            }
        }
    } else if (warp == 1) {
        if (lane == 0 && products > 0) {
            const uint32_t idesc = instruction(TILE);
            // one thread's instructions between products are time that the tensor cores stand still: descriptors differ by addresses in 16 bytes
            const uint64_t dh = umma_desc(smem_addr(h_hi)), db0 = umma_desc(smem_addr(ring));
            constexpr uint64_t BLOCK = BLOCK_BYTES >> 4, STEP = UMMA_K * 2 >> 4;
            Turn turn;
            bool ok = mbar_wait(&h_full, 0, abortp);
            int s = 0, round = 0;
            for (int i = 0; i < products && ok; ++i) {
                const int acc = i % ACCS;
                ok = mbar_wait(&full[s], round & 1, abortp) && (i < ACCS || mbar_wait(&acc_empty[acc], (i / ACCS - 1) & 1, abortp));
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint32_t d = tmem + acc * TILE;
                const uint64_t db = db0 + s * kblocks * BLOCK;
                for (int block = 0; block < kblocks; ++block) {
                    const int steps = min(r - block * TILE_K, TILE_K) / UMMA_K;
#pragma unroll
                    for (int k = 0; k < TILE_K / UMMA_K; ++k)
                        if (k < steps) {
                            umma_bf16(d, dh + block * BLOCK + k * STEP, db + block * BLOCK + k * STEP, idesc, block + k > 0 ? 1u : 0u);
                            umma_bf16(d, dh + (kblocks + block) * BLOCK + k * STEP, db + block * BLOCK + k * STEP, idesc, 1u);
                        }
                }
                umma_commit(&empty[s]);
                umma_commit(&acc_full[by_boxes ? turn.tile % TILE_TURNS * ACCS + turn.adapter : acc]);
                turn.next(by_boxes, j1 - j0, passes);
                if (++s == stages) s = 0, ++round;
            }
            if (*abortp) {                    // products on their way read shared memory and write tensor memory
                umma_commit(&last);
                drain(&last, 0);
            }
        }
    } else if (warp == RESULT_THREADS / 32 - 2) {
        if (lane == 0 && by_boxes && base) {
            const int steps = PER_TILE * (j1 - j0);
            int i = 0;
            for (; i < steps; ++i) {
                const int s = i & depth - 1;
                if (i >= depth && !mbar_wait(&box_empty[s], (i >> depth_log) - 1 & 1, abortp)) break;
                mbar_expect_tx(&box_full[s], BLOCK_BYTES);
                tma_load_2d(box + s * BLOCK_BYTES, &boxes.base[g], &box_full[s], j0 * TILE + i * BOX_COLS, t0);
            }
            if (*abortp)
                for (int k = max(0, i - depth); k < i; ++k) drain(&box_full[k & depth - 1], k >> depth_log & 1);
        }
    } else if (warp == RESULT_THREADS / 32 - 1) {
        // sends boxes off; a box's memory is free when the store after it is on its way and its own has read it
        if (lane == 0 && by_boxes) {
            const int steps = PER_TILE * (j1 - j0), width = n_end - n_first;
            for (int i = 0; i < steps; ++i) {
                const int s = i & depth - 1, c = j0 * TILE + i * BOX_COLS;
                if (!mbar_wait(&box_done[s], i >> depth_log & 1, abortp) || *abortp) break;
                if (c < width) tma_store_2d(&boxes.out[g], box + s * BLOCK_BYTES, c, t0);
                asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                if (i > 0) {
                    asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
                    mbar_arrive(&box_empty[i - 1 & depth - 1]);
                }
            }
            asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
        }
    } else {
        // after a wait that ran out the loops go on, as the barriers of these threads count on all of them, but touch nothing
        const int tid = threadIdx.x - 64, q = warp & 3, part = (warp - 2) >> 2;
        bool ok = true;
        auto wait_for_sums = [&](int barrier, int phase) {
            ok = __all_sync(0xffffffffu, mbar_wait(&acc_full[barrier], phase & 1, abortp)) && ok;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        };
        auto sums_read = [&](int product, int times) {
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0)
                for (int i = 0; i < times; ++i) mbar_arrive(&acc_empty[product % ACCS]);
        };
        if (by_boxes) {
            // A thread has a row of a box; four warps have one, the next four the next.
            // 16 bytes of a row lie at their place xor the row's number: no bank conflicts.  A part has one box of a tile at most.
            constexpr int E = 16 / (int)sizeof(O), COLS = BOX_COLS / 2;
            static_assert(PER_TILE <= PARTS && PARTS % PER_TILE == 0, "a part's boxes are of different tiles");
            const int row = q * 32 + lane, steps = PER_TILE * (j1 - j0);
            int which = -1;                   // the row's adapter among the tile's
            for (int p = 0; p < passes; ++p)
                if (own[row] == list[p]) which = p;
            // of the tile's adapters, those of this warp's rows: a portion's border is seldom among them, so its other products are not loaded
            const uint32_t present = __reduce_or_sync(0xffffffffu, which < 0 ? 0u : 1u << which);
            const bool alone = (present & (present - 1)) == 0;
            const int sole = present ? __ffs(present) - 1 : 0;
#pragma unroll 1
            for (int step = part; step < steps; step += PARTS) {
                const int t = step / PER_TILE, in = step % PER_TILE, s = step & depth - 1;
                for (int p = 0; p < passes; ++p) wait_for_sums(t % TILE_TURNS * ACCS + p, t / TILE_TURNS);
                if (base) {
                    ok = __all_sync(0xffffffffu, mbar_wait(&box_full[s], step >> depth_log & 1, abortp)) && ok;
                } else if (step >= depth) {                        // the stores that had this box's memory have read it
                    ok = __all_sync(0xffffffffu, mbar_wait(&box_empty[s], (step >> depth_log) - 1 & 1, abortp)) && ok;
                }
                auto release = [&]() {
                    for (int p = 0; p < passes; ++p) sums_read(t * passes + p, 1);
                };
                if (ok && (present || !base))                      // rows without an adapter stay as they came, bit by bit
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        float v[COLS];
                        const uint32_t from = tmem + ((uint32_t)(q * 32) << 16) + in * BOX_COLS + half * COLS;
                        if (alone && present) {
                            tmem_load_wide(from + (t * passes + sole) % ACCS * TILE, v);
                            if (which < 0)
#pragma unroll
                                for (int c = 0; c < COLS; ++c) v[c] = 0.f;
                        } else {
#pragma unroll
                            for (int c = 0; c < COLS; ++c) v[c] = 0.f;
#pragma unroll 1
                            for (int p = 0; p < passes; ++p) {
                                if (!(present >> p & 1)) continue;
                                float w[COLS];
                                tmem_load_wide(from + (t * passes + p) % ACCS * TILE, w);
#pragma unroll
                                for (int c = 0; c < COLS; ++c) v[c] = which == p ? w[c] : v[c];
                            }
                        }
                        if (half == 1) release();
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            uint4* at = reinterpret_cast<uint4*>(box + s * BLOCK_BYTES + row * 128 + (((half * 4 + c) ^ (row & 7)) * 16));
                            if (which >= 0 || !base) *at = plus(base ? *at : make_uint4(0, 0, 0, 0), v + c * E, O());
                        }
                    }
                else release();
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(&box_done[s]);
            }
        } else if (warp < 2 + EPI_WARPS) {
            int i = 0;
            for (int p = 0; p < passes; ++p) {
                const int l = list[p];
                // Steps of 64 columns.  What a step adds to is asked for a step ahead: eight columns of four rows a thread.
                const int c = tid % 8 * 8, row0 = tid / 8, steps = 2 * (j1 - j0);
                Eight<O> old[4], ahead[4];
                auto ask = [&](Eight<O> (&e)[4], int step) {
                    const int n0 = n_first + j0 * TILE + step * CHUNK;
                    const bool whole = aligned && n0 % 8 == 0 && step < steps && n0 + c + 8 <= n_end;
#pragma unroll
                    for (int m = 0; m < 4; ++m) {
                        const int row = row0 + 32 * m;
                        e[m].zero();
                        if (whole && base && own[row] == l) e[m].load(base + (size_t)(t0 + row) * ldb + n0 + c);
                    }
                };
                ask(ahead, 0);
#pragma unroll 1
                for (int step = 0; step < steps; ++step) {
                    const int acc = i % ACCS, half = step & 1, n0 = n_first + j0 * TILE + step * CHUNK, wide = min(CHUNK, n_end - n0);
#pragma unroll
                    for (int m = 0; m < 4; ++m) old[m] = ahead[m];
                    ask(ahead, step + 1);
                    if (half == 0) wait_for_sums(acc, i / ACCS);
                    if (wide > 0 && ok) {
                        float v[32];
                        tmem_load<32>(tmem + ((uint32_t)(q * 32) << 16) + acc * TILE + half * CHUNK + part * 32, v);
                        float* row = sums + (q * 32 + lane) * CHUNK_LD + part * 32;
#pragma unroll
                        for (int e = 0; e < 32; e += 4) *reinterpret_cast<float4*>(row + e) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
                    }
                    if (half == 1) sums_read(i++, min(PARTS, PER_TILE) * 4 / EPI_WARPS);
                    epilogue_barrier();
                    if (ok && c < wide) {
                        const bool whole = aligned && n0 % 8 == 0 && c + 8 <= wide;
#pragma unroll
                        for (int m = 0; m < 4; ++m) {
                            const int row = row0 + 32 * m;
                            if (own[row] != l) continue;
                            float v[8], s[8];
                            load8(sums + row * CHUNK_LD + c, s);
                            O* to = out + (size_t)(t0 + row) * ldo + n0 + c;
                            if (whole) {
                                old[m].get(v);
#pragma unroll
                                for (int e = 0; e < 8; ++e) v[e] += s[e];
                                store8(to, v);
                            } else {
                                for (int e = 0; e < min(8, wide - c); ++e)
                                    to[e] = from_float<O>(base ? to_float(base[(size_t)(t0 + row) * ldb + n0 + c + e]) + s[e] : s[e]);
                            }
                        }
                    }
                    epilogue_barrier();
                }
            }
            if ((const O*)out != base) {      // tokens without an adapter
                const int n0 = n_first + j0 * TILE, n1 = min(n_end, n_first + j1 * TILE);
                for (int row = warp - 2; row < TILE; row += EPI_WARPS)
                    if (own[row] < 0 && t0 + row < tokens) {
                        O* to = out + (size_t)(t0 + row) * ldo;
                        const O* from = base ? base + (size_t)(t0 + row) * ldb : nullptr;
                        const bool eights = aligned && n0 % 8 == 0;
#pragma unroll 2
                        for (int n = n0 + lane * 8; eights && n + 8 <= n1; n += 256) {
                            Eight<O> e;
                            e.zero();
                            if (from) e.load(from + n);
                            float v[8];
                            e.get(v);
                            store8(to + n, v);
                        }
                        for (int n = (eights ? n1 - (n1 - n0) % 8 : n0) + lane; n < n1; n += 32) to[n] = from ? from[n] : from_float<O>(0.f);
                    }
            }
        }
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();                             // a warp whose first thread worked alone is whole again: what follows is for whole warps
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}

// Results, one way or the other.  A CTA has some columns of one slice of one tile of tokens.  Or, where `adapters` is given and a tile of tokens has several, all
// CTAs have the same share of the work, parts of neighbouring tiles one after the other: a tile of columns costs more with more adapters, and one tile of tokens
// with two would hold up all others (2,048 tokens in three portions, gate and up of the 7B shape, rank 64: 107 us, shared evenly 92).  To end a part and begin the
// next costs 6 to 8 us (2,048 tokens of one adapter 76 us, shared evenly 84; 1,024 tokens 48 and 54), so this is for several adapters, and for 16
// tiles of columns a CTA and more.  A tile of columns counts 5 with one adapter, 3 + 2 n with up to four, 5 + 5 n with more, where gate and up took (times above) 5, 6 and 10
// with one, two and four, 29, 43 and 82 with 5, 8 and 16.
// Registers are short for float32 results: 164 bytes a thread go through memory (44 for bfloat16 ones), most of it on the way without boxes.
template <typename O>
__global__ void __launch_bounds__(RESULT_THREADS, 1)
low_rank_result_kernel(const __grid_constant__ CUtensorMap map_h, const __grid_constant__ CUtensorMap map_b, const __grid_constant__ Boxes boxes,
                       const int* __restrict__ ids_, const int* __restrict__ adapters_, const O* base, long long ldb, O* out, long long ldo, int by_box, int buffers,
                       int aligned, int tokens, int r, int N, int L, const __grid_constant__ Tiles tiles, int* err) {
    constexpr int PER_TILE = TILE * (int)sizeof(O) / 128;
    __shared__ Shared sh;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        prefetch_map(&map_h), prefetch_map(&map_b);
        sh.abort_flag = 0;
        init_barriers<PER_TILE>(sh);
    }
    pdl_wait();
    const int* ids = pdl_fresh(ids_);
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&sh.tmem_slot)), "r"(ACCS * TILE));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
    }
    const int token_tiles = (tokens + TILE - 1) / TILE, columns = tiles.before[tiles.n], units = tiles.units[tiles.n];
    bool even = false;
    if (adapters_ != nullptr) {
        if (warp == 3) {                      // where a tile of tokens starts in the whole, in fifths of what a tile of columns costs with one adapter
            const int* adapters = pdl_fresh(adapters_);
            int before = 0;
            bool several = false;
            for (int q = 0; q < MOST_EVEN / 32; ++q) {
                const int at = q * 32 + lane, n = at < token_tiles ? adapters[at] : 0;
                int sum = at < token_tiles ? columns * (n <= 1 ? 5 : n <= ACCS ? 3 + 2 * n : 5 + 5 * n) : 0;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int up = __shfl_up_sync(0xffffffffu, sum, o);
                    if (lane >= o) sum += up;
                }
                sh.start[at + 1] = before + sum;
                before += __shfl_sync(0xffffffffu, sum, 31);
                several = __any_sync(0xffffffffu, n > 1) || several;
            }
            if (lane == 0) sh.start[0] = 0, sh.several = several;
        }
        __syncthreads();
        even = sh.several;
    }
    int tile = blockIdx.x / units, g = 0, j0 = 0, j1 = 0, column = 0, low = 0, high = 0;
    if (even) {
        const long long whole = sh.start[token_tiles];
        low = (int)(whole * blockIdx.x / gridDim.x), high = (int)(whole * (blockIdx.x + 1) / gridDim.x);
        tile = 0;
        while (sh.start[tile + 1] <= low) ++tile;
        const int one = (sh.start[tile + 1] - sh.start[tile]) / columns;
        column = (low - sh.start[tile] + one - 1) / one;           // a tile of columns is the CTA's in whose share it starts
    } else {
        const int own = blockIdx.x % units;
        while (own >= tiles.units[g + 1]) ++g;
        const int all = tiles.before[g + 1] - tiles.before[g], mine = tiles.units[g + 1] - tiles.units[g], unit = own - tiles.units[g];
        j0 = (int)((long long)all * unit / mine), j1 = (int)((long long)all * (unit + 1) / mine);
    }
#pragma unroll 1
    for (bool first = true; tile < token_tiles; first = false) {
        if (even) {
            if (sh.start[tile] >= high || sh.abort_flag) break;
            const int one = (sh.start[tile + 1] - sh.start[tile]) / columns, end = min(columns, (high - sh.start[tile] + one - 1) / one);
            if (column >= end) {
                ++tile, column = 0;
                if (first) pdl_trigger();                          // a share that is rounded to nothing
                continue;
            }
            g = 0;
            while (column >= tiles.before[g + 1]) ++g;
            j0 = column - tiles.before[g], column = min(end, tiles.before[g + 1]), j1 = column - tiles.before[g];
            if (!first && threadIdx.x == 0) {
                for (int i = 0; i < BARRIERS; ++i) asm volatile("mbarrier.inval.shared::cta.b64 [%0];" ::"r"(smem_addr(&sh.full[0] + i)) : "memory");
                init_barriers<PER_TILE>(sh);
            }
        }
        result_part<O>(sh, map_h, map_b, boxes, ids, base, ldb, out, ldo, by_box, buffers, aligned, tokens, r, N, L, tiles, tile * TILE, g, j0, j1, first);
        if (!even) break;
    }
    if (threadIdx.x == 0 && sh.abort_flag) report_error(err, PRISM_ERR_WAIT_TIMEOUT);
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(sh.tmem_slot), "r"(ACCS * TILE));
}

// Columns of base or out as boxes of rows of 128 bytes
template <typename O> int make_box_map(CUtensorMap* map, const void* ptr, long long rows, long long cols, long long ld, int box_rows) {
    if (sizeof(O) == 2) return prism::tc::make_map(map, ptr, rows, cols, ld, box_rows);
    EncodeTiledFn fn = encode_fn();
    if (fn == nullptr) return (int)cudaErrorNotSupported;
    cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)ld * 4};
    cuuint32_t size[2] = {32, (cuuint32_t)box_rows};
    cuuint32_t estr[2] = {1, 1};
    const CUresult code = fn(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 2, const_cast<void*>(ptr), dims, strides, size, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return code == CUDA_SUCCESS ? 0 : (int)cudaErrorInvalidValue;
}

template <typename O>
int launch_results(const void* hidden, const int* adapters, const CUtensorMap& map_b, const int* ids, const void* base, long long ldb, void* out, long long ldo, int T, int r, int L,
                   Tiles s, int* err, int sms, cudaStream_t stream) {
    const int tiles = (T + TILE - 1) / TILE, G = s.n, N = s.first[G], kblocks = (r + TILE_K - 1) / TILE_K;
    CUtensorMap map_h;
    int code = prism::tc::make_map(&map_h, hidden, T, 2ll * G * r, 2ll * G * r, TILE);
    if (code != 0) return code;
    Boxes boxes;
    int by_box = 0;
    const long long row_b = T > 1 ? ldb : (N + 7) / 8 * 8, row_o = T > 1 ? ldo : (N + 7) / 8 * 8;
    for (int g = 0; g < G; ++g) {
        const int n0 = s.first[g], wide = s.first[g + 1] - n0;
        const O* b = base ? (const O*)base + n0 : nullptr;
        O* o = (O*)out + n0;
        bool fits = reinterpret_cast<uintptr_t>(b) % 16 == 0 && reinterpret_cast<uintptr_t>(o) % 16 == 0 && row_b * (long long)sizeof(O) % 16 == 0 &&
                    row_o * (long long)sizeof(O) % 16 == 0 && wide * sizeof(O) % 16 == 0;      // a box that ends inside 16 bytes writes more of them
        fits = fits && make_box_map<O>(&boxes.out[g], o, T, wide, row_o, TILE) == 0 &&
               make_box_map<O>(&boxes.base[g], b ? b : o, T, wide, b ? row_b : row_o, TILE) == 0;
        if (fits) by_box |= 1 << g;
        else boxes.out[g] = boxes.base[g] = map_h;                 // never followed
    }
    // a CTA an SM shares the tiles of results; it has some columns of one slice
    int all = 0;
    for (int g = 0; g < G; ++g) all += (s.first[g + 1] - s.first[g] + TILE - 1) / TILE;
    const bool even = tiles > 1 && tiles <= MOST_EVEN && (long long)all * tiles >= 16ll * sms && (long long)all * tiles * (5 + 5 * TILE) < 1ll << 31;
    const double per = all <= sms / tiles ? 1.0 : (double)all * tiles / sms;           // tiles of columns a CTA
    s.units[0] = s.before[0] = 0;
    for (int g = 0; g < G; ++g) {
        const int mine = (s.first[g + 1] - s.first[g] + TILE - 1) / TILE;
        s.before[g + 1] = s.before[g] + mine;
        s.units[g + 1] = s.units[g] + max(1, min(mine, (int)(mine / per)));
    }
    const long long ctas = (long long)s.units[G] * tiles;
    if (ctas >= 1ll << 31) return (int)cudaErrorInvalidValue;
    const int aligned = reinterpret_cast<uintptr_t>(out) % 16 == 0 && reinterpret_cast<uintptr_t>(base) % 16 == 0 &&
                        (T == 1 || (ldo % 8 == 0 && (base == nullptr || ldb % 8 == 0)));
    const int buffers = kblocks == 1 ? 11 : 8;
    const size_t smem = 1024 + (size_t)(2 * kblocks + buffers) * BLOCK_BYTES;
    // one limit for both (it is above open_smem's one value, so every call names the same)
    constexpr size_t MOST = 1024 + 13 * BLOCK_BYTES;
    prism::open_smem(low_rank_result_kernel<O>, MOST);
    return (int)prism::launch_kernel(low_rank_result_kernel<O>, dim3(even ? max(sms, (int)ctas) : (int)ctas), dim3(RESULT_THREADS), smem, stream, map_h, map_b, boxes, ids,
                                     even ? adapters : nullptr, (const O*)base,
                                     ldb, (O*)out, ldo, by_box, buffers, aligned, T, r, N, L, s, err);
}

}  // namespace lowrank_tile
}  // namespace prism

// Whether the tiles take these sizes: x rows that TMA can read, hidden values of all slices in tensor memory.
PRISM_EXPORT int prism_low_rank_tile_supported(int K, int r, int G, int x_aligned) {
    using namespace prism::lowrank_tile;
    return x_aligned && K >= 1 && r >= 16 && r % 16 == 0 && r <= MOST_RANK && G >= 1 && G <= MOST_SLICES && G * r <= MOST_HIDDEN;
}

// bfloat16 x and adapters, all T tokens in tiles; arguments as prism_low_rank_ranked's, ranks may be null.  hidden: 2 T G r bfloat16 of workspace, and an int for each of the
// tiles of 128 tokens.
PRISM_EXPORT int prism_low_rank_tile(const void* x, long long ldx, const void* a, const void* b, const float* scale, const int* ranks, const int* ids,
                                     const void* base, long long ldb, void* out, long long ldo, int out_dtype, int T, int K, int Kp, int r, int L, int G, const int* first,
                                     void* hidden, int sms, int* err, cudaStream_t stream) {
    using namespace prism::lowrank_tile;
    typedef __nv_bfloat16 bf16;
    constexpr int MOST = 65535 * TILE;        // tokens of a launch; the next one's hidden values take the place of its own
    const int size = out_dtype == PRISM_DTYPE_F32 ? 4 : 2;
    for (; T > MOST; T -= MOST) {
        const int code = prism_low_rank_tile(x, ldx, a, b, scale, ranks, ids, base, ldb, out, ldo, out_dtype, MOST, K, Kp, r, L, G, first, hidden, sms, err, stream);
        if (code != 0) return code;
        x = (const bf16*)x + MOST * ldx, ids += MOST, base = base ? (const char*)base + MOST * ldb * size : nullptr, out = (char*)out + MOST * ldo * size;
    }
    if (T <= 0) return 0;
    const bool x_aligned = reinterpret_cast<uintptr_t>(x) % 16 == 0 && (ldx % 8 == 0 || T == 1);
    if (!prism_low_rank_tile_supported(K, r, G, x_aligned) || Kp < K || Kp % 8 || L < 1 || sms < 1)
        return (int)cudaErrorInvalidValue;
    Tiles s;
    s.n = G;
    for (int g = 0; g <= G; ++g) s.first[g] = first[g];
    for (int g = 0; g < G; ++g)
        if (s.first[g] >= s.first[g + 1]) return (int)cudaErrorInvalidValue;
    const int N = first[G], tiles = (T + TILE - 1) / TILE, H = G * r;
    if ((long long)L * N >= 1ll << 31 || (long long)L * H >= 1ll << 31) return (int)cudaErrorInvalidValue;
    int* adapters = reinterpret_cast<int*>((bf16*)hidden + 2ll * T * H);
    CUtensorMap map_x, map_a, map_b;
    // a box of r rows of A: a slice's
    int code = prism::tc::make_map(&map_x, x, T, K, T > 1 ? ldx : (K + 7) / 8 * 8, TILE);
    if (code == 0) code = prism::tc::make_map(&map_a, a, (long long)L * H, Kp, Kp, r);
    if (code == 0) code = prism::tc::make_map(&map_b, b, (long long)L * N, r, r, TILE);
    if (code != 0) return code;

    const int most = max(1, min(4, 256 / H)), sums = TILE * WIDE_LD * 4;           // adapters side by side: in half of tensor memory
    const int least = 2 * (BLOCK_BYTES + most * H * prism::tc::TILE_K * 2);
    int cols = 32;
    while (cols < most * H + H % 32) cols *= 2;         // sums are read 32 columns at a time
    // All of a CTA's memory for copies in flight, or a half of an SM's: of clusters of eight CTAs with an SM each, 15 run at a time on 148 SMs, with half of one 33
    // (2,048 tokens, 16 tiles, down projection of the 7B shape: 55 -> 35 us).
    // CTAs of this kernel that fit an SM have tensor memory side by side, as a cluster's wait for each other: of any two calls, on whatever streams.  None has
    // less than 105 KB, so that there are two at most, of 256 columns, and beside one with 512 columns there is no other.
    const int budget = tiles * CTAS > sms * 5 / 6 ? 104 * 1024 : 198 * 1024;
    const int ring = max(max(budget, least), sums);
    const size_t smem = max(1024 + ring, cols > 256 ? 160 * 1024 : 0);
    prism::open_smem(low_rank_hidden_kernel, smem);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(CTAS, tiles);
    cfg.blockDim = dim3(ALL_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = CTAS, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = prism::pdl_enabled() ? 2 : 1;
    code = (int)cudaLaunchKernelEx(&cfg, low_rank_hidden_kernel, map_x, map_a, scale, ranks, ids, (bf16*)hidden, adapters, T, K, r, G, L, ring, most, cols, err);
    if (code != 0) return code;

    if (out_dtype == PRISM_DTYPE_F32) return launch_results<float>(hidden, adapters, map_b, ids, base, ldb, out, ldo, T, r, L, s, err, sms, stream);
    return launch_results<bf16>(hidden, adapters, map_b, ids, base, ldb, out, ldo, T, r, L, s, err, sms, stream);
}
