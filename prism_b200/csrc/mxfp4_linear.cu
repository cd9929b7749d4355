// y [M, N] = x [M, K] W [N, K]^T (+ bias) with W in microscaled 4-bit floating point (mxfp4.cuh), x in bfloat16 as it is
// (act_bits 16) or brought to 4 bits first (act_bits 4: a block of 32 along a row at a time, as W was).
//
// Both run on the block-scaled tensor-core instructions, which take the codes and scale bytes as they lie in memory: no CUDA
// core ever unpacks a weight.  128 rows of W are the M of a tcgen05.mma, tokens its N, the sums sit in tensor memory in
// float32, the scales beside them (tcgen05.cp).
//
//   act_bits 4   kind::mxf4: 4-bit codes on both sides, a scale for every 32 of either.
//   act_bits 16  kind::mxf8f6f4 multiplies 4-bit codes by 8-bit ones (E4M3).  A bfloat16 value has 8 significant bits, two
//                E4M3 terms of 4 each hold them: x = 2^s (hi + 2^-5 lo), s a block's own, hi the nearest E4M3 of x / 2^s and
//                lo the (exact) rest times 2^5.  Exact for values within 2^-14 of their block's largest; below, off by at
//                most 2^-22 of it.  Up to 64 tokens hi and lo are columns of one instruction, added at the end (W is
//                then read from shared memory once); for tiles of 128 tokens two instructions add to the same sums.
//
// For few tokens it is one kernel, whose CTAs each bring the parts of x that they meet to terms or codes on the way.  For more, a
// first kernel does that once, in the workspace of the call, and clears its counters.  The product is persistent, a CTA an SM:
// warps 0 and 2 issue TMA loads into a ring of stages (W: for 16 bits 128 codes a row, which TMA spreads to a byte each, for 4 bits
// 256; x), warp 1 the scale copies and the products, the warps from 4 on take the sums out.
// All of the product's blocks - (tile of W rows, tile of tokens, stage of K) - are dealt to the CTAs evenly as one long
// line, so that every SM streams the same number of bytes whatever the sizes; a tile that several CTAs have part of is
// added up by the one that comes last, in the order of the CTAs: results do not depend on timing.
//
// What bounds it, with times on the device of calls that follow one another (weights from memory):
//   one tile a CTA and a short K   the way through a launch, the first loads, the code's own first way to the SM and the last sums out:
//                                  4.4 us (1 token x (1,152 x 896)); a shared tile adds some 3 (4,608 x 3,584: 7.5)
//   few tokens, many weights       the products' issue beside the conversion of x: 1 token x (37,888 x 3,584) 16.3 us, 4.4 TB/s of the 6.5
//                                  that a copy reaches; without the products 13.6
//   64 tokens                      the first kernel's 3 us, then the stages' way through the ring: 37,888 x 3,584 21.6 us, tensor cores 42 %
//                                  busy, memory at 3.6 TB/s
//   prompts                        the products and the power that they draw: 2,048 tokens x (28,672 x 4,096) 387 us with 16-bit
//                                  activations (1.24 PFLOP/s, two 8-bit products each), 145 with 4 bits (3.3 PFLOP/s)
// Two SMs that share a tile (cta_group::2, W and x each split between them) took 385 and 226 us there and is not kept.
//
// Every wait is bounded (tcgen05.cuh); on expiry the kernel sets the error word, frees tensor memory and returns.
#include "mxfp4_mma.cuh"
#include "vec.cuh"

namespace prism {
namespace mx {

// ---- x to terms or codes ------------------------------------------------------------------------------------------------

// act 16: terms uint8 [token tile][2 tt][Kp], a tile's hi rows, then its lo rows; scales [token tile][groups][atoms][512],
// the tiles of 128 such rows.  act 4: codes as in mxfp4.cuh, scales [token tile][groups][512].  Rows that have no token are left as
// they are.  A CTA has a group of 128 columns of 32 rows: 16 threads share a row, each has 8 values of two.
template <bool A16>
__global__ void __launch_bounds__(256) prepare_kernel(const __nv_bfloat16* __restrict__ x_in, long long ldx, int M, int K, int groups, int wide,
                                                      int tt, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, int* __restrict__ counters,
                                                      int ncounters) {
    pdl_wait();            // before the trigger: the product, which reads W at once, starts behind all that came before this kernel
    pdl_trigger();
    const __nv_bfloat16* x = pdl_fresh(x_in);
    const int g = blockIdx.x, c = (threadIdx.x & 15) * 8, k = g * GROUP + c, first = blockIdx.y * 32 + (threadIdx.x >> 4);
    const int cta = blockIdx.y * gridDim.x + blockIdx.x;
    for (int i = cta * 256 + threadIdx.x; i < ncounters; i += gridDim.x * gridDim.y * 256) counters[i] = 0;
    uint4 raw[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int r = first + 16 * h;
        raw[h] = r < M ? row8(x + (long long)r * ldx, k, K, wide) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int r = first + 16 * h, tile = r / tt, t = r - tile * tt;
        uint32_t most = magnitude(raw[h]);
        most = __vmaxu2(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = __vmaxu2(most, __shfl_xor_sync(0xffffffffu, most, 2));
        most = max(most << 16, most & 0xffff0000u);
        if (r >= M) continue;
        if (A16) {
            const int byte = term_byte(most), lines = 2 * tt, atoms = (lines + 127) / 128;
            uint32_t hi[2], lo[2];
            terms_of_bf16(raw[h], byte, hi, lo);
            uint8_t* at = codes + ((size_t)tile * lines + t) * ((size_t)groups * GROUP) + k;
            *reinterpret_cast<uint2*>(at) = make_uint2(hi[0], hi[1]);
            *reinterpret_cast<uint2*>(at + (size_t)tt * groups * GROUP) = make_uint2(lo[0], lo[1]);
            if ((threadIdx.x & 3) == 0) {
                uint8_t* s = scales + ((size_t)tile * groups + g) * (atoms * TILE_BYTES) + c / BLOCK;
                const int u = t + tt;
                s[t / 128 * TILE_BYTES + (t & 31) * 16 + (t & 127) / 32 * 4] = (uint8_t)byte;
                s[u / 128 * TILE_BYTES + (u & 31) * 16 + (u & 127) / 32 * 4] = low_byte(byte);
            }
        } else {
            const int byte = scale_byte(most);
            *reinterpret_cast<uint32_t*>(codes + (size_t)r * (groups * (GROUP / 2)) + k / 2) = codes_of_bf16(raw[h], byte);
            if ((threadIdx.x & 3) == 0)
                scales[((size_t)tile * groups + g) * TILE_BYTES + (t & 31) * 16 + t / 32 * 4 + c / BLOCK] = (uint8_t)byte;
        }
    }
}

// ---- the product --------------------------------------------------------------------------------------------------------

constexpr int STAGE_OUT = 16 * 128 * 2;        // bytes of sixteen tokens' results of 128 features in bfloat16

// FUSED: the product brings x to terms itself (no first kernel)
template <bool A16_, int TT_, int W_, int GS_, bool FUSED_> struct Cfg {
    static constexpr bool A16 = A16_, FUSED = FUSED_;
    static constexpr int TT = TT_, W = W_;                         // tokens of a tile; tiles of 128 rows of W that share it
    static constexpr bool SIDE = A16 && TT <= 64;                  // hi and lo side by side as columns
    static constexpr int GS = GS_;                                 // groups of 128 along K in a stage
    static constexpr int SUBS = A16 ? GS : GS / 2;                 // tiles of 128 bytes a row that hold them
    static constexpr int XR = A16 ? 2 * TT : TT;                   // rows of x's tile
    static constexpr int NCOL = SIDE ? 2 * TT : TT;                // N of the instruction
    static constexpr int ATOMS = (XR + 127) / 128;                 // tiles of scales of x
    static constexpr int W_BYTES = W * SUBS * 16384, X_BYTES = SUBS * XR * 128, STAGE = W_BYTES + X_BYTES;
    // bytes that W's loads of a stage report: codes that TMA spreads count as they are in memory, 64 bytes a row
    static constexpr int W_ARRIVE = W * SUBS * (A16 ? 8192 : 16384);
    static constexpr int SF = GS * TILE_BYTES * (W + ATOMS);       // scale bytes of a stage
    static constexpr int FIT = (216 * 1024) / (STAGE + SF);
    static constexpr int SF_COLS = GS * 4 * (W + ATOMS);           // their columns in tensor memory: every stage has its own
    static constexpr int STAGES = FIT > 10 ? 10 : FIT;
    static constexpr int BUFS = 2 * W * NCOL + STAGES * SF_COLS <= 512 ? 2 : 1;
    static constexpr int COLS_USED = BUFS * W * NCOL + STAGES * SF_COLS;
    static constexpr int COLS = COLS_USED <= 64 ? 64 : COLS_USED <= 128 ? 128 : COLS_USED <= 256 ? 256 : 512;
    static constexpr int EPI_WARPS = 4 * W, FIRST_X = 4 + EPI_WARPS, X_WARPS = 8, TEAMS = 2;       // teams of X_WARPS take the stages in turn
    static constexpr int THREADS = 32 * (4 + EPI_WARPS + (FUSED ? TEAMS * X_WARPS : 0));
    static constexpr size_t SMEM = (size_t)STAGES * (STAGE + SF) + 1024 + 512 + W * STAGE_OUT;
    static_assert(COLS_USED <= 512 && STAGES >= 3 && (A16 || GS % 2 == 0) && (!FUSED || TT <= 16) && (!FUSED || GS * TT / 2 % X_WARPS == 0), "tensor memory, shared memory or form");
};

// 8 or 16 columns of a warp's lanes, without the wait
__device__ __forceinline__ void tmem_get(uint32_t (&r)[8], uint32_t taddr) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "r"(taddr));
}
__device__ __forceinline__ void tmem_get(uint32_t (&r)[16], uint32_t taddr) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
                   "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]) : "r"(taddr));
}
// Instruction descriptor: element kinds (mxf8f6f4: A E2M1 = 5, B E4M3 = 0; mxf4: E2M1 = 1 on both sides), N / 8, scales E8M0,
// M / 128; `id`: which byte of a scale column the instruction begins at.
template <typename C> __device__ __forceinline__ constexpr uint32_t idesc_of(int id) {
    return (C::A16 ? 5u << 7 : 1u << 7 | 1u << 10) | (uint32_t)(C::NCOL >> 3) << 17 | 1u << 23 | 1u << 27 | (uint32_t)id << 4 | (uint32_t)id << 29;
}

struct Product {
    const uint8_t *w_scales, *x_scales;
    const __nv_bfloat16* x;    // (fused) as it is
    long long ldx;
    int K, wide;
    const void* bias;
    void* y;
    float* part;               // [P][2][W][TT][128]
    int *counters, *err;
    long long ldy;
    Split split;
    int M, N, groups, mtiles, ntiles, bias_bf16, out_bf16, wide_out;       // wide_out: rows of the result in bfloat16 at multiples of 16 bytes
};

// Sixteen tokens' results of 128 features, a feature a thread of four warps, to memory: as bfloat16 through `stage` (4 KB), so that
// 16 threads store a token's 256 bytes 16 bytes each.  Stores of 2 bytes a lane took 16 cycles a warp: 11,000 cycles a tile of 256 x 128
// beside 166,000 of products in 12 tiles.  `bar`: a barrier of the four warps.
__device__ __forceinline__ void store_sixteen(const Product& p, unsigned char* stage, int bar, int m0, int t0, int tokens, int f0, int row, const float (&v)[16]) {
    if (p.wide_out) {
        __nv_bfloat16* to = reinterpret_cast<__nv_bfloat16*>(stage) + row;
#pragma unroll
        for (int j = 0; j < 16; ++j) to[j * 128] = __float2bfloat16_rn(v[j]);
        asm volatile("bar.sync %0, 128;" ::"r"(bar) : "memory");
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int t = h * 8 + row / 16, f = f0 + row % 16 * 8;
            if (t0 + t < tokens && f < p.N)
                *reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(p.y) + (long long)(m0 + t0 + t) * p.ldy + f) =
                    *reinterpret_cast<const uint4*>(stage + t * 256 + row % 16 * 16);
        }
        asm volatile("bar.sync %0, 128;" ::"r"(bar) : "memory");
        return;
    }
    if (f0 + row >= p.N) return;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
        if (t0 + j >= tokens) return;
        const long long at = (long long)(m0 + t0 + j) * p.ldy + f0 + row;
        if (p.out_bf16) reinterpret_cast<__nv_bfloat16*>(p.y)[at] = __float2bfloat16_rn(v[j]);
        else reinterpret_cast<float*>(p.y)[at] = v[j];
    }
}

template <typename C>
__global__ void __launch_bounds__(C::THREADS, 1)
product_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const __grid_constant__ Product p) {
    constexpr int TT = C::TT, W = C::W, STAGES = C::STAGES;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* tiles = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    unsigned char* sf = tiles + (size_t)STAGES * C::STAGE;
    uint64_t* full = reinterpret_cast<uint64_t*>(sf + STAGES * C::SF);
    uint64_t *empty = full + STAGES, *acc_full = empty + STAGES, *acc_empty = acc_full + C::BUFS;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + C::BUFS);
    unsigned char* staging = reinterpret_cast<unsigned char*>(full) + 512;
    __shared__ int abort_flag, is_last, gone;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, cta = blockIdx.x;
    if (threadIdx.x == 0) {
        abort_flag = 0;
        for (int s = 0; s < STAGES; ++s) { mbar_init(&full[s], C::FUSED ? 1 + C::X_WARPS : 2); mbar_init(&empty[s], 1); }
        for (int s = 0; s < C::BUFS; ++s) { mbar_init(&acc_full[s], 1); mbar_init(&acc_empty[s], C::EPI_WARPS); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_slot)), "r"(C::COLS));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = *tmem_slot, tmem_sf = tmem + C::BUFS * W * C::NCOL;
    volatile int* abortp = &abort_flag;
    const int b0 = p.split.start(cta), n = p.split.start(cta + 1) - b0, kb = p.split.kb;

    // unit u: token tile u % mtiles of the W tiles W (u / mtiles) .. + W - 1.  The loops below carry their place along: one
    // thread's integer divisions would take longer than a block's products.
    if (warp == 0 || (warp == 2 && !C::FUSED)) {
        // warp 0: W and its scales; warp 2: x's.  W waits for nobody where the kernel before this one is x's own, which began
        // after everything before it had ended
        const bool is_w = C::FUSED || warp == 0;
        const int u0 = b0 / kb;
        int k = b0 - u0 * kb, m = u0 % p.mtiles, t0 = u0 / p.mtiles * W;
        if (C::FUSED || !is_w) pdl_wait();
        uint32_t parity = 1;                                             // the first round passes at once
        int s = 0, i = 0;
        for (; i < n; ++i) {
            if (!warp_wait(&empty[s], parity, abortp)) break;
            const int gs = C::GS == 1 ? 1 : min(C::GS, p.groups - k * C::GS);             // groups that exist of this stage's
            unsigned char *st = tiles + s * C::STAGE, *ss = sf + s * C::SF;
            if (is_w) {
                if (elect_one()) {
                    mbar_expect_tx(&full[s], C::W_ARRIVE + gs * TILE_BYTES * W);
#pragma unroll
                    for (int w = 0; w < W; ++w) {
#pragma unroll
                        for (int b = 0; b < C::SUBS; ++b)
                            tma_load_2d(st + (w * C::SUBS + b) * 16384, &map_w, &full[s], (k * C::SUBS + b) * 128, (t0 + w) * 128);
                        const int t = min(t0 + w, p.ntiles - 1);         // the last tile may have no partner: its scales again, never stored
                        bulk_load(ss + w * C::GS * TILE_BYTES, p.w_scales + ((size_t)t * p.groups + k * C::GS) * TILE_BYTES, gs * TILE_BYTES, &full[s]);
                    }
                }
            } else if (elect_one()) {
                mbar_expect_tx(&full[s], C::X_BYTES + gs * TILE_BYTES * C::ATOMS);
#pragma unroll
                for (int b = 0; b < C::SUBS; ++b)
                    tma_load_2d(st + C::W_BYTES + b * (C::XR * 128), &map_x, &full[s], (k * C::SUBS + b) * 128, m * C::XR);
                bulk_load(ss + W * C::GS * TILE_BYTES, p.x_scales + ((size_t)m * p.groups + k * C::GS) * (C::ATOMS * TILE_BYTES),
                          gs * C::ATOMS * TILE_BYTES, &full[s]);
            }
            __syncwarp();
            if (++k == kb) {
                k = 0;
                if (++m == p.mtiles) { m = 0; t0 += W; }
            }
            if (++s == STAGES) { s = 0; parity ^= 1; }
        }
        if (is_w) pdl_trigger_gemm();
        if (*abortp)                                                     // what is in flight gets a bounded chance to land
            for (int j = max(0, i - STAGES); j < i; ++j) mbar_wait(&full[j % STAGES], (j / STAGES) & 1, abortp);
    } else if (C::FUSED && warp >= C::FIRST_X) {
        // A team's warps share a stage: an item is two tokens' values of a group, 8 to a lane; its next stage's are on their way.
        constexpr int ITEMS = C::GS * TT / 2 / C::X_WARPS;
        pdl_wait();
        const __nv_bfloat16* x = pdl_fresh(p.x);
        const int c = (lane & 15) * 8, first = (warp - C::FIRST_X) % C::X_WARPS, team = (warp - C::FIRST_X) / C::X_WARPS;
        uint4 raw[2][ITEMS];
        int kl = (b0 + team) % kb, il = team;                            // the next stage to be asked for
        auto ask = [&](uint4 (&to)[ITEMS]) {
            if (il >= n) return;
#pragma unroll
            for (int j = 0; j < ITEMS; ++j) {
                const int item = first + C::X_WARPS * j, t = item % (TT / 2) * 2 + (lane >> 4), at = (kl * C::GS + item / (TT / 2)) * GROUP + c;
                to[j] = t < p.M ? row8(x + (long long)t * p.ldx, at, p.K, p.wide) : make_uint4(0, 0, 0, 0);
            }
            il += C::TEAMS;
            kl = (kl + C::TEAMS) % kb;
        };
        ask(raw[0]);
        uint32_t parity = 1;
        int s = team;
        bool ok = true;
#pragma unroll 1
        for (int i = team; i < n && ok; i += 2 * C::TEAMS) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (i + h * C::TEAMS >= n) break;
                ask(raw[1 - h]);
                ok = warp_wait(&empty[s], parity, abortp);
                if (!ok) break;
                unsigned char *xt = tiles + s * C::STAGE + C::W_BYTES, *ss = sf + s * C::SF + W * C::GS * TILE_BYTES;
#pragma unroll
                for (int j = 0; j < ITEMS; ++j) {
                    const int item = first + C::X_WARPS * j, t = item % (TT / 2) * 2 + (lane >> 4), g = item / (TT / 2);
                    uint32_t most = magnitude(raw[h][j]);
                    most = __vmaxu2(most, __shfl_xor_sync(0xffffffffu, most, 1));
                    most = __vmaxu2(most, __shfl_xor_sync(0xffffffffu, most, 2));
                    most = max(most << 16, most & 0xffff0000u);          // as float32 bits
                    unsigned char* sc = ss + g * C::ATOMS * TILE_BYTES + (lane & 15) / 4;
                    if (C::A16) {                                        // 16-byte pieces of a row change places by the row's number
                        const int byte = term_byte(most);
                        uint32_t hi[2], lo[2];
                        terms_of_bf16(raw[h][j], byte, hi, lo);
                        unsigned char* to = xt + g * (C::XR * 128) + t * 128 + ((((lane & 15) >> 1) ^ (t & 7)) << 4) + (lane & 1) * 8;
                        *reinterpret_cast<uint2*>(to) = make_uint2(hi[0], hi[1]);
                        *reinterpret_cast<uint2*>(to + TT * 128) = make_uint2(lo[0], lo[1]);
                        if ((lane & 3) == 0) {
                            sc[(t & 31) * 16 + t / 32 * 4] = (uint8_t)byte;
                            sc[((t + TT) & 31) * 16 + (t + TT) / 32 * 4] = low_byte(byte);
                        }
                    } else {
                        const int byte = scale_byte(most);
                        *reinterpret_cast<uint32_t*>(xt + g / 2 * (C::XR * 128) + t * 128 + ((((g & 1) * 4 + (lane & 15) / 4) ^ (t & 7)) << 4) +
                                                     (lane & 3) * 4) = codes_of_bf16(raw[h][j], byte);
                        if ((lane & 3) == 0) sc[(t & 31) * 16 + t / 32 * 4] = (uint8_t)byte;
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(&full[s]);
                if ((s += C::TEAMS) >= STAGES) { s -= STAGES; parity ^= 1; }
            }
        }
    } else if (warp == 1) {
        const uint64_t desc0 = umma_desc(smem_addr(tiles));              // (offsets stay within the address field: 16-byte steps of 227 KB)
        const uint32_t sf0 = smem_addr(sf);
        int k = b0 % kb, s = 0, buf = 0;
        uint32_t parity = 0, acc_parity = 1;                             // the first wait for each accumulator passes at once
        bool fresh = true, ready = false;
        for (int i = 0; i < n; ++i) {
            if (fresh && !warp_wait(&acc_empty[buf], acc_parity, abortp)) break;
            if (!__all_sync(0xffffffffu, ready) && !warp_wait(&full[s], parity, abortp)) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t ss = sf0 + s * C::SF, tsf = tmem_sf + s * C::SF_COLS;
            const int gs = C::GS == 1 ? 1 : min(C::GS, p.groups - k * C::GS);
            const uint64_t da = desc0 + (uint32_t)(s * (C::STAGE >> 4)), db = da + (C::W_BYTES >> 4);
            const uint32_t d = tmem + buf * W * C::NCOL;
            const bool done = ++k == kb || i == n - 1;
            const int s_now = s;
            if (++s == STAGES) { s = 0; parity ^= 1; }
            ready = i + 1 < n && mbar_test(&full[s], parity);            // the next stage: the answer comes while products are issued
            if (elect_one()) {
                uint32_t more = !fresh;
#pragma unroll
                for (int g = 0; g < C::GS; ++g) {
                    if (g >= gs) break;
#pragma unroll
                    for (int w = 0; w < W; ++w) scales_to_tmem(tsf + (w * C::GS + g) * 4, ss + (w * C::GS + g) * TILE_BYTES);
#pragma unroll
                    for (int a = 0; a < C::ATOMS; ++a)
                        scales_to_tmem(tsf + (W * C::GS + g * C::ATOMS + a) * 4, ss + (W * C::GS + g * C::ATOMS + a) * TILE_BYTES);
                    const int sub = C::A16 ? g : g / 2;
                    const uint32_t sa = tsf + g * 4, sb = tsf + (W * C::GS + g * C::ATOMS) * 4;
                    uint64_t a = da + sub * 1024 + (C::A16 ? 0 : (g & 1) * 4), b = db + sub * (C::XR * 128 >> 4) + (C::A16 ? 0 : (g & 1) * 4);
                    uint32_t id = 0;
#pragma unroll
                    for (int j = 0; j < (C::A16 ? 4 : 2); ++j) {         // 32 bytes of a row each: 32 or 64 elements
                        const uint32_t idesc = idesc_of<C>(0) | id << 4 | id << 29;
#pragma unroll
                        for (int w = 0; w < W; ++w) {
                            umma_scaled<C::A16>(d + w * C::NCOL, a + w * (C::SUBS * 1024), b, idesc, sa + w * (C::GS * 4), sb, more);
                            if (C::A16 && !C::SIDE)
                                umma_scaled<C::A16>(d + w * C::NCOL, a + w * (C::SUBS * 1024), b + (TT * 128 >> 4), idesc, sa + w * (C::GS * 4), sb + 4, 1);
                        }
                        more = 1;
                        id += C::A16 ? 1 : 2;
                        a += 2;
                        b += 2;
                    }
                }
                umma_commit(&empty[s_now]);
                if (done) umma_commit(&acc_full[buf]);
            }
            __syncwarp();
            fresh = done;
            if (done) {
                k = 0;
                if (++buf == C::BUFS) { buf = 0; acc_parity ^= 1; }
            }
        }
    } else if (warp >= 4 && warp < C::FIRST_X) {
        // warps of one tile of W rows: 4 + 4 w .. 7 + 4 w; TMEM lanes (warp % 4) * 32 .. + 31
        const int w = (warp - 4) / 4, q = warp & 3, row = q * 32 + lane;
        pdl_wait();
        int seg = 0;
        for (int i = 0; i < n; ++seg) {
            const int u = (b0 + i) / kb, k0 = b0 + i - u * kb, k1 = min(kb, k0 + n - i), buf = seg % C::BUFS;
            i += k1 - k0;
            mbar_wait(&acc_full[buf], (seg / C::BUFS) & 1, abortp);
            // one thread reads the flag for all of these warps: they leave together or not at all
            asm volatile("bar.sync 1, %0;" ::"n"(C::EPI_WARPS * 32) : "memory");
            if (threadIdx.x == 128) gone = *abortp;
            asm volatile("bar.sync 1, %0;" ::"n"(C::EPI_WARPS * 32) : "memory");
            if (gone) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const int m0 = u % p.mtiles * TT, f = (u / p.mtiles * W + w) * 128 + row;      // first token, this thread's output feature
            const int tokens = min(TT, p.M - m0);
            const uint32_t d = tmem + ((uint32_t)(q * 32) << 16) + (buf * W + w) * C::NCOL;
            const bool whole = k0 == 0 && k1 == kb;
            const float bias = p.bias != nullptr && f < p.N ? load_param(p.bias, p.bias_bf16, f) : 0.f;
            auto store = [&](int t0, auto& v) {
                constexpr int count = (int)(sizeof(v) / sizeof(float));
#pragma unroll
                for (int j = 0; j < count; ++j) v[j] += bias;
                if constexpr (count == 16) {
                    store_sixteen(p, staging + w * STAGE_OUT, 2 + w, m0, t0, tokens, f - row, row, v);
                } else {
                    if (f >= p.N) return;
#pragma unroll
                    for (int j = 0; j < count; ++j) {
                        if (t0 + j >= tokens) return;
                        const long long at = (long long)(m0 + t0 + j) * p.ldy + f;
                        if (p.out_bf16) reinterpret_cast<__nv_bfloat16*>(p.y)[at] = __float2bfloat16_rn(v[j]);
                        else reinterpret_cast<float*>(p.y)[at] = v[j];
                    }
                }
            };
            float* mine = p.part + (((size_t)cta * 2 + p.split.place(cta, u)) * W + w) * (TT * 128) + row;
            auto release = [&]() {                                       // the sums are out: the next unit's may begin
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(&acc_empty[buf]);
            };
            if constexpr (TT == 128) {
                // one set of sums, and many: all into registers before the first is stored (2,048 tokens x (28,672 x 4,096) in 4
                // bits 173 -> 152 us; tiles of 64 tokens, of fewer blocks each, lost by as much to the code that this takes)
                uint32_t r[TT / 16][16];
#pragma unroll
                for (int c = 0; c < TT / 16; ++c) {
                    tmem_get(r[c], d + 16 * c);
                }
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                for (int c = 0; c < TT / 16; ++c)
#pragma unroll
                    for (int j = 0; j < 16; ++j) asm volatile("" : "+r"(r[c][j]));       // not before the wait
                release();
#pragma unroll
                for (int c = 0; c < TT / 16; ++c) {
                    if (16 * c >= tokens) break;
                    float v[16];
#pragma unroll
                    for (int j = 0; j < 16; ++j) v[j] = __uint_as_float(r[c][j]);
                    if (whole) store(16 * c, v);
                    else
#pragma unroll
                        for (int j = 0; j < 16; ++j) mine[(16 * c + j) * 128] = v[j];
                }
            } else {
                constexpr int TAKE = C::FUSED ? 8 : 16;
#pragma unroll 1
                for (int t0 = 0; t0 < tokens; t0 += TAKE) {
                    uint32_t r[TAKE], l[TAKE];
                    tmem_get(r, d + t0);
                    if (C::SIDE) tmem_get(l, d + TT + t0);
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                    float v[TAKE];
#pragma unroll
                    for (int j = 0; j < TAKE; ++j) {
                        asm volatile("" : "+r"(r[j]));                   // not before the wait
                        if (C::SIDE) asm volatile("" : "+r"(l[j]));
                        v[j] = __uint_as_float(r[j]) + (C::SIDE ? __uint_as_float(l[j]) : 0.f);
                    }
                    if (whole) store(t0, v);
                    else
#pragma unroll
                        for (int j = 0; j < TAKE; ++j) mine[(t0 + j) * 128] = v[j];
                }
                release();
            }
            if (whole) continue;
            const int c0 = p.split.owner(u * kb), c1 = p.split.owner((u + 1) * kb - 1);
            asm volatile("bar.sync 1, %0;" ::"n"(C::EPI_WARPS * 32) : "memory");
            if (threadIdx.x == 128) is_last = add_acq_rel(&p.counters[u], 1) == c1 - c0;       // (two fences of all threads: 0.4 us more)
            asm volatile("bar.sync 1, %0;" ::"n"(C::EPI_WARPS * 32) : "memory");
            if (!is_last) continue;
            if (C::FUSED && threadIdx.x == 128) p.counters[u] = 0;        // as the next launch expects it
            // one CTA's share after another's, the loads of eight of them at once
            constexpr int SHARES = 8, JOIN = C::FUSED ? 4 : 8;          // as many registers as there are
#pragma unroll 1
            for (int t0 = 0; t0 < tokens; t0 += JOIN) {
                float v[JOIN] = {};
#pragma unroll 1
                for (int c = c0; c <= c1; c += SHARES) {
                    float part[SHARES][JOIN];
#pragma unroll
                    for (int k = 0; k < SHARES; ++k) {
                        const bool there = c + k <= c1;
                        const float* from = p.part + (((size_t)(c + k) * 2 + p.split.place(c + k, u)) * W + w) * (TT * 128) + row + t0 * 128;
#pragma unroll
                        for (int j = 0; j < JOIN; ++j) part[k][j] = there ? __ldcg(from + j * 128) : 0.f;
                    }
#pragma unroll
                    for (int k = 0; k < SHARES; ++k)
#pragma unroll
                        for (int j = 0; j < JOIN; ++j) v[j] += part[k][j];
                }
                store(t0, v);
            }
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0 && abort_flag) report_error(p.err, PRISM_ERR_WAIT_TIMEOUT);
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::COLS));
    }
}

// ---- host side ----------------------------------------------------------------------------------------------------------

constexpr int MOST_COUNTERS = 4096;       // tiles of the fused form: counters of the stream's, which the kernel leaves at zero

// A form of the product and how many CTAs share its blocks
struct Plan {
    int tt, w, gs, groups, mtiles, ntiles, kb, P;
    bool fused;
    long long units, codes, scales, parts, counters, bytes;       // bytes from the workspace's start
};
// Few tokens go through the fused form of their size, one launch: up to 16 with 16-bit activations (1 token x (3,584 x 18,944) 12.0 us, with
// a first kernel 15.7; 16 tokens 16.3 and 17.2; x (3,584 x 3,584) 9.8 and 8.6, the one size tried that loses), up to 8 with 4-bit ones
// (8 tokens x (896 x 4,864) 7.6 and 9.0; 16 tokens x (3,584 x 18,944) 15.3 and 13.5).  For more, tiles of 32 to 128 tokens by one or two of
// W's.  What is chosen, tile and CTAs that share a unit's K, takes least by this estimate (us): blocks of the busiest CTA times a
// block's time (W and x from memory, or the products), and where K is shared 2 for handing over and the bytes of the shares at 100 KB
// a us.  Measured, tiles of 32, 64, 64 by two and 128 by two: 64 tokens x (37,888 x 3,584) 36.9, 23.7, 21.8, 32.5 us, x (9,728 x 896) in
// 4 bits 10.8, 5.8, 6.6, 7.3; 159 x 777 x 4,407 14.7, 17.5, 20.3, 29.7; 2,048 x 28,672 x 4,096 in 4 bits 467, 259, 191, 145.  One, two, four
// and (all SMs) six CTAs a unit: 1 token x (3,584 x 18,944) 37, 22, 14.4, 12.6; 64 tokens x (4,608 x 3,584) 12.0, 13.7, 13.4, 13.4.
inline Plan plan_for(int M, int N, int K, int act_bits) {
    struct Form { int tt, w; float block16, block4; };
    static const Form few[] = {{8, 1, .40f, .40f}, {16, 1, .50f, 0.f}};
    static const Form many[] = {{32, 1, .26f, .30f}, {64, 1, .32f, .38f}, {64, 2, .58f, .63f}, {128, 2, 1.0f, .80f}};
    Plan best;
    float best_us = 1e30f;
    const bool a16 = act_bits == 16;
    const int sms = sm_count();
    const bool fused = M <= (a16 ? 16 : 8) && N <= MOST_COUNTERS * 128LL;       // as many tiles as the fused form has counters for
    const Form* forms = fused ? &few[M <= 8 ? 0 : 1] : many;
    for (int i = 0; i < (fused ? 1 : 4); ++i) {
        Plan q;
        q.tt = forms[i].tt;
        q.w = forms[i].w;
        q.gs = !a16 || q.tt <= 16 ? 2 : 1;
        q.fused = fused;
        q.groups = groups_of(K);
        q.mtiles = (M + q.tt - 1) / q.tt;
        q.ntiles = (N + 127) / 128;
        q.kb = (q.groups + q.gs - 1) / q.gs;
        q.units = (long long)((q.ntiles + q.w - 1) / q.w) * q.mtiles;
        const long long total = q.units * q.kb;
        const float block = a16 ? forms[i].block16 : forms[i].block4;
        const float share = (float)(q.tt * q.w) * (512.f / 100e3f);
        for (int split = 1; split <= q.kb; split += split < 4 ? 1 : split / 4) {
            const long long want = q.units * split;
            q.P = (int)(want < sms ? want : sms);
            if (q.P > total) q.P = (int)total;
            const long long each = (total + q.P - 1) / q.P;
            const int shares = each >= q.kb && total % q.P == 0 ? 1 : (int)((q.kb + each - 1) / each) + (want > sms);
            const float us = each * block + (shares > 1 ? 2 * (1.5f + (1 + shares) * share) : 0.f);
            if (us < best_us) { best_us = us; best = q; }
            if (want >= sms) break;
        }
    }
    Plan& q = best;
    const int xr = a16 ? 2 * q.tt : q.tt, atoms = (xr + 127) / 128;
    auto up = [](long long b) { return (b + 1023) / 1024 * 1024; };
    q.codes = 0;
    q.scales = q.fused ? 0 : up(a16 ? (long long)q.mtiles * xr * q.groups * GROUP : (long long)M * q.groups * (GROUP / 2));
    q.parts = q.scales + (q.fused ? 0 : up((long long)q.mtiles * q.groups * atoms * TILE_BYTES));
    q.counters = q.parts + up((long long)q.P * 2 * q.w * q.tt * 128 * 4);
    q.bytes = q.counters + (q.fused ? 0 : up(q.units * 4));
    return q;
}

template <typename C> int run_product(const CUtensorMap& mw, const CUtensorMap& mx, const Product& p, cudaStream_t stream) {
    auto kern = product_kernel<C>;
    static unsigned char done[64] = {};
    open_once(kern, C::SMEM, done);
    return (int)launch_kernel(kern, dim3(p.split.P), dim3(C::THREADS), C::SMEM, stream, mw, mx, p);
}

}  // namespace mx
}  // namespace prism

// what prism_mxfp4_linear needs for these sizes: bytes of workspace, into need[0], and counters, into need[1]
PRISM_EXPORT int prism_mxfp4_linear_workspace(int M, int N, int K, int act_bits, long long* need) {
    if (M <= 0 || N <= 0 || K <= 0 || (act_bits != 16 && act_bits != 4)) return (int)cudaErrorInvalidValue;
    const prism::mx::Plan q = prism::mx::plan_for(M, N, K, act_bits);
    need[0] = q.bytes;
    need[1] = q.fused ? q.units : 0;
    return q.units * q.kb > 0x7fffffffLL ? (int)cudaErrorInvalidValue : 0;
}

// x [M, K] bfloat16 (row stride ldx); codes, scales: W [N, K]; y [M, N] of `out_dtype` (row stride ldy); act_bits 16 or 4;
// ws: workspace of the call, 256-byte aligned; nothing is launched and -1 returned where its ws_bytes are fewer than
// prism_mxfp4_linear_workspace says on this device; counters: as many ints as it says there (4,096 always
// suffice), zero before the first launch (the kernel leaves them zero), of one stream's launches at a time
PRISM_EXPORT int prism_mxfp4_linear(void* ws, long long ws_bytes, int* counters, const void* x, long long ldx, const void* codes, const void* scales,
                                    const void* bias, int bias_dtype, void* y, int out_dtype, long long ldy, int M, int N, int K, int act_bits,
                                    int* err, cudaStream_t stream) {
    using namespace prism;
    using namespace prism::mx;
    if (M <= 0 || N <= 0) return 0;
    if (K <= 0 || (act_bits != 16 && act_bits != 4) || ((uintptr_t)codes & 31) || ((uintptr_t)scales & 15) || ((uintptr_t)ws & 255))
        return (int)cudaErrorInvalidValue;
    const Plan q = plan_for(M, N, K, act_bits);
    if (q.units * q.kb > 0x7fffffffLL) return (int)cudaErrorInvalidValue;
    if (ws_bytes < q.bytes) return WORKSPACE_TOO_SMALL;
    uint8_t* base = static_cast<uint8_t*>(ws);
    const bool a16 = act_bits == 16;
    CUtensorMap mw, mx;
    int rc = byte_map(&mw, codes, N, (long long)q.groups * (GROUP / 2), 128, a16);
    if (rc) return rc;
    Product p;
    p.w_scales = static_cast<const uint8_t*>(scales);
    p.x_scales = base + q.scales;
    p.x = static_cast<const __nv_bfloat16*>(x);
    p.ldx = ldx;
    p.K = K;
    p.wide = ((uintptr_t)x & 15) == 0 && ldx % 8 == 0;
    p.bias = bias;
    p.y = y;
    p.part = reinterpret_cast<float*>(base + q.parts);
    p.counters = q.fused ? counters : reinterpret_cast<int*>(base + q.counters);
    p.err = err;
    p.ldy = ldy;
    p.split = Split((int)(q.units * q.kb), q.P, q.kb);
    p.M = M, p.N = N, p.groups = q.groups, p.mtiles = q.mtiles, p.ntiles = q.ntiles;
    p.bias_bf16 = bias_dtype == PRISM_DTYPE_BF16, p.out_bf16 = out_dtype == PRISM_DTYPE_BF16;
    p.wide_out = p.out_bf16 && N % 8 == 0 && ldy % 8 == 0 && ((uintptr_t)y & 15) == 0;
    if (q.fused) {
        if (!a16) return run_product<Cfg<false, 8, 1, 2, true>>(mw, mw, p, stream);
        return q.tt == 8 ? run_product<Cfg<true, 8, 1, 2, true>>(mw, mw, p, stream) : run_product<Cfg<true, 16, 1, 2, true>>(mw, mw, p, stream);
    }
    const int xr = a16 ? 2 * q.tt : q.tt;
    rc = a16 ? byte_map(&mx, base + q.codes, (long long)q.mtiles * xr, (long long)q.groups * GROUP, xr, false)
             : byte_map(&mx, base + q.codes, M, (long long)q.groups * (GROUP / 2), xr, false);
    if (rc) return rc;
    if ((M + 31) / 32 > 65535) return (int)cudaErrorInvalidValue;
    rc = (int)launch_kernel(a16 ? prepare_kernel<true> : prepare_kernel<false>, dim3(q.groups, (M + 31) / 32), dim3(256), 0, stream, p.x, ldx, M, K,
                            q.groups, p.wide, q.tt, base + q.codes, base + q.scales, p.counters, (int)q.units);
    if (rc) return rc;
    const int form = q.tt * 10 + q.w;
    if (a16) {
        switch (form) {
            case 321: return run_product<Cfg<true, 32, 1, 1, false>>(mw, mx, p, stream);
            case 641: return run_product<Cfg<true, 64, 1, 1, false>>(mw, mx, p, stream);
            case 642: return run_product<Cfg<true, 64, 2, 1, false>>(mw, mx, p, stream);
            default: return run_product<Cfg<true, 128, 2, 1, false>>(mw, mx, p, stream);
        }
    }
    switch (form) {
        case 321: return run_product<Cfg<false, 32, 1, 2, false>>(mw, mx, p, stream);
        case 641: return run_product<Cfg<false, 64, 1, 2, false>>(mw, mx, p, stream);
        case 642: return run_product<Cfg<false, 64, 2, 2, false>>(mw, mx, p, stream);
        default: return run_product<Cfg<false, 128, 2, 2, false>>(mw, mx, p, stream);
    }
}
