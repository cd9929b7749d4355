// Block-scaled tensor-core products of 4-bit codes (tcgen05.mma kind::mxf4, kind::mxf8f6f4): two 8-bit terms that hold a 16-bit
// value, scales on their way to tensor memory, how a product's blocks are dealt to CTAs, tensor maps.
#pragma once

#include "mxfp4.cuh"
#include "tcgen05.cuh"

namespace prism {
namespace mx {

using tc::mbar_expect_tx;
using tc::mbar_init;
using tc::mbar_wait;
using tc::smem_addr;
using tc::tma_load_2d;
using tc::umma_commit;
using tc::umma_desc;

// ---- a bfloat16 value as two E4M3 terms: x = 2^(byte - 127) (hi + 2^-5 lo) -----------------------------------------------
// The byte of a block of 32 from the bits of its largest magnitude: values scaled to below 256; at least 5, so that the low
// terms' byte, 5 less, exists; 255 (both) for a block with an infinity or NaN.

__device__ __forceinline__ uint32_t pack_e4m3(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;" : "=h"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void unpack_e4m3(uint32_t p, float& lo, float& hi) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)p));
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.f32.f16 %0, a;\n\tcvt.f32.f16 %1, b;\n\t}" : "=f"(lo), "=f"(hi) : "r"(h));
}

__device__ __forceinline__ int term_byte(uint32_t most) { return most >= 0x7f800000u ? 255 : max((int)(most >> 23) - 7, 5); }
__device__ __forceinline__ uint8_t low_byte(int byte) { return (uint8_t)(byte == 255 ? 255 : byte - 5); }
// A float32 value as three such terms, 2^(byte - 127) (t0 + 2^-5 t1 + 2^-10 t2): each takes what the one before left over, at most
// half a step of it, 8 of 256.  So off by at most 2^-14 of the value (8 of 2^10 beside 128), or, where the last is below E4M3's
// normal numbers, by 2^-27 of the block's largest.  The last one's byte is 10 less, so a block's is at least 10.
__device__ __forceinline__ int three_term_byte(uint32_t most) { return most >= 0x7f800000u ? 255 : max((int)(most >> 23) - 7, 10); }
__device__ __forceinline__ void three_terms(float v, int byte, uint32_t (&term)[3]) {
    float rest = byte == 255 ? 0.f : v * __uint_as_float((uint32_t)(254 - byte) << 23);
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        float held, none;
        term[i] = pack_e4m3(rest, 0.f);
        unpack_e4m3(term[i], held, none);
        rest = (rest - held) * 32.f;
    }
}
// The terms of eight bfloat16 values as they lie in memory, in half precision where two share an instruction (exact: a scaled
// value has 8 significant bits and is below 256; what half precision drops is below 2^-24, which no E4M3 term of it holds).
__device__ __forceinline__ uint32_t magnitude(const uint4& raw) {       // the largest, as bfloat16 bits, in either half of the word
    const uint32_t m = 0x7fff7fffu;
    return __vmaxu2(__vmaxu2(raw.x & m, raw.y & m), __vmaxu2(raw.z & m, raw.w & m));
}
__device__ __forceinline__ void terms_of_bf16(const uint4& raw, int byte, uint32_t (&hi)[2], uint32_t (&lo)[2]) {
    const float f = byte == 255 ? 0.f : __uint_as_float((uint32_t)(254 - byte) << 23);
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
    uint16_t h8[4], l8[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float a = __uint_as_float(w[i] << 16) * f, b = __uint_as_float(w[i] & 0xffff0000u) * f;
        uint32_t x, back, rest;
        asm("cvt.rn.f16x2.f32 %0, %2, %1;" : "=r"(x) : "f"(a), "f"(b));
        asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(h8[i]) : "r"(x));
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(back) : "h"(h8[i]));
        asm("{\n\t.reg .b32 d;\n\tsub.f16x2 d, %1, %2;\n\tmul.f16x2 %0, d, %3;\n\t}" : "=r"(rest) : "r"(x), "r"(back), "r"(0x50005000u));     // 32, 32
        asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(l8[i]) : "r"(rest));
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        hi[i] = byte == 255 ? 0 : h8[2 * i] | (uint32_t)h8[2 * i + 1] << 16;
        lo[i] = byte == 255 ? 0 : l8[2 * i] | (uint32_t)l8[2 * i + 1] << 16;
    }
}

// the same eight as 4-bit codes under their block's scale byte
__device__ __forceinline__ uint32_t codes_of_bf16(const uint4& raw, int byte) {
    const float inv = scale_inverse(byte);
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
    uint32_t word = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) word |= pack2(__uint_as_float(w[i] << 16) * inv, __uint_as_float(w[i] & 0xffff0000u) * inv) << (8 * i);
    return byte == 255 ? 0 : word;
}
// eight of a row's values from column c, zero beyond K
__device__ __forceinline__ uint4 row8(const __nv_bfloat16* row, int c, int K, int wide) {
    if (wide && c + 8 <= K) return *reinterpret_cast<const uint4*>(row + c);
    __nv_bfloat16 v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = c + j < K ? row[c + j] : __nv_bfloat16(0.f);
    return *reinterpret_cast<const uint4*>(v);
}

// ---- pieces of the products -----------------------------------------------------------------------------------------------

// How `total` blocks are dealt to P CTAs as one line: the first `more` have one block more than the others.  A unit is kb
// neighbouring blocks; a CTA that does not begin within a unit has its first blocks in the second of its two places for
// sums that are not whole (it can only share the unit it begins in and the unit it ends in with others).
struct Split {
    int total, P, kb, base, more;
    __host__ __device__ Split() {}
    __host__ __device__ Split(int total_, int P_, int kb_) : total(total_), P(P_), kb(kb_), base(total_ / P_), more(total_ - total_ / P_ * P_) {}
    __device__ __forceinline__ int start(int c) const { return c * base + min(c, more); }
    __device__ __forceinline__ int owner(int b) const {
        const int edge = more * (base + 1);
        return b < edge ? b / (base + 1) : more + (b - edge) / base;
    }
    __device__ __forceinline__ int place(int c, int unit) const { return start(c) >= unit * kb ? 0 : 1; }
};

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(smem_addr(dst)), "l"(src), "r"(bytes), "r"(smem_addr(bar)) : "memory");
}
// To a counter in memory, behind all that the calling thread's CTA wrote before it met at a barrier that the thread was at; and (acq)
// ahead of all that is read behind the barrier after it.  A barrier and one thread's release order as much as a fence of every
// thread does and cost less.
__device__ __forceinline__ void add_release(int* p, int v) { asm volatile("red.release.gpu.global.add.s32 [%0], %1;" ::"l"(p), "r"(v) : "memory"); }
__device__ __forceinline__ int add_acq_rel(int* p, int v) {
    int before;
    asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], %2;" : "=r"(before) : "l"(p), "r"(v) : "memory");
    return before;
}
// The warps that issue loads and products run their loops as a whole, and one lane of them issues: operands then stay in the
// uniform registers that these instructions take them from.  A single lane's loop moves them over for every instruction (a
// product of 128 x 32 x 32: 115 cycles against 42, of 128 x 128 x 32 65).
__device__ __forceinline__ bool elect_one() {
    uint32_t e;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(e));
    return e != 0;
}
// Whether a barrier's phase is over, at once: a try_wait may hold the warp for microseconds where it is not (the product of 8 tokens with
// 9,728 x 896 in 4 bits, which asked for the stage behind its last one that way: 10.0 us, so 4.8)
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred P1;\n\tmbarrier.test_wait.parity.shared::cta.b64 P1, [%1], %2;\n\tselp.b32 %0, 1, 0, P1;\n\t}"
                 : "=r"(ok) : "r"(smem_addr(bar)), "r"(parity) : "memory");
    return ok != 0;
}
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abortp) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, abortp));
}
// 512 bytes of scales, 32 rows of 16 without swizzle, to four columns of tensor memory, the same in every quarter of its lanes
__device__ __forceinline__ void scales_to_tmem(uint32_t taddr, uint32_t saddr) {
    const uint64_t d = (uint64_t)((saddr >> 4) & 0x3FFF) | (uint64_t)8 << 32 | (uint64_t)1 << 46;
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(d) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory");
}
template <bool A16>
__device__ __forceinline__ void umma_scaled(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
    if (A16)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
            ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate) : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
            ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate) : "memory");
}
// ---- host side ------------------------------------------------------------------------------------------------------------

// a matrix of bytes (or of 4-bit codes that TMA spreads to a byte each: `spread`, 128 of them a box row), boxes of 128 bytes in shared memory
inline int byte_map(CUtensorMap* map, const void* ptr, long long rows, long long row_bytes, int box_rows, bool spread) {
    tc::EncodeTiledFn fn = tc::encode_fn();
    if (fn == nullptr) return (int)cudaErrorNotSupported;
    cuuint64_t dims[2] = {(cuuint64_t)(spread ? row_bytes * 2 : row_bytes), (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)row_bytes};
    cuuint32_t box[2] = {128, (cuuint32_t)box_rows}, estr[2] = {1, 1};
    CUresult r = fn(map, spread ? CU_TENSOR_MAP_DATA_TYPE_16U4_ALIGN16B : CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(ptr), dims, strides, box,
                    estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? 0 : (int)cudaErrorInvalidValue;
}

inline int current_device() {
    int dev = 0;
    cudaGetDevice(&dev);
    return dev;
}
inline int sm_count() {
    static int n[64] = {};
    const int dev = current_device();
    if (dev < 0 || dev >= 64) return 148;
    if (!n[dev]) cudaDeviceGetAttribute(&n[dev], cudaDevAttrMultiProcessorCount, dev);
    return n[dev];
}
// A kernel's limit of shared memory, always the same value: asked for once on a device
template <typename... KArgs> inline void open_once(void (*kern)(KArgs...), size_t smem, unsigned char (&done)[64]) {
    const int dev = current_device();
    if (dev >= 0 && dev < 64 && done[dev]) return;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) == cudaSuccess && dev >= 0 && dev < 64) done[dev] = 1;
}

}  // namespace mx
}  // namespace prism
