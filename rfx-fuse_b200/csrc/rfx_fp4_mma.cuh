// tcgen05 block-scaled 4-bit products: operands, scales and instruction descriptors.
//
// One step multiplies 64 columns: A 128 rows, B up to 256 rows, both K-major in shared memory
// (32 bytes of a row a step), scales in TMEM.  nvfp4 reads four scales a row and step (one atom
// of 128 rows x 4), mxfp4 two: an atom serves two steps, and the scale id in the instruction
// descriptor picks its half.
#pragma once
#include "rfx_fp4_dev.cuh"
#include "rfx_tc.cuh"

namespace rfx {

namespace {

// K-major rows of kBytes (32 or 128) under the swizzle of that width; a descriptor moves by one
// step with + 2 (32 bytes).
template <int kBytes>
__device__ __forceinline__ uint64_t f4_operand_desc(uint32_t addr) {
    uint64_t d = (uint64_t)((addr & 0x3FFFFu) >> 4);
    d |= (uint64_t)1 << 16;
    d |= (uint64_t)((8 * kBytes) >> 4) << 32;           // 8-row groups follow one another
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)(kBytes == 128 ? 2 : 6) << 61;       // 128- or 32-byte swizzle
    return d;
}

// A scale atom in shared memory: 32 rows of 16 bytes, no swizzle.
__device__ __forceinline__ uint64_t f4_atom_desc(uint32_t addr) {
    uint64_t d = (uint64_t)((addr & 0x3FFFFu) >> 4);
    d |= (uint64_t)1 << 16;
    d |= (uint64_t)(128 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    return d;
}

// Four TMEM columns from an atom, repeated over the four lane quarters.
__device__ __forceinline__ void f4_copy_atom(uint32_t tmem, uint64_t desc) {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
}

// Both operands e2m1, fp32 accumulators, M = 128, N = n; `half` picks an atom's half (mxfp4).
template <int kNv>
__device__ __forceinline__ uint32_t f4_idesc(int n, int half) {
    uint32_t d = (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((128u >> 4) << 24);
    if (!kNv) d |= (1u << 23) | ((uint32_t)(2 * half) << 4) | ((uint32_t)(2 * half) << 29);
    return d;
}

template <int kNv>
__device__ __forceinline__ void f4_mma(uint32_t d, uint64_t da, uint64_t db, uint32_t idesc,
                                       uint32_t sa, uint32_t sb, uint32_t acc) {
    if (kNv) {
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X "
            "[%0], %1, %2, %3, [%4], [%5], p;\n\t}\n" ::"r"(d),
            "l"(da), "l"(db), "r"(idesc), "r"(sa), "r"(sb), "r"(acc)
            : "memory");
    } else {
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X "
            "[%0], %1, %2, %3, [%4], [%5], p;\n\t}\n" ::"r"(d),
            "l"(da), "l"(db), "r"(idesc), "r"(sa), "r"(sb), "r"(acc)
            : "memory");
    }
}

// The two matrices' scales as factors of an accumulator, x * lead * rest.  Their product alone may
// leave fp32 where the result does not (0 * inf, 2^20 * 2^-160): then the larger comes first, so that
// x * lead is infinite only if the result is (rest >= 1) and small only by an exact power of two.
struct F4Alpha {
    float lead, rest;
};
__device__ __forceinline__ F4Alpha f4_alpha(const float* ga, const float* gb) {
    const float x = __ldg(ga), y = __ldg(gb);
    const float lead = x > y ? x : y, rest = x > y ? y : x, both = lead * rest;
    if (both >= 1.17549435e-38f && both <= 3.40282347e38f) return {both, 1.0f};
    return {lead, rest};
}

// Untiled copy of `bytes` (a multiple of 16) into shared memory, completing on `bar`.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
        "l"(src), "r"(bytes), "r"(bar)
        : "memory");
}

}  // namespace

}  // namespace rfx
