// Building blocks of the tensor-core kernels (rfx_topk.cu, rfx_fp4_product.cu, rfx_fp4_topk.cu):
// bounded mbarrier waits, TMA loads, tcgen05 commits, fences and accumulator reads.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <cstdint>

namespace rfx {

namespace {

constexpr unsigned long long kWaitNs = 1000000000ull;
// A sleeping waiter stays in try_wait until the phase completes or this many nanoseconds pass.
constexpr uint32_t kSuspendNs = 2000;

__device__ __forceinline__ uint32_t smem_u32(const void* p) {
    return (uint32_t)__cvta_generic_to_shared(p);
}

__device__ __forceinline__ unsigned long long now_ns() {
    unsigned long long t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}

template <bool kSleep>
__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    if (kSleep) {
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}\n"
            : "=r"(ok)
            : "r"(bar), "r"(parity), "r"(kSuspendNs)
            : "memory");
    } else {
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}\n"
            : "=r"(ok)
            : "r"(bar), "r"(parity)
            : "memory");
    }
    return ok != 0;
}

// Wait for the phase of `parity` to complete.  Returns kWaitOk, or kWaitFail on timeout or
// when another role of the CTA has aborted (abort may be null: wait regardless), or
// kWaitStop once step `it` is at or beyond the CTA's stop limit (limit may be null).
constexpr int kWaitFail = 0, kWaitOk = 1, kWaitStop = 2;

template <bool kSleep = true>
__device__ int mbar_wait(uint32_t bar, uint32_t parity, volatile int* abort,
                         unsigned long long* polls = nullptr, volatile int* limit = nullptr,
                         int it = 0) {
    unsigned long long t0 = 0;  // read at the 16th poll: most waits end before it
    for (uint32_t spin = 1;; ++spin) {
        if (polls) ++*polls;
        if (mbar_try<kSleep>(bar, parity)) return kWaitOk;
        if (limit && it >= *limit) return kWaitStop;
        if (abort && *abort) return kWaitFail;
        if ((spin & 15u) == 0) {
            const unsigned long long t = now_ns();
            if (t0 == 0) t0 = t;
            else if (t - t0 > kWaitNs) return kWaitFail;
        }
    }
}

// mbar_wait for the roles that may not lose cycles: one inlined poll, the bounded loop behind it.
// True when the phase has completed.
__device__ __noinline__ bool mbar_wait_slow(uint32_t bar, uint32_t parity, volatile int* abort) {
    return mbar_wait<false>(bar, parity, abort) == kWaitOk;
}
__device__ __forceinline__ bool mbar_wait_fast(uint32_t bar, uint32_t parity, volatile int* abort) {
    return mbar_try<false>(bar, parity) || mbar_wait_slow(bar, parity, abort);
}

// For the issuing warps: no result, so that their control flow stays uniform.  A wait that runs out
// records `code` in *err and sets *abort, after which every wait returns at once: the warp runs
// through the rest of its loop on whatever the buffers hold, and the call ends with its error.
__device__ __noinline__ void mbar_wait_issue_slow(uint32_t bar, uint32_t parity, volatile int* abort, int* err, int code) {
    if (mbar_wait<false>(bar, parity, abort) != kWaitOk && !*abort) {
        atomicExch(err, code);
        *abort = 1;
    }
}
__device__ __forceinline__ void mbar_wait_issue(uint32_t bar, uint32_t parity, volatile int* abort, int* err, int code) {
    if (!mbar_try<false>(bar, parity)) mbar_wait_issue_slow(bar, parity, abort, err, code);
    __syncwarp();
}

// True in one lane of a converged warp.  The single-issuer roles run their loops in the whole warp
// and issue under this predicate: addresses and descriptors then stay in uniform registers, which
// the TMA and tcgen05 instructions take (a loop inside one lane moves each of them there first).
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xFFFFFFFF;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}\n"
        : "=r"(p));
    return p != 0;
}

// A position in a ring of n slots: its slot and the parity of the round.
struct RingPos {
    int slot = 0;
    uint32_t parity = 0;
    __device__ __forceinline__ void next(int n) {
        if (++slot == n) {
            slot = 0;
            parity ^= 1u;
        }
    }
};

// mbar_wait that also adds the cycles it spent to *cyc.
template <bool kSleep = true>
__device__ __forceinline__ int mbar_wait_t(uint32_t bar, uint32_t parity, volatile int* abort,
                                           unsigned long long* polls, unsigned long long* cyc,
                                           volatile int* limit = nullptr, int it = 0) {
    const long long t0 = clock64();
    const int r = mbar_wait<kSleep>(bar, parity, abort, polls, limit, it);
    *cyc += (unsigned long long)(clock64() - t0);
    return r;
}

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}

__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes)
                 : "memory");
}

__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}

// Programmatic dependent launch: a kernel lets the next one's blocks start, and a kernel started so
// waits for the one before (its memory included) to end.
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
// What the kernel before left, after wait_for_previous(): an ordinary load.  Not __ldg, which promises
// that nobody writes the data while this kernel runs; the compiler may then place it above the wait.
template <class T>
__device__ __forceinline__ T load_left(const T* p) {
    return *p;
}

// Work by cluster launch control: a running block takes over the index of one that has not started.
// The 16-byte answer arrives in shared memory at `slot`, completing on `bar`.
__device__ __forceinline__ void clc_request(uint32_t slot, uint32_t bar) {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // after the last answer's readers
    mbar_expect_tx(bar, 16);
    asm volatile(
        "clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(slot),
        "r"(bar)
        : "memory");
}
// The block index taken over, or -1 when none was left (no further request may follow).
__device__ __forceinline__ int clc_answer(uint32_t slot) {
    uint32_t ok, x;
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b128 h;\n\t.reg .b32 y, z, w;\n\t"
        "ld.shared.b128 h, [%2];\n\t"
        "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t"
        "mov.u32 %1, 0;\n\t"
        "@p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%1, y, z, w}, h;\n\t}\n"
        : "=r"(ok), "=r"(x)
        : "r"(slot)
        : "memory");
    return ok ? (int)x : -1;
}

// 2-D tiled TMA load of a map's box into shared memory, completing on `bar`; x times the element size
// is a multiple of 16 bytes.
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* tm, int x, int y,
                                         uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
        "l"((unsigned long long)tm), "r"(x), "r"(y), "r"(bar)
        : "memory");
}

// Shared-memory matrix descriptor: K-major, 128-byte swizzle, 8-row groups 1024 bytes apart.
__device__ __forceinline__ uint64_t sw128_desc(uint32_t addr) {
    uint64_t d = (uint64_t)((addr & 0x3FFFFu) >> 4);  // start address
    d |= (uint64_t)1 << 16;                           // leading offset (unused when swizzled)
    d |= (uint64_t)(1024 >> 4) << 32;                 // stride offset
    d |= (uint64_t)1 << 46;                           // descriptor version
    d |= (uint64_t)2 << 61;                           // 128-byte swizzle
    return d;
}

__device__ __forceinline__ void mma_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar)
                 : "memory");
}

__device__ __forceinline__ void tc_fence_before() {
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tc_fence_after() {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}

// Issue a load of 32 consecutive fp32 accumulator columns of this thread's TMEM lane; the
// registers are valid after tmem_wait().
__device__ __forceinline__ void tmem_ld32_issue(uint32_t taddr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
          "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
          "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
          "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]),
          "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
}

__device__ __forceinline__ void tmem_wait() {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

// Ties 32 loaded registers to a point after tmem_wait() so no use moves above the wait.
__device__ __forceinline__ void tmem_pin32(uint32_t* r) {
    asm volatile(""
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]),
                   "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]),
                   "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]),
                   "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                   "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),
                   "+r"(r[30]), "+r"(r[31]));
}

// Largest of three floats (the three-input max.f32 of sm_100).
__device__ __forceinline__ float fmax3(float x, float y, float z) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(x), "f"(y), "f"(z));
    return d;
}

}  // namespace

}  // namespace rfx
