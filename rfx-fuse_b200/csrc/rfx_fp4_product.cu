// Product of two matrices in microscaled 4 bits, out[i][j] = a_i . b_j, on the block-scaled
// tcgen05 tensor cores (fp32 accumulation, one rounding to the output type).
//
// The 128 rows of the instruction's A are rows of b (columns of the output): an accumulator lane
// is then an output column, so a warp's store of one register is 32 neighbouring outputs and
// needs no transpose; the instruction's N holds up to 256 rows of a, and shrinks to the rows
// there are (16 at least), so that a product of a few rows only reads b.
//
// A block takes the unit (p.group neighbouring tiles) of its index, then the units of blocks that have
// not started yet, by cluster launch control: some SMs store at three quarters of the others' rate,
// and equal shares of 43 tiles left those running for 50 us of 185 (1,024 x 200,000 fp32 outputs).
//   warps 0-7  read an accumulator (quarter warp & 3) and store it.  With tiles of up to 128 rows of
//              a the accumulators form a ring and the two groups of four warps take alternate tiles;
//              with more, both take the one accumulator, half the columns each, and release it as
//              soon as it is in registers, so the next tile's products run under the stores;
//   warp 8     loads code rows by TMA and scale atoms by bulk copies into a ring of
//              chunks of 256 columns (64 when the matrix has no more);
//   warp 9     allocates TMEM; copies the chunk's atoms to TMEM (its columns belong to
//              the ring stage, so a stage's "empty" barrier also frees them) and multiplies.
// Every wait is bounded; on expiry the CTA records it in *err, drains its copies, frees TMEM and
// returns.
#include <algorithm>

#include "rfx_fp4_mma.cuh"

namespace rfx {

namespace {

constexpr int kPThreads = 320;
constexpr int kPMaxStage = 16;
constexpr int kPSmem = 227 * 1024;
constexpr int kPSched = 4;
constexpr int kPBars = 1024;  // barriers and flags

template <int kNv, int kCB, class T>
__global__ void __launch_bounds__(kPThreads, 1)
k_f4_product(const __grid_constant__ CUtensorMap tma, const __grid_constant__ CUtensorMap tmb, F4ProductArgs p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* sm = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint64_t* bars = (uint64_t*)sm;
    // full[16], empty[16], acc_full[8], acc_empty[8]
    uint32_t* tmem_slot = (uint32_t*)(bars + 48);
    volatile int* abort = (volatile int*)(tmem_slot + 1);
    const uint32_t bar0 = smem_u32(bars);
    auto full = [&](int s) { return bar0 + 8u * s; };
    auto empty = [&](int s) { return bar0 + 8u * (16 + s); };
    auto accf = [&](int b) { return bar0 + 8u * (32 + b); };
    auto acce = [&](int b) { return bar0 + 8u * (40 + b); };
    // answers of the tile scheduler: 4 slots of 16 bytes, their full and empty barriers
    auto sslot = [&](int s) { return bar0 + 512u + 16u * s; };
    auto sfull = [&](int s) { return bar0 + 576u + 8u * s; };
    auto sempty = [&](int s) { return bar0 + 608u + 8u * s; };
    const uint32_t stage0 = bar0 + kPBars;
    constexpr int kAtoms = kCB == 32 ? 1 : (kNv ? 4 : 2);  // scale atoms of a whole chunk
    const int nrt = p.bn > kF4Tile ? 2 : 1;                // scale tiles of a's rows
    const uint32_t off_b = 128 * kCB;
    const uint32_t off_sb = off_b + (uint32_t)((p.bn * kCB + 1023) / 1024 * 1024);  // scales of b, then of a
    const uint32_t off_sa = off_sb + kAtoms * kF4Atom;
    const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int s = 0; s < p.nstage; ++s) {
            mbar_init(full(s), 1);
            mbar_init(empty(s), 1);
        }
        for (int b = 0; b < p.nacc; ++b) {
            mbar_init(accf(b), 1);
            mbar_init(acce(b), p.nacc > 1 ? 4 : 8);  // one arrival a warp
        }
        for (int s = 0; s < kPSched; ++s) {
            mbar_init(sfull(s), 1);
            mbar_init(sempty(s), 10);  // every warp
        }
        *abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                         smem_u32(tmem_slot)),
                     "r"(512)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    constexpr uint32_t tmem = 0;  // all 512 columns are this block's: they start at column 0
    RingPos sched;
    bool ok = true;
    // the next unit of this warp, or -1
    auto next_unit = [&]() {
        if (!__all_sync(0xFFFFFFFFu, mbar_wait_fast(sfull(sched.slot), sched.parity, abort))) {
            ok = false;
            return -1;
        }
        const int t = __shfl_sync(0xFFFFFFFFu, clc_answer(sslot(sched.slot)), 0);
        __syncwarp();
        if (lane == 0) mbar_arrive(sempty(sched.slot));
        sched.next(kPSched);
        return t;
    };

    if (warp == 8) {
        int step = 0;
        RingPos st;
        bool asked = false;
        for (int unit = blockIdx.x; ok && unit >= 0; unit = ok ? next_unit() : -1) {
            ok = __all_sync(0xFFFFFFFFu, mbar_wait_fast(sempty(sched.slot), sched.parity ^ 1u, abort));
            if (!ok) break;
            if (elect_one()) clc_request(sslot(sched.slot), sfull(sched.slot));
            asked = true;
            for (int t = unit * p.group, te = min(t + p.group, p.ntiles); ok && t < te; ++t) {
                const int jt = t % p.njt, i0 = t / p.njt * p.bn;
                const int rt0 = i0 / kF4Tile;
                const int rts = min(nrt, p.a.tiles() - rt0);
                const uint8_t* sb = p.b.scales + (long long)jt * p.b.natoms * kF4Atom;
                const uint8_t* sa = p.a.scales + (long long)rt0 * p.a.natoms * kF4Atom;
                int left = p.b.Kp / 64;  // steps to go
                for (int c = 0; c < p.nchunk; ++c, ++step) {
                    ok = __all_sync(0xFFFFFFFFu, mbar_wait_fast(empty(st.slot), st.parity ^ 1u, abort));
                    if (!ok) break;
                    const int steps = min(left, kCB / 32);
                    left -= steps;
                    if (elect_one()) {
                        const uint32_t dst = stage0 + (uint32_t)(st.slot * p.stage_bytes), bar = full(st.slot);
                        const uint32_t sfb = (uint32_t)((kNv ? steps : (steps + 1) / 2) * kF4Atom);
                        mbar_expect_tx(bar, (uint32_t)((128 + p.bn) * kCB) + sfb * (1 + rts));
                        tma_load(dst, &tmb, c * kCB, jt * 128, bar);
                        tma_load(dst + off_b, &tma, c * kCB, i0, bar);
                        bulk_load(dst + off_sb, sb, sfb, bar);
                        bulk_load(dst + off_sa, sa, sfb, bar);
                        if (rts > 1)
                            bulk_load(dst + off_sa + kAtoms * kF4Atom, sa + (long long)p.a.natoms * kF4Atom, sfb, bar);
                    }
                    sb += kAtoms * kF4Atom;
                    sa += kAtoms * kF4Atom;
                    st.next(p.nstage);
                }
            }
        }
        if (!ok && lane == 0) {
            if (!*abort) atomicExch(p.err, 1);
            *abort = 1;
        }
        // drain this warp's answer and copies still in flight (after next_unit the answer has been read)
        if (!ok && asked) mbar_wait<false>(sfull(sched.slot), sched.parity, nullptr);
        for (int i = step > p.nstage ? step - p.nstage : 0; i < step; ++i)
            mbar_wait<false>(full(i % p.nstage), (uint32_t)(i / p.nstage) & 1u, nullptr);
        __syncwarp();
    } else if (warp == 9) {
        RingPos st, ac;
        int last = -1;
        uint32_t last_parity = 0;
        const uint32_t sfc = (uint32_t)(4 * kAtoms * (1 + nrt));  // TMEM columns of a stage's scales
        for (int unit = blockIdx.x; unit >= 0; unit = next_unit()) {
            for (int t = unit * p.group, te = min(t + p.group, p.ntiles); t < te; ++t) {
                mbar_wait_issue(acce(ac.slot), ac.parity ^ 1u, abort, p.err, 2);
                tc_fence_after();
                const uint32_t d = tmem + (uint32_t)(ac.slot * p.acc_cols);
                int left = p.b.Kp / 64;
                for (int c = 0; c < p.nchunk; ++c) {
                    mbar_wait_issue(full(st.slot), st.parity, abort, p.err, 2);
                    tc_fence_after();
                    const uint32_t src = stage0 + (uint32_t)(st.slot * p.stage_bytes);
                    const int steps = min(left, kCB / 32);
                    left -= steps;
                    const int atoms = kNv ? steps : (steps + 1) / 2;
                    const uint32_t tsb = tmem + 256u + (uint32_t)st.slot * sfc, tsa = tsb + 4 * kAtoms;
                    const uint64_t db = f4_operand_desc<kCB>(src), da = f4_operand_desc<kCB>(src + off_b);
                    const uint64_t dsb = f4_atom_desc(src + off_sb), dsa = f4_atom_desc(src + off_sa);
                    if (elect_one()) {
#pragma unroll
                        for (int k = 0; k < kAtoms; ++k) {
                            if (k >= atoms) break;
                            f4_copy_atom(tsb + 4 * k, dsb + k * (kF4Atom >> 4));
                            f4_copy_atom(tsa + 4 * k * nrt, dsa + k * (kF4Atom >> 4));
                            if (nrt > 1) f4_copy_atom(tsa + 8 * k + 4, dsa + (kAtoms + k) * (kF4Atom >> 4));
                        }
#pragma unroll
                        for (int k = 0; k < kCB / 32; ++k) {
                            if (k >= steps) break;
                            const int at = kNv ? k : k >> 1;
                            f4_mma<kNv>(d, db + 2 * k, da + 2 * k, f4_idesc<kNv>(p.bn, kNv ? 0 : k & 1),
                                        tsb + 4 * at, tsa + 4 * nrt * at, (c | k) ? 1u : 0u);
                        }
                        mma_commit(empty(st.slot));
                        if (c == p.nchunk - 1) mma_commit(accf(ac.slot));
                    }
                    __syncwarp();
                    last = st.slot;
                    last_parity = st.parity;
                    st.next(p.nstage);
                }
                ac.next(p.nacc);
            }
        }
        if (!ok && lane == 0) {
            if (!*abort) atomicExch(p.err, 2);
            *abort = 1;
        }
        // the last products must finish before the accumulators are freed
        if (last >= 0) mbar_wait<false>(empty(last), last_parity, nullptr);
        __syncwarp();
    } else {
        const int group = warp >> 2;
        const int jl = 32 * (warp & 3) + lane;
        const uint32_t lane_addr = (uint32_t)(32 * (warp & 3)) << 16;
        const F4Alpha alpha = f4_alpha(p.a.gs, p.b.gs);
        T* out = (T*)p.out;
        RingPos ac;
        int n = 0;
        for (int unit = blockIdx.x; ok && unit >= 0; unit = ok ? next_unit() : -1) {
            for (int t = unit * p.group, te = min(t + p.group, p.ntiles); t < te; ++t, ++n, ac.next(p.nacc)) {
                if (p.nacc > 1 && (n & 1) != group) continue;
                const int b = ac.slot;
                ok = __all_sync(0xFFFFFFFFu, mbar_wait_fast(accf(b), ac.parity, abort));
                if (!ok) break;
                tc_fence_after();
                const int jt = t % p.njt, i0 = t / p.njt * p.bn;
                const int cb = p.nacc > 1 ? 0 : 128 * group;   // first of this warp's columns (rows of a)
                const int ce = min(min(p.bn, cb + 128), p.a.rows - i0);
                uint32_t r[4][32];
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    if (cb + 32 * c < ce) tmem_ld32_issue(tmem + lane_addr + (uint32_t)(b * p.acc_cols + cb + 32 * c), r[c]);
                tmem_wait();
#pragma unroll
                for (int c = 0; c < 4; ++c) tmem_pin32(r[c]);
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(acce(b));
                const long long j = (long long)jt * 128 + jl;
                if (j < p.b.rows) {
                    T* o = out + (long long)(i0 + cb) * p.ld + j;
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const int rows = ce - cb - 32 * c;
                        if (rows >= 32) {
#pragma unroll
                            for (int e = 0; e < 32; ++e, o += p.ld) *o = from_f32<T>(__uint_as_float(r[c][e]) * alpha.lead * alpha.rest);
                        } else if (rows > 0) {
#pragma unroll
                            for (int f = 0; f < 32; f += 4) {  // few rows leave most of these branches
                                if (f < rows) {
#pragma unroll
                                    for (int e = f; e < f + 4; ++e, o += p.ld)
                                        if (e < rows) *o = from_f32<T>(__uint_as_float(r[c][e]) * alpha.lead * alpha.rest);
                                }
                            }
                        }
                    }
                }
                __syncwarp();
            }
        }
        if (!ok && lane == 0) {
            if (!*abort) atomicExch(p.err, 3);
            *abort = 1;
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 9) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(*tmem_slot), "r"(512)
                     : "memory");
    }
}

// Few rows of a (up to 32) of at most 256 columns: the product only streams b, and what a tile costs
// beside its bytes bounds it.  So a stays in shared memory and TMEM, a stage is four tiles of b
// (their scales one copy), and the four tiles' outputs of kBn rows sit side by side in accumulators
// of 32 columns, 32 / kBn tiles in each: one wait, one TMEM load and one release for all of them.
// One row against 1,000,000 x 64: 28 us in the general kernel (issue-bound at 670 cycles a tile).
//   warps 0-7  read accumulators (quarter warp & 3; the two groups of four take alternate ones);
//   warp 8     loads; warp 9 allocates TMEM, copies scales and multiplies.
constexpr int kSGroup = 4;   // tiles of a stage
constexpr int kSAcc = 8;     // accumulators of 32 columns
constexpr int rows_stages(int cb) { return cb == 32 ? 8 : 3; }
constexpr int rows_stage(int nv, int cb) { return kSGroup * (128 * cb + (cb == 32 ? 1 : nv ? 4 : 2) * kF4Atom); }

template <int kNv, int kCB, class T, int kBn>
__global__ void __launch_bounds__(kPThreads, 1)
k_f4_product_rows(const __grid_constant__ CUtensorMap tma, const __grid_constant__ CUtensorMap tmb, F4ProductArgs p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* sm = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint64_t* bars = (uint64_t*)sm;
    // full[8], empty[8], acc_full[8], acc_empty[8], a_full
    uint32_t* tmem_slot = (uint32_t*)(bars + 40);
    volatile int* abort = (volatile int*)(tmem_slot + 1);
    const uint32_t bar0 = smem_u32(bars);
    auto full = [&](int s) { return bar0 + 8u * s; };
    auto empty = [&](int s) { return bar0 + 8u * (8 + s); };
    auto accf = [&](int b) { return bar0 + 8u * (16 + b); };
    auto acce = [&](int b) { return bar0 + 8u * (24 + b); };
    const uint32_t afull = bar0 + 8u * 32;
    constexpr int kAtoms = kCB == 32 ? 1 : (kNv ? 4 : 2);
    constexpr int kBox = 128 * kCB;
    constexpr int kStages = rows_stages(kCB), kStage = rows_stage(kNv, kCB);
    constexpr int kPer = 32 / kBn;                      // tiles of an accumulator
    const uint32_t s_a = bar0 + kPBars, s_sa = s_a + 32 * kCB, ring0 = s_a + 8192;
    const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int ngroups = (p.njt + kSGroup - 1) / kSGroup;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(full(s), 1);
            mbar_init(empty(s), 1);
        }
        for (int b = 0; b < kSAcc; ++b) {
            mbar_init(accf(b), 1);
            mbar_init(acce(b), 4);  // one arrival a warp
        }
        mbar_init(afull, 1);
        *abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                         smem_u32(tmem_slot)),
                     "r"(512)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    constexpr uint32_t tmem = 0;  // all 512 columns are this block's: they start at column 0
    const int steps = p.b.Kp / 64;
    const int atoms = kNv ? steps : (steps + 1) / 2;
    bool ok = true;

    if (warp == 8) {
        const uint32_t sfb = (uint32_t)(atoms * kF4Atom);
        RingPos st;
        int n = 0;
        if (elect_one()) {
            mbar_expect_tx(afull, (uint32_t)(kBn * kCB) + sfb);
            tma_load(s_a, &tma, 0, 0, afull);
            bulk_load(s_sa, p.a.scales, sfb, afull);
        }
        for (int g = blockIdx.x; g < ngroups; g += gridDim.x, ++n) {
            ok = __all_sync(0xFFFFFFFFu, mbar_wait_fast(empty(st.slot), st.parity ^ 1u, abort));
            if (!ok) break;
            if (elect_one()) {
                const uint32_t dst = ring0 + (uint32_t)(st.slot * kStage), bar = full(st.slot);
                const int t = g * kSGroup, nt = min(kSGroup, p.njt - t);
                const uint32_t sc = (uint32_t)nt * sfb;  // the tiles' scales follow one another
                mbar_expect_tx(bar, (nt > 2 ? 4u : 2u) * kBox + sc);
                tma_load(dst, &tmb, 0, t * 128, bar);
                if (nt > 2) tma_load(dst + 2 * kBox, &tmb, 0, t * 128 + 256, bar);
                bulk_load(dst + kSGroup * kBox, p.b.scales + (long long)t * p.b.natoms * kF4Atom, sc, bar);
            }
            st.next(kStages);
        }
        if (!ok && lane == 0) {
            if (!*abort) atomicExch(p.err, 1);
            *abort = 1;
        }
        // drain this warp's copies still in flight
        mbar_wait<false>(afull, 0, nullptr);
        for (int i = n > kStages ? n - kStages : 0; i < n; ++i)
            mbar_wait<false>(full(i % kStages), (uint32_t)(i / kStages) & 1u, nullptr);
        __syncwarp();
    } else if (warp == 9) {
        RingPos st, ac;
        int last = -1;
        uint32_t last_parity = 0;
        mbar_wait_issue(afull, 0, abort, p.err, 2);
        const uint32_t tsa = tmem + 256u;
        const uint64_t da = f4_operand_desc<kCB>(s_a);
        tc_fence_after();
        if (elect_one())
            for (int k = 0; k < atoms; ++k) f4_copy_atom(tsa + 4 * k, f4_atom_desc(s_sa + k * kF4Atom));
        __syncwarp();
        for (int g = blockIdx.x; g < ngroups; g += gridDim.x) {
            mbar_wait_issue(full(st.slot), st.parity, abort, p.err, 2);
            tc_fence_after();
            const uint32_t src = ring0 + (uint32_t)(st.slot * kStage);
            const uint32_t tsb = tmem + 272u + (uint32_t)(st.slot * kSGroup * 4 * kAtoms);
            const int nt = min(kSGroup, p.njt - g * kSGroup);
#pragma unroll
            for (int h0 = 0; h0 < kSGroup; h0 += kPer) {
                if (h0 >= nt) break;
                mbar_wait_issue(acce(ac.slot), ac.parity ^ 1u, abort, p.err, 2);
                tc_fence_after();
                if (elect_one()) {
#pragma unroll
                    for (int h = h0; h < h0 + kPer; ++h) {
                        if (h >= nt) break;
                        const uint32_t d = tmem + (uint32_t)(32 * ac.slot + (h - h0) * kBn);
                        const uint32_t tsh = tsb + 4 * kAtoms * h;
                        const uint64_t db = f4_operand_desc<kCB>(src + h * kBox);
                        const uint64_t dsc = f4_atom_desc(src + kSGroup * kBox + h * atoms * kF4Atom);
                        if (kCB == 32) {
                            f4_copy_atom(tsh, dsc);
                            f4_mma<kNv>(d, db, da, f4_idesc<kNv>(kBn, 0), tsh, tsa, 0u);
                        } else {
                            for (int k = 0; k < atoms; ++k) f4_copy_atom(tsh + 4 * k, dsc + k * (kF4Atom >> 4));
                            for (int k = 0; k < steps; ++k) {
                                const int at = kNv ? k : k >> 1;
                                f4_mma<kNv>(d, db + 2 * k, da + 2 * k, f4_idesc<kNv>(kBn, kNv ? 0 : k & 1), tsh + 4 * at,
                                            tsa + 4 * at, k ? 1u : 0u);
                            }
                        }
                    }
                    mma_commit(accf(ac.slot));
                    if (h0 + kPer >= nt) mma_commit(empty(st.slot));
                }
                __syncwarp();
                last = ac.slot;
                last_parity = ac.parity;
                ac.next(kSAcc);
            }
            st.next(kStages);
        }
        // the last products must finish before the accumulators are freed
        if (last >= 0) mbar_wait<false>(accf(last), last_parity, nullptr);
        __syncwarp();
    } else {
        const int set = warp >> 2;
        const int jl = 32 * (warp & 3) + lane;
        const uint32_t lane_addr = tmem + ((uint32_t)(32 * (warp & 3)) << 16);
        const F4Alpha alpha = f4_alpha(p.a.gs, p.b.gs);
        T* out = (T*)p.out;
        RingPos ac;
        for (int g = blockIdx.x; ok && g < ngroups; g += gridDim.x) {
            const int nt = min(kSGroup, p.njt - g * kSGroup);
#pragma unroll
            for (int h = 0; h < kSGroup; h += kPer) {
                if (h >= nt || !ok) break;
                if ((ac.slot & 1) == set) {  // the ring's length is even: a set keeps its accumulators
                    ok = __all_sync(0xFFFFFFFFu, mbar_wait_fast(accf(ac.slot), ac.parity, abort));
                    if (!ok) break;
                    tc_fence_after();
                    uint32_t r[32];
                    tmem_ld32_issue(lane_addr + (uint32_t)(32 * ac.slot), r);
                    tmem_wait();
                    tmem_pin32(r);
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(acce(ac.slot));
                    const long long j = ((long long)g * kSGroup + h) * 128 + jl;
                    T* o = out + j;
#pragma unroll
                    for (int i = 0; i < kBn; ++i, o += p.ld) {
                        if (i < p.a.rows) {
#pragma unroll
                            for (int e = 0; e < kPer; ++e)
                                if (j + 128 * e < p.b.rows)
                                    o[128 * e] = from_f32<T>(__uint_as_float(r[e * kBn + i]) * alpha.lead * alpha.rest);
                        }
                    }
                }
                ac.next(kSAcc);
            }
        }
        if (!ok && lane == 0) {
            if (!*abort) atomicExch(p.err, 3);
            *abort = 1;
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 9) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(*tmem_slot), "r"(512)
                     : "memory");
    }
}

template <int kNv, int kCB, class T, int kBn>
cudaError_t launch_rows_bn(const CUtensorMap& ta, const CUtensorMap& tb, const F4ProductArgs& p, int grid, cudaStream_t st) {
    const int smem = 1024 + kPBars + 8192 + rows_stages(kCB) * rows_stage(kNv, kCB);
    auto f = k_f4_product_rows<kNv, kCB, T, kBn>;
    cudaError_t e = cudaFuncSetAttribute((const void*)f, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    f<<<grid, kPThreads, smem, st>>>(ta, tb, p);
    return cudaGetLastError();
}

template <int kNv, int kCB, class T>
cudaError_t launch_rows(const CUtensorMap& ta, const CUtensorMap& tb, const F4ProductArgs& p, int grid, cudaStream_t st) {
    if (p.bn == 8) return launch_rows_bn<kNv, kCB, T, 8>(ta, tb, p, grid, st);
    if (p.bn == 16) return launch_rows_bn<kNv, kCB, T, 16>(ta, tb, p, grid, st);
    return launch_rows_bn<kNv, kCB, T, 32>(ta, tb, p, grid, st);
}

// Few rows of a over a long inner axis give few tiles: the blocks of a cluster split the axis of one
// tile, leave their fp32 sums in shared memory and each adds up a share of the rows over the
// cluster's blocks, in the order of their shares of the axis (no atomics: the same sums every time).
// 16 x 8,192 x 8,192: 14.3 us in the general kernel, where 64 tiles keep 64 of 148 SMs busy.
//   warps 0-3  accumulator to shared memory, then the sums; warp 4 loads; warp 5 multiplies.
constexpr int kXThreads = 192;
constexpr int kXRows = 64;   // rows of a at most
constexpr int kXStages = 6;

template <int kNv, class T>
__global__ void __launch_bounds__(kXThreads, 1)
k_f4_product_split(const __grid_constant__ CUtensorMap tma, const __grid_constant__ CUtensorMap tmb, F4ProductArgs p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* sm = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint64_t* bars = (uint64_t*)sm;
    // full[6], empty[6], acc_full
    uint32_t* tmem_slot = (uint32_t*)(bars + 16);
    volatile int* abort = (volatile int*)(tmem_slot + 1);
    const uint32_t bar0 = smem_u32(bars);
    auto full = [&](int s) { return bar0 + 8u * s; };
    auto empty = [&](int s) { return bar0 + 8u * (kXStages + s); };
    const uint32_t accf = bar0 + 8u * 12;
    constexpr int kCB = 128, kAtoms = kNv ? 4 : 2;
    const uint32_t stage0 = bar0 + kPBars;
    const uint32_t off_b = 128 * kCB, off_sb = off_b + kXRows * kCB, off_sa = off_sb + kAtoms * kF4Atom;
    constexpr uint32_t kStage = (128 + kXRows) * kCB + 2 * kAtoms * kF4Atom;
    const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int part = blockIdx.x % p.split, jt = blockIdx.x / p.split;
    const int c0 = p.nchunk * part / p.split, c1 = p.nchunk * (part + 1) / p.split;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kXStages; ++s) {
            mbar_init(full(s), 1);
            mbar_init(empty(s), 1);
        }
        mbar_init(accf, 1);
        *abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 5) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                         smem_u32(tmem_slot)),
                     "r"(512)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    constexpr uint32_t tmem = 0;  // all 512 columns are this block's: they start at column 0
    bool ok = true;

    if (warp == 4) {
        RingPos st;
        int n = 0;
        const uint8_t* sb = p.b.scales + ((long long)jt * p.b.natoms + c0 * kAtoms) * kF4Atom;
        const uint8_t* sa = p.a.scales + (long long)c0 * kAtoms * kF4Atom;
        for (int c = c0; c < c1; ++c, ++n) {
            ok = __all_sync(0xFFFFFFFFu, mbar_wait_fast(empty(st.slot), st.parity ^ 1u, abort));
            if (!ok) break;
            const int steps = min(p.b.Kp / 64 - 4 * c, 4);
            if (elect_one()) {
                const uint32_t dst = stage0 + (uint32_t)st.slot * kStage, bar = full(st.slot);
                const uint32_t sfb = (uint32_t)((kNv ? steps : (steps + 1) / 2) * kF4Atom);
                mbar_expect_tx(bar, (uint32_t)((128 + p.bn) * kCB) + 2 * sfb);
                tma_load(dst, &tmb, c * kCB, jt * 128, bar);
                tma_load(dst + off_b, &tma, c * kCB, 0, bar);
                bulk_load(dst + off_sb, sb, sfb, bar);
                bulk_load(dst + off_sa, sa, sfb, bar);
            }
            sb += kAtoms * kF4Atom;
            sa += kAtoms * kF4Atom;
            st.next(kXStages);
        }
        if (!ok && lane == 0) {
            if (!*abort) atomicExch(p.err, 1);
            *abort = 1;
        }
        // drain this warp's copies still in flight
        for (int i = n > kXStages ? n - kXStages : 0; i < n; ++i)
            mbar_wait<false>(full(i % kXStages), (uint32_t)(i / kXStages) & 1u, nullptr);
        __syncwarp();
    } else if (warp == 5) {
        RingPos st;
        for (int c = c0; c < c1; ++c) {
            mbar_wait_issue(full(st.slot), st.parity, abort, p.err, 2);
            tc_fence_after();
            const uint32_t src = stage0 + (uint32_t)st.slot * kStage;
            const int steps = min(p.b.Kp / 64 - 4 * c, 4);
            const int atoms = kNv ? steps : (steps + 1) / 2;
            const uint32_t tsb = 64u + (uint32_t)(st.slot * 8 * kAtoms), tsa = tsb + 4 * kAtoms;
            const uint64_t db = f4_operand_desc<kCB>(src), da = f4_operand_desc<kCB>(src + off_b);
            const uint64_t dsb = f4_atom_desc(src + off_sb), dsa = f4_atom_desc(src + off_sa);
            if (elect_one()) {
#pragma unroll
                for (int k = 0; k < kAtoms; ++k) {
                    if (k >= atoms) break;
                    f4_copy_atom(tsb + 4 * k, dsb + k * (kF4Atom >> 4));
                    f4_copy_atom(tsa + 4 * k, dsa + k * (kF4Atom >> 4));
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    if (k >= steps) break;
                    const int at = kNv ? k : k >> 1;
                    f4_mma<kNv>(tmem, db + 2 * k, da + 2 * k, f4_idesc<kNv>(p.bn, kNv ? 0 : k & 1), tsb + 4 * at,
                                tsa + 4 * at, (c > c0 || k) ? 1u : 0u);
                }
                mma_commit(empty(st.slot));
                if (c == c1 - 1) mma_commit(accf);
            }
            __syncwarp();
            st.next(kXStages);
        }
        // the products must finish before the accumulator is freed
        mbar_wait<false>(accf, 0, nullptr);
        __syncwarp();
    }
    // every copy has landed and every product is done: the ring's memory takes the sums
    if (warp < 4) {
        ok = __all_sync(0xFFFFFFFFu, mbar_wait_fast(accf, 0, abort));
        if (!ok && lane == 0) {
            if (!*abort) atomicExch(p.err, 3);
            *abort = 1;
        }
    }
    __syncwarp();
    __syncthreads();
    float* sums = (float*)(sm + kPBars);  // [row of a][128]
    if (warp < 4) {
        tc_fence_after();
#pragma unroll
        for (int h = 0; h < kXRows / 32; ++h) {
            if (32 * h >= p.bn) break;
            uint32_t r[32];
            tmem_ld32_issue(tmem + ((uint32_t)(32 * warp) << 16) + 32 * h, r);
            tmem_wait();
            tmem_pin32(r);
#pragma unroll
            for (int e = 0; e < 32; ++e) sums[(32 * h + e) * 128 + 32 * warp + lane] = __uint_as_float(r[e]);
        }
        tc_fence_before();
    }
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    {
        const F4Alpha alpha = f4_alpha(p.a.gs, p.b.gs);
        T* out = (T*)p.out;
        const uint32_t mine = smem_u32(sums);
        // four outputs at a time, all their parts on the way before the first is added
        const int step = p.split * kXThreads, n = p.a.rows * 128;
        for (int t0 = part * kXThreads + threadIdx.x; t0 < n; t0 += 4 * step) {
            float x[4][8];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int t = min(t0 + e * step, n - 1);
#pragma unroll
                for (int s = 0; s < 8; ++s) {
                    x[e][s] = 0.0f;
                    if (s < p.split) {
                        uint32_t at;
                        asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(mine + 4u * (uint32_t)t), "r"(s));
                        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x[e][s]) : "r"(at) : "memory");
                    }
                }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int t = t0 + e * step;
                const long long j = (long long)jt * 128 + (t & 127);
                if (t >= n || j >= p.b.rows) continue;
                float v = 0.0f;
#pragma unroll
                for (int s = 0; s < 8; ++s) v += x[e][s];
                out[(long long)(t >> 7) * p.ld + j] = from_f32<T>(v * alpha.lead * alpha.rest);
            }
        }
    }
    __syncwarp();
    // no block leaves while another reads its sums
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (warp == 5) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(*tmem_slot), "r"(512)
                     : "memory");
    }
}

template <int kNv, class T>
cudaError_t launch_split(const CUtensorMap& ta, const CUtensorMap& tb, const F4ProductArgs& p, cudaStream_t st) {
    constexpr int kAtoms = kNv ? 4 : 2;
    const int smem = 1024 + kPBars + kXStages * ((128 + kXRows) * 128 + 2 * kAtoms * kF4Atom);
    auto f = k_f4_product_split<kNv, T>;
    cudaError_t e = cudaFuncSetAttribute((const void*)f, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(p.njt * p.split));
    cfg.blockDim = dim3((unsigned)kXThreads);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)p.split;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, f, ta, tb, p);
}

template <int kNv, int kCB, class T>
cudaError_t launch(const CUtensorMap& ta, const CUtensorMap& tb, const F4ProductArgs& p, int grid, cudaStream_t st) {
    const int smem = 1024 + kPBars + p.nstage * p.stage_bytes;
    auto f = k_f4_product<kNv, kCB, T>;
    cudaError_t e = cudaFuncSetAttribute((const void*)f, cudaFuncAttributeMaxDynamicSharedMemorySize, kPSmem);
    if (e != cudaSuccess) return e;
    f<<<grid, kPThreads, smem, st>>>(ta, tb, p);
    return cudaGetLastError();
}

template <int kNv>
cudaError_t launch_split_t(const CUtensorMap& ta, const CUtensorMap& tb, const F4ProductArgs& p, cudaStream_t st) {
    if (p.dtype == RFX_F32) return launch_split<kNv, float>(ta, tb, p, st);
    if (p.dtype == RFX_BF16) return launch_split<kNv, __nv_bfloat16>(ta, tb, p, st);
    return launch_split<kNv, __half>(ta, tb, p, st);
}

template <int kNv, int kCB>
cudaError_t launch_rows_t(const CUtensorMap& ta, const CUtensorMap& tb, const F4ProductArgs& p, int grid, cudaStream_t st) {
    if (p.dtype == RFX_F32) return launch_rows<kNv, kCB, float>(ta, tb, p, grid, st);
    if (p.dtype == RFX_BF16) return launch_rows<kNv, kCB, __nv_bfloat16>(ta, tb, p, grid, st);
    return launch_rows<kNv, kCB, __half>(ta, tb, p, grid, st);
}

template <int kNv, int kCB>
cudaError_t launch_t(const CUtensorMap& ta, const CUtensorMap& tb, const F4ProductArgs& p, int grid, cudaStream_t st) {
    if (p.dtype == RFX_F32) return launch<kNv, kCB, float>(ta, tb, p, grid, st);
    if (p.dtype == RFX_BF16) return launch<kNv, kCB, __nv_bfloat16>(ta, tb, p, grid, st);
    return launch<kNv, kCB, __half>(ta, tb, p, grid, st);
}

}  // namespace

cudaError_t f4_product(const F4& a, const F4& b, void* out, int dtype, long long ld, int* err, int sms,
                       cudaStream_t st, int* launches) {
    F4ProductArgs p;
    p.a = a;
    p.b = b;
    p.out = out;
    p.ld = ld;
    p.dtype = dtype;
    p.err = err;
    // Up to 512 columns the stores bound a tile, and tiles of 128 rows overlap them better (two
    // accumulators); beyond, the products do, and tiles of 256 rows read b half as often.  1,024 x
    // 40,000 fp32 outputs, 128 against 256 rows: 64 columns 33.5 / 38.9 us, 512 36.9 / 38.9,
    // 1,024 48.2 / 44.9, 4,096 143 / 105.
    p.bn = std::min(b.Kp <= 512 ? 128 : 256, (a.rows + 15) / 16 * 16);
    p.nit = (int)(((long long)a.rows + p.bn - 1) / p.bn);
    p.njt = b.tiles();
    const int cb = b.Kp == 64 ? 32 : 128;
    // few rows of few columns stream b; both ways give the same sums (the steps' order is the same)
    if (a.rows <= 32 && b.Kp <= 256) {
        p.bn = a.rows <= 8 ? 8 : a.rows <= 16 ? 16 : 32;
        CUtensorMap ta, tb;
        if (!f4_map(&ta, a, p.bn, cb) || !f4_map(&tb, b, 256, cb)) return cudaErrorInvalidValue;
        const int grid = std::min((p.njt + kSGroup - 1) / kSGroup, sms);
        *launches += 1;
        if (cb == 32) return b.nv ? launch_rows_t<1, 32>(ta, tb, p, grid, st) : launch_rows_t<0, 32>(ta, tb, p, grid, st);
        return b.nv ? launch_rows_t<1, 128>(ta, tb, p, grid, st) : launch_rows_t<0, 128>(ta, tb, p, grid, st);
    }
    p.nchunk = (b.Kp + 2 * cb - 1) / (2 * cb);
    // at most half the SMs' tiles, and at least four chunks (1,024 columns) for every block of a cluster
    const int most = std::min(std::min(8, sms / p.njt), p.nchunk / 4);
    p.split = most >= 8 ? 8 : most >= 4 ? 4 : most >= 2 ? 2 : 1;
    if (a.rows <= kXRows && p.split >= 2) {
        CUtensorMap ta, tb;
        if (!f4_map(&ta, a, p.bn, cb) || !f4_map(&tb, b, 128, cb)) return cudaErrorInvalidValue;
        *launches += 1;
        return b.nv ? launch_split_t<1>(ta, tb, p, st) : launch_split_t<0>(ta, tb, p, st);
    }
    const int atoms = cb == 32 ? 1 : (b.nv ? 4 : 2);
    const int nrt = p.bn > kF4Tile ? 2 : 1;
    p.stage_bytes = ((128 * cb + (p.bn * cb + 1023) / 1024 * 1024 + atoms * kF4Atom * (1 + nrt)) + 1023) / 1024 * 1024;
    const int sfc = 4 * atoms * (1 + nrt);
    p.nstage = std::min(std::min(kPMaxStage, 256 / sfc), (kPSmem - 1024 - kPBars) / p.stage_bytes);
    p.acc_cols = 32;
    while (p.acc_cols < p.bn) p.acc_cols *= 2;
    p.nacc = 256 / p.acc_cols;
    const long long ntiles = (long long)p.nit * p.njt;
    p.ntiles = (int)ntiles;
    // a tile of few rows takes less than a request for the next one: several to a unit, eight units
    // a block; else single tiles, which balance best
    p.group = p.bn > 64 ? 1 : (int)std::max(1ll, std::min(8ll, ntiles / (8ll * sms)));
    const int grid = (p.ntiles + p.group - 1) / p.group;
    CUtensorMap ta, tb;
    if (!f4_map(&ta, a, p.bn, cb) || !f4_map(&tb, b, 128, cb)) return cudaErrorInvalidValue;
    *launches += 1;
    if (cb == 32) return b.nv ? launch_t<1, 32>(ta, tb, p, grid, st) : launch_t<0, 32>(ta, tb, p, grid, st);
    return b.nv ? launch_t<1, 128>(ta, tb, p, grid, st) : launch_t<0, 128>(ta, tb, p, grid, st);
}

}  // namespace rfx
