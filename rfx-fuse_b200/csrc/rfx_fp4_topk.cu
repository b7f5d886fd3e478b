// The k nearest rows under the product of two 4-bit matrices, without the product.
//
// The answer is exact: the value of a pair is the sum over its blocks, in order, of scale times
// scale times the blocks' integer dot product, in 64 bits (for nvfp4 that sum has no rounding at
// all), and rows rank by (value descending, index ascending).  The tensor cores only decide which
// pairs are worth that evaluation: an fp32 accumulator lies within err = kEps |a_i| |b_j| of the
// value (Cauchy-Schwarz bounds the sum of the terms' magnitudes; the largest error measured is 2^-22.4
// of it, for 130 x 3,000 rows of 256 columns in nvfp4 among rows of 16 to 256 columns in both formats,
// with scales over 3 and over up to 61 binades and with sums that cancel; kEps = 2^-15 leaves a factor
// of 2^7, and a test holds the accumulators to it).  The norms' bounds come with the matrices, one for
// 128 rows.
//
//   k_f4_keys  products of 128 rows of a with b's tiles of 128 rows (tcgen05, block-scaled); of
//              every row's 32 neighbouring accumulators only the maximum is kept, as the upper 16
//              bits of its order-preserving integer (rounded down).
//   k_f4_pick  a block per row of a (k_f4_pick_warp: a warp, for many rows with few keys).  The
//              keys are dealt to groups; the k-th largest of the groups' largest keys, L, is a lower
//              bound of the k-th largest accumulator: k columns have L or more, so the k-th value is
//              at least L - err, and a column of the answer has an accumulator of at least L - 2 err.  Of the chunks whose key reaches that
//              (about k, 1.2 k where groups are few) every column is estimated in fp32; what
//              reaches L - 2 err is evaluated exactly and ranked by counting who is better.
//
// What the first kernel leaves is 2 bytes for 32 pairs.  Rows are taken in batches of 256 MB of keys
// (4,096 x 1,000,000 in one; when that took 441 us, batches of 120 MB took 490: each ends with idle SMs).
// k_f4_keys: 300 cycles a tile of 128 x 128, of which the ALU's 128 for maxima (a 3-input maximum
// takes two issue slots) and 90 for keys and bookkeeping; k_f4_pick: two thirds of the issue slots,
// latency of its barriers and loads between them.  Alone and cold at 4,096 x 1,000,000 they take 305
// and 141 us, together 417.
// err is one number for a batch, from its largest bound of a tile of a times its largest of a tile of b:
// rows of very different norms keep the answer and lose the filter (one row of b of 10 times the
// others' norm: 421 us; of 100 times: 38 ms; of 1,000: 231 ms).
#include <algorithm>

#include "rfx_fp4_mma.cuh"

namespace rfx {

namespace {

constexpr int kKThreads = 448;
constexpr int kSpan = 6;                     // tiles of b in a unit of work: two for each of three groups of warps
constexpr int kSpanKeys = 4 * kSpan;         // keys of a row and a span
constexpr float kEps = 1.0f / 32768.0f;
constexpr uint32_t kAlways = 0xFFFFu;        // key of a chunk that has to be looked at (no float's)
constexpr int kWarpKeys = 1024;              // keys of a row that a warp can hold

struct KeysArgs {
    F4 a, b;
    int q0;               // first row tile of a in this batch
    int nq;               // row tiles of a in it
    int ntiles, nspan;    // tiles of b, and spans of them
    uint32_t* keys;       // [rows of the batch][nspan][12] pairs of keys
    float* errs;          // [grid] largest err of a block's tiles; negative: some tiles have none
    int* err;
};

struct PickArgs {
    F4 a, b;
    int row0;             // first row of the batch
    int k;
    long long self;       // row of b that is row 0 of a and left out for it (and so on); -1: none
    int nspan;
    const uint32_t* keys;
    const float* errs;
    int nerrs;
    int* idx;             // [rows of a][k]
    float* val;
};

// Order-preserving integer of a float, its upper 16 bits; the lowest float of a key.
__device__ __forceinline__ uint32_t key_of(float v) {
    const uint32_t b = __float_as_uint(v);
    return ((b & 0x80000000u) ? ~b : b | 0x80000000u) >> 16;
}
__device__ __forceinline__ float key_floor(uint32_t key) {
    const uint32_t u = key << 16;
    return __uint_as_float((u & 0x80000000u) ? u & 0x7FFFFFFFu : ~u);
}

// The ring of b's tiles, two to a stage; TMEM has room for three stages' scales at 128 bytes a row.
constexpr int kAccs = 3;
constexpr int keys_stages(int cb) { return cb == 32 ? 8 : 3; }
constexpr int keys_stage(int nv, int cb) {
    return (2 * (128 * cb + (cb == 32 ? 1 : nv ? 4 : 2) * kF4Atom) + 1023) / 1024 * 1024;
}

// A CTA takes the units [u0, u1) of (row tile of a, span of b), b fastest.
//   warps 0-11 quarter warp & 3 of the rows, every third tile, always of the same accumulator;
//   warp 12    loads the row tile of a into one of two slots, b's tiles into a ring;
//   warp 13    allocates TMEM, copies scales to TMEM and multiplies into three
//              accumulators of 128 columns.
// Every wait is bounded; on expiry the CTA records it in *err, drains its copies, frees TMEM and
// returns.
template <int kNv, int kCB>
__global__ void __launch_bounds__(kKThreads, 1)
k_f4_keys(const __grid_constant__ CUtensorMap tma, const __grid_constant__ CUtensorMap tmb, KeysArgs p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* sm = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    constexpr int kAtoms = kCB == 32 ? 1 : (kNv ? 4 : 2);
    constexpr int kBox = 128 * kCB;
    constexpr int kSlot = kBox + 2048;
    constexpr int kStages = keys_stages(kCB), kStage = keys_stage(kNv, kCB);  // two tiles of b each
    uint64_t* bars = (uint64_t*)sm;
    // full[16], empty[16], acc_full[3], acc_empty[3], a_full[2], a_empty[2]
    uint32_t* tmem_slot = (uint32_t*)(bars + 42);
    volatile int* abort = (volatile int*)(tmem_slot + 1);
    const uint32_t bar0 = smem_u32(bars);
    auto full = [&](int s) { return bar0 + 8u * s; };
    auto empty = [&](int s) { return bar0 + 8u * (16 + s); };
    auto accf = [&](int b) { return bar0 + 8u * (32 + b); };
    auto acce = [&](int b) { return bar0 + 8u * (35 + b); };
    auto afull = [&](int b) { return bar0 + 8u * (38 + b); };
    auto aempty = [&](int b) { return bar0 + 8u * (40 + b); };
    const uint32_t slot0 = bar0 + 1024u;
    const uint32_t ring0 = slot0 + 2 * kSlot;

    const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const long long units = (long long)p.nq * p.nspan;
    const long long u0 = units * blockIdx.x / gridDim.x;
    const int nu = (int)(units * (blockIdx.x + 1) / gridDim.x - u0);

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(full(s), 1);
            mbar_init(empty(s), 1);
        }
        for (int b = 0; b < kAccs; ++b) {
            mbar_init(accf(b), 1);
            mbar_init(acce(b), 4);  // one arrival a warp
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(afull(b), 1);
            mbar_init(aempty(b), 1);
        }
        *abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 13) {
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
    let_next_start();  // k_f4_pick's blocks take the places of the blocks that end

    if (warp == 12) {
        const uint32_t sfb = (uint32_t)(atoms * kF4Atom);
        int n = 0, na = 0;
        RingPos st, sl;
        bool ok = true;
        int qt = p.q0 + (int)(u0 / p.nspan), span = (int)(u0 % p.nspan);
        for (int u = 0; ok && u < nu; ++u) {
            if (u == 0 || span == 0) {
                ok = __all_sync(0xFFFFFFFFu, mbar_wait_fast(aempty(sl.slot), sl.parity ^ 1u, abort));
                if (!ok) break;
                if (elect_one()) {
                    const uint32_t dst = slot0 + (uint32_t)(sl.slot * kSlot);
                    mbar_expect_tx(afull(sl.slot), (uint32_t)kBox + sfb);
                    tma_load(dst, &tma, 0, qt * 128, afull(sl.slot));
                    bulk_load(dst + kBox, p.a.scales + (long long)qt * p.a.natoms * kF4Atom, sfb, afull(sl.slot));
                }
                sl.next(2);
                ++na;
            }
            const int te = min(p.ntiles, span * kSpan + kSpan);
            for (int t = span * kSpan; t < te; t += 2, ++n) {
                ok = __all_sync(0xFFFFFFFFu, mbar_wait_fast(empty(st.slot), st.parity ^ 1u, abort));
                if (!ok) break;
                if (elect_one()) {
                    const uint32_t dst = ring0 + (uint32_t)(st.slot * kStage);
                    const uint32_t sc = t + 1 < te ? 2 * sfb : sfb;  // two tiles' scales follow one another
                    mbar_expect_tx(full(st.slot), 2u * kBox + sc);
                    tma_load(dst, &tmb, 0, t * 128, full(st.slot));
                    bulk_load(dst + 2 * kBox, p.b.scales + (long long)t * p.b.natoms * kF4Atom, sc, full(st.slot));
                }
                st.next(kStages);
            }
            if (++span == p.nspan) {
                span = 0;
                ++qt;
            }
        }
        if (!ok && lane == 0) {
            if (!*abort) atomicExch(p.err, 1);
            *abort = 1;
        }
        // drain this warp's copies still in flight
        for (int i = na > 2 ? na - 2 : 0; i < na; ++i) mbar_wait<false>(afull(i & 1), (uint32_t)(i >> 1) & 1u, nullptr);
        for (int i = n > kStages ? n - kStages : 0; i < n; ++i)
            mbar_wait<false>(full(i % kStages), (uint32_t)(i / kStages) & 1u, nullptr);
        __syncwarp();
    } else if (warp == 13) {
        RingPos st, sl;
        uint32_t uses = 0;  // a parity bit for every accumulator
        int last = -1;
        uint32_t tsa = 0;
        uint64_t da = 0;
        int span = (int)(u0 % p.nspan);
        for (int u = 0; u < nu; ++u) {
            if (u == 0 || span == 0) {
                mbar_wait_issue(afull(sl.slot), sl.parity, abort, p.err, 2);
                tc_fence_after();
                const uint32_t src = slot0 + (uint32_t)(sl.slot * kSlot);
                tsa = 384u + (uint32_t)(4 * kAtoms * sl.slot);
                if (elect_one())
                    for (int k0 = 0; k0 < atoms; ++k0) f4_copy_atom(tsa + 4 * k0, f4_atom_desc(src + kBox + k0 * kF4Atom));
                da = f4_operand_desc<kCB>(src);
            }
            const int nt = min(kSpan, p.ntiles - span * kSpan);
#pragma unroll
            for (int t = 0; t < kSpan; t += 2) {
                if (t >= nt) break;
                mbar_wait_issue(full(st.slot), st.parity, abort, p.err, 2);
                const uint32_t src = ring0 + (uint32_t)(st.slot * kStage);
                const uint32_t tsb = 384u + (uint32_t)(8 * kAtoms * (1 + st.slot));
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if (t + h >= nt) break;
                    const int ac = (t + h) % kAccs;
                    mbar_wait_issue(acce(ac), ((uses >> ac) & 1u) ^ 1u, abort, p.err, 2);
                    tc_fence_after();
                    if (elect_one()) {
                        const uint32_t tsh = tsb + 4 * kAtoms * h;
                        const uint64_t dsc = f4_atom_desc(src + 2 * kBox + h * atoms * kF4Atom);
                        const uint64_t db = f4_operand_desc<kCB>(src + h * kBox);
                        const uint32_t d = (uint32_t)(128 * ac);
                        if (kCB == 32) {
                            f4_copy_atom(tsh, dsc);
                            f4_mma<kNv>(d, da, db, f4_idesc<kNv>(128, 0), tsa, tsh, 0u);
                        } else {
                            for (int k0 = 0; k0 < atoms; ++k0) f4_copy_atom(tsh + 4 * k0, dsc + k0 * (kF4Atom >> 4));
                            for (int k0 = 0; k0 < steps; ++k0) {
                                const int at = kNv ? k0 : k0 >> 1;
                                f4_mma<kNv>(d, da + 2 * k0, db + 2 * k0, f4_idesc<kNv>(128, kNv ? 0 : k0 & 1),
                                            tsa + 4 * at, tsh + 4 * at, k0 ? 1u : 0u);
                            }
                        }
                        mma_commit(accf(ac));
                        if (h == 1 || t + 1 >= nt) mma_commit(empty(st.slot));
                    }
                    __syncwarp();
                    last = ac;
                    uses ^= 1u << ac;
                }
                st.next(kStages);
            }
            if (++span == p.nspan) span = 0;
            if (span == 0 || u == nu - 1) {
                if (elect_one()) mma_commit(aempty(sl.slot));
                __syncwarp();
                sl.next(2);
            }
        }
        // the last products must finish before the accumulators are freed
        if (last >= 0) mbar_wait<false>(accf(last), ((uses >> last) & 1u) ^ 1u, nullptr);
        __syncwarp();
    } else {
        const int quarter = warp & 3, phase = warp >> 2;
        const uint32_t lane_addr = tmem + ((uint32_t)(32 * quarter) << 16) + (uint32_t)(128 * phase);
        const float kNegInf = -__int_as_float(0x7f800000);
        float worst = 0.0f;  // largest bound of this block's tiles that the filter can use
        bool some_forced = false;
        uint32_t parity = 0;
        bool ok = true;
        int qt = p.q0 + (int)(u0 / p.nspan), span = (int)(u0 % p.nspan);
        float bd = lane < min(kSpan, p.ntiles - span * kSpan) ? __ldg(p.b.bounds + span * kSpan + lane) : 0.0f;
        float bq = nu > 0 ? __ldg(p.a.bounds + qt) : 0.0f;
        for (int u = 0; ok && u < nu; ++u) {
            const long long row = (long long)qt * 128 + 32 * quarter + lane;
            const bool any = (long long)qt * 128 + 32 * quarter < p.a.rows;  // of this warp's rows
            const int nt = min(kSpan, p.ntiles - span * kSpan);
            // a sum of such terms can overflow fp32 and lose its sign: those tiles are looked at
            const uint32_t forced = __ballot_sync(0xFFFFFFFFu, !(bq * bd * kEps < 1e30f));
            if (forced) some_forced = true;
            if (!((forced >> lane) & 1u)) worst = fmaxf(worst, bq * bd * (kEps * 1.000001f));
            const int ncols = min(kSpan * 128, p.b.rows - span * kSpan * 128);  // columns that exist
            const bool plain = forced == 0 && ncols == kSpan * 128;
            uint32_t* out = p.keys + ((row - (long long)p.q0 * 128) * p.nspan + span) * (kSpanKeys / 2) + 4 * phase;
            // the next unit's bounds, under this one's work
            int span1 = span + 1, qt1 = qt;
            if (span1 == p.nspan) {
                span1 = 0;
                ++qt1;
            }
            if (u + 1 < nu) {
                bd = lane < min(kSpan, p.ntiles - span1 * kSpan) ? __ldg(p.b.bounds + span1 * kSpan + lane) : 0.0f;
                bq = __ldg(p.a.bounds + qt1);
            }
            uint32_t keys[4] = {0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < kSpan / kAccs; ++i) {
                const int t = kAccs * i + phase;
                if (t >= nt || !ok) continue;
                const bool got = mbar_wait_fast(accf(phase), parity, abort);
                parity ^= 1u;
                if (!__all_sync(0xFFFFFFFFu, got)) {
                    ok = false;
                    continue;
                }
                if (any) {
                    // 32 columns are read while the maximum of the 32 before is taken
                    uint32_t r[2][32];
                    float top[4];
                    tc_fence_after();
                    tmem_ld32_issue(lane_addr, r[0]);
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        tmem_wait();
                        tmem_pin32(r[c & 1]);
                        if (c < 3) {
                            tmem_ld32_issue(lane_addr + 32 * (c + 1), r[(c + 1) & 1]);
                        } else {
                            tc_fence_before();
                            __syncwarp();
                            if (lane == 0) mbar_arrive(acce(phase));
                        }
                        uint32_t* x = r[c & 1];
                        if (!plain) {
                            const int ncol = ncols - 128 * t - 32 * c;
#pragma unroll
                            for (int e = 0; e < 32; ++e)
                                if (e >= ncol) x[e] = __float_as_uint(kNegInf);
                        }
                        float m[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) m[e] = __uint_as_float(x[e]);
#pragma unroll
                        for (int e = 4; e < 28; e += 8) {
#pragma unroll
                            for (int f = 0; f < 4; ++f)
                                m[f] = fmax3(m[f], __uint_as_float(x[e + 2 * f]), __uint_as_float(x[e + 2 * f + 1]));
                        }
                        m[0] = fmax3(m[0], __uint_as_float(x[28]), __uint_as_float(x[29]));
                        m[1] = fmax3(m[1], __uint_as_float(x[30]), __uint_as_float(x[31]));
                        // NaN alone becomes -inf: nobody's neighbours
                        top[c] = fmax3(fmax3(m[0], m[1], m[2]), m[3], kNegInf);
                    }
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        // key_of both: the upper halves, all bits flipped under a sign, else the sign
                        uint32_t pair = __byte_perm(__float_as_uint(top[2 * c]), __float_as_uint(top[2 * c + 1]), 0x7632);
                        uint32_t neg;
                        asm("prmt.b32 %0, %1, %2, %3;" : "=r"(neg) : "r"(pair), "r"(0u), "r"(0xBB99u));
                        pair ^= neg | 0x80008000u;
                        if (!plain) {
                            const int ncol = ncols - 128 * t - 64 * c;
                            if ((forced >> t) & 1u) pair = kAlways << 16 | kAlways;
                            if (ncol <= 32) pair &= 0xFFFFu;
                            if (ncol <= 0) pair = 0;
                        }
                        keys[2 * i + c] = pair;
                    }
                } else if (lane == 0) {
                    mbar_arrive(acce(phase));
                }
            }
            if (ok && row < p.a.rows) *reinterpret_cast<uint4*>(out) = make_uint4(keys[0], keys[1], keys[2], keys[3]);
            span = span1;
            qt = qt1;
        }
        if (!ok && lane == 0) {
            if (!*abort) atomicExch(p.err, 3);
            *abort = 1;
        }
        if (warp == 0) {
            for (int o = 16; o; o >>= 1) worst = fmaxf(worst, __shfl_xor_sync(0xFFFFFFFFu, worst, o));
            if (lane == 0) p.errs[blockIdx.x] = some_forced ? -fmaxf(worst, 1e-37f) : worst;
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 13) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(*tmem_slot), "r"(512)
                     : "memory");
    }
}

__device__ __forceinline__ bool f4_better(double va, int ja, double vb, int jb) {
    return va > vb || (va == vb && ja < jb);
}

// Four times the exact value of the row (decoded in qa, scales in sa) with a row of b (codes cb,
// first scale sb), without the matrix scales; NaN when a scale is.
template <int kNv>
__device__ __noinline__ double f4_exact(const int* qa, const float* sa, const uint4* cb, const uint8_t* sb, int steps) {
    double v = 0.0;
    for (int c = 0; c < steps; ++c) {
        uint32_t wb = __ldg(reinterpret_cast<const uint32_t*>(sb + (kNv ? c : c >> 1) * kF4Atom));
        if (!kNv && (c & 1)) wb >>= 16;
#pragma unroll
        for (int h = 0; h < 2; ++h) {  // 32 columns
            const uint4 y = __ldg(cb + 2 * c + h);
            const int4* q = reinterpret_cast<const int4*>(qa + 16 * c + 8 * h);
            const int lo = e2m1_dot16(q[0], y.x, y.y, 0), hi = e2m1_dot16(q[1], y.z, y.w, 0);
            if (kNv) {
                // e4m3 times e4m3 times the integer: exact, and so is every sum
                v += (double)sa[4 * c + 2 * h] * (double)e4m3_value((wb >> (16 * h)) & 0xFFu) * (double)lo;
                v += (double)sa[4 * c + 2 * h + 1] * (double)e4m3_value((wb >> (16 * h + 8)) & 0xFFu) * (double)hi;
            } else {
                const uint32_t eb = (wb >> (8 * h)) & 0xFFu;
                const double s = eb == 255u ? __longlong_as_double(0x7ff8000000000000ll)
                                            : __longlong_as_double((long long)(eb + 896u) << 52);  // 2^(eb - 127)
                v += (double)sa[2 * c + h] * s * (double)(lo + hi);
            }
        }
    }
    return v;
}

// 64 columns of the same (four times the value) in fp32, added to v: within the accumulators' own bound (at most 16 blocks,
// a few units of 2^-24 of the terms' sum), so that the same err covers it.
template <int kNv>
__device__ __forceinline__ float f4_estimate64(const int* qa, const float* sa, uint4 y0, uint4 y1, uint32_t wb, float v) {
    // an integer dot product added to the bits of 1.5 * 2^23 is a float, less 1.5 * 2^23
    constexpr int kMagic = 0x4B400000;
    constexpr float kMagicF = 12582912.0f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const uint4 y = h ? y1 : y0;
        const int4* q = reinterpret_cast<const int4*>(qa + 8 * h);
        if (kNv) {
            const float2 sb = e4m3_pair(wb >> (16 * h));
            v = fmaf(sa[2 * h] * sb.x, __int_as_float(e2m1_dot16(q[0], y.x, y.y, kMagic)) - kMagicF, v);
            v = fmaf(sa[2 * h + 1] * sb.y, __int_as_float(e2m1_dot16(q[1], y.z, y.w, kMagic)) - kMagicF, v);
        } else {
            const int dot = e2m1_dot16(q[1], y.z, y.w, e2m1_dot16(q[0], y.x, y.y, kMagic));
            v = fmaf(sa[h] * e8m0_value((wb >> (8 * h)) & 0xFFu), __int_as_float(dot) - kMagicF, v);
        }
    }
    return v;
}

// Every product is NaN.
__device__ __forceinline__ bool nan_scale(const F4& a, const F4& b) {
    const float x = __ldg(a.gs), y = __ldg(b.gs);
    return !(x == x && y == y);
}

// kT threads a row: 128, eight rows an SM, which hide one another's waits for memory and barriers
// (both kernels at 4,096 x 1,000,000, top 50: 417 us, 439 with 256 threads; 100,000 rows: 131, 150); 1024
// when there are too few rows to fill the GPU.  128 threads are held to 64 registers and spill 84 bytes
// (nvfp4) or 60 (mxfp4).
template <int kNv, int kT>
__global__ void __launch_bounds__(kT, kT == 1024 ? 1 : 1024 / kT)
k_f4_pick(PickArgs p) {
    constexpr int kUnits = kT == 128 ? 2048 : 4096;  // units of keys: a key, or every kUnits-th vector of 8
    constexpr int kFound = kT == 128 ? 512 : 1024;         // columns waiting to be ranked
    constexpr int kScan = kT == 128 ? 128 : 256;           // units a round turns into chunks
    constexpr int kList = 8 * kScan + 256;  // chunks waiting to be looked at
    __shared__ __align__(16) int qa[kF4TopkK / 4];
    __shared__ float sa[kF4TopkK / 16];
    __shared__ double fv[kFound];       // found: values (4 x) of the first n_known, columns of all
    __shared__ int fj[kFound];
    __shared__ uint32_t list[kList];    // chunks to look at
    __shared__ __align__(16) uint16_t tops[kUnits];  // a unit's largest key
    __shared__ uint16_t ulist[kUnits];  // units to look at
    __shared__ int n_list, n_found, n_units, n_valid;
    __shared__ float s_err;
    __shared__ int s_forced;
    __shared__ uint32_t s_l;
    const double kNegInf = -__longlong_as_double(0x7ff0000000000000ll);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const long long i = (long long)p.row0 + blockIdx.x;
    const int kp = p.self >= 0 ? p.k + 1 : p.k;  // the row itself may be one of the k columns
    const int self = p.self >= 0 ? (int)(p.self + i) : -1;
    const uint4* keys = reinterpret_cast<const uint4*>(p.keys + (long long)blockIdx.x * p.nspan * (kSpanKeys / 2));
    const int nvec = p.nspan * (kSpanKeys / 8);    // 8 keys each
    const uint8_t* b_codes = p.b.codes;
    const uint8_t* b_scales = p.b.scales;
    const int pitch = p.b.pitch(), tile_bytes = p.b.natoms * kF4Atom, steps = p.b.Kp / 64;
    auto codes_of = [=](int j) { return reinterpret_cast<const uint4*>(b_codes + (long long)j * pitch); };
    auto scales_of = [=](int j) {
        return b_scales + (long long)(j >> 7) * tile_bytes + (j & 31) * 16 + ((j >> 5) & 3) * 4;
    };
    const bool small = nvec * 8 <= kUnits;  // a unit is a key
    const int nunits = small ? nvec * 8 : min(nvec, kUnits);

    // the row, decoded, and its scales
    for (int t = tid; t < p.a.Kp / 4; t += kT) {
        const uint32_t w = *reinterpret_cast<const uint16_t*>(p.a.codes + i * p.a.pitch() + 2 * t);
        int d = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) d |= ((int)(2.0f * e2m1_value((w >> (4 * e)) & 15u)) & 0xFF) << (8 * e);
        qa[t] = d;
    }
    float s0 = 0.0f;
    if (tid < p.a.Kp / (kNv ? 16 : 32)) sa[tid] = s0 = f4_scale_value(kNv, p.a.scales[f4_scale_at(p.a, i, tid)]);
    if (tid == 0 && nan_scale(p.a, p.b)) s0 = __int_as_float(0x7fc00000);
    wait_for_previous();  // the keys
    if (__syncthreads_or(!(s0 == s0))) {  // a NaN row is nobody's neighbour and has none
        for (int s = tid; s < p.k; s += kT) {
            p.idx[i * p.k + s] = -1;
            p.val[i * p.k + s] = -__int_as_float(0x7f800000);
        }
        return;
    }
    // the largest key of every unit, four vectors in flight; thread t owns the units t, t + kT, ...
    for (int t0 = tid; t0 < nvec; t0 += 4 * kT) {
        uint4 x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
            x[e] = t0 + e * kT < nvec ? load_left(keys + t0 + e * kT) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int t = t0 + e * kT;
            if (t >= nvec) continue;
            if (small) {
                reinterpret_cast<uint4*>(tops)[t] = x[e];
            } else {
                const uint32_t m = __vmaxu2(__vmaxu2(x[e].x, x[e].y), __vmaxu2(x[e].z, x[e].w));
                uint32_t best = max(m & 0xFFFFu, m >> 16);
                if (t >= kUnits) best = max(best, (uint32_t)tops[t % kUnits]);
                tops[t % kUnits] = (uint16_t)best;
            }
        }
    }
    if (warp == kT / 32 - 1) {
        float e = 0.0f;
        bool f = false;
        for (int t = lane; t < p.nerrs; t += 32) {
            const float x = load_left(p.errs + t);
            f |= x < 0.0f;
            e = fmaxf(e, fabsf(x));
        }
        for (int o = 16; o; o >>= 1) e = fmaxf(e, __shfl_xor_sync(0xFFFFFFFFu, e, o));
        f = __any_sync(0xFFFFFFFFu, f);
        if (lane == 0) {
            s_err = fmaxf(e, 1e-37f);
            s_forced = f;
            n_list = n_found = n_units = 0;
        }
    }
    __syncthreads();
    const bool forced = s_forced != 0;
    // the units are dealt to groups: L is the kp-th largest of the groups' largest keys, by bisection of
    // its 16 bits (0: there are fewer), or a little less, as soon as kp groups have it
    // Fewer chunks than kp bound nothing, and every column would be ranked: then the columns' estimates
    // are the keys (one row against 1,000, top 50: 19 us, 59 without).
    const uint16_t* from = tops;
    int nfrom = nunits;
    if (p.b.rows < 32 * kp && p.b.rows <= 2048 && !forced) {
        for (int j = tid; j < p.b.rows; j += kT) {
            float v = 0.0f;
            for (int st = 0; st < steps; ++st) {
                const uint32_t w = __ldg(reinterpret_cast<const uint32_t*>(scales_of(j) + (kNv ? st : st >> 1) * kF4Atom));
                v = f4_estimate64<kNv>(qa + 16 * st, sa + (kNv ? 4 : 2) * st, __ldg(codes_of(j) + 2 * st),
                                       __ldg(codes_of(j) + 2 * st + 1), !kNv && (st & 1) ? w >> 16 : w, v);
            }
            ulist[j] = j != self && v == v ? (uint16_t)key_of(0.25f * v) : 0;  // (four times the value)
        }
        __syncthreads();
        from = ulist;
        nfrom = p.b.rows;
    }
    uint32_t s_key = 0;
    {
        constexpr int kGroups = 256;  // with 128: an eighth more chunks to look at for 50 neighbours
        constexpr int kTops = kT < kGroups ? kGroups : kT;
        __shared__ __align__(16) uint16_t top[kTops];  // a group: those at its number plus multiples of kGroups
#pragma unroll
        for (int h = 0; h < kTops; h += kT) {
            uint32_t most = 0;
            for (int t = tid + h; t < nfrom; t += kTops) {
                const uint32_t key = from[t];
                if (key != kAlways) most = max(most, key);
            }
            top[tid + h] = (uint16_t)most;
        }
        __syncthreads();
        // four warps find L each for itself, which costs less than a barrier a bit; of 32 one does
        if (kT == 128 || warp == 0) {
            constexpr int kW = kGroups / 64;  // words of two groups a lane
            uint32_t x[kW];
#pragma unroll
            for (int e = 0; e < kW; ++e) {
                x[e] = reinterpret_cast<const uint32_t*>(top)[lane + 32 * e];
#pragma unroll
                for (int h = 1; h < kTops / kGroups; ++h)
                    x[e] = __vmaxu2(x[e], reinterpret_cast<const uint32_t*>(top)[lane + 32 * e + h * (kGroups / 2)]);
            }
            for (uint32_t bit = 0x8000u; bit; bit >>= 1) {
                const uint32_t want = s_key | bit;
                int c = 0;
#pragma unroll
                for (int e = 0; e < kW; ++e) c += ((x[e] & 0xFFFFu) >= want) + (x[e] >= want << 16);
                c = __reduce_add_sync(0xFFFFFFFFu, c);
                if (c >= kp) s_key = want;
                if (c == kp) break;
            }
        }
        if (kT != 128) {
            if (tid == 0) s_l = s_key;
            __syncthreads();
            s_key = s_l;
        }
    }
    const double err = (double)s_err;
    // the k-th value is at least this
    double floor_v = s_key > key_of(-__int_as_float(0x7f800000)) ? (double)key_floor(s_key) - err : kNegInf;
    // an accumulator, or an estimate, of the answer is at least floor - err
    auto bar_of = [&]() { return max(key_of(__double2float_rd(floor_v - err)), 1u); };
    {
        const uint32_t bar = bar_of();
        for (int t = tid; t < nunits; t += kT)
            if (tops[t] >= bar) ulist[atomicAdd(&n_units, 1)] = (uint16_t)t;
    }
    __syncthreads();

    // Evaluates what was found exactly, ranks it, keeps the best k at the front and raises the floor.
    int n_known = 0;
    auto rank_found = [&]() {
        __syncthreads();
        const int n = n_found;
        if (tid == 0) n_valid = 0;
        for (int t = n_known + tid; t < n; t += kT) {
            const double x = f4_exact<kNv>(qa, sa, codes_of(fj[t]), scales_of(fj[t]), steps);
            const bool in = x * 0.25 >= floor_v;  // false for NaN
            fv[t] = in ? x : kNegInf;
            if (!in) fj[t] = 0x7FFFFFFF;
        }
        __syncthreads();
        constexpr int kE = (kFound + kT - 1) / kT;
        double v[kE];
        int j[kE], r[kE];
#pragma unroll
        for (int e = 0; e < kE; ++e) {
            const int t = tid + e * kT;
            r[e] = kFound;
            if (t >= n || fj[t] == 0x7FFFFFFF) continue;
            v[e] = fv[t];
            j[e] = fj[t];
            int c = 0;
            for (int o = 0; o < n; ++o) c += f4_better(fv[o], fj[o], v[e], j[e]);
            r[e] = c;
            if (c < p.k) atomicAdd(&n_valid, 1);
        }
        __syncthreads();
#pragma unroll
        for (int e = 0; e < kE; ++e)
            if (r[e] < p.k) {
                fv[r[e]] = v[e];
                fj[r[e]] = j[e];
            }
        if (tid == 0) n_found = n_valid;
        __syncthreads();
        n_known = n_found;
        if (n_known == p.k) floor_v = fmax(floor_v, 0.25 * fv[p.k - 1]);
        __syncthreads();
    };
    // Looks at the chunks [c0, c1) of the list, a warp a chunk, a lane a column; what overflows is
    // only counted.
    auto look_at = [&](int c0, int c1) {
        const float least = 4.0f * __double2float_rd(floor_v - err);
        // the next chunk's first 64 columns are loaded under this one's arithmetic
        uint4 y0, y1;
        uint32_t sc;
        auto fetch = [&](int c) {
            const int j = min((int)list[c] * 32 + lane, p.b.rows - 1);
            y0 = __ldg(codes_of(j));
            y1 = __ldg(codes_of(j) + 1);
            sc = __ldg(reinterpret_cast<const uint32_t*>(scales_of(j)));
        };
        if (c0 + warp < c1) fetch(c0 + warp);
        for (int c = c0 + warp; c < c1; c += kT / 32) {
            const int j = (int)list[c] * 32 + lane;
            const uint4 z0 = y0, z1 = y1;
            const uint32_t zs = sc;
            if (c + kT / 32 < c1) fetch(c + kT / 32);
            float v = f4_estimate64<kNv>(qa, sa, z0, z1, zs, 0.0f);
            for (int st = 1; st < steps; ++st) {
                const int jc = min(j, p.b.rows - 1);
                const uint32_t w = __ldg(reinterpret_cast<const uint32_t*>(scales_of(jc) + (kNv ? st : st >> 1) * kF4Atom));
                v = f4_estimate64<kNv>(qa + 16 * st, sa + (kNv ? 4 : 2) * st, __ldg(codes_of(jc) + 2 * st),
                                       __ldg(codes_of(jc) + 2 * st + 1), !kNv && (st & 1) ? w >> 16 : w, v);
            }
            // without a bound on the terms fp32 could overflow: rank_found decides
            if (j < p.b.rows && j != self && (forced || v >= least)) {
                const int at = atomicAdd(&n_found, 1);
                if (at < kFound) fj[at] = j;
            }
        }
        __syncthreads();
    };
    // The whole list; where that finds more than there is room for (ties in masses), again from the
    // start, as many chunks at a time as surely have room.
    auto look = [&]() {
        __syncthreads();
        const int n = n_list, before = n_found;
        __syncthreads();  // everyone has read n_found before anyone adds to it
        look_at(0, n);
        if (n_found > kFound) {
            __syncthreads();
            if (tid == 0) n_found = before;
            __syncthreads();
            for (int c0 = 0; c0 < n;) {
                const int c1 = min(n, c0 + (kFound - n_found) / 32);
                __syncthreads();
                look_at(c0, c1);
                c0 = c1;
                rank_found();
            }
        }
        if (tid == 0) n_list = 0;
        __syncthreads();
    };
    // the units' chunks that may hold a column of the answer
    const int per = small ? 1 : (nvec + kUnits - 1) / kUnits;  // vectors of a unit
    const int ntask = n_units * per;
    for (int t0 = 0; t0 < ntask; t0 += kScan) {
        const uint32_t bar = bar_of();
        const int t = t0 + tid;
        if (tid < kScan && t < ntask) {
            const int unit = ulist[t / per];
            const int vec = small ? unit >> 3 : unit + t % per * kUnits;
            if (vec < nvec) {
                // keys 8 vec ..: [span][tile % 3][tile / 3][4 chunks of the tile]
                const int chunk0 = (vec / kAccs * kSpan + vec % kAccs) * 4;
                if (small) {
                    const int e = unit & 7;
                    if (tops[unit] >= bar) list[atomicAdd(&n_list, 1)] = (uint32_t)(chunk0 + 4 * kAccs * (e >> 2) + (e & 3));
                } else {
                    const uint4 x = load_left(keys + vec);
                    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (((w[e >> 1] >> (16 * (e & 1))) & 0xFFFFu) >= bar)
                            list[atomicAdd(&n_list, 1)] = (uint32_t)(chunk0 + 4 * kAccs * (e >> 2) + (e & 3));
                }
            }
        }
        __syncthreads();
        const bool room = n_list <= 256;
        __syncthreads();  // everyone has read n_list before anyone adds to it
        if (!room) look();
    }
    look();
    rank_found();
    const double g = (double)__ldg(p.a.gs) * (double)__ldg(p.b.gs);
    for (int s = tid; s < p.k; s += kT) {
        const bool in = s < n_known;
        p.idx[i * p.k + s] = in ? fj[s] : -1;
        p.val[i * p.k + s] = in ? (float)(fv[s] * 0.25 * g) : -__int_as_float(0x7f800000);
    }
}

// The same for rows with few keys, a warp a row: the keys stay in registers, nothing waits for a
// barrier, and an SM works on 32 rows (10,000 x 10,000, top 10, both kernels: 67 us, 105 with a block of
// 128 threads a row; alone and cold it takes 60, at 0.83 instructions a cycle and scheduler, 4,800 a row,
// half of them estimates).  A group is a word of two keys.
constexpr int kWFound = 128;  // columns waiting to be ranked: 32 more always fit beside the best 64

template <int kNv>
__global__ void __launch_bounds__(128, 8)
k_f4_pick_warp(PickArgs p, int rows) {
    __shared__ __align__(16) int s_qa[4][kF4TopkK / 4];
    __shared__ float s_sa[4][kF4TopkK / 16];
    __shared__ double s_fv[4][kWFound];  // as in k_f4_pick
    __shared__ int s_fj[4][kWFound];
    __shared__ uint16_t s_list[4][kWarpKeys];
    constexpr uint32_t kAll = 0xFFFFFFFFu;
    const double kNegInf = -__longlong_as_double(0x7ff0000000000000ll);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int* qa = s_qa[warp];
    float* sa = s_sa[warp];
    double* fv = s_fv[warp];
    int* fj = s_fj[warp];
    uint16_t* list = s_list[warp];
    const int q = blockIdx.x * 4 + warp;  // row of the batch
    const long long i = (long long)p.row0 + q;
    if (q >= rows) return;
    const int kp = p.self >= 0 ? p.k + 1 : p.k;
    const int self = p.self >= 0 ? (int)(p.self + i) : -1;
    const uint4* keys = reinterpret_cast<const uint4*>(p.keys + (long long)q * p.nspan * (kSpanKeys / 2));
    const int nvec = p.nspan * (kSpanKeys / 8), steps = p.b.Kp / 64;
    auto codes_of = [&](int j) { return reinterpret_cast<const uint4*>(p.b.codes + (long long)j * p.b.pitch()); };
    auto scales_of = [&](int j) {
        return p.b.scales + (long long)(j >> 7) * (p.b.natoms * kF4Atom) + (j & 31) * 16 + ((j >> 5) & 3) * 4;
    };

    for (int t = lane; t < p.a.Kp / 4; t += 32) {
        const uint32_t w = *reinterpret_cast<const uint16_t*>(p.a.codes + i * p.a.pitch() + 2 * t);
        int d = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) d |= ((int)(2.0f * e2m1_value((w >> (4 * e)) & 15u)) & 0xFF) << (8 * e);
        qa[t] = d;
    }
    float s0 = 0.0f;
    if (lane < p.a.Kp / (kNv ? 16 : 32)) sa[lane] = s0 = f4_scale_value(kNv, p.a.scales[f4_scale_at(p.a, i, lane)]);
    if (lane == 0 && nan_scale(p.a, p.b)) s0 = __int_as_float(0x7fc00000);
    wait_for_previous();  // the keys
    int n_known = 0, n_found = 0;
    if (!__any_sync(kAll, !(s0 == s0))) {  // a NaN row is nobody's neighbour and has none
        uint32_t x[16];  // words of two keys
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint4 y = lane + 32 * e < nvec ? load_left(keys + lane + 32 * e) : make_uint4(0, 0, 0, 0);
            x[4 * e] = y.x;
            x[4 * e + 1] = y.y;
            x[4 * e + 2] = y.z;
            x[4 * e + 3] = y.w;
        }
        float worst = 0.0f;
        bool forced = false;
        for (int t = lane; t < p.nerrs; t += 32) {
            const float y = load_left(p.errs + t);
            forced |= y < 0.0f;
            worst = fmaxf(worst, fabsf(y));
        }
        for (int o = 16; o; o >>= 1) worst = fmaxf(worst, __shfl_xor_sync(kAll, worst, o));
        forced = __any_sync(kAll, forced);
        const double err = (double)fmaxf(worst, 1e-37f);
        // L: the kp-th largest of the words' larger keys, by bisection as in k_f4_pick
        uint32_t s_key = 0;
        {
            uint32_t top[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const uint32_t lo = x[e] & 0xFFFFu, hi = x[e] >> 16;
                top[e] = max(lo == kAlways ? 0u : lo, hi == kAlways ? 0u : hi);
            }
            for (uint32_t bit = 0x8000u; bit; bit >>= 1) {
                int c = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (32 * e < nvec) {
#pragma unroll
                        for (int h = 0; h < 4; ++h) c += top[4 * e + h] >= (s_key | bit);
                    }
                }
                c = __reduce_add_sync(kAll, c);
                if (c >= kp) s_key |= bit;
                if (c == kp) break;
            }
        }
        double floor_v = s_key > key_of(-__int_as_float(0x7f800000)) ? (double)key_floor(s_key) - err : kNegInf;
        int n_list = 0;
        {
            const uint32_t bar = max(key_of(__double2float_rd(floor_v - err)), 1u);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (32 * e < nvec) {
                    const int vec = lane + 32 * e;
                    const int chunk0 = (vec / kAccs * kSpan + vec % kAccs) * 4;  // as in k_f4_pick
#pragma unroll
                    for (int h = 0; h < 8; ++h) {
                        const bool in = (h & 1 ? x[4 * e + h / 2] >> 16 : x[4 * e + h / 2] & 0xFFFFu) >= bar;
                        const uint32_t who = __ballot_sync(kAll, in);
                        if (in) list[n_list + __popc(who & ((1u << lane) - 1))] = (uint16_t)(chunk0 + 4 * kAccs * (h >> 2) + (h & 3));
                        n_list += __popc(who);
                    }
                }
            }
        }
        __syncwarp();
        float least = 4.0f * __double2float_rd(floor_v - err);  // of an estimate
        // Evaluates what was found exactly, ranks it, keeps the best k at the front, raises the floor.
        auto rank_found = [&]() {
            __syncwarp();
            for (int t = n_known + lane; t < n_found; t += 32) {
                const double y = f4_exact<kNv>(qa, sa, codes_of(fj[t]), scales_of(fj[t]), steps);
                const bool in = y * 0.25 >= floor_v;  // false for NaN
                fv[t] = in ? y : kNegInf;
                if (!in) fj[t] = 0x7FFFFFFF;
            }
            __syncwarp();
            double v[kWFound / 32];
            int j[kWFound / 32], r[kWFound / 32], kept = 0;
#pragma unroll
            for (int e = 0; e < kWFound / 32; ++e) {
                const int t = lane + 32 * e;
                v[e] = t < n_found ? fv[t] : kNegInf;
                j[e] = t < n_found ? fj[t] : 0x7FFFFFFF;
                r[e] = 0;
            }
#pragma unroll
            for (int e = 0; e < kWFound / 32; ++e) {
                if (32 * e < n_found) {
                    int c = 0;
#pragma unroll 4
                    for (int o = 0; o < n_found; ++o) c += f4_better(fv[o], fj[o], v[e], j[e]);
                    r[e] = c;
                }
                if (j[e] == 0x7FFFFFFF) r[e] = kWFound;
                kept += r[e] < p.k;
            }
            __syncwarp();
#pragma unroll
            for (int e = 0; e < kWFound / 32; ++e)
                if (r[e] < p.k) {
                    fv[r[e]] = v[e];
                    fj[r[e]] = j[e];
                }
            n_known = n_found = __reduce_add_sync(kAll, kept);
            __syncwarp();
            if (n_known == p.k) floor_v = fmax(floor_v, 0.25 * fv[p.k - 1]);
            least = 4.0f * __double2float_rd(floor_v - err);
        };
        // the listed chunks, a lane a column; the next chunk's first 64 columns are loaded under
        // this one's arithmetic
        const int most = min(kWFound, 2 * p.k + 32) - 32;  // the cost of ranking grows as its square
        uint4 y0, y1;
        uint32_t sc;
        auto fetch = [&](int c) {
            const int j = min((int)list[c] * 32 + lane, p.b.rows - 1);
            y0 = __ldg(codes_of(j));
            y1 = __ldg(codes_of(j) + 1);
            sc = __ldg(reinterpret_cast<const uint32_t*>(scales_of(j)));
        };
        if (n_list > 0) fetch(0);
        for (int c = 0; c < n_list; ++c) {
            const int j = (int)list[c] * 32 + lane;
            const uint4 z0 = y0, z1 = y1;
            const uint32_t zs = sc;
            if (c + 1 < n_list) fetch(c + 1);
            float v = f4_estimate64<kNv>(qa, sa, z0, z1, zs, 0.0f);
            for (int st = 1; st < steps; ++st) {
                const int jc = min(j, p.b.rows - 1);
                const uint32_t w = __ldg(reinterpret_cast<const uint32_t*>(scales_of(jc) + (kNv ? st : st >> 1) * kF4Atom));
                v = f4_estimate64<kNv>(qa + 16 * st, sa + (kNv ? 4 : 2) * st, __ldg(codes_of(jc) + 2 * st),
                                       __ldg(codes_of(jc) + 2 * st + 1), !kNv && (st & 1) ? w >> 16 : w, v);
            }
            if (n_found > most) rank_found();
            // without a bound on the terms fp32 could overflow: rank_found decides
            const bool in = j < p.b.rows && j != self && (forced || v >= least);
            const uint32_t who = __ballot_sync(kAll, in);
            if (in) fj[n_found + __popc(who & ((1u << lane) - 1))] = j;
            n_found += __popc(who);
        }
        rank_found();
    }
    const double g = (double)__ldg(p.a.gs) * (double)__ldg(p.b.gs);
    for (int s = lane; s < p.k; s += 32) {
        const bool in = s < n_known;
        p.idx[i * p.k + s] = in ? fj[s] : -1;
        p.val[i * p.k + s] = in ? (float)(fv[s] * 0.25 * g) : -__int_as_float(0x7f800000);
    }
}

__global__ void k_f4_topk_none(long long n, int* idx, float* val) {
    for (long long t = (long long)blockIdx.x * blockDim.x + threadIdx.x; t < n; t += (long long)gridDim.x * blockDim.x) {
        idx[t] = -1;
        val[t] = -__int_as_float(0x7f800000);
    }
}

// Rows of a whose keys are made before they are read: whole tiles, about kKeyMB of keys.
constexpr long long kKeyMB = 256;
struct TopkPlan {
    int nspan, rows;
    long long key_bytes;
};
TopkPlan topk_plan(const F4& a, const F4& b) {
    TopkPlan t;
    t.nspan = (b.tiles() + kSpan - 1) / kSpan;
    const long long row = (long long)t.nspan * kSpanKeys * 2;
    const long long tiles = std::max(1ll, (kKeyMB << 20) / (row * 128));
    t.rows = (int)std::min<long long>(a.rows, tiles * 128);
    t.key_bytes = (row * t.rows + 255) / 256 * 256;
    return t;
}

template <int kNv, int kCB>
cudaError_t launch_keys(const CUtensorMap& ta, const CUtensorMap& tb, KeysArgs& p, int grid, cudaStream_t st) {
    const int smem = 1024 + 1024 + 2 * (128 * kCB + 2048) + keys_stages(kCB) * keys_stage(kNv, kCB);
    auto f = k_f4_keys<kNv, kCB>;
    cudaError_t e = cudaFuncSetAttribute((const void*)f, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    f<<<grid, kKThreads, smem, st>>>(ta, tb, p);
    return cudaGetLastError();
}

template <int kNv, int kT>
cudaError_t launch_pick(const PickArgs& q, int rows, cudaStream_t st) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)rows);
    cfg.blockDim = dim3((unsigned)kT);
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, k_f4_pick<kNv, kT>, q);
}

template <int kNv>
cudaError_t launch_pick_warp(const PickArgs& q, int rows, cudaStream_t st) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((rows + 3) / 4));
    cfg.blockDim = dim3(128);
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, k_f4_pick_warp<kNv>, q, rows);
}

}  // namespace

long long f4_topk_workspace(const F4& a, const F4& b, int k, int sms) {
    if (a.rows == 0 || b.rows == 0) return 0;
    return topk_plan(a, b).key_bytes + 4ll * sms;
}

cudaError_t f4_topk(const F4& a, const F4& b, int k, long long self, int* idx, float* val, void* ws,
                    int* err, int sms, cudaStream_t st, int* launches) {
    if (b.rows == 0) {
        const long long n = (long long)a.rows * k;
        k_f4_topk_none<<<(int)std::min<long long>((n + 255) / 256, 4096), 256, 0, st>>>(n, idx, val);
        *launches += 1;
        return cudaGetLastError();
    }
    const TopkPlan plan = topk_plan(a, b);
    const int cb = b.Kp == 64 ? 32 : 128;
    CUtensorMap ta, tb;
    if (!f4_map(&ta, a, 128, cb) || !f4_map(&tb, b, 256, cb)) return cudaErrorInvalidValue;
    KeysArgs p;
    p.a = a;
    p.b = b;
    p.ntiles = b.tiles();
    p.nspan = plan.nspan;
    p.keys = (uint32_t*)ws;
    p.errs = (float*)((uint8_t*)ws + plan.key_bytes);
    p.err = err;
    PickArgs q;
    q.a = a;
    q.b = b;
    q.k = k;
    q.self = self;
    q.nspan = plan.nspan;
    q.keys = p.keys;
    q.errs = p.errs;
    q.idx = idx;
    q.val = val;
    for (long long r0 = 0; r0 < a.rows; r0 += plan.rows) {
        const int rows = (int)std::min<long long>(plan.rows, a.rows - r0);
        p.q0 = (int)(r0 / 128);
        p.nq = (rows + 127) / 128;
        const int grid = (int)std::min<long long>((long long)p.nq * p.nspan, sms);
        cudaError_t e;
        if (cb == 32) e = b.nv ? launch_keys<1, 32>(ta, tb, p, grid, st) : launch_keys<0, 32>(ta, tb, p, grid, st);
        else e = b.nv ? launch_keys<1, 128>(ta, tb, p, grid, st) : launch_keys<0, 128>(ta, tb, p, grid, st);
        if (e != cudaSuccess) return e;
        q.row0 = (int)r0;
        q.nerrs = grid;
        const bool few_keys = plan.nspan * kSpanKeys <= kWarpKeys;
        // A warp is slow for one row, so the warps' kernel needs an SM nearly full of rows.  Both kernels,
        // a warp a row against 128 threads (mxfp4, rank 48, top 10): 1,200 x 10,000 33.8 / 25.6 us, 2,400
        // 35.6 / 35.8, 4,000 37.9 / 50.2, 10,000 66.6 / 105; 1,200 x 32,000 39.7 / 31.6, 4,000 48.1 / 60.4;
        // 20,000 x 20,000 132 / 212.  And its groups of 64 columns have to outnumber k: 10,000 x 1,700,
        // top 50 369 / 241; 10,000 x 1,000, top 10 60.4 / 91.1.  Few rows, 128 against 1,024 threads (1,000,000
        // x 64, top 50): one 37.9 / 29.5 us, 148 63.5 / 39.9, 296 74.5 / 62.3, 592 93.2 / 103.
        const int threads = rows <= 2 * sms ? 1024 : few_keys && rows >= 24 * sms && b.rows >= 96 * k ? 32 : 128;
        if (threads == 32) e = b.nv ? launch_pick_warp<1>(q, rows, st) : launch_pick_warp<0>(q, rows, st);
        else if (threads == 128) e = b.nv ? launch_pick<1, 128>(q, rows, st) : launch_pick<0, 128>(q, rows, st);
        else e = b.nv ? launch_pick<1, 1024>(q, rows, st) : launch_pick<0, 1024>(q, rows, st);
        if (e != cudaSuccess) return e;
        *launches += 2;
        if ((e = cudaGetLastError()) != cudaSuccess) return e;
    }
    return cudaSuccess;
}

}  // namespace rfx
