// The k nearest rows under the product of two 4-bit matrices, without the product: tcgen05
// block-scaled products as a filter, the exact value of what passes it, one heap a row.
//
// The answer is exact: the value of a pair is the sum over its blocks, in order, of scale times
// scale times the blocks' integer dot product, in 64 bits (for nvfp4 that sum has no rounding at
// all), and rows rank by (value descending, index ascending).  The fp32 accumulator only decides
// what is worth that evaluation: it lies within kEps |a_i| |b_j| of the value (Cauchy-Schwarz
// bounds the terms; kEps = 2^-13 leaves a factor of 2^8 over 64-column steps added in fp32), so
// no pair below the row's current k-th value less that bound can belong to the answer.  The norms'
// bounds come with the matrices, a tile of 128 rows each.
//
// CTA = 128 rows of a (accumulator lanes) against the tiles [t0, t1) of 128 rows of b:
//   warps 0-7   filter: a lane holds one row's accumulators; the maximum of 32 columns decides
//               whether they are looked at one by one.  Groups of four warps take alternate tiles.
//               What passes goes into the quarter's queue as (row, column);
//   warps 8-11  select: a lane takes one queued pair, evaluates it exactly from the codes, and
//               puts it into its row's heap (lanes of the same row one after another), raising
//               the row's bar for the filter;
//   warp 12     loads the rows of a once and b's tiles through a ring (TMA, bulk copies);
//   warp 13     copies scales to TMEM and multiplies, into three accumulators of 128 columns.
// With few rows of a, b is split over CTAs; k_f4_merge joins the sorted lists of the splits.
// Waits on barriers and on queue space are bounded; the select warps end when the filter warps
// have ended.  On expiry the CTA records it in *err, drains its copies, frees TMEM and returns.
#include <algorithm>

#include "rfx_fp4_mma.cuh"

namespace rfx {

namespace {

constexpr int kKThreads = 448;
constexpr int kQueue = 2048;                 // entries of a quarter's queue
constexpr uint32_t kNoEntry = 0xFFFFFFFFu;
constexpr int kColBits = 27;                 // column within the split in a queue entry
constexpr float kEps = 1.0f / 8192.0f;
constexpr int kMaxSplit = 160;
constexpr int kBarBytes = 512;

struct TopkF4Args {
    F4 a, b;
    int k;
    long long self;       // row of b that is row 0 of a and left out for it (and so on); -1: none
    int ntiles, splits;
    int nstage, stage_bytes;
    int* out_idx;         // [rows of a][k], one split
    float* out_val;
    double* ws_v;         // [rows of a][splits][k], several
    int* ws_j;
    int* err;
};

__device__ __forceinline__ bool f4_better(double va, int ja, double vb, int jb) {
    return va > vb || (va == vb && ja < jb);
}

// A row's best k are a 4-ary heap in shared memory, the worst at its root; entry s sits at
// v[s * 128], j[s * 128] (1 + 4 + 16 + 64 slots hold 64 entries in four levels).
__device__ __forceinline__ void f4_heap_insert(double* v, int* j, int n, double val, int col) {
    int i = n;
#pragma unroll
    for (int l = 0; l < 3; ++l) {
        const int p = (i - 1) >> 2;
        if (i > 0 && f4_better(v[p * 128], j[p * 128], val, col)) {
            v[i * 128] = v[p * 128];
            j[i * 128] = j[p * 128];
            i = p;
        }
    }
    v[i * 128] = val;
    j[i * 128] = col;
}

__device__ __forceinline__ void f4_heap_replace_root(double* v, int* j, int n, double val, int col) {
    int i = 0;
#pragma unroll
    for (int l = 0; l < 3; ++l) {
        const int c0 = 4 * i + 1;
        int w = -1;
        double wv = 0.0;
        int wj = 0;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (c0 + u < n) {
                const double cv = v[(c0 + u) * 128];
                const int cj = j[(c0 + u) * 128];
                if (w < 0 || f4_better(wv, wj, cv, cj)) {
                    w = c0 + u;
                    wv = cv;
                    wj = cj;
                }
            }
        }
        if (w >= 0 && f4_better(val, col, wv, wj)) {
            v[i * 128] = wv;
            j[i * 128] = wj;
            i = w;
        }
    }
    v[i * 128] = val;
    j[i * 128] = col;
}

// Four times the exact value of a_i . b_j without the matrix scales; NaN when a scale is.
template <int kNv>
__device__ double f4_exact(const F4& a, const F4& b, long long i, long long j) {
    const uint4* ca = reinterpret_cast<const uint4*>(a.codes + i * a.pitch());
    const uint4* cb = reinterpret_cast<const uint4*>(b.codes + j * b.pitch());
    const uint8_t* sa = a.scales + f4_scale_at(a, i, 0);
    const uint8_t* sb = b.scales + f4_scale_at(b, j, 0);
    double v = 0.0;
    for (int c = 0; c < a.Kp / 64; ++c) {
        const int at = kNv ? c : c >> 1;
        uint32_t wa = __ldg(reinterpret_cast<const uint32_t*>(sa + at * kF4Atom));
        uint32_t wb = __ldg(reinterpret_cast<const uint32_t*>(sb + at * kF4Atom));
        if (!kNv && (c & 1)) {
            wa >>= 16;
            wb >>= 16;
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {  // 32 columns
            const uint4 x = __ldg(ca + 2 * c + h), y = __ldg(cb + 2 * c + h);
            int lo = e2m1_dot8(x.x, y.x, 0);
            lo = e2m1_dot8(x.y, y.y, lo);
            int hi = e2m1_dot8(x.z, y.z, 0);
            hi = e2m1_dot8(x.w, y.w, hi);
            if (kNv) {
                const double s0 = (double)(e4m3_value((wa >> (16 * h)) & 0xFFu) * e4m3_value((wb >> (16 * h)) & 0xFFu));
                const double s1 = (double)(e4m3_value((wa >> (16 * h + 8)) & 0xFFu) * e4m3_value((wb >> (16 * h + 8)) & 0xFFu));
                v += s0 * (double)lo;
                v += s1 * (double)hi;
            } else {
                const uint32_t ea = (wa >> (8 * h)) & 0xFFu, eb = (wb >> (8 * h)) & 0xFFu;
                // 2^(ea + eb - 254) as bits; a byte of 255 is NaN
                const double s = ea == 255u || eb == 255u ? __longlong_as_double(0x7ff8000000000000ll)
                                                          : __longlong_as_double((long long)(ea + eb + 769u) << 52);
                v += s * (double)(lo + hi);
            }
        }
    }
    return v;
}

__device__ __forceinline__ float f4_final(double v4, double g) { return (float)(v4 * 0.25 * g); }

template <int kNv, int kCB>
__global__ void __launch_bounds__(kKThreads, 1)
k_f4_topk(const __grid_constant__ CUtensorMap tma, const __grid_constant__ CUtensorMap tmb, TopkF4Args p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* sm = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    constexpr int kAtoms = kCB == 32 ? 1 : (kNv ? 4 : 2);
    constexpr int kBox = 128 * kCB;
    const int k = p.k;
    // rows of a, ring, heaps, queues, then barriers and per-row state
    uint8_t* s_a = sm;
    uint8_t* s_sa = sm + kBox;
    uint8_t* s_ring = sm + kBox + 2048;
    double* heap_v = (double*)(s_ring + p.nstage * p.stage_bytes);      // [k][128]
    int* heap_j = (int*)(heap_v + k * 128);                             // [k][128]
    uint32_t* queue = (uint32_t*)(heap_j + k * 128);                    // [4][kQueue]
    volatile float* thr = (volatile float*)(queue + 4 * kQueue);        // [128] bars
    int* cnt = (int*)(thr + 128);                                       // [128] heap entries
    uint64_t* bars = (uint64_t*)(cnt + 128);
    // full[16], empty[16], acc_full[3], acc_empty[3], a_full
    uint32_t* tmem_slot = (uint32_t*)(bars + 40);
    volatile int* abort = (volatile int*)(tmem_slot + 1);
    volatile int* ended = (volatile int*)(tmem_slot + 2);               // [4] filter warps that ended
    volatile uint32_t* q_head = (volatile uint32_t*)(tmem_slot + 6);    // [4]
    uint32_t* q_tail = tmem_slot + 10;                                  // [4]
    const uint32_t bar0 = smem_u32(bars);
    auto full = [&](int s) { return bar0 + 8u * s; };
    auto empty = [&](int s) { return bar0 + 8u * (16 + s); };
    auto accf = [&](int b) { return bar0 + 8u * (32 + b); };
    auto acce = [&](int b) { return bar0 + 8u * (35 + b); };
    const uint32_t afull = bar0 + 8u * 38;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long i0 = (long long)blockIdx.x * 128;
    const int t0 = (int)((long long)p.ntiles * blockIdx.y / p.splits);
    const int t1 = (int)((long long)p.ntiles * (blockIdx.y + 1) / p.splits);

    if (threadIdx.x == 0) {
        for (int s = 0; s < p.nstage; ++s) {
            mbar_init(full(s), 1);
            mbar_init(empty(s), 1);
        }
        for (int b = 0; b < 3; ++b) {
            mbar_init(accf(b), 1);
            mbar_init(acce(b), 128);
        }
        mbar_init(afull, 1);
        *abort = 0;
        for (int q = 0; q < 4; ++q) {
            ended[q] = 0;
            q_head[q] = 0;
            q_tail[q] = 0;
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    for (int i = threadIdx.x; i < 4 * kQueue; i += kKThreads) queue[i] = kNoEntry;
    if (threadIdx.x < 128) {
        cnt[threadIdx.x] = 0;
        thr[threadIdx.x] = i0 + threadIdx.x < p.a.rows ? -__int_as_float(0x7f800000) : __int_as_float(0x7f800000);
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
    const uint32_t tmem = *tmem_slot;
    const int steps = p.b.Kp / 64;
    const int atoms = kNv ? steps : (steps + 1) / 2;

    if (warp == 12) {
        if (lane == 0) {
            const uint32_t sfb = (uint32_t)(atoms * kF4Atom);
            mbar_expect_tx(afull, (uint32_t)kBox + sfb);
            tma_load(smem_u32(s_a), &tma, 0, (int)i0, afull);
            bulk_load(smem_u32(s_sa), p.a.scales + (long long)blockIdx.x * p.a.natoms * kF4Atom, sfb, afull);
            int n = 0;
            for (int t = t0; t < t1; ++t, ++n) {
                const int s = n % p.nstage;
                if (mbar_wait(empty(s), ((uint32_t)(n / p.nstage) & 1u) ^ 1u, abort) != kWaitOk) {
                    if (!*abort) atomicExch(p.err, 1);
                    *abort = 1;
                    break;
                }
                const uint32_t st = smem_u32(s_ring + s * p.stage_bytes);
                mbar_expect_tx(full(s), (uint32_t)kBox + sfb);
                tma_load(st, &tmb, 0, t * 128, full(s));
                bulk_load(st + kBox, p.b.scales + (long long)t * p.b.natoms * kF4Atom, sfb, full(s));
            }
            // drain this thread's copies still in flight
            mbar_wait(afull, 0, nullptr);
            for (int i = n > p.nstage ? n - p.nstage : 0; i < n; ++i)
                mbar_wait(full(i % p.nstage), (uint32_t)(i / p.nstage) & 1u, nullptr);
        }
        __syncwarp();
    } else if (warp == 13) {
        if (lane == 0) {
            bool ok = mbar_wait(afull, 0, abort) == kWaitOk;
            const uint32_t tsa = tmem + 384u;
            int n = 0;
            if (ok) {
                tc_fence_after();
                for (int k0 = 0; k0 < atoms; ++k0) f4_copy_atom(tsa + 4 * k0, f4_atom_desc(smem_u32(s_sa) + k0 * kF4Atom));
            }
            const uint64_t da = f4_operand_desc<kCB>(smem_u32(s_a));
            for (int t = t0; ok && t < t1; ++t) {
                const int s = n % p.nstage, b = n % 3;
                if (mbar_wait(acce(b), ((uint32_t)(n / 3) & 1u) ^ 1u, abort) != kWaitOk ||
                    mbar_wait(full(s), (uint32_t)(n / p.nstage) & 1u, abort) != kWaitOk) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t st = smem_u32(s_ring + s * p.stage_bytes);
                const uint32_t tsb = tmem + 400u + (uint32_t)(s * 4 * kAtoms);
                for (int k0 = 0; k0 < atoms; ++k0) f4_copy_atom(tsb + 4 * k0, f4_atom_desc(st + kBox + k0 * kF4Atom));
                const uint64_t db = f4_operand_desc<kCB>(st);
                for (int k0 = 0; k0 < steps; ++k0) {
                    const int at = kNv ? k0 : k0 >> 1;
                    f4_mma<kNv>(tmem + (uint32_t)(128 * b), da + 2 * k0, db + 2 * k0, f4_idesc<kNv>(128, kNv ? 0 : k0 & 1),
                                tsa + 4 * at, tsb + 4 * at, k0 ? 1u : 0u);
                }
                mma_commit(empty(s));
                mma_commit(accf(b));
                ++n;
            }
            if (!ok) {
                if (!*abort) atomicExch(p.err, 2);
                *abort = 1;
            }
            // the last products must finish before the accumulators are freed
            if (n > 0) mbar_wait(accf((n - 1) % 3), (uint32_t)((n - 1) / 3) & 1u, nullptr);
        }
        __syncwarp();
    } else if (warp < 8) {
        // ---------------- filter ----------------
        const int group = warp >> 2, quarter = warp & 3;
        const int rl = 32 * quarter + lane;
        const uint32_t lane_addr = (uint32_t)(32 * quarter) << 16;
        const bool valid = i0 + rl < p.a.rows;
        const float bq = __ldg(p.a.bounds + blockIdx.x) * (kEps * 1.000001f);
        uint32_t* qu = queue + quarter * kQueue;
        bool ok = true;
        int n = group;
        float bd = t0 + group < t1 ? __ldg(p.b.bounds + t0 + group) : 0.0f;
        for (int t = t0 + group; t < t1; t += 2, n += 2) {
            const int b = n % 3;
            const float slack = fmaxf(bq * bd, 1e-37f);
            if (t + 2 < t1) bd = __ldg(p.b.bounds + t + 2);
            const int w = mbar_wait<false>(accf(b), (uint32_t)(n / 3) & 1u, abort);
            if (__any_sync(0xFFFFFFFFu, w != kWaitOk)) {
                ok = false;
                break;
            }
            tc_fence_after();
            // a sum of such terms can overflow fp32 and lose its sign: look at every column
            const bool force = !(slack < 1e30f) && valid;
            const float bar = __fsub_rd(thr[rl], slack);
            const int ncol = p.b.rows - t * 128;  // columns that exist
#pragma unroll 1
            for (int h = 0; h < 2 && ok; ++h) {
                uint32_t r[2][32];
                __syncwarp();
#pragma unroll
                for (int c = 0; c < 2; ++c) tmem_ld32_issue(tmem + lane_addr + (uint32_t)(128 * b + 64 * h + 32 * c), r[c]);
                tmem_wait();
#pragma unroll
                for (int c = 0; c < 2; ++c) tmem_pin32(r[c]);
                if (h == 1) {
                    tc_fence_before();
                    mbar_arrive(acce(b));
                }
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    float m0 = __uint_as_float(r[c][0]), m1 = __uint_as_float(r[c][1]);
#pragma unroll
                    for (int e = 2; e < 30; e += 4) {
                        m0 = fmax3(m0, __uint_as_float(r[c][e]), __uint_as_float(r[c][e + 1]));
                        m1 = fmax3(m1, __uint_as_float(r[c][e + 2]), __uint_as_float(r[c][e + 3]));
                    }
                    m0 = fmax3(m0, __uint_as_float(r[c][30]), __uint_as_float(r[c][31]));
                    m0 = fmaxf(m0, m1);
                    const int left = ncol - (64 * h + 32 * c);
                    if (!__any_sync(0xFFFFFFFFu, (m0 >= bar || force) && left > 0)) continue;
                    uint32_t mask = 0;
#pragma unroll
                    for (int e = 0; e < 32; ++e) mask |= (__uint_as_float(r[c][e]) >= bar ? 1u : 0u) << e;
                    if (force) mask = 0xFFFFFFFFu;
                    if (left < 32) mask &= left > 0 ? (1u << left) - 1u : 0u;
                    const int mine = __popc(mask);
                    int upto = mine;
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const int v = __shfl_up_sync(0xFFFFFFFFu, upto, o);
                        if (lane >= o) upto += v;
                    }
                    const int total = __shfl_sync(0xFFFFFFFFu, upto, 31);
                    if (total == 0) continue;
                    uint32_t pos = 0;
                    if (lane == 0) pos = atomicAdd(&q_tail[quarter], (uint32_t)total);
                    pos = __shfl_sync(0xFFFFFFFFu, pos, 0);
                    // room: the select warp has taken everything kQueue entries back
                    bool room = true;
                    const unsigned long long w0 = now_ns();
                    while (pos + (uint32_t)total - q_head[quarter] > (uint32_t)kQueue) {
                        if (*abort || now_ns() - w0 > kWaitNs) {
                            room = false;
                            break;
                        }
                        __nanosleep(100);
                    }
                    if (!__all_sync(0xFFFFFFFFu, room)) {
                        ok = false;
                        break;
                    }
                    pos += (uint32_t)(upto - mine);
                    const uint32_t base = ((uint32_t)lane << kColBits) | (uint32_t)((t - t0) * 128 + 64 * h + 32 * c);
                    while (mask) {
                        const int e = __ffs(mask) - 1;
                        mask &= mask - 1;
                        ((volatile uint32_t*)qu)[pos % kQueue] = base + (uint32_t)e;
                        ++pos;
                    }
                }
            }
            if (!ok) break;
        }
        if (!ok) {
            if (lane == 0) {
                if (!*abort) atomicExch(p.err, 3);
                *abort = 1;
            }
        }
        __threadfence_block();
        __syncwarp();
        if (lane == 0) atomicAdd((int*)&ended[quarter], 1);
    } else {
        // ---------------- select ----------------
        const int quarter = warp & 3;
        volatile uint32_t* qu = queue + quarter * kQueue;
        uint32_t head = 0;
        int idle = 0;
        while (true) {
            // ended first: what was queued before it is then visible
            const bool done = ended[quarter] == 2;
            __threadfence_block();
            const uint32_t ent = qu[(head + lane) % kQueue];
            const uint32_t have = __ballot_sync(0xFFFFFFFFu, ent != kNoEntry);
            const int n = have == 0xFFFFFFFFu ? 32 : __ffs(~have) - 1;
            const bool stop = __all_sync(0xFFFFFFFFu, done);
            if (n == 0) {
                if (stop) break;
                __nanosleep(64);
                idle = 0;
                continue;
            }
            if (n < 32 && !stop && ++idle < 4) {  // a fuller batch costs the same
                __nanosleep(64);
                continue;
            }
            idle = 0;
            const bool mine = lane < n;
            if (mine) qu[(head + lane) % kQueue] = kNoEntry;
            __threadfence_block();
            __syncwarp();
            head += (uint32_t)n;
            if (lane == 0) q_head[quarter] = head;
            const int rl = 32 * quarter + (int)(ent >> kColBits);
            const long long i = i0 + rl;
            const long long col = (long long)t0 * 128 + (ent & ((1u << kColBits) - 1u));
            double v = 0.0;
            bool take = mine && !(p.self >= 0 && col == p.self + i);
            if (take) {
                v = f4_exact<kNv>(p.a, p.b, i, col);
                take = v == v;
            }
            uint32_t todo = __ballot_sync(0xFFFFFFFFu, take);
            const uint32_t peers = __match_any_sync(0xFFFFFFFFu, take ? rl : -1 - lane);
            while (todo) {
                // the lowest waiting lane of every row
                const bool go = take && (__ffs(peers & todo) - 1) == lane;
                if (go) {
                    double* hv = heap_v + rl;
                    int* hj = heap_j + rl;
                    const int c = cnt[rl];
                    if (c < k) {
                        f4_heap_insert(hv, hj, c, v, (int)col);
                        cnt[rl] = c + 1;
                        if (c + 1 == k) thr[rl] = __double2float_rd(hv[0] * 0.25);
                    } else if (f4_better(v, (int)col, hv[0], hj[0])) {
                        f4_heap_replace_root(hv, hj, k, v, (int)col);
                        thr[rl] = __double2float_rd(hv[0] * 0.25);
                    }
                }
                __syncwarp();
                const uint32_t went = __ballot_sync(0xFFFFFFFFu, go);
                todo &= ~went;
                if (go) take = false;
            }
        }
        // best first: the root (worst) goes to the back
        const int rl = 32 * quarter + lane;
        const long long i = i0 + rl;
        if (i < p.a.rows && !*abort) {
            double* hv = heap_v + rl;
            int* hj = heap_j + rl;
            const int c = cnt[rl];
            for (int n = c; n > 1; --n) {
                const double wv = hv[0];
                const int wj = hj[0];
                f4_heap_replace_root(hv, hj, n - 1, hv[(n - 1) * 128], hj[(n - 1) * 128]);
                hv[(n - 1) * 128] = wv;
                hj[(n - 1) * 128] = wj;
            }
            const double g = (double)__ldg(p.a.gs) * (double)__ldg(p.b.gs);
            for (int s = 0; s < k; ++s) {
                const bool in = s < c;
                if (p.splits == 1) {
                    p.out_idx[i * k + s] = in ? hj[s * 128] : -1;
                    p.out_val[i * k + s] = in ? f4_final(hv[s * 128], g) : -__int_as_float(0x7f800000);
                } else {
                    const long long o = (i * p.splits + blockIdx.y) * k + s;
                    p.ws_j[o] = in ? hj[s * 128] : -1;
                    p.ws_v[o] = in ? hv[s * 128] : 0.0;
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 13) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512)
                     : "memory");
    }
}

// Joins the sorted lists of a row's splits: a warp per row, a lane keeps the heads of up to five
// lists; every round the best head of the warp is the next neighbour.
constexpr int kMergeLists = (kMaxSplit + 31) / 32;
__global__ void k_f4_merge(const double* __restrict__ ws_v, const int* __restrict__ ws_j, int rows, int splits,
                           int k, const float* ga, const float* gb, int* __restrict__ idx, float* __restrict__ val) {
    const int row = (int)((blockIdx.x * blockDim.x + threadIdx.x) >> 5), lane = threadIdx.x & 31;
    if (row >= rows) return;
    const double g = (double)__ldg(ga) * (double)__ldg(gb);
    const double* v = ws_v + (long long)row * splits * k;
    const int* j = ws_j + (long long)row * splits * k;
    double hv[kMergeLists];
    int hj[kMergeLists], at[kMergeLists];
#pragma unroll
    for (int l = 0; l < kMergeLists; ++l) {
        const int s = lane + 32 * l;
        at[l] = 0;
        hj[l] = s < splits ? j[(long long)s * k] : -1;
        hv[l] = s < splits ? v[(long long)s * k] : 0.0;
    }
    for (int o = 0; o < k; ++o) {
        int bl = -1, bj = -1;
        double bv = 0.0;
#pragma unroll
        for (int l = 0; l < kMergeLists; ++l)
            if (hj[l] >= 0 && (bj < 0 || f4_better(hv[l], hj[l], bv, bj))) {
                bl = l;
                bj = hj[l];
                bv = hv[l];
            }
        const int mine = bj;
#pragma unroll
        for (int d = 16; d; d >>= 1) {
            const double ov = __shfl_xor_sync(0xFFFFFFFFu, bv, d);
            const int oj = __shfl_xor_sync(0xFFFFFFFFu, bj, d);
            if (oj >= 0 && (bj < 0 || f4_better(ov, oj, bv, bj))) {
                bv = ov;
                bj = oj;
            }
        }
        if (lane == 0) {
            idx[(long long)row * k + o] = bj;
            val[(long long)row * k + o] = bj >= 0 ? f4_final(bv, g) : -__int_as_float(0x7f800000);
        }
        if (bj >= 0 && mine == bj) {  // columns are unique over the splits
#pragma unroll
            for (int l = 0; l < kMergeLists; ++l)
                if (l == bl) {
                    const long long s = lane + 32 * l;
                    const int a = ++at[l];
                    hj[l] = a < k ? j[s * k + a] : -1;
                    hv[l] = a < k ? v[s * k + a] : 0.0;
                }
        }
    }
}

__global__ void k_f4_topk_none(long long n, int* idx, float* val) {
    for (long long t = (long long)blockIdx.x * blockDim.x + threadIdx.x; t < n; t += (long long)gridDim.x * blockDim.x) {
        idx[t] = -1;
        val[t] = -__int_as_float(0x7f800000);
    }
}

int topk_splits(const F4& a, const F4& b, int sms) {
    const int nq = a.tiles(), nt = b.tiles();
    int s = std::max(1, std::min(std::min(sms / std::max(1, nq), nt), kMaxSplit));
    // a queue entry holds a column of the split in kColBits bits
    const int need = (int)(((long long)nt * 128 + (1ll << kColBits) - 1) / ((1ll << kColBits) - 128));
    return std::max(s, need);
}

template <int kNv, int kCB>
cudaError_t launch_topk(const CUtensorMap& ta, const CUtensorMap& tb, TopkF4Args& p, cudaStream_t st) {
    constexpr int kAtoms = kCB == 32 ? 1 : (kNv ? 4 : 2);
    p.stage_bytes = (128 * kCB + kAtoms * kF4Atom + 1023) / 1024 * 1024;
    p.nstage = kCB == 32 ? 12 : 4;
    const int smem = 1024 + 128 * kCB + 2048 + p.nstage * p.stage_bytes + p.k * 128 * 12 + 4 * kQueue * 4 +
                     128 * 8 + kBarBytes;
    auto f = k_f4_topk<kNv, kCB>;
    cudaError_t e = cudaFuncSetAttribute((const void*)f, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    f<<<dim3((unsigned)p.a.tiles(), (unsigned)p.splits), kKThreads, smem, st>>>(ta, tb, p);
    return cudaGetLastError();
}

}  // namespace

long long f4_topk_workspace(const F4& a, const F4& b, int k, int sms) {
    if (a.rows == 0 || b.rows == 0) return 0;
    const int s = topk_splits(a, b, sms);
    return s == 1 ? 0 : (long long)a.rows * s * k * 12;
}

cudaError_t f4_topk(const F4& a, const F4& b, int k, long long self, int* idx, float* val, void* ws,
                    int* err, int sms, cudaStream_t st, int* launches) {
    if (b.rows == 0) {
        const long long n = (long long)a.rows * k;
        k_f4_topk_none<<<(int)std::min<long long>((n + 255) / 256, 4096), 256, 0, st>>>(n, idx, val);
        *launches += 1;
        return cudaGetLastError();
    }
    TopkF4Args p;
    p.a = a;
    p.b = b;
    p.k = k;
    p.self = self;
    p.ntiles = b.tiles();
    p.splits = topk_splits(a, b, sms);
    p.out_idx = idx;
    p.out_val = val;
    p.ws_v = (double*)ws;
    p.ws_j = p.splits > 1 ? (int*)(p.ws_v + (long long)a.rows * p.splits * k) : nullptr;
    p.err = err;
    const int cb = b.Kp == 64 ? 32 : 128;
    CUtensorMap ta, tb;
    if (!f4_map(&ta, a, 128, cb) || !f4_map(&tb, b, 128, cb)) return cudaErrorInvalidValue;
    cudaError_t e;
    if (cb == 32) e = b.nv ? launch_topk<1, 32>(ta, tb, p, st) : launch_topk<0, 32>(ta, tb, p, st);
    else e = b.nv ? launch_topk<1, 128>(ta, tb, p, st) : launch_topk<0, 128>(ta, tb, p, st);
    *launches += 1;
    if (e != cudaSuccess || p.splits == 1) return e;
    k_f4_merge<<<(a.rows + 3) / 4, 128, 0, st>>>(p.ws_v, p.ws_j, a.rows, p.splits, k, a.gs, b.gs, idx, val);
    *launches += 1;
    return cudaGetLastError();
}

}  // namespace rfx
