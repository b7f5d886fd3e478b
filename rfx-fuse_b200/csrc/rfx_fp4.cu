// Quantisation to microscaled 4 bits, its inverse, and the exchange with row-major codes and
// scales.  All are copies with a little arithmetic: DRAM bounds them.
//
// mxfp4: a block's scale is 2^E, E the smallest with max |x| <= 6 * 2^E (not below -127), so no
// value saturates.  nvfp4: the matrix scale g is the smallest power of two with max |x| <=
// 6 * 448 g (not below 2^-126; 1 for a matrix of zeros), and a block's scale is e4m3(max |x| /
// (6 g)).  With g a power of two, scale times code has 6 significant bits: values come back
// exactly in fp32 and bf16 (but where they reach 2^128, or lie below 2^-128), and the 24-bit input's quotients decide every rounding exactly as
// real arithmetic does (max |x| / 6 and x / scale, rounded once to fp32, are never a false tie:
// the divisors have at most 4 bits).  Codes round to the nearest, ties to the even code.
// A block that holds an infinity or NaN gets a NaN scale; g ignores such values.
#include <algorithm>

#include "rfx_fp4_dev.cuh"

namespace rfx {

namespace {

constexpr int kQThreads = 256;
constexpr int kQChunk = 256;  // columns of a block of the grid

// Division of n < 2^31 by a constant as a multiplication and a shift (Granlund and Montgomery,
// Division by invariant integers using multiplication, PLDI 1994).
struct FastDiv {
    uint32_t m, s, d;
    explicit FastDiv(uint32_t div) : d(div) {
        s = 0;
        while ((1ull << s) < div) ++s;
        m = (uint32_t)((((1ull << s) - div) << 32) / div + 1);
    }
    __device__ __forceinline__ uint32_t quo(uint32_t n) const { return (__umulhi(m, n) + n) >> s; }
};

// The matrix scale for the largest finite |x| (its bits).
__device__ __forceinline__ float nv_matrix_scale(uint32_t bits) {
    if (bits == 0) return 1.0f;
    int e = (int)(bits >> 23) - 127;                          // 2^e <= max < 2^(e+1) when normal
    e = (bits & 0x7FFFFFu) <= 0x280000u ? e - 11 : e - 10;    // 2688 = 1.3125 * 2^11
    if (e < -126) e = -126;
    return __int_as_float((e + 127) << 23);
}

__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

// Elements of a 16-byte vector.
template <class T> constexpr int kVecOf = 16 / (int)sizeof(T);

// Columns [c, c + kN) of a row of `cols` into v, zeros from cols on.
template <class T, bool kVec, int kN>
__device__ __forceinline__ void load_cols(const T* row, int c, int cols, float* v) {
    if (kVec && c + kN <= cols) {
#pragma unroll
        for (int h = 0; h < kN; h += kVecOf<T>) {
            const uint4 a = __ldg(reinterpret_cast<const uint4*>(row + c + h));
            T t[kVecOf<T>];
            memcpy(t, &a, 16);
#pragma unroll
            for (int i = 0; i < kVecOf<T>; ++i) v[h + i] = to_f32<T>(t[i]);
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < kN; ++i) v[i] = c + i < cols ? to_f32<T>(row[c + i]) : 0.0f;
}

// Largest finite |x|, by integer maximum (the order of the atomics does not matter).  Rows
// [0, rows) of U vectors each, rows * U < 2^31.
template <class T, bool kVec>
__global__ void k_f4_amax(const T* __restrict__ x, long long ld, int rows, int cols, FastDiv U, bool flat, uint32_t* out) {
    const uint32_t total = (uint32_t)rows * U.d;
    const uint32_t step = gridDim.x * blockDim.x;
    uint32_t m = 0;
#pragma unroll 4
    for (uint32_t t = blockIdx.x * blockDim.x + threadIdx.x; t < total; t += step) {
        float v[kVecOf<T>];
        const uint32_t r = flat ? 0u : U.quo(t);  // flat: rows of whole vectors that follow one another
        load_cols<T, kVec, kVecOf<T>>(x + (long long)r * ld, (int)(t - r * U.d) * kVecOf<T>, flat ? 0x7FFFFFFF : cols, v);
#pragma unroll
        for (int i = 0; i < kVecOf<T>; ++i) {
            const uint32_t b = abs_bits(v[i]);
            if (b < 0x7F800000u) m = max(m, b);
        }
    }
    m = __reduce_max_sync(0xFFFFFFFFu, m);
    if ((threadIdx.x & 31) == 0 && m) atomicMax(out, m);
}

// Four times the squared norm of eight codes, 4 at least: a norm bound is then never below a
// scale, so that no product of two scales overflows where the bounds' product does not.
__device__ __forceinline__ int mag2(uint32_t w) {
    const uint32_t m0 = e2m1_mag4(w), m1 = e2m1_mag4(w >> 16);
    return max(4, (int)__dp4a(m1, m1, __dp4a(m0, m0, 0u)));
}

// Scale in a norm's bound: not below 2^-60, so that no square underflows (a bound may be larger
// than the norm, and infinite where a square overflows).
__device__ __forceinline__ float bound_scale(float s) { return s < 8.673617379884035e-19f ? 8.673617379884035e-19f : s; }

// Bound of the tile's row norms from the units' sums of (2 x)^2, n2[unit][row] (padded to 129
// rows); rows with a NaN scale are left out, they are nobody's neighbour.
__device__ void tile_bound(const float* n2, int U, int rows, float* out) {
    __shared__ float worst[4];
    float m = 0.0f;
    if (threadIdx.x < kF4Tile) {
        if ((int)threadIdx.x < rows) {
            float s = 0.0f;
            for (int u = 0; u < U; ++u) s += n2[u * 129 + threadIdx.x];
            m = s >= 0.0f ? s : 0.0f;
        }
        for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
        if ((threadIdx.x & 31) == 0) worst[threadIdx.x >> 5] = m;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        m = fmaxf(fmaxf(worst[0], worst[1]), fmaxf(worst[2], worst[3]));
        *out = sqrtf(m) * 0.50001f;  // at most 64 additions, each off by 2^-24
    }
}

// max(a, |b|), NaN when either is.
__device__ __forceinline__ float max_abs_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(fabsf(b)));
    return d;
}

// One block: 128 rows x up to kQChunk columns, a lane 8 columns; a block of columns is 2 or 4
// neighbouring lanes.  Codes leave as 4 bytes a lane, scales through shared memory in the atoms'
// order.  kSelf: the grid is this block alone, which then finds the matrix scale itself (one
// launch for small matrices).  Tiles run from the last to the first: k_f4_amax has just read the
// last ones into L2.  Integer operations issue at half the rate of fp32 ones here, and they bound
// the kernel: hence the fp32 maxima, the table of scales and no division per lane.
template <class T, bool kVec, int kNv, bool kSelf>
__global__ void __launch_bounds__(kQThreads)
k_f4_quantize(const T* __restrict__ x, long long ld, F4 m) {
    __shared__ uint32_t sf[kQChunk / 64 * kF4Atom / 4];
    __shared__ float2 table[kNv ? 128 : 1];  // e4m3 values and their reciprocals
    __shared__ uint32_t s_amax;
    extern __shared__ float n2[];
    const int tile = gridDim.x - 1 - blockIdx.x;
    const int c0 = blockIdx.y * kQChunk;
    const int kc = min(kQChunk, m.Kp - c0);  // columns of this block (multiple of 64)
    const int U = kc / 8;
    const int r0 = tile * kF4Tile;
    const int nr = min(kF4Tile, m.rows - r0);
    const bool bounds = m.Kp <= kF4TopkK;
    const int atoms = kNv ? kc / 64 : (kc + 127) / 128;
    for (int i = threadIdx.x; i < atoms * (kF4Atom / 4); i += kQThreads) sf[i] = 0;
    if (kNv && threadIdx.x < 128) {
        const float s = e4m3_value(threadIdx.x);
        table[threadIdx.x] = make_float2(s, s > 0.0f ? 1.0f / s : 0.0f);
    }
    if (kSelf && threadIdx.x == 0) s_amax = 0;
    __syncthreads();
    const T* src = x + (long long)r0 * ld;
    // a thread keeps its columns and walks down the rows
    const int groups = kQThreads / U, grp = threadIdx.x / U, u = threadIdx.x - grp * U;
    const bool active = grp < groups;
    float g = 1.0f;
    if (kNv) {
        uint32_t amax = 0;
        if (kSelf) {
            for (int q = active ? grp : nr; q < nr; q += groups) {
                float v[8];
                load_cols<T, kVec, 8>(src + (long long)q * ld, c0 + 8 * u, m.cols, v);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const uint32_t b = abs_bits(v[i]);
                    if (b < 0x7F800000u) amax = max(amax, b);
                }
            }
            if (amax) atomicMax(&s_amax, amax);
            __syncthreads();
            amax = s_amax;
        } else {
            amax = __ldg(reinterpret_cast<const uint32_t*>(m.gs) + 1);
        }
        g = nv_matrix_scale(amax);
    }
    if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) m.gs[0] = g;
    const float inv_g = 1.0f / g;
    constexpr int kLanes = kNv ? 2 : 4;  // lanes of a block of columns
    uint8_t* dst = m.codes + (long long)r0 * m.pitch() + c0 / 2;
    // U is a multiple of 8, so a block of columns never straddles a warp's end, and every lane of
    // a warp makes the same number of rounds
    const int rounds = (kF4Tile + groups - 1) / groups;
    int q = grp;
#pragma unroll 4
    for (int round = 0; round < rounds; ++round, q += groups) {
        const bool live = active && q < nr;
        float v[8];
        if (live) {
            load_cols<T, kVec, 8>(src + (long long)q * ld, c0 + 8 * u, m.cols, v);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = 0.0f;
        }
        float amax = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) amax = max_abs_nan(amax, v[i]);
#pragma unroll
        for (int o = 1; o < kLanes; o <<= 1) amax = max_abs_nan(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, o));
        const bool bad = !(amax < __int_as_float(0x7f800000));
        uint32_t byte;
        float s;  // the scale in units of g
        if (kNv) {
            // amax / (6 g) and x / s correctly rounded from rounded reciprocals (Markstein, IBM
            // Journal of Research and Development 34(1), 1990)
            constexpr float r6 = 1.0f / 6.0f;
            const float w = amax * inv_g;
            const float z = w * r6;
            byte = cvt_e4m3x2(fmaf(fmaf(-z, 6.0f, w), r6, z), 0.0f) & 0x7Fu;
            const float2 sr = table[byte];
            s = sr.x;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float xs = v[i] * inv_g;
                const float y = xs * sr.y;
                v[i] = fmaf(fmaf(-y, s, xs), sr.y, y);
            }
        } else {
            const uint32_t bits = __float_as_uint(amax);
            int e = (int)(bits >> 23) - 127;
            e = (bits & 0x7FFFFFu) <= 0x400000u ? e - 2 : e - 1;  // 6 = 1.5 * 2^2
            if (e < -127) e = -127;
            byte = (uint32_t)(e + 127);
            s = e8m0_value(byte);
            const float r = __int_as_float((127 - e) << 23);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] *= r;
        }
        uint32_t w = cvt_e2m1x8(v);
        if (bad || (kNv && s == 0.0f)) w = 0;
        if (bad) {
            byte = kNv ? 0x7Fu : 0xFFu;
            s = __int_as_float(0x7fc00000);
        }
        if (live) {
            reinterpret_cast<uint32_t*>(dst + (long long)q * m.pitch())[u] = w;
            if (u % kLanes == 0 && c0 + 8 * u < m.cols) {
                const int blk = u / kLanes;
                reinterpret_cast<uint8_t*>(sf)[blk / 4 * kF4Atom + (q % 32) * 16 + q / 32 * 4 + blk % 4] = (uint8_t)byte;
            }
            if (bounds) {
                const float b = bound_scale(s);
                n2[u * 129 + q] = (float)mag2(w) * (b * b);
            }
        }
    }
    __syncthreads();
    uint32_t* out = reinterpret_cast<uint32_t*>(m.scales + ((long long)tile * m.natoms + c0 / (kNv ? 64 : 128)) * kF4Atom);
    for (int i = threadIdx.x; i < atoms * (kF4Atom / 4); i += kQThreads) out[i] = sf[i];
    if (bounds) tile_bound(n2, U, nr, m.bounds + tile);
}

// x g, rounded once to T.  A 16-bit T from the nearest fp32 would be rounded twice: the fp32 is cut
// off instead and its last bit set where that lost anything (rounding to odd: Boldo and Melquiond,
// IEEE Transactions on Computers 57(4), 2008), then the second rounding decides as the only one
// would.  x has 6 significant bits, so the product is exact in 64.
template <class T>
__device__ __forceinline__ T scaled_once(float x, float g) {
    if (sizeof(T) == 4) return from_f32<T>(x * g);
    float v = __fmul_rz(x, g);
    if ((double)v != (double)x * (double)g) v = __uint_as_float(__float_as_uint(v) | 1u);
    return from_f32<T>(v);
}

// Values of rows [r0, r1) into out (row r0 first).  A block takes 128 rows x up to kQChunk columns:
// their codes come into shared memory by 16-byte loads, all in flight at once, their scales decoded
// beside them.  A thread then writes kV elements at a time: 16 bytes, 4, or one element, as columns
// and alignment allow; neighbouring threads write neighbouring elements and walk down the rows.
template <class T, int kNv, int kV>
__global__ void __launch_bounds__(kQThreads)
k_f4_dequantize(F4 m, int r0, int r1, T* __restrict__ out, long long ld) {
    constexpr int sh = kNv ? 4 : 5;
    constexpr int kBlocks = kQChunk >> sh;     // scales of a row here
    constexpr int kRow = kQChunk / 2 + 16;     // bytes of a row of codes, padded against conflicts
    __shared__ __align__(16) uint8_t cs[kF4Tile * kRow];
    __shared__ float sc[kF4Tile * (kBlocks + 1)];
    __shared__ float lut[16];                  // the codes' values, for one element at a time
    const int tile = r0 / kF4Tile + blockIdx.x;
    const int c0 = blockIdx.y * kQChunk;
    const int kc = min(kQChunk, m.cols - c0);
    const int nb = (kc + (1 << sh) - 1) >> sh;
    const int qa = max(0, r0 - tile * kF4Tile), qb = min(kF4Tile, r1 - tile * kF4Tile);
    const float g = __ldg(m.gs);
    {
        const uint8_t* codes = m.codes + (long long)tile * kF4Tile * m.pitch() + c0 / 2;
        const int words = (min(kQChunk, m.Kp - c0) / 2) / 16;  // 16-byte words of a row: 2, 4, 6 or 8
        for (int t = threadIdx.x; t < kF4Tile * words; t += kQThreads) {
            const int q = t / words, w = t - q * words;
            if (q >= qa && q < qb)
                *reinterpret_cast<uint4*>(cs + q * kRow + 16 * w) =
                    __ldg(reinterpret_cast<const uint4*>(codes + (long long)q * m.pitch()) + w);
        }
        if (kV < 4 && threadIdx.x < 16) lut[threadIdx.x] = e2m1_value(threadIdx.x);
        const uint8_t* atoms = m.scales + ((long long)tile * m.natoms + c0 / (kNv ? 64 : 128)) * kF4Atom;
        for (int t = threadIdx.x; t < kF4Tile * nb; t += kQThreads) {
            const int b = t >> 7, r = t & 127;
            sc[r * (kBlocks + 1) + b] =
                f4_scale_value(kNv, __ldg(atoms + b / 4 * kF4Atom + (r % 32) * 16 + r / 32 * 4 + b % 4));
        }
    }
    __syncthreads();
    const int U = kc / kV, groups = kQThreads / U;
    const int grp = threadIdx.x / U, u = threadIdx.x - grp * U;
    if (grp >= groups) return;
    const uint8_t* p = cs + (u * kV) / 2;
    const float* s = sc + ((u * kV) >> sh);
    T* o = out + ((long long)tile * kF4Tile - r0 + qa + grp) * ld + c0 + u * kV;
    const long long step = groups * ld;
    const int shift = (u & 1) * 4;
    auto rows = [&](auto value) {
#pragma unroll 4
        for (int q = qa + grp; q < qb; q += groups, o += step) {
            const float sv = s[q * (kBlocks + 1)];
            if constexpr (kV >= 4) {
                uint32_t w;
                if constexpr (kV == 8) w = *reinterpret_cast<const uint32_t*>(p + q * kRow);
                else w = *reinterpret_cast<const uint16_t*>(p + q * kRow);
                float f[kV];
                e2m1_values<kV>(w, f);
                T v[kV];
#pragma unroll
                for (int i = 0; i < kV; ++i) v[i] = value(f[i] * sv);
                uint4 x;
                memcpy(&x, v, 16);
                *reinterpret_cast<uint4*>(o) = x;
            } else {
                const uint32_t w = p[q * kRow];
                if constexpr (kV == 2) {
                    T v[2] = {value(lut[w & 15u] * sv), value(lut[w >> 4] * sv)};
                    uint32_t x;
                    memcpy(&x, v, 4);
                    *reinterpret_cast<uint32_t*>(o) = x;
                } else {
                    *o = value(lut[w >> shift & 15u] * sv);
                }
            }
        }
    };
    // a power of two, as the quantiser's, only shifts (where it does not, the 16-bit result is 0)
    if (sizeof(T) == 4 || (__float_as_uint(g) & 0x7FFFFFu) == 0) rows([=](float x) { return from_f32<T>(x * g); });
    else rows([=](float x) { return scaled_once<T>(x, g); });
}

// A caller's matrix scale, NaN unless positive and finite: no order of the products without their
// scales is that of the products with such a one, and products and values are then NaN as well.
__device__ __forceinline__ float usable_scale(float g) {
    return g > 0.0f && g < __int_as_float(0x7f800000) ? g : __int_as_float(0x7fc00000);
}

// Row-major codes [rows][(cols + 1) / 2] and scales [rows][nblocks] into the layout above.  A
// block takes 128 rows x up to kQChunk columns, like the quantiser.
__global__ void __launch_bounds__(kQThreads)
k_f4_pack(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, const float* g, F4 m) {
    __shared__ uint32_t sf[kQChunk / 64 * kF4Atom / 4];
    extern __shared__ float n2[];
    const int tile = blockIdx.x;
    const int c0 = blockIdx.y * kQChunk;
    const int kc = min(kQChunk, m.Kp - c0);
    const int U = kc / 8;
    const int r0 = tile * kF4Tile;
    const int nr = min(kF4Tile, m.rows - r0);
    const int sh = m.nv ? 1 : 2;  // units of a block of columns, log2
    const int atoms = m.nv ? kc / 64 : (kc + 127) / 128;
    const bool bounds = m.Kp <= kF4TopkK;
    const int in_pitch = (m.cols + 1) / 2;
    const bool words = in_pitch % 4 == 0 && (uintptr_t)codes % 4 == 0;  // rows of whole 4-byte words
    for (int i = threadIdx.x; i < atoms * (kF4Atom / 4); i += kQThreads) sf[i] = 0;
    __syncthreads();
#pragma unroll 4
    for (int t = threadIdx.x; t < nr * U; t += kQThreads) {
        const int q = t / U, u = t - q * U;
        const uint8_t* src = codes + (long long)(r0 + q) * in_pitch;
        uint32_t w = 0;
        if (words && c0 + 8 * u + 8 <= m.cols) {
            w = __ldg(reinterpret_cast<const uint32_t*>(src + c0 / 2) + u);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int c = c0 + 8 * u + 2 * i;
                if (c < m.cols) {
                    uint32_t b = src[c / 2];
                    if (c + 1 >= m.cols) b &= 15u;
                    w |= b << (8 * i);
                }
            }
        }
        reinterpret_cast<uint32_t*>(m.codes + (long long)(r0 + q) * m.pitch() + c0 / 2)[u] = w;
        const int blk = u >> sh, gblk = (m.nv ? c0 / 16 : c0 / 32) + blk;
        uint32_t byte = gblk < m.nblocks ? scales[(long long)(r0 + q) * m.nblocks + gblk] : 0u;
        if (m.nv) byte &= 0x7Fu;  // unsigned e4m3
        if ((u & ((1 << sh) - 1)) == 0)
            reinterpret_cast<uint8_t*>(sf)[blk / 4 * kF4Atom + (q % 32) * 16 + q / 32 * 4 + blk % 4] = (uint8_t)byte;
        if (bounds) {
            const float s = bound_scale(f4_scale_value(m.nv, byte));
            n2[u * 129 + q] = (float)mag2(w) * (s * s);
        }
    }
    __syncthreads();
    uint32_t* dst = reinterpret_cast<uint32_t*>(m.scales + ((long long)tile * m.natoms + c0 / (m.nv ? 64 : 128)) * kF4Atom);
    for (int i = threadIdx.x; i < atoms * (kF4Atom / 4); i += kQThreads) dst[i] = sf[i];
    if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) m.gs[0] = g ? usable_scale(*g) : 1.0f;
    if (bounds) tile_bound(n2, U, nr, m.bounds + tile);
}

// The inverse of k_f4_pack: a thread per byte of a row's codes, then of its scales.
__global__ void k_f4_unpack(F4 m, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
    const int pc = (m.cols + 1) / 2, w = pc + m.nblocks;
    const long long n = (long long)m.rows * w;
    const long long step = (long long)gridDim.x * blockDim.x;
    for (long long t = (long long)blockIdx.x * blockDim.x + threadIdx.x; t < n; t += step) {
        const long long r = t / w;
        const int c = (int)(t - r * w);
        if (c < pc) codes[r * pc + c] = m.codes[r * m.pitch() + c];
        else scales[r * m.nblocks + (c - pc)] = m.scales[f4_scale_at(m, r, c - pc)];
    }
}

__global__ void k_f4_unit_scale(float* gs) { gs[0] = 1.0f; }

size_t bound_smem(const F4& m, int width) {
    return m.Kp <= kF4TopkK ? (size_t)(m.Kp / width) * 129 * sizeof(float) : 0;
}

template <class T, bool kVec>
cudaError_t quantize_t(const T* x, long long ld, const F4& m, int sms, cudaStream_t st, int* launches) {
    const dim3 grid((unsigned)m.tiles(), (unsigned)((m.Kp + kQChunk - 1) / kQChunk));
    const size_t smem = bound_smem(m, 8);
    const bool self = grid.x == 1 && grid.y == 1;
    if (!m.nv) {
        k_f4_quantize<T, kVec, 0, false><<<grid, kQThreads, smem, st>>>(x, ld, m);
        *launches += 1;
    } else if (self) {
        k_f4_quantize<T, kVec, 1, true><<<grid, kQThreads, smem, st>>>(x, ld, m);
        *launches += 1;
    } else {
        cudaError_t e = cudaMemsetAsync(m.gs + 1, 0, 4, st);
        if (e != cudaSuccess) return e;
        const FastDiv vecs((uint32_t)((m.cols + kVecOf<T> - 1) / kVecOf<T>));
        const int most = (int)std::min<long long>(m.rows, (1ll << 27) / vecs.d);  // rows of a launch
        const bool flat = kVec && ld == m.cols && m.cols % kVecOf<T> == 0;
        for (int r0 = 0; r0 < m.rows; r0 += std::min(most, m.rows - r0)) {
            const int rows = std::min(most, m.rows - r0);
            const int blocks = (int)std::min<long long>(((long long)rows * vecs.d + 255) / 256, (long long)sms * 8);
            k_f4_amax<T, kVec><<<blocks, 256, 0, st>>>(x + (long long)r0 * ld, ld, rows, m.cols, vecs, flat,
                                                      reinterpret_cast<uint32_t*>(m.gs) + 1);
            *launches += 1;
        }
        k_f4_quantize<T, kVec, 1, false><<<grid, kQThreads, smem, st>>>(x, ld, m);
        *launches += 1;
    }
    return cudaGetLastError();
}

template <class T>
cudaError_t quantize_d(const void* x, long long ld, const F4& m, int sms, cudaStream_t st, int* launches) {
    const bool vec = ((uintptr_t)x & 15) == 0 && (ld * (long long)sizeof(T)) % 16 == 0;
    return vec ? quantize_t<T, true>((const T*)x, ld, m, sms, st, launches)
               : quantize_t<T, false>((const T*)x, ld, m, sms, st, launches);
}

template <class T, int kV>
cudaError_t dequantize_v(const F4& m, int r0, int r1, T* out, long long ld, cudaStream_t st) {
    const dim3 grid((unsigned)((r1 - 1) / kF4Tile - r0 / kF4Tile + 1), (unsigned)((m.cols + kQChunk - 1) / kQChunk));
    if (m.nv) k_f4_dequantize<T, 1, kV><<<grid, kQThreads, 0, st>>>(m, r0, r1, out, ld);
    else k_f4_dequantize<T, 0, kV><<<grid, kQThreads, 0, st>>>(m, r0, r1, out, ld);
    return cudaGetLastError();
}

template <class T>
cudaError_t dequantize_d(const F4& m, int r0, int r1, T* out, long long ld, cudaStream_t st) {
    auto fits = [&](int bytes) {
        return m.cols * (int)sizeof(T) % bytes == 0 && (uintptr_t)out % bytes == 0 && ld * (long long)sizeof(T) % bytes == 0;
    };
    if (m.cols % kVecOf<T> == 0 && fits(16)) return dequantize_v<T, kVecOf<T>>(m, r0, r1, out, ld, st);
    if (sizeof(T) == 2 && fits(4)) return dequantize_v<T, 2>(m, r0, r1, out, ld, st);
    return dequantize_v<T, 1>(m, r0, r1, out, ld, st);
}

}  // namespace

// The matrix scale of a matrix without rows.
cudaError_t f4_unit_scale(const F4& m, cudaStream_t st) {
    k_f4_unit_scale<<<1, 1, 0, st>>>(m.gs);
    return cudaGetLastError();
}

cudaError_t f4_quantize(const void* x, int dtype, long long ld, const F4& m, int sms, cudaStream_t st,
                        int* launches) {
    if (dtype == RFX_F32) return quantize_d<float>(x, ld, m, sms, st, launches);
    if (dtype == RFX_BF16) return quantize_d<__nv_bfloat16>(x, ld, m, sms, st, launches);
    return quantize_d<__half>(x, ld, m, sms, st, launches);
}

cudaError_t f4_dequantize(const F4& m, int r0, int r1, void* out, int dtype, long long ld, cudaStream_t st) {
    if (dtype == RFX_F32) return dequantize_d<float>(m, r0, r1, (float*)out, ld, st);
    if (dtype == RFX_BF16) return dequantize_d<__nv_bfloat16>(m, r0, r1, (__nv_bfloat16*)out, ld, st);
    return dequantize_d<__half>(m, r0, r1, (__half*)out, ld, st);
}

cudaError_t f4_pack(const uint8_t* codes, const uint8_t* scales, const float* g, const F4& m, cudaStream_t st) {
    const dim3 grid((unsigned)m.tiles(), (unsigned)((m.Kp + kQChunk - 1) / kQChunk));
    const size_t smem = bound_smem(m, 8);
    k_f4_pack<<<grid, kQThreads, smem, st>>>(codes, scales, g, m);
    return cudaGetLastError();
}

cudaError_t f4_unpack(const F4& m, uint8_t* codes, uint8_t* scales, cudaStream_t st) {
    const long long n = (long long)m.rows * ((m.cols + 1) / 2 + m.nblocks);
    k_f4_unpack<<<(int)std::min<long long>((n + 255) / 256, 1 << 16), 256, 0, st>>>(m, codes, scales);
    return cudaGetLastError();
}

}  // namespace rfx
