// Quantisation to microscaled 4 bits, its inverse, and the exchange with row-major codes and
// scales.  All are copies with a little arithmetic: DRAM bounds them.
//
// mxfp4: a block's scale is 2^E, E the smallest with max |x| <= 6 * 2^E (not below -127), so no
// value saturates.  nvfp4: the matrix scale g is the smallest power of two with max |x| <=
// 6 * 448 g (not below 2^-126; 1 for a matrix of zeros), and a block's scale is e4m3(max |x| /
// (6 g)).  With g a power of two, scale times code has 6 significant bits: values come back
// exactly in fp32 and bf16, and the 24-bit input's quotients decide every rounding exactly as
// real arithmetic does (max |x| / 6 and x / scale, rounded once to fp32, are never a false tie:
// the divisors have at most 4 bits).  Codes round to the nearest, ties to the even code.
// A block that holds an infinity or NaN gets a NaN scale; g ignores such values.
#include <algorithm>

#include "rfx_fp4_dev.cuh"

namespace rfx {

namespace {

constexpr int kQThreads = 256;
constexpr int kQChunk = 512;  // columns of a block of the grid, for matrices wider than kF4TopkK

// The matrix scale for the largest finite |x| (its bits).
__device__ __forceinline__ float nv_matrix_scale(uint32_t bits) {
    if (bits == 0) return 1.0f;
    int e = (int)(bits >> 23) - 127;                          // 2^e <= max < 2^(e+1) when normal
    e = (bits & 0x7FFFFFu) <= 0x280000u ? e - 11 : e - 10;    // 2688 = 1.3125 * 2^11
    if (e < -126) e = -126;
    return __int_as_float((e + 127) << 23);
}

__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

// Columns [c, c + 8) of a row of `cols` into v, zeros from cols on.
template <class T, bool kVec>
__device__ __forceinline__ void load8(const T* row, int c, int cols, float* v) {
    if (kVec && c + 8 <= cols) {
        if (sizeof(T) == 4) {
            const float4 a = __ldg(reinterpret_cast<const float4*>(row + c));
            const float4 b = __ldg(reinterpret_cast<const float4*>(row + c) + 1);
            v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
            v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
        } else {
            const uint4 a = __ldg(reinterpret_cast<const uint4*>(row + c));
            T t[8];
            *reinterpret_cast<uint4*>(t) = a;
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = to_f32<T>(t[i]);
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c + i < cols ? to_f32<T>(row[c + i]) : 0.0f;
}

// Largest finite |x|, by integer maximum (the order of the atomics does not matter).
template <class T, bool kVec>
__global__ void k_f4_amax(const T* __restrict__ x, long long ld, int rows, int cols, uint32_t* out) {
    const int U = (cols + 7) / 8;
    const long long total = (long long)rows * U;
    const long long step = (long long)gridDim.x * blockDim.x;
    uint32_t m = 0;
    for (long long t = (long long)blockIdx.x * blockDim.x + threadIdx.x; t < total; t += step) {
        long long r;
        int u;
        if (total < (1ll << 31)) {
            r = (uint32_t)t / (uint32_t)U;
            u = (int)((uint32_t)t % (uint32_t)U);
        } else {
            r = t / U;
            u = (int)(t % U);
        }
        float v[8];
        load8<T, kVec>(x + r * ld, 8 * u, cols, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
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

// Bound of the tile's row norms from the units' sums of squares n2[row][U] (doubles, so that no
// scale's square underflows); rows with a NaN scale are left out, they are nobody's neighbour.
__device__ void tile_bound(const double* n2, int U, int rows, float* out) {
    __shared__ double worst[4];
    double m = 0.0;
    if (threadIdx.x < kF4Tile) {
        if ((int)threadIdx.x < rows) {
            double s = 0.0;
            for (int u = 0; u < U; ++u) s += n2[threadIdx.x * U + u];
            m = s >= 0.0 ? s : 0.0;
        }
        for (int o = 16; o; o >>= 1) m = fmax(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
        if ((threadIdx.x & 31) == 0) worst[threadIdx.x >> 5] = m;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        m = fmax(fmax(worst[0], worst[1]), fmax(worst[2], worst[3]));
        *out = __double2float_ru(sqrt(m) * 0.5 * 1.000001);
    }
}

// One block: 128 rows x up to kQChunk columns (all of them when the matrix has at most
// kF4TopkK).  A lane holds 8 columns; a block of columns is 2 or 4 neighbouring lanes.  Codes
// leave as 4 bytes a lane, scales through shared memory in the atoms' order.  kSelf: the grid is
// this block alone, which then finds the matrix scale itself (one launch for small matrices).
// Tiles run from the last to the first: k_f4_amax has just read the last ones into L2.
template <class T, bool kVec, int kNv, bool kSelf>
__global__ void __launch_bounds__(kQThreads)
k_f4_quantize(const T* __restrict__ x, long long ld, F4 m) {
    __shared__ uint32_t sf[kQChunk / 64 * kF4Atom / 4];
    __shared__ uint32_t s_amax;
    extern __shared__ double n2[];
    const int tile = gridDim.x - 1 - blockIdx.x;
    const int c0 = blockIdx.y * kQChunk;
    const int kc = min(kQChunk, m.Kp - c0);  // columns of this block (multiple of 64)
    const int U = kc / 8;
    const int r0 = tile * kF4Tile;
    const int nr = min(kF4Tile, m.rows - r0);
    const bool bounds = m.Kp <= kF4TopkK;
    const int atoms = kNv ? kc / 64 : (kc + 127) / 128;
    for (int i = threadIdx.x; i < atoms * (kF4Atom / 4); i += kQThreads) sf[i] = 0;
    if (kSelf && threadIdx.x == 0) s_amax = 0;
    __syncthreads();
    float g = 1.0f;
    if (kNv) {
        uint32_t amax = 0;
        if (kSelf) {
            for (int t = threadIdx.x; t < nr * U; t += kQThreads) {
                const int q = t / U, u = t - q * U;
                float v[8];
                load8<T, kVec>(x + (long long)(r0 + q) * ld, c0 + 8 * u, m.cols, v);
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
    // U is a multiple of 8, so a block of columns never straddles a warp's end; every lane of a
    // warp makes the same number of rounds
    for (int t = threadIdx.x; t < kF4Tile * U; t += kQThreads) {
        const int q = t / U, u = t - q * U;
        const bool live = q < nr;
        float v[8];
        if (live) {
            load8<T, kVec>(x + (long long)(r0 + q) * ld, c0 + 8 * u, m.cols, v);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = 0.0f;
        }
        uint32_t amax = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) amax = max(amax, abs_bits(v[i]));
#pragma unroll
        for (int o = 1; o < kLanes; o <<= 1) amax = max(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, o));
        uint32_t byte;
        float s;  // the scale in units of g
        if (kNv) {
            byte = cvt_e4m3x2(__uint_as_float(amax) * inv_g / 6.0f, 0.0f) & 0xFFu;
            s = e4m3_value(byte);
            // x / s correctly rounded from the rounded reciprocal (Markstein, IBM Journal of
            // Research and Development 34(1), 1990)
            const float r = s > 0.0f ? 1.0f / s : 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float xs = v[i] * inv_g;
                const float y = xs * r;
                v[i] = fmaf(fmaf(-y, s, xs), r, y);
            }
        } else {
            int e = (int)(amax >> 23) - 127;
            e = (amax & 0x7FFFFFu) <= 0x400000u ? e - 2 : e - 1;  // 6 = 1.5 * 2^2
            if (e < -127) e = -127;
            byte = (uint32_t)(e + 127);
            s = e8m0_value(byte);
            const float r = __int_as_float((127 - e) << 23);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] *= r;
        }
        uint32_t w = cvt_e2m1x8(v);
        if (kNv && s == 0.0f) w = 0;
        if (amax >= 0x7F800000u) {
            byte = kNv ? 0x7Fu : 0xFFu;
            w = 0;
            s = __int_as_float(0x7fc00000);
        }
        if (live) {
            reinterpret_cast<uint32_t*>(m.codes + (long long)(r0 + q) * m.pitch() + c0 / 2)[u] = w;
            if (u % kLanes == 0 && c0 + 8 * u < m.cols) {
                const int blk = u / kLanes;
                reinterpret_cast<uint8_t*>(sf)[blk / 4 * kF4Atom + (q % 32) * 16 + q / 32 * 4 + blk % 4] = (uint8_t)byte;
            }
            if (bounds) n2[q * U + u] = (double)mag2(w) * ((double)s * (double)s);
        }
    }
    __syncthreads();
    uint32_t* dst = reinterpret_cast<uint32_t*>(m.scales + ((long long)tile * m.natoms + c0 / (kNv ? 64 : 128)) * kF4Atom);
    for (int i = threadIdx.x; i < atoms * (kF4Atom / 4); i += kQThreads) dst[i] = sf[i];
    if (bounds) tile_bound(n2, U, nr, m.bounds + tile);
}

// Values of rows [r0, r1): a thread per element, so that any leading dimension stores coalesced.
template <class T>
__global__ void k_f4_dequantize_any(F4 m, int r0, long long n, T* __restrict__ out, long long ld) {
    const long long step = (long long)gridDim.x * blockDim.x;
    const float g = __ldg(m.gs);
    const int sh = m.nv ? 4 : 5;
    for (long long t = (long long)blockIdx.x * blockDim.x + threadIdx.x; t < n; t += step) {
        long long r;
        int c;
        if (n < (1ll << 31)) {
            r = (uint32_t)t / (uint32_t)m.cols;
            c = (int)((uint32_t)t - (uint32_t)r * (uint32_t)m.cols);
        } else {
            r = t / m.cols;
            c = (int)(t - r * m.cols);
        }
        const uint32_t b = __ldg(m.codes + (r0 + r) * m.pitch() + c / 2);
        const float s = f4_scale_value(m.nv, __ldg(m.scales + f4_scale_at(m, r0 + r, c >> sh)));
        out[r * ld + c] = from_f32<T>(e2m1_value((c & 1) ? b >> 4 : b & 15u) * s * g);
    }
}

// The same for rows whose 8-column pieces are all whole and 16-byte aligned.
template <class T>
__global__ void k_f4_dequantize_vec(F4 m, int r0, long long n, T* __restrict__ out, long long ld) {
    const int U = m.cols / 8;
    const long long step = (long long)gridDim.x * blockDim.x;
    const float g = __ldg(m.gs);
    const int sh = m.nv ? 1 : 2;
    for (long long t = (long long)blockIdx.x * blockDim.x + threadIdx.x; t < n; t += step) {
        long long r;
        int u;
        if (n < (1ll << 31)) {
            r = (uint32_t)t / (uint32_t)U;
            u = (int)((uint32_t)t - (uint32_t)r * (uint32_t)U);
        } else {
            r = t / U;
            u = (int)(t - r * U);
        }
        const uint32_t w = __ldg(reinterpret_cast<const uint32_t*>(m.codes + (r0 + r) * m.pitch()) + u);
        const float s = f4_scale_value(m.nv, __ldg(m.scales + f4_scale_at(m, r0 + r, u >> sh)));
        T v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = from_f32<T>(e2m1_value((w >> (4 * i)) & 15u) * s * g);
        uint4* o = reinterpret_cast<uint4*>(out + r * ld + 8 * u);
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) o[i] = reinterpret_cast<const uint4*>(v)[i];
    }
}

// Row-major codes [rows][(cols + 1) / 2] and scales [rows][nblocks] into the layout above.  A
// block takes 128 rows x up to kQChunk columns, like the quantiser.
__global__ void __launch_bounds__(kQThreads)
k_f4_pack(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, const float* g, F4 m) {
    __shared__ uint32_t sf[kQChunk / 64 * kF4Atom / 4];
    extern __shared__ double n2[];
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
    for (int i = threadIdx.x; i < atoms * (kF4Atom / 4); i += kQThreads) sf[i] = 0;
    __syncthreads();
    for (int t = threadIdx.x; t < nr * U; t += kQThreads) {
        const int q = t / U, u = t - q * U;
        const uint8_t* src = codes + (long long)(r0 + q) * in_pitch;
        uint32_t w = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int c = c0 + 8 * u + 2 * i;
            if (c < m.cols) {
                uint32_t b = src[c / 2];
                if (c + 1 >= m.cols) b &= 15u;
                w |= b << (8 * i);
            }
        }
        reinterpret_cast<uint32_t*>(m.codes + (long long)(r0 + q) * m.pitch() + c0 / 2)[u] = w;
        const int blk = u >> sh, gblk = (m.nv ? c0 / 16 : c0 / 32) + blk;
        uint32_t byte = gblk < m.nblocks ? scales[(long long)(r0 + q) * m.nblocks + gblk] : 0u;
        if (m.nv) byte &= 0x7Fu;  // unsigned e4m3
        if ((u & ((1 << sh) - 1)) == 0)
            reinterpret_cast<uint8_t*>(sf)[blk / 4 * kF4Atom + (q % 32) * 16 + q / 32 * 4 + blk % 4] = (uint8_t)byte;
        if (bounds) {
            const double s = (double)f4_scale_value(m.nv, byte);
            n2[q * U + u] = (double)mag2(w) * (s * s);
        }
    }
    __syncthreads();
    uint32_t* dst = reinterpret_cast<uint32_t*>(m.scales + ((long long)tile * m.natoms + c0 / (m.nv ? 64 : 128)) * kF4Atom);
    for (int i = threadIdx.x; i < atoms * (kF4Atom / 4); i += kQThreads) dst[i] = sf[i];
    if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) m.gs[0] = g ? *g : 1.0f;
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

template <class T, bool kVec>
cudaError_t quantize_t(const T* x, long long ld, const F4& m, int sms, cudaStream_t st, int* launches) {
    const dim3 grid((unsigned)m.tiles(), (unsigned)((m.Kp + kQChunk - 1) / kQChunk));
    const size_t smem = m.Kp <= kF4TopkK ? (size_t)kF4Tile * (m.Kp / 8) * sizeof(double) : 0;
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
        const long long units = (long long)m.rows * ((m.cols + 7) / 8);
        const int blocks = (int)std::min<long long>((units + 255) / 256, (long long)sms * 8);
        k_f4_amax<T, kVec><<<blocks, 256, 0, st>>>(x, ld, m.rows, m.cols, reinterpret_cast<uint32_t*>(m.gs) + 1);
        k_f4_quantize<T, kVec, 1, false><<<grid, kQThreads, smem, st>>>(x, ld, m);
        *launches += 2;
    }
    return cudaGetLastError();
}

template <class T>
cudaError_t quantize_d(const void* x, long long ld, const F4& m, int sms, cudaStream_t st, int* launches) {
    const bool vec = ((uintptr_t)x & 15) == 0 && (ld * (long long)sizeof(T)) % 16 == 0;
    return vec ? quantize_t<T, true>((const T*)x, ld, m, sms, st, launches)
               : quantize_t<T, false>((const T*)x, ld, m, sms, st, launches);
}

template <class T>
cudaError_t dequantize_d(const F4& m, int r0, int r1, void* out, long long ld, cudaStream_t st) {
    const bool vec = m.cols % 8 == 0 && ((uintptr_t)out & 15) == 0 && (ld * (long long)sizeof(T)) % 16 == 0;
    const long long n = (long long)(r1 - r0) * (vec ? m.cols / 8 : m.cols);
    const int blocks = (int)std::min<long long>((n + 255) / 256, 1ll << 20);
    if (vec) k_f4_dequantize_vec<T><<<blocks, 256, 0, st>>>(m, r0, n, (T*)out, ld);
    else k_f4_dequantize_any<T><<<blocks, 256, 0, st>>>(m, r0, n, (T*)out, ld);
    return cudaGetLastError();
}

}  // namespace

cudaError_t f4_quantize(const void* x, int dtype, long long ld, const F4& m, int sms, cudaStream_t st,
                        int* launches) {
    if (dtype == RFX_F32) return quantize_d<float>(x, ld, m, sms, st, launches);
    if (dtype == RFX_BF16) return quantize_d<__nv_bfloat16>(x, ld, m, sms, st, launches);
    return quantize_d<__half>(x, ld, m, sms, st, launches);
}

cudaError_t f4_dequantize(const F4& m, int r0, int r1, void* out, int dtype, long long ld, cudaStream_t st) {
    if (dtype == RFX_F32) return dequantize_d<float>(m, r0, r1, out, ld, st);
    if (dtype == RFX_BF16) return dequantize_d<__nv_bfloat16>(m, r0, r1, out, ld, st);
    return dequantize_d<__half>(m, r0, r1, out, ld, st);
}

cudaError_t f4_pack(const uint8_t* codes, const uint8_t* scales, const float* g, const F4& m, cudaStream_t st) {
    const dim3 grid((unsigned)m.tiles(), (unsigned)((m.Kp + kQChunk - 1) / kQChunk));
    const size_t smem = m.Kp <= kF4TopkK ? (size_t)kF4Tile * (m.Kp / 8) * sizeof(double) : 0;
    k_f4_pack<<<grid, kQThreads, smem, st>>>(codes, scales, g, m);
    return cudaGetLastError();
}

cudaError_t f4_unpack(const F4& m, uint8_t* codes, uint8_t* scales, cudaStream_t st) {
    const long long n = (long long)m.rows * ((m.cols + 1) / 2 + m.nblocks);
    k_f4_unpack<<<(int)std::min<long long>((n + 255) / 256, 1 << 16), 256, 0, st>>>(m, codes, scales);
    return cudaGetLastError();
}

}  // namespace rfx
