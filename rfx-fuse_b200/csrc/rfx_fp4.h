// Matrices in microscaled 4 bits: layout, kernels and launchers (rfx_fp4.cu, rfx_fp4_product.cu,
// rfx_fp4_topk.cu; C ABI in rfx_fp4_host.cu).
//
// codes   [rows][pitch] bytes, two e2m1 codes a byte (even column low); pitch = Kp / 2 with
//         Kp = cols rounded up to 64, so that every row starts on 32 bytes (TMA) and a tensor-core
//         step of 64 columns never leaves it; the columns from cols on hold code 0.
// scales  [row tile of 128][atom][512]: an atom is 128 rows x 4 scales in the order in which
//         tcgen05.cp spreads scales over TMEM (row r, scale b at (r % 32) * 16 + r / 32 * 4 + b),
//         so a tile's scales are one contiguous copy.  Rows and scales that do not exist hold 0.
// gs      [0] matrix scale g, [1] scratch of the quantiser.
// bounds  [row tile] a bound of the tile's row norms in units of g (inf: none); only matrices
//         with Kp <= kF4TopkK have it.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <cstdint>

#include "../../include/rfx_b200.h"

namespace rfx {

constexpr int kF4Tile = 128;    // rows of a scale tile
constexpr int kF4Atom = 512;    // bytes of a scale atom
constexpr int kF4TopkK = 256;   // widest matrix of the top-k (one shared-memory row)
constexpr int kF4TopMax = 64;   // neighbours at most

struct F4 {
    int nv;        // 1: nvfp4 (16-column blocks, e4m3), 0: mxfp4 (32-column blocks, e8m0)
    int rows, cols;
    int Kp;        // padded columns
    int natoms;    // scale atoms of a row tile
    int nblocks;   // scales of a row, ceil(cols / block)
    uint8_t* codes;
    uint8_t* scales;
    float* gs;
    float* bounds;
    __host__ __device__ int pitch() const { return Kp / 2; }
    __host__ __device__ int tiles() const { return (int)(((long long)rows + kF4Tile - 1) / kF4Tile); }
};

inline F4 f4_of(const rfx_fp4_matrix& m) {
    F4 f;
    f.nv = m.format == RFX_FP4_NV;
    f.rows = m.rows;
    f.cols = m.cols;
    f.Kp = (m.cols + 63) / 64 * 64;
    f.natoms = f.nv ? f.Kp / 64 : (f.Kp + 127) / 128;
    const int bs = f.nv ? 16 : 32;
    f.nblocks = (m.cols + bs - 1) / bs;
    f.codes = m.codes_dev;
    f.scales = m.scales_dev;
    f.gs = m.scale_dev;
    f.bounds = m.bounds_dev;
    return f;
}

// Byte of scale `blk` of row `r`.
__host__ __device__ inline long long f4_scale_at(const F4& m, long long r, int blk) {
    const int q = (int)(r % kF4Tile);
    return ((r / kF4Tile) * m.natoms + blk / 4) * kF4Atom + (q % 32) * 16 + q / 32 * 4 + blk % 4;
}

// Launchers: enqueue on `st`, return the launch status.
cudaError_t f4_unit_scale(const F4& m, cudaStream_t st);
cudaError_t f4_quantize(const void* x, int dtype, long long ld, const F4& m, int sms, cudaStream_t st,
                        int* launches);
cudaError_t f4_dequantize(const F4& m, int r0, int r1, void* out, int dtype, long long ld, cudaStream_t st);
cudaError_t f4_pack(const uint8_t* codes, const uint8_t* scales, const float* g, const F4& m, cudaStream_t st);
cudaError_t f4_unpack(const F4& m, uint8_t* codes, uint8_t* scales, cudaStream_t st);

// Tensor map of a matrix's code rows: boxes of `box_rows` rows x `box_bytes` bytes (32 or 128,
// swizzled over the box row).  False when the driver refuses it.
bool f4_map(CUtensorMap* tm, const F4& m, int box_rows, int box_bytes);

struct F4ProductArgs {
    F4 a, b;          // out[i][j] = a_i . b_j
    void* out;
    long long ld;
    int dtype;        // RFX_F32 / RFX_BF16 / RFX_F16
    int bn;           // rows of a in a tile (multiple of 16, <= 256)
    int njt, nit;     // tiles of b and of a (njt * nit < 2^31)
    int ntiles, group; // their number, tiles of a unit of scheduling
    int nchunk;       // chunks of the inner axis
    int split;        // blocks of a cluster that share one tile's inner axis
    int nstage, nacc; // shared-memory ring, accumulator ring
    int acc_cols;     // TMEM columns of an accumulator
    int stage_bytes;
    int* err;
};
cudaError_t f4_product(const F4& a, const F4& b, void* out, int dtype, long long ld, int* err, int sms,
                       cudaStream_t st, int* launches);

long long f4_topk_workspace(const F4& a, const F4& b, int k, int sms);
cudaError_t f4_topk(const F4& a, const F4& b, int k, long long self, int* idx, float* val, void* ws,
                    int* err, int sms, cudaStream_t st, int* launches);

}  // namespace rfx
