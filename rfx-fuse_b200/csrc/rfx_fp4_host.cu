// C ABI of the microscaled 4-bit matrices (include/rfx_b200.h) and of the low-rank proximity
// held in them; kernels in rfx_fp4.cu, rfx_fp4_product.cu, rfx_fp4_topk.cu.
#include <cstring>
#include <mutex>

#include "rfx_ctx.h"
#include "rfx_fp4.h"
#include "rfx_tma_host.h"

namespace rfx {

bool f4_map(CUtensorMap* tm, const F4& m, int box_rows, int box_bytes) {
    std::memset(tm, 0, sizeof(*tm));
    const cuuint64_t dims[2] = {(cuuint64_t)m.pitch(), (cuuint64_t)m.rows};
    const cuuint64_t strides[1] = {(cuuint64_t)m.pitch()};
    const cuuint32_t box[2] = {(cuuint32_t)box_bytes, (cuuint32_t)box_rows};
    const cuuint32_t es[2] = {1, 1};
    return rfxh::encode_fn()(tm, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, m.codes, dims, strides, box, es,
                             CU_TENSOR_MAP_INTERLEAVE_NONE,
                             box_bytes == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_32B,
                             CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace rfx

namespace rfxh {

namespace {

using rfx::F4;

// [0] set by a kernel of the calls without a context whose pipeline wait timed out, taken by
// rfx_fp4_status; [1] what that took.  Contexts have words of their own.
__device__ int g_f4_err[4];

// Reads and clears in one step: a code that is set meanwhile is in this answer or the next.
__global__ void k_f4_take_err(int* err) { err[1] = atomicExch(err, 0); }

constexpr int kMaxDevices = 64;
constexpr int kMaxCols = 65535 * 256;  // a grid's second axis of 256 columns a block

// What a call needs to know about the current device, looked up once per device.
struct DeviceInfo {
    int sms = 0;
    int* err = nullptr;
};

DeviceInfo device_info() {
    static std::mutex mu;
    static DeviceInfo known[kMaxDevices];
    int dev = 0;
    RFX_CUDA(cudaGetDevice(&dev));
    require(dev >= 0 && dev < kMaxDevices, RFX_ERR_ARG, "device index out of range");
    std::lock_guard<std::mutex> lock(mu);
    DeviceInfo& d = known[dev];
    if (!d.err) {
        void* p = nullptr;
        RFX_CUDA(cudaGetSymbolAddress(&p, g_f4_err));
        RFX_CUDA(cudaDeviceGetAttribute(&d.sms, cudaDevAttrMultiProcessorCount, dev));
        d.err = (int*)p;
    }
    return d;
}

bool aligned(const void* p, size_t a) { return ((uintptr_t)p & (a - 1)) == 0; }

void check_shape(int format, int rows, int cols) {
    require(format == RFX_FP4_MX || format == RFX_FP4_NV, RFX_ERR_ARG, "format must be RFX_FP4_MX or RFX_FP4_NV");
    require(rows >= 0 && rows <= 0x7fffff00, RFX_ERR_ARG, "rows out of range");
    require(cols >= 1 && cols <= kMaxCols, RFX_ERR_ARG, "cols must be in [1, 16776960]");
}

F4 matrix_of(const rfx_fp4_matrix* m, const char* what) {
    require(m != nullptr, RFX_ERR_ARG, std::string(what) + ": null matrix");
    check_shape(m->format, m->rows, m->cols);
    const F4 f = rfx::f4_of(*m);
    require(m->scale_dev && aligned(m->scale_dev, 8), RFX_ERR_ARG, std::string(what) + ": null or unaligned scale");
    if (m->rows > 0) {
        require(m->codes_dev && m->scales_dev && aligned(m->codes_dev, 16) && aligned(m->scales_dev, 16),
                RFX_ERR_ARG, std::string(what) + ": null or unaligned codes or scales");
        require(f.Kp > rfx::kF4TopkK || (m->bounds_dev && aligned(m->bounds_dev, 4)), RFX_ERR_ARG,
                std::string(what) + ": null or unaligned bounds");
    }
    return f;
}

void check_dtype(int dtype) {
    require(dtype == RFX_F32 || dtype == RFX_BF16 || dtype == RFX_F16, RFX_ERR_ARG,
            "dtype must be RFX_F32, RFX_BF16 or RFX_F16");
}

void check_elements(const void* p, int dtype, const char* what) {
    require(p && aligned(p, dtype == RFX_F32 ? 4 : 2), RFX_ERR_ARG, std::string(what) + " is null or unaligned");
}

void check_pair(const F4& a, const F4& b) {
    require(a.nv == b.nv && a.cols == b.cols, RFX_ERR_ARG, "a and b must share format and cols");
}

void check_launch(cudaError_t e, const char* what) {
    if (e != cudaSuccess) throw RfxError(RFX_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(e));
}

void product(const F4& a, const F4& b, void* out, int dtype, long long ld, int* err, cudaStream_t st, int* launches) {
    check_launch(rfx::f4_product(a, b, out, dtype, ld, err, device_info().sms, st, launches), "rfx_fp4_product");
}

long long topk_bytes(const F4& a, const F4& b, int k) { return rfx::f4_topk_workspace(a, b, k, device_info().sms); }

void check_topk(const F4& a, const F4& b, int k) {
    check_pair(a, b);
    require(k >= 1 && k <= rfx::kF4TopMax, RFX_ERR_ARG, "k must be in [1, 64]");
    require(a.Kp <= rfx::kF4TopkK, RFX_ERR_UNSUPPORTED, "top-k needs at most 256 columns");
}

void topk(const F4& a, const F4& b, int k, long long self, int* idx, float* val, void* ws, int* err,
          cudaStream_t st, int* launches) {
    check_launch(rfx::f4_topk(a, b, k, self, idx, val, ws, err, device_info().sms, st, launches), "rfx_fp4_topk");
}

// Waits for the stream and throws if *err says that a wait of its kernels timed out.
void raise_if_timed_out(const int* err, cudaStream_t st) {
    int h = 0;
    RFX_CUDA(cudaMemcpyAsync(&h, err, 4, cudaMemcpyDeviceToHost, st));
    RFX_CUDA(cudaStreamSynchronize(st));
    if (h != 0)
        throw RfxError(RFX_ERR_DEVICE, "4-bit product kernel: a pipeline wait timed out (code " + std::to_string(h) + ")");
}

// A context's error word, cleared for a call.
int* ctx_err(Ctx& c) {
    int* err = (int*)c.lr_err.get(16);
    RFX_CUDA(cudaMemsetAsync(err, 0, 16, c.st));
    return err;
}

// The low-rank factors of a context in 4 bits.
F4 ctx_matrix(Ctx& c) {
    require(c.lr_ready && c.lr4_ready, RFX_ERR_STATE, "4-bit low-rank factors have not been made");
    return rfx::f4_of(c.lr4_m);
}

// Rows [r0, r1) widened to whole tiles at the front; *skip rows of the result are not asked for.
F4 rows_of(const F4& m, int r0, int r1, int* skip) {
    F4 v = m;
    const int b = r0 / rfx::kF4Tile * rfx::kF4Tile;
    *skip = r0 - b;
    v.rows = r1 - b;
    v.codes += (long long)b * m.pitch();
    v.scales += (long long)(b / rfx::kF4Tile) * m.natoms * rfx::kF4Atom;
    v.bounds += b / rfx::kF4Tile;
    return v;
}

}  // namespace

}  // namespace rfxh

using namespace rfxh;

extern "C" {

int rfx_fp4_sizes(int format, int rows, int cols, rfx_fp4_layout* out) {
    return guarded([&] {
        check_shape(format, rows, cols);
        require(out != nullptr, RFX_ERR_ARG, "null output");
        rfx_fp4_matrix m{};
        m.format = format;
        m.rows = rows;
        m.cols = cols;
        const F4 f = rfx::f4_of(m);
        out->pitch = f.pitch();
        out->tile_bytes = (long long)f.natoms * rfx::kF4Atom;
        out->codes = (long long)rows * out->pitch;
        out->scales = (long long)f.tiles() * out->tile_bytes;
        out->scale = 8;
        out->bounds = f.Kp <= rfx::kF4TopkK ? 4ll * f.tiles() : 0;
    });
}

int rfx_fp4_quantize(const void* x_dev, int dtype, long long row_stride, const rfx_fp4_matrix* out, void* stream) {
    return guarded([&] {
        const F4 m = matrix_of(out, "out");
        check_dtype(dtype);
        require(row_stride >= m.cols, RFX_ERR_ARG, "row_stride must be at least cols");
        cudaStream_t st = static_cast<cudaStream_t>(stream);
        int launches = 0;
        if (m.rows == 0) return check_launch(rfx::f4_unit_scale(m, st), "rfx_fp4_quantize");
        check_elements(x_dev, dtype, "x");
        check_launch(rfx::f4_quantize(x_dev, dtype, row_stride, m, device_info().sms, st, &launches), "rfx_fp4_quantize");
    });
}

int rfx_fp4_dequantize(const rfx_fp4_matrix* mat, int row_begin, int row_end, void* out_dev, int dtype,
                       long long ld, void* stream) {
    return guarded([&] {
        const F4 m = matrix_of(mat, "matrix");
        check_dtype(dtype);
        require(row_begin >= 0 && row_begin <= row_end && row_end <= m.rows, RFX_ERR_ARG, "bad row range");
        require(ld >= m.cols, RFX_ERR_ARG, "ld must be at least cols");
        if (row_begin == row_end) return;
        check_elements(out_dev, dtype, "out");
        check_launch(rfx::f4_dequantize(m, row_begin, row_end, out_dev, dtype, ld, static_cast<cudaStream_t>(stream)),
                     "rfx_fp4_dequantize");
    });
}

int rfx_fp4_pack(const uint8_t* codes_dev, const uint8_t* scales_dev, const float* scale_dev,
                 const rfx_fp4_matrix* out, void* stream) {
    return guarded([&] {
        const F4 m = matrix_of(out, "out");
        if (m.rows == 0) return check_launch(rfx::f4_unit_scale(m, static_cast<cudaStream_t>(stream)), "rfx_fp4_pack");
        require(codes_dev && scales_dev, RFX_ERR_ARG, "null codes or scales");
        require(!scale_dev || aligned(scale_dev, 4), RFX_ERR_ARG, "unaligned scale");
        check_launch(rfx::f4_pack(codes_dev, scales_dev, scale_dev, m, static_cast<cudaStream_t>(stream)), "rfx_fp4_pack");
    });
}

int rfx_fp4_unpack(const rfx_fp4_matrix* mat, uint8_t* codes_dev, uint8_t* scales_dev, void* stream) {
    return guarded([&] {
        const F4 m = matrix_of(mat, "matrix");
        if (m.rows == 0) return;
        require(codes_dev && scales_dev, RFX_ERR_ARG, "null output");
        check_launch(rfx::f4_unpack(m, codes_dev, scales_dev, static_cast<cudaStream_t>(stream)), "rfx_fp4_unpack");
    });
}

int rfx_fp4_product(const rfx_fp4_matrix* a_, const rfx_fp4_matrix* b_, void* out_dev, int dtype, long long ld,
                    void* stream) {
    return guarded([&] {
        const F4 a = matrix_of(a_, "a"), b = matrix_of(b_, "b");
        check_pair(a, b);
        check_dtype(dtype);
        require(ld >= b.rows, RFX_ERR_ARG, "ld must be at least b.rows");
        if (a.rows == 0 || b.rows == 0) return;
        check_elements(out_dev, dtype, "out");
        require(((long long)a.tiles() + 1) * b.tiles() < (1ll << 31), RFX_ERR_UNSUPPORTED, "product too large");
        int launches = 0;
        product(a, b, out_dev, dtype, ld, device_info().err, static_cast<cudaStream_t>(stream), &launches);
    });
}

int rfx_fp4_topk_workspace(const rfx_fp4_matrix* a_, const rfx_fp4_matrix* b_, int k, long long* bytes) {
    return guarded([&] {
        const F4 a = matrix_of(a_, "a"), b = matrix_of(b_, "b");
        check_topk(a, b, k);
        require(bytes != nullptr, RFX_ERR_ARG, "null output");
        *bytes = topk_bytes(a, b, k);
    });
}

int rfx_fp4_topk(const rfx_fp4_matrix* a_, const rfx_fp4_matrix* b_, int k, long long self, int* idx_dev,
                 float* val_dev, void* ws_dev, long long ws_bytes, void* stream) {
    return guarded([&] {
        const F4 a = matrix_of(a_, "a"), b = matrix_of(b_, "b");
        check_topk(a, b, k);
        require(self == -1 || (self >= 0 && self + a.rows <= b.rows), RFX_ERR_ARG,
                "self must be -1 or the first of a.rows rows of b");
        if (a.rows == 0) return;
        require(idx_dev && val_dev && aligned(idx_dev, 4) && aligned(val_dev, 4), RFX_ERR_ARG, "null or unaligned output");
        const long long need = topk_bytes(a, b, k);
        require(ws_bytes >= need && (need == 0 || (ws_dev && aligned(ws_dev, 16))), RFX_ERR_ARG,
                "the workspace is smaller than rfx_fp4_topk_workspace, null or unaligned");
        int launches = 0;
        topk(a, b, k, self, idx_dev, val_dev, ws_dev, device_info().err, static_cast<cudaStream_t>(stream), &launches);
    });
}

int rfx_fp4_status(void) {
    return guarded([&] {
        static std::mutex mu;  // of what k_f4_take_err leaves
        std::lock_guard<std::mutex> lock(mu);
        int* err = device_info().err;
        RFX_CUDA(cudaDeviceSynchronize());
        k_f4_take_err<<<1, 1>>>(err);
        check_launch(cudaGetLastError(), "rfx_fp4_status");
        raise_if_timed_out(err + 1, nullptr);
    });
}

int rfx_fp4_status_word(int** word_dev) {
    return guarded([&] {
        require(word_dev != nullptr, RFX_ERR_ARG, "null output");
        *word_dev = device_info().err;
    });
}

int rfx_lowrank_pack4(void* ctx, int format) {
    return guarded([&] {
        Ctx& c = *as_ctx(ctx);
        require(format == RFX_FP4_MX || format == RFX_FP4_NV, RFX_ERR_ARG, "format must be RFX_FP4_MX or RFX_FP4_NV");
        require(c.lr_ready && c.lr_float, RFX_ERR_STATE, "the float low-rank factors are gone: build them first");
        rfx_fp4_matrix m{};
        m.format = format;
        m.rows = c.lr_R;
        m.cols = c.lr_k;
        const F4 f = rfx::f4_of(m);
        const size_t codes = round_up((size_t)m.rows * f.pitch(), 256);
        const size_t scales = (size_t)f.tiles() * f.natoms * rfx::kF4Atom;
        c.lr4_ready = false;  // until the new factors are there
        uint8_t* p = (uint8_t*)c.lr4_buf.get(codes + scales + 256 + (size_t)f.tiles() * 4);
        m.codes_dev = p;
        m.scales_dev = p + codes;
        m.scale_dev = (float*)(p + codes + scales);
        m.bounds_dev = (float*)(p + codes + scales + 256);
        int launches = 0;
        check_launch(rfx::f4_quantize(c.lr_X.p, RFX_F32, c.lr_k, rfx::f4_of(m), c.sm_count, c.st, &launches),
                     "rfx_lowrank_pack4");
        c.launches += launches;
        RFX_CUDA(cudaStreamSynchronize(c.st));
        c.lr4_m = m;
        c.lr4_ready = true;
    });
}

int rfx_lowrank4_factors(void* ctx, float* A_host, int* rank_out, int* rows_out) {
    return guarded([&] {
        Ctx& c = *as_ctx(ctx);
        const F4 m = ctx_matrix(c);
        if (A_host) {
            const size_t n = (size_t)m.rows * m.cols * 4;
            float* out = (float*)c.lr_out_v.get(n);
            check_launch(rfx::f4_dequantize(m, 0, m.rows, out, RFX_F32, m.cols, c.st), "rfx_lowrank4_factors");
            c.launches += 1;
            RFX_CUDA(cudaMemcpyAsync(A_host, out, n, cudaMemcpyDeviceToHost, c.st));
            RFX_CUDA(cudaStreamSynchronize(c.st));
        }
        if (rank_out) *rank_out = m.cols;
        if (rows_out) *rows_out = m.rows;
    });
}

int rfx_lowrank4_topk(void* ctx, int k, int row_begin, int row_end, int* idx_host, float* val_host) {
    return guarded([&] {
        Ctx& c = *as_ctx(ctx);
        const F4 m = ctx_matrix(c);
        require(row_begin >= 0 && row_begin <= row_end && row_end <= m.rows, RFX_ERR_ARG, "bad row range");
        check_topk(m, m, k);
        require(idx_host && val_host, RFX_ERR_ARG, "null output");
        if (row_begin == row_end) return;
        int skip = 0;
        const F4 a = rows_of(m, row_begin, row_end, &skip);
        int* oi = (int*)c.lr_out_i.get((size_t)a.rows * k * 4);
        float* ov = (float*)c.lr_out_v.get((size_t)a.rows * k * 4);
        void* ws = c.lr_part.get((size_t)topk_bytes(a, m, k));
        int* err = ctx_err(c);
        int launches = 0;
        topk(a, m, k, row_begin - skip, oi, ov, ws, err, c.st, &launches);
        c.launches += launches;
        const size_t n = (size_t)(row_end - row_begin) * k * 4;
        RFX_CUDA(cudaMemcpyAsync(idx_host, oi + (size_t)skip * k, n, cudaMemcpyDeviceToHost, c.st));
        RFX_CUDA(cudaMemcpyAsync(val_host, ov + (size_t)skip * k, n, cudaMemcpyDeviceToHost, c.st));
        raise_if_timed_out(err, c.st);
    });
}

int rfx_lowrank4_product(void* ctx, int row_begin, int row_end, float* out_host) {
    return guarded([&] {
        Ctx& c = *as_ctx(ctx);
        const F4 m = ctx_matrix(c);
        require(row_begin >= 0 && row_begin <= row_end && row_end <= m.rows, RFX_ERR_ARG, "bad row range");
        require(out_host, RFX_ERR_ARG, "null output");
        if (row_begin == row_end) return;
        const int R = m.rows;
        // blocks of whole tiles of rows, so that only the first computes rows that are not asked for:
        // up to 256 MB of device scratch, or one tile's rows where those take more
        const int chunk = (int)std::max<long long>(1, ((long long)256 << 20) / ((long long)R * 4 * rfx::kF4Tile)) * rfx::kF4Tile;
        const int first = row_begin / rfx::kF4Tile * rfx::kF4Tile;
        int* err = ctx_err(c);
        float* buf = (float*)c.lr_out_v.get((size_t)std::min(chunk, row_end - first) * R * 4);
        for (int b0 = first; b0 < row_end; b0 += std::min(chunk, row_end - b0)) {
            const int r0 = std::max(b0, row_begin), r1 = b0 + std::min(chunk, row_end - b0);
            int skip = 0;
            const F4 a = rows_of(m, r0, r1, &skip);
            int launches = 0;
            product(a, m, buf, RFX_F32, R, err, c.st, &launches);
            c.launches += launches;
            RFX_CUDA(cudaMemcpyAsync(out_host + (size_t)(r0 - row_begin) * R, buf + (size_t)skip * R,
                                     (size_t)(r1 - r0) * R * 4, cudaMemcpyDeviceToHost, c.st));
            raise_if_timed_out(err, c.st);
        }
    });
}

}  // extern "C"
