// psgdk_mx.hip -- the C ABI of the microscaled (MX) operators but the product (include/psgdk.h, "microscaled numbers"): argument checks, choice of
// kernel, launches.  Nothing here shares state with a plan; every call is stream-ordered and keeps nothing.
#include <type_traits>
#include "mx_host.hiph"

// calls f with a null pointer of the element type
template <typename F>
static int mx_by_dtype(int d, F&& f) {
    return d == PSGDK_BF16 ? f((bf16_t*)nullptr) : d == PSGDK_F32 ? f((float*)nullptr) : f((mx_half*)nullptr);
}

template <typename T, int FMT, bool NOISE>
static int mx_launch_round(const MxJobs& a, unsigned grid, bool rows, bool cols, hipStream_t st) {
    if (!cols) mx_rows_kernel<T, FMT, NOISE><<<grid, 256, 0, st>>>(a);
    else if (rows) mx_tile_kernel<T, FMT, true, NOISE, false><<<grid, 128 * sizeof(T), 0, st>>>(a, MxNormArgs{nullptr, nullptr, 0});
    else mx_tile_kernel<T, FMT, false, NOISE, false><<<grid, 128 * sizeof(T), 0, st>>>(a, MxNormArgs{nullptr, nullptr, 0});
    MX_LAUNCHED();
    return PSGDK_OK;
}

template <typename T, int FMT, int THREADS, int CH>
static void mx_norm_one(const void* x, const void* res, const void* gain, int gdt, void* s, float* inv, uint8_t* codes, uint8_t* scales, int rows,
                        int cols, float eps, hipStream_t st) {
    const unsigned grid = THREADS == 64 ? (rows + 3) / 4 : rows;
    rms_norm_mx_kernel<T, FMT, THREADS, CH><<<grid, 256, 0, st>>>((const T*)x, (const T*)res, gain, gdt, (T*)s, inv, codes, scales, rows, cols, 1.0 / cols, eps);
}
// one wave a row up to 2048 columns, a workgroup a row up to 16384
template <typename T, int FMT, typename... A>
static void mx_norm_by_cols(int cols, A... a) {
    if (cols <= 512) mx_norm_one<T, FMT, 64, 1>(a...);
    else if (cols <= 1024) mx_norm_one<T, FMT, 64, 2>(a...);
    else if (cols <= 2048) mx_norm_one<T, FMT, 64, 4>(a...);
    else if (cols <= 4096) mx_norm_one<T, FMT, 256, 2>(a...);
    else if (cols <= 8192) mx_norm_one<T, FMT, 256, 4>(a...);
    else mx_norm_one<T, FMT, 256, 8>(a...);
}

template <typename T, typename TD, int THREADS, int CH>
static void mx_norm_back_one(unsigned grid, const void* dy, const void* s, const void* gain, int gdt, const float* inv, const void* ds, void* dx,
                             float* part, int rows, int cols, hipStream_t st) {
    rms_norm_mx_backward_kernel<T, TD, THREADS, CH>
        <<<grid, 256, 0, st>>>((const TD*)dy, (const T*)s, gain, gdt, inv, (const T*)ds, (T*)dx, part, rows, cols);
}
template <typename T, typename TD, typename... A>
static void mx_norm_back_by_cols(int cols, A... a) {
    if (cols <= 512) mx_norm_back_one<T, TD, 64, 1>(a...);
    else if (cols <= 1024) mx_norm_back_one<T, TD, 64, 2>(a...);
    else if (cols <= 2048) mx_norm_back_one<T, TD, 64, 4>(a...);
    else if (cols <= 4096) mx_norm_back_one<T, TD, 256, 2>(a...);
    else if (cols <= 8192) mx_norm_back_one<T, TD, 256, 4>(a...);
    else mx_norm_back_one<T, TD, 256, 8>(a...);
}
// lines of the gain gradient's shares: enough workgroups to fill the chip, no more (every line costs 8 bytes a column)
static int mx_back_lines(int64_t rows, int64_t cols) {
    const int64_t per = cols <= 2048 ? 4 : 1, want = (rows + per - 1) / per;
    return (int)(want < 512 ? want : 512);
}

extern "C" {

int psgdk_mx_storage(int64_t rows, int64_t cols, int fmt, int64_t* code_bytes, int64_t* scale_bytes) {
    if (rows < 0 || cols < 0 || rows > kMaxDim || cols > kMaxDim || !mx_fmt_ok(fmt) || !code_bytes || !scale_bytes) return PSGDK_ERR_INVALID;
    *code_bytes = rows * (mx_pad(cols) * fmt / 8);
    *scale_bytes = rows * (mx_pad(cols) / MX_BLOCK);
    return PSGDK_OK;
}

int psgdk_mx_quantize(int count, const psgdk_mx_tensor* t, int dtype, int fmt, void* stream) {
    if (count < 0 || (count && !t) || !mx_dtype_ok(dtype) || !mx_fmt_ok(fmt)) return PSGDK_ERR_INVALID;
    for (int i = 0; i < count; ++i)
        if (t[i].rows < 0 || t[i].cols < 0 || t[i].rows > kMaxDim || t[i].cols > kMaxDim || t[i].ld < t[i].cols) return PSGDK_ERR_INVALID;
    if (count == 0) return PSGDK_OK;
    int f = 0;                                            // the first tensor that has elements says what is written; the others agree
    while (f < count - 1 && (t[f].rows == 0 || t[f].cols == 0)) ++f;
    if (t[f].rows == 0 || t[f].cols == 0) return PSGDK_OK;
    const bool rows = t[f].codes != nullptr, cols = t[f].codes_t != nullptr, noise = t[f].noise != nullptr;
    if ((!rows && !cols) || (noise && fmt != PSGDK_MX_FP4)) return PSGDK_ERR_INVALID;
    const int64_t most = kMaxThreads / (cols ? 128 * mx_size(dtype) : 256);      // workgroups of a launch
    // rows: units of 256 elements, 8 a workgroup; tiles: 128 x 128 over the padded extent of what is written
    const auto across = [&](const psgdk_mx_tensor& q) { return cols ? (rows ? mx_pad(q.cols) : q.cols + 127) / 128 : mx_pad(q.cols) / MX_PAD; };
    const auto needs = [&](const psgdk_mx_tensor& q) { return cols ? mx_pad(q.rows) / 128 * across(q) : (q.rows * across(q) + 7) / 8; };
    for (int i = 0; i < count; ++i) {
        const psgdk_mx_tensor& q = t[i];
        if (q.rows == 0 || q.cols == 0) continue;
        if (!q.x || (q.codes != nullptr) != rows || (q.codes_t != nullptr) != cols || (q.noise != nullptr) != noise) return PSGDK_ERR_INVALID;
        if ((rows && !q.scales) || (cols && !q.scales_t)) return PSGDK_ERR_INVALID;
        if (!mx_aligned(q.x, mx_size(dtype)) || !mx_aligned(q.codes, 16) || !mx_aligned(q.codes_t, 16)) return PSGDK_ERR_INVALID;
    }
    for (int i = 0; i < count; ++i)
        if (t[i].rows && t[i].cols && needs(t[i]) > most) return PSGDK_ERR_UNSUPPORTED;          // (before the first launch: all of the tensors or none)
    const hipStream_t st = (hipStream_t)stream;
    for (int i = 0; i < count;) {
        MxJobs a;
        a.n = 0;
        int64_t wgs = 0;
        for (; i < count && a.n < MX_JOBS; ++i) {
            const psgdk_mx_tensor& q = t[i];
            if (q.rows == 0 || q.cols == 0) continue;
            const int64_t need = needs(q);
            if (wgs + need > most) break;
            MxJob& j = a.j[a.n++];
            j = MxJob{q.x, (const uint8_t*)q.noise, (uint8_t*)q.codes, (uint8_t*)q.scales, (uint8_t*)q.codes_t, (uint8_t*)q.scales_t, q.ld, (int)q.rows,
                      (int)q.cols, (unsigned)wgs, FastDiv::make((unsigned)across(q))};
            wgs += need;
        }
        if (a.n == 0) continue;
        const int rc = mx_by_dtype(dtype, [&](auto* e) {
            using T = std::remove_pointer_t<decltype(e)>;
            if (fmt == PSGDK_MX_FP8) return mx_launch_round<T, 8, false>(a, (unsigned)wgs, rows, cols, st);
            return noise ? mx_launch_round<T, 4, true>(a, (unsigned)wgs, rows, cols, st) : mx_launch_round<T, 4, false>(a, (unsigned)wgs, rows, cols, st);
        });
        if (rc != PSGDK_OK) return rc;
    }
    return PSGDK_OK;
}

int psgdk_mx_dequantize(const void* codes, const void* scales, int64_t rows, int64_t cols, int fmt, void* out, int out_dtype, void* stream) {
    if (rows < 0 || cols < 0 || rows > kMaxDim || cols > kMaxDim || !mx_fmt_ok(fmt) || !mx_dtype_ok(out_dtype)) return PSGDK_ERR_INVALID;
    if (rows == 0 || cols == 0) return PSGDK_OK;
    if (!codes || !scales || !out || !mx_aligned(codes, 16) || !mx_aligned(out, mx_size(out_dtype))) return PSGDK_ERR_INVALID;
    const int64_t units = mx_pad(cols) / MX_PAD, need = (rows * units + 7) / 8;
    if (need > kMaxThreads / 256) return PSGDK_ERR_UNSUPPORTED;
    const FastDiv div = FastDiv::make((unsigned)units);
    const hipStream_t st = (hipStream_t)stream;
    return mx_by_dtype(out_dtype, [&](auto* e) {
        using T = std::remove_pointer_t<decltype(e)>;
#define MX_DEQ(F) mx_dequantize_kernel<T, F><<<(unsigned)need, 256, 0, st>>>((const uint8_t*)codes, (const uint8_t*)scales, (T*)out, (int)rows, (int)cols, div)
        if (fmt == PSGDK_MX_FP4) MX_DEQ(4);
        else MX_DEQ(8);
#undef MX_DEQ
        MX_LAUNCHED();
        return (int)PSGDK_OK;
    });
}

int psgdk_rms_norm_mx(const void* x, const void* residual, const void* gain, int gain_dtype, int64_t rows, int64_t cols, int dtype, float eps, int fmt,
                      void* s, float* inv, void* codes, void* scales, void* codes_t, void* scales_t, void* stream) {
    if (rows < 0 || cols < 1 || rows > kMaxDim || !mx_dtype_ok(dtype) || !mx_dtype_ok(gain_dtype) || !mx_fmt_ok(fmt) || !(eps >= 0.0f)) return PSGDK_ERR_INVALID;
    if (cols > PSGDK_NORM_MAX_COLS) return PSGDK_ERR_UNSUPPORTED;
    if (rows == 0) return PSGDK_OK;
    if (!x || !gain || !inv || (residual && !s) || (!codes && !codes_t) || (codes && !scales) || (codes_t && !scales_t)) return PSGDK_ERR_INVALID;
    const int size = mx_size(dtype);
    if (!mx_aligned(x, size) || !mx_aligned(residual, size) || !mx_aligned(s, size) || !mx_aligned(gain, mx_size(gain_dtype)) || !mx_aligned(inv, 4) ||
        !mx_aligned(codes, 16) || !mx_aligned(codes_t, 16)) return PSGDK_ERR_INVALID;
    const hipStream_t st = (hipStream_t)stream;
    const int64_t tiles_n = (cols + 127) / 128, tiles = mx_pad(rows) / 128 * tiles_n;
    if ((cols <= 2048 ? (rows + 3) / 4 : rows) > kMaxThreads / 256 || (codes_t && tiles > kMaxThreads / (128 * size))) return PSGDK_ERR_UNSUPPORTED;
    return mx_by_dtype(dtype, [&](auto* e) {
        using T = std::remove_pointer_t<decltype(e)>;
#define MX_NORM(F) mx_norm_by_cols<T, F>((int)cols, x, residual, gain, gain_dtype, s, inv, (uint8_t*)codes, (uint8_t*)scales, (int)rows, (int)cols, eps, st)
        if (!codes) MX_NORM(0);
        else if (fmt == PSGDK_MX_FP4) MX_NORM(4);
        else MX_NORM(8);
#undef MX_NORM
        MX_LAUNCHED();
        if (codes_t) {
            MxJobs a;
            a.n = 1;
            a.j[0] = MxJob{residual ? s : x, nullptr, nullptr, nullptr, (uint8_t*)codes_t, (uint8_t*)scales_t, cols, (int)rows, (int)cols, 0u,
                           FastDiv::make((unsigned)tiles_n)};
            const MxNormArgs n{inv, gain, gain_dtype};
#define MX_NT(F) mx_tile_kernel<T, F, false, false, true><<<(unsigned)tiles, 128 * sizeof(T), 0, st>>>(a, n)
            if (fmt == PSGDK_MX_FP4) MX_NT(4);
            else MX_NT(8);
#undef MX_NT
            MX_LAUNCHED();
        }
        return (int)PSGDK_OK;
    });
}

int psgdk_rms_norm_mx_backward_work_bytes(int64_t rows, int64_t cols, size_t* bytes) {
    if (rows < 0 || cols < 1 || rows > kMaxDim || !bytes) return PSGDK_ERR_INVALID;
    if (cols > PSGDK_NORM_MAX_COLS) return PSGDK_ERR_UNSUPPORTED;
    *bytes = (size_t)mx_back_lines(rows, cols) * cols * 4;
    return PSGDK_OK;
}

int psgdk_rms_norm_mx_backward(const void* dy, int dy_dtype, const void* s, const void* gain, int gain_dtype, const float* inv, const void* ds,
                               int64_t rows, int64_t cols, int dtype, void* dx, float* dgain, void* work, size_t work_bytes, void* stream) {
    if (rows < 0 || cols < 1 || rows > kMaxDim || !mx_dtype_ok(dtype) || !mx_dtype_ok(gain_dtype)) return PSGDK_ERR_INVALID;
    if (dy_dtype != dtype && dy_dtype != PSGDK_F32) return PSGDK_ERR_INVALID;
    if (cols > PSGDK_NORM_MAX_COLS) return PSGDK_ERR_UNSUPPORTED;
    if (!dgain || !mx_aligned(dgain, 4)) return PSGDK_ERR_INVALID;
    const int lines = mx_back_lines(rows, cols), size = mx_size(dtype);
    if (rows > 0) {
        if (!dy || !s || !gain || !inv || !dx || !work || work_bytes < (size_t)lines * cols * 4 || !mx_aligned(work, 4)) return PSGDK_ERR_INVALID;
        if (!mx_aligned(dy, mx_size(dy_dtype)) || !mx_aligned(s, size) || !mx_aligned(ds, size) || !mx_aligned(dx, size) || !mx_aligned(inv, 4) ||
            !mx_aligned(gain, mx_size(gain_dtype))) return PSGDK_ERR_INVALID;
    }
    const hipStream_t st = (hipStream_t)stream;
    if (rows > 0) {
        const int rc = mx_by_dtype(dtype, [&](auto* e) {
            using T = std::remove_pointer_t<decltype(e)>;
#define MX_BACK(TD) mx_norm_back_by_cols<T, TD>((int)cols, (unsigned)lines, dy, s, gain, gain_dtype, inv, ds, dx, (float*)work, (int)rows, (int)cols, st)
            if (dy_dtype == PSGDK_F32) MX_BACK(float);
            else MX_BACK(T);
#undef MX_BACK
            MX_LAUNCHED();
            return (int)PSGDK_OK;
        });
        if (rc != PSGDK_OK) return rc;
    }
    rms_norm_mx_dgain_kernel<<<(unsigned)((cols + 31) / 32), 1024, 0, st>>>((const float*)work, dgain, rows > 0 ? lines : 0, (int)cols);
    MX_LAUNCHED();
    return PSGDK_OK;
}

}  // extern "C"
