// psgdk_mx_gemm.hip -- psgdk_mx_matmul (include/psgdk.h, "microscaled numbers"): argument checks, choice of kernel, launches.
#include <cmath>
#include "../../include/psgdk_test.h"
#include "mx_host.hiph"
#include "gemm_mx.hiph"

// a 32-bit output with an 8-bit operand: fp32 sums through bf16 products (gemm_mx.hiph)
static bool mx_wide(int a_fmt, int b_fmt, int out_dtype) { return out_dtype == PSGDK_F32 && (a_fmt == PSGDK_MX_FP8 || b_fmt == PSGDK_MX_FP8); }
struct MxPlan { bool skinny; int mt, kw, bm, bn, splits; };
static MxPlan mx_plan(int64_t M, int64_t N, int64_t KS, int a_fmt, int b_fmt, bool wide) {
    MxPlan p{};
    p.splits = 1;
    // Few rows: the kernel without LDS reads A anew for every 16 rows of B, the tiles once for 128.  Measured (fp8 x fp4, us, without / tiles): M = 5:
    // N = K = 4096 4.8 / 8.8, 8192 13.3 / 13.4; M = 16: 6.0 / 9.4, 17.4 / 13.9, 50257 x 768 10.9 / 8.2; M = 64: 12.8 / 12.7, 42.7 / 18.0; M = 1:
    // 50257 x 768 6.8 without (A's one row costs nothing).
    const int64_t mt = (M + 15) / 16;
    if (M <= 4 || (M <= 64 && mt * N * KS <= (1ll << 25) / 256)) {
        p.skinny = true;
        p.mt = (int)mt;
        p.kw = 1;                                        // two waves a SIMD or more, none without a share of K
        while (p.kw < 8 && (N + 15) / 16 * p.kw < 2048 && p.kw < KS) p.kw *= 2;
        return p;
    }
    // Tiles: the size and the number of splits of K with the smallest estimated time.  Microseconds for 256 elements of K, measured at 4096 x 4096 and
    // 2048 x 2048: a workgroup alone on its CU, and (128 rows) each of two; for the prologue and stores of a round of tiles; a split adds a launch and
    // fp32 sums that are written and read once.
    const bool four = a_fmt == PSGDK_MX_FP4 && b_fmt == PSGDK_MX_FP4;
    const double big = four ? 1.9 : 2.8, alone = wide ? 1.9 : four ? 0.8 : 1.3, pair = wide ? 3.0 : four ? 1.04 : 1.67;
    double best = 1e30;
    for (int bm = 256; bm >= 64; bm /= 2) {
        if ((bm == 64) != (M <= 64) || (bm == 256 && wide)) continue;
        const int bn = bm == 256 ? 256 : 128;
        const double tiles = (double)((M + bm - 1) / bm) * ((N + bn - 1) / bn);
        for (int splits = 1; splits <= 16 && (splits == 1 || splits * 2 <= KS); splits *= 2) {
            const double wgs = tiles * splits, blocks = (double)((KS + splits - 1) / splits);
            double t = bm == 256 ? std::ceil(wgs / 256) * (blocks * big + 6.0)
                                 : (wgs <= 256 ? blocks * alone + 2.2 : std::ceil(wgs / 512) * (blocks * pair + 2.2)) * (bm == 64 ? 0.7 : 1.0);
            if (splits > 1) t += 4.0 + (double)M * N * splits * 8 / 4.5e6;
            if (t < best) { best = t; p.bm = bm; p.bn = bn; p.splits = splits; }
        }
    }
    return p;
}

template <int FA, int FB, bool WIDE>
static int mx_launch_product(const MxGemm& g, const MxPlan& p, hipStream_t st) {
    if (p.skinny) {
        const int64_t groups = ((int64_t)g.N + 15) / 16;
        const int waves = p.kw == 8 ? 8 : 4;
        const unsigned grid = (unsigned)((groups * p.kw + waves - 1) / waves), lds = p.kw > 1 ? waves * p.mt * 1024 : 0;
#define MX_SKINNY(MT) if (p.mt == MT) mx_skinny_kernel<FA, FB, WIDE, MT><<<grid, waves * 64, lds, st>>>(g, p.kw);
        MX_SKINNY(1) MX_SKINNY(2) MX_SKINNY(3) MX_SKINNY(4)
#undef MX_SKINNY
    } else {
        const unsigned grid = (unsigned)((int64_t)g.tiles_m * g.tiles_n * g.splits);
        if constexpr (!WIDE) if (p.bm == 256) mx_tile_gemm_kernel<FA, FB, WIDE, 256, 256, 2><<<grid, 256, 0, st>>>(g);
        if (p.bm == 128) mx_tile_gemm_kernel<FA, FB, WIDE, 128, 128, 2><<<grid, 256, 0, st>>>(g);
        if (p.bm == 64) mx_tile_gemm_kernel<FA, FB, WIDE, 64, 128, 2><<<grid, 256, 0, st>>>(g);
    }
    MX_LAUNCHED();
    if (g.part) {
        const int64_t total = (int64_t)g.M * g.N;
        mx_join_kernel<<<(unsigned)((total + 1023) / 1024), 256, 0, st>>>(g.part, g.out, g.out_dtype, g.splits, total);
        MX_LAUNCHED();
    }
    return PSGDK_OK;
}

extern "C" {

int psgdk_mx_matmul_work_bytes(int64_t m, int64_t n, int64_t k, int a_fmt, int b_fmt, int out_dtype, size_t* bytes) {
    if (m < 0 || n < 0 || k < 0 || m > kMaxDim || n > kMaxDim || k > kMaxDim || !bytes) return PSGDK_ERR_INVALID;
    if (!mx_fmt_ok(a_fmt) || !mx_fmt_ok(b_fmt) || !mx_dtype_ok(out_dtype)) return PSGDK_ERR_INVALID;
    const MxPlan p = mx_plan(m, n, mx_pad(k) / MX_PAD, a_fmt, b_fmt, mx_wide(a_fmt, b_fmt, out_dtype));
    *bytes = p.splits > 1 ? (size_t)p.splits * m * n * 4 : 0;
    return PSGDK_OK;
}

int psgdk_mx_matmul(const void* a_codes, const void* a_scales, int64_t m, int a_fmt, const void* b_codes, const void* b_scales, int64_t n, int b_fmt,
                    int64_t k, void* out, int out_dtype, void* work, size_t work_bytes, void* stream) {
    if (m < 0 || n < 0 || k < 0 || m > kMaxDim || n > kMaxDim || k > kMaxDim) return PSGDK_ERR_INVALID;
    if (!mx_fmt_ok(a_fmt) || !mx_fmt_ok(b_fmt) || !mx_dtype_ok(out_dtype)) return PSGDK_ERR_INVALID;
    if (k > kMaxK || n > kMaxN) return PSGDK_ERR_UNSUPPORTED;
    if (m == 0 || n == 0) return PSGDK_OK;
    if (!out || !mx_aligned(out, mx_size(out_dtype))) return PSGDK_ERR_INVALID;
    if (k > 0 && (!a_codes || !a_scales || !b_codes || !b_scales)) return PSGDK_ERR_INVALID;
    if (!mx_aligned(a_codes, 16) || !mx_aligned(b_codes, 16) || !mx_aligned(a_scales, 8) || !mx_aligned(b_scales, 8)) return PSGDK_ERR_INVALID;
    const int64_t KS = mx_pad(k) / MX_PAD;
    const bool wide = mx_wide(a_fmt, b_fmt, out_dtype);
    const MxPlan p = mx_plan(m, n, KS, a_fmt, b_fmt, wide);
    const size_t need = p.splits > 1 ? (size_t)p.splits * m * n * 4 : 0;
    if (need && (!work || work_bytes < need || !mx_aligned(work, 16))) return PSGDK_ERR_INVALID;
    const int64_t tm = p.skinny ? 1 : (m + p.bm - 1) / p.bm, tn = p.skinny ? 1 : (n + p.bn - 1) / p.bn;
    if (tm * tn * p.splits > kMaxThreads / 256 || (need && (m * n + 1023) / 1024 > kMaxThreads / 256)) return PSGDK_ERR_UNSUPPORTED;
    const MxGemm g{(const uint8_t*)a_codes, (const uint8_t*)a_scales, (const uint8_t*)b_codes, (const uint8_t*)b_scales, out, need ? (float*)work : nullptr, n,
                   (int)m, (int)n, (int)KS, out_dtype, p.splits, (int)tm, (int)tn};
    const hipStream_t st = (hipStream_t)stream;
    if (a_fmt == PSGDK_MX_FP4 && b_fmt == PSGDK_MX_FP4) return mx_launch_product<4, 4, false>(g, p, st);
    if (wide) {
        if (a_fmt == PSGDK_MX_FP4) return mx_launch_product<4, 8, true>(g, p, st);
        return b_fmt == PSGDK_MX_FP4 ? mx_launch_product<8, 4, true>(g, p, st) : mx_launch_product<8, 8, true>(g, p, st);
    }
    if (a_fmt == PSGDK_MX_FP4) return mx_launch_product<4, 8, false>(g, p, st);
    return b_fmt == PSGDK_MX_FP4 ? mx_launch_product<8, 4, false>(g, p, st) : mx_launch_product<8, 8, false>(g, p, st);
}

int psgdk_test_mx_plan(int64_t m, int64_t n, int64_t k, int a_fmt, int b_fmt, int out_dtype, int* rows, int* cols, int* splits, int* wide) {
    if (m < 1 || n < 1 || k < 0 || m > kMaxDim || n > kMaxDim || k > kMaxDim || !rows || !cols || !splits || !wide) return PSGDK_ERR_INVALID;
    if (!mx_fmt_ok(a_fmt) || !mx_fmt_ok(b_fmt) || !mx_dtype_ok(out_dtype)) return PSGDK_ERR_INVALID;
    *wide = mx_wide(a_fmt, b_fmt, out_dtype);
    const MxPlan p = mx_plan(m, n, mx_pad(k) / MX_PAD, a_fmt, b_fmt, *wide);
    *rows = p.skinny ? 16 * p.mt : p.bm;
    *cols = p.skinny ? 0 : p.bn;
    *splits = p.skinny ? p.kw : p.splits;
    return PSGDK_OK;
}

}  // extern "C"
