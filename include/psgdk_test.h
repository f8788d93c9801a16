/*
 * psgdk_test.h -- kernel-level TEST and BENCHMARK hooks of libpsgdk.so (used by tests/, tools/ and bench.py only).
 *
 * They are exported by the same shared library as the drop-in ABI (include/psgdk.h) but are not part of it: nothing here
 * replaces a function of the reference, and a maintainer binding the library into the reference needs none of it.
 */
#ifndef PSGDK_TEST_H
#define PSGDK_TEST_H

#include "psgdk.h"

#ifdef __cplusplus
extern "C" {
#endif

/* The draws of the PRODUCTION noise path, written out so that an oracle can replay them: what psgdk_accumulate's fused damping
 * branch / the update's own damping stage (psgd.py:402-403: randn_like(G)) and the norm-bound start blocks (psgd.py:62 and :87:
 * randn(32, d) per dense factor) draw from the built-in Philox stream for (seed, offset) -- generated by the SAME device
 * functions the fused kernels call (tile_noise / nlb_philox4), in the same tile mapping, then scattered to logical layout.
 *   g_out[t]                      : numel(t) values of the preconditioner dtype, logical (row-major) order; NULL entries are skipped
 *   spd_out[t*PSGDK_MAX_DIMS+i]   : 32 x d_i values for dense factor i of tensor t (chain 0, psgd.py:62); NULL entries are skipped
 *   skh_out[t*PSGDK_MAX_DIMS+i]   : the same for chain 1 (psgd.py:87)
 * All three are HOST arrays of DEVICE pointers (the layout of psgdk_noise); any of the three arrays may be NULL.
 * pro_iter: -1, or the rotation number of PRO4P whose start blocks are wanted (psgd.py:447-450). */
int psgdk_test_dump_noise(psgdk_plan* plan, uint64_t seed, uint64_t offset, void* const* g_out, void* const* spd_out,
                          void* const* skh_out, int pro_iter, void* stream);

/* (psgdk_test_peaks and psgdk_test_clock are exported by libpsgdk_probe.so -- csrc/psgdk_probe.hip, a tool library of its own: the
 *  product library carries no probe kernels.)
 * Ceilings of THIS chip, measured in-process in well under a second (bench.py's roofline.peak_measured; SURVEY 8d "re-verify on the
 * box"): out4[0] = TFLOP/s of back-to-back v_mfma_f32_16x16x32_bf16 on register operands (the shape the engine's main loops
 * issue), out4[1] = the same with v_mfma_f32_32x32x16_bf16, out4[2] = GB/s (read + write) of a streaming 16-byte copy of half the
 * scratch buffer into the other half, out4[3] = GB/s of a streaming read.  out4: HOST memory; scratch: device memory, >= 64 MiB
 * (use >= 1 GiB so that the copy exceeds the 256 MiB Infinity Cache).  Synchronises the stream. */
int psgdk_test_peaks(float* out4, void* scratch, size_t scratch_bytes, void* stream);
/* the shader clock (MHz) the chip sustains while every CU issues dependent matrix instructions for ~2 ms: shader-clock ticks (s_memtime)
 * over the 100 MHz wall clock (s_memrealtime), read by one lane per workgroup around the loop; the median over the workgroups */
int psgdk_test_clock(float* shader_mhz, void* stream);

/* kernel launches issued by the library in this process since the last reset (host counter, every launch site; memsets and copies are
 * not kernels and not counted): bench.py divides it by the steps for the latency-bound small plans (launches / step) */
int psgdk_test_launch_count(int64_t* count, int reset);

/* on = 0: psgdk_precond_grad_apply takes its two-call route (precond_grad + apply_update) on this plan -- A/B runs and the parity test of
 * the fused parameter update; on = 1 (default): fused where a tensor allows it */
int psgdk_test_fuse_mode(psgdk_plan* plan, int on, int stagger_ticks);      /* stagger_ticks >= 0: GemmUpdArgs::stagger of the fused launches (100 MHz ticks); -1: unchanged */

/* measurement switch of the momentum pass (tools/ew_bench.py, tools/ew_check.py): mode 1 = damped input without its noise (wrong results:
 * the pass's HBM floor), 2 = the general path for every tile (bit-identical to the compile-time-resolved path), 0 = production */
int psgdk_test_ew_mode(psgdk_plan* plan, int mode);

/* test hook: ONE norm lower bound (psgd.py:46-93; chain 0 = spd on term1, 1 = skh on R) of every dense factor on the plan's
 * CURRENT work arena (i.e. after a psgdk_update_precond_q0p5eq1p5 call), by the cooperative launch (route 1) or the multi-launch
 * route (route 0), Philox noise (seed, offset).  Copies the four products' row sums of squares ([F][4][32] fp32) to out_vsq and
 * the last two subspace blocks ([F][2][32][max_dense_dim] of the preconditioner dtype: products 4 and 3; rows padded with zeros) to out_v (device
 * pointers, either may be NULL).  inject_fault != 0 makes member 1 of every multi-member factor skip its arrivals, to exercise
 * the timeout path (route 1 only). */
int psgdk_test_nlb(psgdk_plan* plan, int chain, int route, uint64_t seed, uint64_t offset, float* out_vsq, void* out_v,
                   int inject_fault, void* stream);
/* Where a cooperative norm-bound launch spends its time (tools/nlb_stamps.py): runs the bound of `chain` once on the plan's current
 * work state with the INSTRUMENTED instantiation of nlb_coop_kernel (phases fenced, lane 0 of every workgroup stamps the 100 MHz wall clock
 * at each phase boundary) and copies 32 words per workgroup to `out` (host memory, >= max_blocks * 32 words; synchronises the stream):
 * words 0..29 = (clock << 8) | phase code in the order they were taken (0 = unused slot), word 30 = HW_REG_XCC_ID, word 31 = (factor << 32) |
 * (member << 8) | members.  Phase codes: kernels_dense.hiph (NLB_STAMP).  The production instantiation carries none of this. */
int psgdk_test_nlb_stamps(psgdk_plan* plan, int chain, uint64_t seed, uint64_t offset, unsigned long long* out, int max_blocks,
                          int* n_blocks, void* stream);
/* C[M,N] = A[M,K] * B[N,K]^T on padded row-major operands (all dims multiples of 64), same kernel the engine uses. */
int psgdk_test_gemm_nt(const void* A, const void* B, void* C, void* Ct, int dtype, int M, int N, int K, int lda,
                       int ldb, int ldc, int ldct, int symmetric, void* stream);
/* times `iters` launches of a batch of identical dense problems (contiguous operands) with hipEvents: avg ms/launch */
int psgdk_test_stage_bench(psgdk_plan* plan, int which, int variant, int iters, float* avg_ms, void* stream);
int psgdk_test_gemm_launch(const void* A, const void* B, void* C, void* Ct, int dtype, int M, int N, int K, int flags, void* stream);
int psgdk_test_gemm_bench(const void* A, const void* B, void* C, void* Ct, int dtype, int M, int N, int K, int batch,
                          int symmetric, int iters, float* avg_ms, void* stream);

/* X = Y * inv(U) for an upper-triangular U [d x d, row stride ld_u] and Y [rows x d, row stride ld] (the fp32 right
 * solve of psgd.py:288-293), same kernel the EQ update uses; dp = roundup(d, 64) must equal ld_u and ld, buffers padded
 * with zeros to multiples of 64 in both extents.  out_nat [rows_p x dp] and/or out_t [dp x rows_p] (either may be NULL).
 * Ut: NULL -> the fp32-matrix-core kernel (every dtype); U^T [dp x dp] -> the bf16 kernel the EQ update uses for bf16 state
 * (panel resident in LDS, updates on the bf16 matrix cores; dtype must be PSGDK_BF16, dp <= 1088). */
int psgdk_test_trsm_right(const void* Y, const void* U, const void* Ut, void* out_nat, void* out_t, int dtype, int rows, int d,
                          void* stream);
/* Timing of the solve kernels alone (bf16; tools/trsm_bench.py): average of `iters` launches between two events.  Ut as above;
 * dbg (bf16 LDS-panel kernel only): 1 = without the update loop, 2 = without the diagonal step, 4 = without the stores,
 * 8 = 64-row panels (one workgroup per CU) instead of 32-row ones, 16 = the first panel's thread 0 writes shader-clock stamps of
 * its phase boundaries (2 + 4 per 64-column block + 2, int64) into `stamps` (device memory, >= 1 KiB). */
int psgdk_test_trsm_bench(const void* Y, const void* U, const void* Ut, void* out_nat, void* out_t, int rows, int d, int iters, int dbg,
                          float* avg_ms, void* stamps, void* stream);

/* Host-only: builds the tile table the grouped GEMM would use for `n` dense problems C[M,N] (K each; sym[i] != 0: upper
 * tiles only) on the 128x128 (big = 0) or 256x256 (big = 1) tiling and reports, per XCD queue, its tile count and its summed
 * cost (K per tile), plus the length of the interleaved table.  No device call: the scheduling rules (queues cut at equal
 * cumulative cost, long tiles first, block b -> XCD b % 8) can be checked without a GPU. */
int psgdk_test_tile_queues(int n, const int32_t* M, const int32_t* N, const int32_t* K, const int32_t* sym, int big,
                           int64_t* queue_tiles, int64_t* queue_cost, int64_t* table_len);

/* Host-only: what psgdk_mx_matmul chooses for a product.  rows x cols: its tile (cols = 0: the few-rows kernel, rows = the rows of A
 * it holds); splits: the parts K is cut in (the few-rows kernel: waves that share a group of rows of B); wide: 1 where 8-bit elements
 * are multiplied as bf16. */
int psgdk_test_mx_plan(int64_t m, int64_t n, int64_t k, int a_fmt, int b_fmt, int out_dtype, int* rows, int* cols, int* splits, int* wide);

#ifdef __cplusplus
}
#endif
#endif /* PSGDK_TEST_H */
