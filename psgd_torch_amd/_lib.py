"""ctypes binding of libpsgdk.so (include/psgdk.h).  There is NO fallback: if the HIP library is missing or a
call fails, this raises."""
import ctypes as C
import os

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "libpsgdk.so")

PSGDK_OK, PSGDK_ERR_INVALID, PSGDK_ERR_UNSUPPORTED, PSGDK_ERR_HIP, PSGDK_ERR_STATE, PSGDK_ERR_NLB_TIMEOUT = 0, 1, 2, 3, 4, 5
INFO_NLB_COOP, INFO_NLB_FALLBACKS, INFO_DENSE_FACTORS, INFO_MAX_DENSE_DIM, INFO_HSUMSQ_OFFSET, INFO_BALNORM_OFFSET, INFO_UPDATE_FUSED = 0, 1, 2, 3, 4, 5, 6
INFO_NLB_MEMBER_COLS = 7
LRA_INFO_PACKED_ROWS, LRA_INFO_GRAM_AGE = 0, 1
BF16, F32 = 0, 1
F16 = 2                # psgdk_mx_* and psgdk_rms_norm_mx* only
DIAG, DENSE, SCALAR = 0, 1, 2
GEOM_Q0P5EQ1P5, GEOM_EQ, GEOM_QEQ, GEOM_QUAD, GEOM_QEP, GEOM_QUAD4P, GEOM_PRO4P = 0, 1, 2, 3, 4, 5, 6
SRC_EMA, SRC_GRAD = 0, 1
ABI_VERSION = 405      # PSGDK_VERSION this binding was written against (checked at load)
MAX_DIMS = 26          # PSGDK_MAX_DIMS: noise pointer slots per tensor (include/psgdk.h)


class PsgdkError(RuntimeError):
    def __init__(self, status, what):
        self.status = status
        super().__init__(what)


class Noise(C.Structure):
    _fields_ = [("g_noise", C.POINTER(C.c_void_p)), ("spd_noise", C.POINTER(C.c_void_p)),
                ("skh_noise", C.POINTER(C.c_void_p))]


class Damp(C.Structure):
    _fields_ = [("source", C.c_int), ("damping", C.c_float), ("noise", C.POINTER(Noise)), ("seed", C.c_uint64),
                ("offset", C.c_uint64)]


class MxTensorArg(C.Structure):
    _fields_ = [("x", C.c_void_p), ("noise", C.c_void_p), ("codes", C.c_void_p), ("scales", C.c_void_p), ("codes_t", C.c_void_p),
                ("scales_t", C.c_void_p), ("rows", C.c_int64), ("cols", C.c_int64), ("ld", C.c_int64)]


_lib = None

# name -> (restype, argtypes); every symbol include/psgdk.h declares (the drop-in ABI)
SIGNATURES = {
    "psgdk_version": (C.c_int, []),
    "psgdk_strerror": (C.c_char_p, [C.c_int]),
    "psgdk_last_hip_error": (C.c_int, []),
    "psgdk_plan_create": (C.c_int, [C.POINTER(C.c_void_p), C.c_int, C.POINTER(C.c_int32), C.POINTER(C.c_int64),
                                    C.c_double, C.c_double, C.c_int, C.c_int]),
    "psgdk_plan_destroy": (C.c_int, [C.c_void_p]),
    "psgdk_plan_set_stream_ids": (C.c_int, [C.c_void_p, C.POINTER(C.c_uint32)]),
    "psgdk_plan_set_geometry": (C.c_int, [C.c_void_p, C.c_int]),
    "psgdk_plan_arena_bytes": (C.c_int, [C.c_void_p, C.POINTER(C.c_size_t), C.POINTER(C.c_size_t)]),
    "psgdk_plan_bind": (C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p]),
    "psgdk_plan_num_factors": (C.c_int, [C.c_void_p, C.c_int, C.POINTER(C.c_int)]),
    "psgdk_plan_factor_view": (C.c_int, [C.c_void_p, C.c_int, C.c_int, C.POINTER(C.c_int), C.POINTER(C.c_size_t),
                                         C.POINTER(C.c_int64), C.POINTER(C.c_int64), C.POINTER(C.c_size_t)]),
    "psgdk_plan_ema_view": (C.c_int, [C.c_void_p, C.c_int, C.POINTER(C.c_size_t), C.POINTER(C.c_int64),
                                      C.POINTER(C.c_int64), C.POINTER(C.c_int64), C.POINTER(C.c_int)]),
    "psgdk_init_state": (C.c_int, [C.c_void_p, C.c_double, C.c_void_p]),
    "psgdk_state_changed": (C.c_int, [C.c_void_p, C.c_void_p]),
    "psgdk_accumulate": (C.c_int, [C.c_void_p, C.POINTER(C.c_void_p), C.c_int, C.POINTER(C.c_void_p), C.c_int,
                                   C.c_float, C.c_float, C.c_int, C.POINTER(Damp), C.c_void_p]),
    "psgdk_update_precond_q0p5eq1p5": (C.c_int, [C.c_void_p, C.c_int, C.c_float, C.c_float, C.c_float,
                                                 C.POINTER(Noise), C.c_uint64, C.c_uint64, C.POINTER(C.c_uint8),
                                                 C.c_void_p]),
    "psgdk_update_precond_qeq": (C.c_int, [C.c_void_p, C.c_int, C.c_float, C.c_float, C.c_float,
                                           C.POINTER(Noise), C.c_uint64, C.c_uint64, C.POINTER(C.c_uint8), C.c_void_p]),
    "psgdk_update_precond_quad": (C.c_int, [C.c_void_p, C.c_int, C.c_float, C.c_float, C.c_float,
                                            C.POINTER(Noise), C.c_uint64, C.c_uint64, C.POINTER(C.c_uint8), C.c_void_p]),
    "psgdk_update_precond_quad4p": (C.c_int, [C.c_void_p, C.c_int, C.c_float, C.c_float, C.c_float,
                                              C.POINTER(Noise), C.c_uint64, C.c_uint64, C.POINTER(C.c_uint8), C.c_void_p]),
    "psgdk_update_precond_pro4p": (C.c_int, [C.c_void_p, C.c_int, C.c_float, C.c_float, C.c_float,
                                             C.POINTER(Noise), C.c_uint64, C.c_uint64, C.POINTER(C.c_uint8), C.c_void_p]),
    "psgdk_update_precond_qep": (C.c_int, [C.c_void_p, C.c_int, C.c_float, C.c_float, C.c_float,
                                           C.POINTER(Noise), C.c_uint64, C.c_uint64, C.c_void_p]),
    "psgdk_update_precond_eq": (C.c_int, [C.c_void_p, C.c_int, C.c_float, C.c_float, C.c_float,
                                          C.POINTER(Noise), C.c_uint64, C.c_uint64, C.POINTER(C.c_uint8), C.c_void_p]),
    "psgdk_precond_grad": (C.c_int, [C.c_void_p, C.c_int, C.c_void_p]),
    "psgdk_apply_update": (C.c_int, [C.c_void_p, C.POINTER(C.c_void_p), C.c_int, C.c_float, C.c_float, C.c_float,
                                     C.c_float, C.c_void_p]),
    "psgdk_precond_grad_apply": (C.c_int, [C.c_void_p, C.c_int, C.POINTER(C.c_void_p), C.c_int, C.c_float, C.c_float, C.c_float,
                                           C.c_float, C.c_void_p]),
    "psgdk_export_precond_grad": (C.c_int, [C.c_void_p, C.POINTER(C.c_void_p), C.c_int, C.c_int, C.c_float, C.c_float, C.c_void_p]),
    "psgdk_read_precond_grad": (C.c_int, [C.c_void_p, C.c_int, C.c_void_p, C.c_int, C.c_int, C.c_float, C.c_float,
                                          C.c_void_p]),
    "psgdk_lra_create": (C.c_int, [C.POINTER(C.c_void_p), C.c_int64, C.c_int, C.c_int]),
    "psgdk_lra_destroy": (C.c_int, [C.c_void_p]),
    "psgdk_lra_work_bytes": (C.c_int, [C.c_void_p, C.POINTER(C.c_size_t)]),
    "psgdk_lra_bind": (C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p]),
    "psgdk_lra_set_gram_recurrence": (C.c_int, [C.c_void_p, C.c_int]),
    "psgdk_lra_state_changed": (C.c_int, [C.c_void_p]),
    "psgdk_lra_update_whiten": (C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_uint64, C.c_uint64, C.c_int, C.c_float,
                                          C.c_float, C.c_float, C.c_void_p]),
    "psgdk_lra_precond_grad": (C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p]),
    "psgdk_plan_info": (C.c_int, [C.c_void_p, C.c_int, C.POINTER(C.c_int64)]),
    "psgdk_profile_enable": (C.c_int, [C.c_void_p, C.c_int]),
    "psgdk_profile_read": (C.c_int, [C.c_void_p, C.POINTER(C.c_double), C.POINTER(C.c_int64), C.c_int]),
    "psgdk_profile_read_fused": (C.c_int, [C.c_void_p, C.POINTER(C.c_double), C.POINTER(C.c_int64)]),
    "psgdk_profile_read_calls": (C.c_int, [C.c_void_p, C.POINTER(C.c_double), C.POINTER(C.c_int64), C.c_int]),
    "psgdk_plan_set_row_shard": (C.c_int, [C.c_void_p, C.c_int, C.c_int64, C.c_int64, C.c_int, C.c_int]),
    "psgdk_plan_exchange_bytes": (C.c_int, [C.c_void_p, C.POINTER(C.c_size_t)]),
    "psgdk_update_precond_begin": (C.c_int, [C.c_void_p, C.c_int, C.c_float, C.c_float, C.c_float, C.POINTER(Noise), C.c_uint64, C.c_uint64,
                                             C.c_void_p, C.c_void_p]),
    "psgdk_update_precond_finish": (C.c_int, [C.c_void_p, C.c_int, C.c_float, C.c_float, C.c_float, C.POINTER(Noise), C.c_uint64, C.c_uint64,
                                              C.c_void_p, C.POINTER(C.c_uint8), C.c_void_p]),
    "psgdk_balance_phase": (C.c_int, [C.c_void_p, C.POINTER(C.c_uint8), C.c_int, C.c_void_p]),
    "psgdk_flat_create": (C.c_int, [C.POINTER(C.c_void_p), C.c_int, C.POINTER(C.c_int64), C.POINTER(C.c_int64)]),
    "psgdk_flat_destroy": (C.c_int, [C.c_void_p]),
    "psgdk_flat_apply": (C.c_int, [C.c_void_p, C.POINTER(C.c_void_p), C.c_int, C.c_void_p, C.c_int, C.c_float, C.c_float,
                                   C.c_void_p]),
    "psgdk_flat_set_clip_groups": (C.c_int, [C.c_void_p, C.c_int, C.POINTER(C.c_int32), C.POINTER(C.c_int64), C.c_int64, C.c_int, C.POINTER(C.c_int64)]),
    "psgdk_flat_apply_groups": (C.c_int, [C.c_void_p, C.POINTER(C.c_void_p), C.c_int, C.c_void_p, C.c_int, C.c_float, C.c_float, C.c_float, C.c_float,
                                          C.c_void_p]),
    "psgdk_flat_gather": (C.c_int, [C.c_void_p, C.POINTER(C.c_void_p), C.c_int, C.c_void_p, C.c_int, C.c_void_p, C.c_float, C.c_void_p,
                                    C.c_void_p]),
    "psgdk_flat_apply_clipped": (C.c_int, [C.c_void_p, C.POINTER(C.c_void_p), C.c_int, C.c_void_p, C.c_int, C.c_float, C.c_void_p, C.c_int64,
                                           C.c_float, C.c_float, C.c_void_p]),
    "psgdk_lra_last_sumsq": (C.c_int, [C.c_void_p, C.POINTER(C.c_void_p)]),
    "psgdk_lra_info": (C.c_int, [C.c_void_p, C.c_int, C.POINTER(C.c_int64)]),
    "psgdk_lra_set_row_shard": (C.c_int, [C.c_void_p, C.c_int64]),
    "psgdk_lra_update_phase": (C.c_int, [C.c_void_p, C.c_int, C.c_void_p, C.c_void_p, C.c_uint64, C.c_uint64, C.c_int, C.c_float, C.c_float,
                                         C.c_float, C.c_void_p]),
    "psgdk_lra_apply_phase": (C.c_int, [C.c_void_p, C.c_int, C.c_void_p, C.c_void_p, C.c_void_p]),
    "psgdk_lra_phase_segments": (C.c_int, [C.c_void_p, C.c_int, C.c_int, C.POINTER(C.c_int), C.POINTER(C.c_int64), C.POINTER(C.c_int),
                                           C.POINTER(C.c_int)]),
    "psgdk_mx_storage": (C.c_int, [C.c_int64, C.c_int64, C.c_int, C.POINTER(C.c_int64), C.POINTER(C.c_int64)]),
    "psgdk_mx_quantize": (C.c_int, [C.c_int, C.POINTER(MxTensorArg), C.c_int, C.c_int, C.c_void_p]),
    "psgdk_mx_dequantize": (C.c_int, [C.c_void_p, C.c_void_p, C.c_int64, C.c_int64, C.c_int, C.c_void_p, C.c_int, C.c_void_p]),
    "psgdk_mx_matmul_work_bytes": (C.c_int, [C.c_int64, C.c_int64, C.c_int64, C.c_int, C.c_int, C.c_int, C.POINTER(C.c_size_t)]),
    "psgdk_mx_matmul": (C.c_int, [C.c_void_p, C.c_void_p, C.c_int64, C.c_int, C.c_void_p, C.c_void_p, C.c_int64, C.c_int, C.c_int64, C.c_void_p,
                                  C.c_int, C.c_void_p, C.c_size_t, C.c_void_p]),
    "psgdk_rms_norm_mx": (C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_int, C.c_int64, C.c_int64, C.c_int, C.c_float, C.c_int, C.c_void_p,
                                    C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p]),
    "psgdk_rms_norm_mx_backward_work_bytes": (C.c_int, [C.c_int64, C.c_int64, C.POINTER(C.c_size_t)]),
    "psgdk_rms_norm_mx_backward": (C.c_int, [C.c_void_p, C.c_int, C.c_void_p, C.c_void_p, C.c_int, C.c_void_p, C.c_void_p, C.c_int64, C.c_int64,
                                             C.c_int, C.c_void_p, C.c_void_p, C.c_void_p, C.c_size_t, C.c_void_p]),
    "psgdk_fill_normal": (C.c_int, [C.c_void_p, C.c_int, C.c_int64, C.c_uint64, C.c_uint64, C.c_uint32, C.c_void_p]),
}

# include/psgdk_test.h: kernel-level test / benchmark hooks (same library, not part of the drop-in ABI)
TEST_SIGNATURES = {
    "psgdk_test_ew_mode": (C.c_int, [C.c_void_p, C.c_int]),
    "psgdk_test_fuse_mode": (C.c_int, [C.c_void_p, C.c_int, C.c_int]),
    "psgdk_test_launch_count": (C.c_int, [C.POINTER(C.c_int64), C.c_int]),
    "psgdk_test_dump_noise": (C.c_int, [C.c_void_p, C.c_uint64, C.c_uint64, C.POINTER(C.c_void_p), C.POINTER(C.c_void_p),
                                        C.POINTER(C.c_void_p), C.c_int, C.c_void_p]),
    "psgdk_test_nlb_stamps": (C.c_int, [C.c_void_p, C.c_int, C.c_uint64, C.c_uint64, C.c_void_p, C.c_int, C.c_void_p, C.c_void_p]),
    "psgdk_test_nlb": (C.c_int, [C.c_void_p, C.c_int, C.c_int, C.c_uint64, C.c_uint64, C.c_void_p, C.c_void_p, C.c_int, C.c_void_p]),
    "psgdk_test_gemm_nt": (C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_int, C.c_int, C.c_int,
                                     C.c_int, C.c_int, C.c_int, C.c_int, C.c_int, C.c_int, C.c_void_p]),
    "psgdk_test_stage_bench": (C.c_int, [C.c_void_p, C.c_int, C.c_int, C.c_int, C.POINTER(C.c_float), C.c_void_p]),
    "psgdk_test_gemm_launch": (C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_int, C.c_int, C.c_int, C.c_int, C.c_int, C.c_void_p]),
    "psgdk_test_gemm_bench": (C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_int, C.c_int, C.c_int,
                                        C.c_int, C.c_int, C.c_int, C.c_int, C.POINTER(C.c_float), C.c_void_p]),
    "psgdk_test_tile_queues": (C.c_int, [C.c_int, C.POINTER(C.c_int32), C.POINTER(C.c_int32), C.POINTER(C.c_int32), C.POINTER(C.c_int32),
                                        C.c_int, C.POINTER(C.c_int64), C.POINTER(C.c_int64), C.POINTER(C.c_int64)]),
    "psgdk_test_mx_plan": (C.c_int, [C.c_int64, C.c_int64, C.c_int64, C.c_int, C.c_int, C.c_int, C.POINTER(C.c_int), C.POINTER(C.c_int),
                                     C.POINTER(C.c_int), C.POINTER(C.c_int)]),
    "psgdk_test_trsm_bench": (C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_int, C.c_int, C.c_int, C.c_int,
                                        C.POINTER(C.c_float), C.c_void_p, C.c_void_p]),
    "psgdk_test_trsm_right": (C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_int, C.c_int, C.c_int,
                                        C.c_void_p]),
}


# libpsgdk_probe.so (csrc/psgdk_probe.hip): the chip's measured ceilings for bench.py -- a tool library, not in the product
PROBE_LIB_PATH = os.path.join(_HERE, "libpsgdk_probe.so")
PROBE_SIGNATURES = {
    "psgdk_test_peaks": (C.c_int, [C.POINTER(C.c_float), C.c_void_p, C.c_size_t, C.c_void_p]),
    "psgdk_test_clock": (C.c_int, [C.POINTER(C.c_float), C.c_void_p]),
}
_probe = None


def probe_lib():
    global _probe
    if _probe is None:
        if not os.path.exists(PROBE_LIB_PATH):
            raise PsgdkError(-1, f"{PROBE_LIB_PATH} is missing: build it with `python -m psgd_torch_amd.build`")
        import torch  # noqa: F401
        L = C.CDLL(PROBE_LIB_PATH)
        for name, (res, args) in PROBE_SIGNATURES.items():
            fn = getattr(L, name)
            fn.restype, fn.argtypes = res, args
        _probe = L
    return _probe


def lib():
    """Loads libpsgdk.so (importing torch first so that the HIP runtime already in the process is reused)."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise PsgdkError(-1, f"{LIB_PATH} is missing: build it with `python -m psgd_torch_amd.build` "
                             "(there is no CPU fallback for the HIP engine)")
    import torch  # noqa: F401  (loads libamdhip64.so.7 so the same runtime instance serves both)
    L = C.CDLL(LIB_PATH)
    for name, (res, args) in list(SIGNATURES.items()) + list(TEST_SIGNATURES.items()):
        fn = getattr(L, name)
        fn.restype, fn.argtypes = res, args
    if L.psgdk_version() != ABI_VERSION:       # a stale libpsgdk.so next to newer Python: its layouts (noise slots per tensor) differ
        raise PsgdkError(-1, f"{LIB_PATH} has ABI version {L.psgdk_version()}, this package expects {ABI_VERSION}: rebuild it with "
                             "`python -m psgd_torch_amd.build`")
    _lib = L
    return L


def check(status, what=""):
    if status != PSGDK_OK:
        L = lib()
        msg = L.psgdk_strerror(status).decode()
        if status == PSGDK_ERR_HIP:
            msg += f" (hipError {L.psgdk_last_hip_error()})"
        raise PsgdkError(status, f"psgdk: {what}: {msg}")


def dtype_code(dt):
    import torch
    if dt == torch.bfloat16:
        return BF16
    if dt == torch.float32:
        return F32
    raise PsgdkError(PSGDK_ERR_INVALID, f"unsupported dtype {dt} (bf16 and fp32 only)")


def ptr_array(tensors):
    arr = (C.c_void_p * len(tensors))()
    for i, t in enumerate(tensors):
        arr[i] = None if t is None else t.data_ptr()
    return arr


def current_stream():
    import torch
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)
