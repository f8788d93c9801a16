"""CPU side of the microscaled operators: the C calls' refusals and sizes, the Python layer's checks, the oracle's own rounding."""
import ctypes as C
import math

import pytest
import torch

import mx_oracle as O


@pytest.fixture(scope="module")
def lib():
    from psgd_torch_amd import _lib, build
    build.build()
    return _lib.lib()


def test_storage(lib):
    a, b = C.c_int64(), C.c_int64()
    for rows, cols, fmt, want in ((3, 1, 4, (3 * 128, 3 * 8)), (5, 256, 8, (5 * 256, 5 * 8)), (2, 257, 4, (2 * 256, 2 * 16)), (0, 7, 8, (0, 0)), (7, 0, 8, (0, 0))):
        assert lib.psgdk_mx_storage(rows, cols, fmt, C.byref(a), C.byref(b)) == 0 and (a.value, b.value) == want
    assert lib.psgdk_mx_storage(-1, 4, 4, C.byref(a), C.byref(b)) == 1
    assert lib.psgdk_mx_storage(4, 4, 6, C.byref(a), C.byref(b)) == 1
    assert lib.psgdk_mx_storage(4, 4, 4, None, C.byref(b)) == 1


def _arg(**kw):
    from psgd_torch_amd import _lib
    t = _lib.MxTensorArg()
    t.rows, t.cols, t.ld = 4, 64, 64
    t.x, t.codes, t.scales = 4096, 8192, 16384          # (never reached: every call below is refused before a launch)
    for k, v in kw.items():
        setattr(t, k, v)
    return t


@pytest.mark.parametrize("kw,dtype,fmt", [
    (dict(), 3, 4), (dict(), 0, 5), (dict(x=None), 0, 4), (dict(codes=None), 0, 4), (dict(scales=None), 0, 4), (dict(rows=-1), 0, 4), (dict(cols=-1), 0, 4),
    (dict(ld=63), 0, 4), (dict(noise=4096), 0, 8), (dict(codes=8200), 0, 4), (dict(x=4097), 0, 4), (dict(x=4098), 1, 4), (dict(rows=1 << 31), 0, 4),
    (dict(codes_t=8192, scales_t=None), 0, 4)])
def test_quantize_refuses(lib, kw, dtype, fmt):
    t = _arg(**kw)
    assert lib.psgdk_mx_quantize(1, C.byref(t), dtype, fmt, None) == 1


def test_quantize_jobs_have_to_agree(lib):
    from psgd_torch_amd import _lib
    for kw in (dict(codes_t=8192, scales_t=8192), dict(noise=4096), dict(codes=None, codes_t=8192, scales_t=8192)):
        ts = (_lib.MxTensorArg * 2)(_arg(), _arg(**kw))
        assert lib.psgdk_mx_quantize(2, ts, 0, 4, None) == 1
    assert lib.psgdk_mx_quantize(-1, None, 0, 4, None) == 1 and lib.psgdk_mx_quantize(1, None, 0, 4, None) == 1
    assert lib.psgdk_mx_quantize(0, None, 0, 4, None) == 0
    empty = (_lib.MxTensorArg * 2)(_arg(rows=0), _arg(cols=0, x=None))
    assert lib.psgdk_mx_quantize(2, empty, 0, 4, None) == 0                       # nothing to do: no launch


def test_dequantize_refuses(lib):
    ok = [4096, 4096, 4, 64, 4, 8192, 0, None]
    for i, v in ((0, None), (1, None), (2, -1), (3, -1), (4, 7), (5, None), (6, 9), (0, 4104), (5, 8193)):
        a = list(ok)
        a[i] = v
        assert lib.psgdk_mx_dequantize(*a) == 1, (i, v)
    assert lib.psgdk_mx_dequantize(None, None, 0, 64, 4, None, 0, None) == 0


def test_matmul_refuses(lib):
    ok = [4096, 4096, 70, 4, 4096, 4096, 40, 8, 512, 8192, 0, 65536, 1 << 30, None]
    bad = [(2, -1), (6, -1), (8, -1), (3, 5), (7, 5), (10, 3), (9, None), (0, None), (1, None), (4, None), (5, None), (0, 4104), (4, 4104), (1, 4100), (5, 4100), (9, 8193),
           (2, 1 << 31), (6, 1 << 31), (8, 1 << 31)]
    for i, v in bad:
        a = list(ok)
        a[i] = v
        assert lib.psgdk_mx_matmul(*a) == 1, (i, v)
    wb = C.c_size_t()
    assert lib.psgdk_mx_matmul_work_bytes(128, 128, 1 << 16, 4, 8, 0, C.byref(wb)) == 0 and wb.value > 0
    split = [4096, 4096, 128, 4, 4096, 4096, 128, 8, 1 << 16, 8192, 0, None, 0, None]
    assert lib.psgdk_mx_matmul(*split) == 1                                         # split sums without a workspace
    split[11], split[12] = 65536, wb.value - 1
    assert lib.psgdk_mx_matmul(*split) == 1
    assert lib.psgdk_mx_matmul_work_bytes(1, 1, -1, 4, 4, 0, C.byref(wb)) == 1 and lib.psgdk_mx_matmul_work_bytes(1, 1, 1, 4, 4, 0, None) == 1
    for i, v in ((6, (1 << 22) + 1), (8, (1 << 23) + 1)):
        a = list(ok)
        a[i] = v
        assert lib.psgdk_mx_matmul(*a) == 2, (i, v)
    assert lib.psgdk_mx_matmul(None, None, 0, 4, None, None, 40, 4, 64, None, 0, None, 0, None) == 0


def test_norm_refuses(lib):
    #      x     res   gain gdt rows cols dt  eps   fmt  s     inv   codes scales codes_t scales_t
    ok = [4096, 4096, 4096, 1, 4, 64, 0, 1e-5, 8, 8192, 8192, 8192, 8192, None, None, None]
    for i, v in ((0, None), (2, None), (3, 4), (4, -1), (5, 0), (6, 4), (7, -1.0), (7, math.nan), (8, 3), (9, None), (10, None), (11, None), (12, None), (13, 8192), (0, 4097),
                 (2, 4098), (11, 8200)):
        a = list(ok)
        a[i] = v
        assert lib.psgdk_rms_norm_mx(*a) == 1, (i, v)
    a = list(ok)
    a[5] = 16385
    assert lib.psgdk_rms_norm_mx(*a) == 2
    assert lib.psgdk_rms_norm_mx(None, None, None, 1, 0, 64, 0, 1e-5, 8, None, None, None, None, None, None, None) == 0
    #       dy   dydt  s    gain gdt inv  ds   rows cols dt dx   dgain work bytes
    okb = [4096, 1, 4096, 4096, 1, 4096, None, 4, 64, 0, 8192, 8192, 8192, 1 << 20, None]
    for i, v in ((0, None), (1, 2), (1, 5), (2, None), (3, None), (4, 3), (5, None), (7, -1), (8, 0), (9, 3), (10, None), (11, None), (12, None), (13, 0), (2, 4097)):
        b = list(okb)
        b[i] = v
        assert lib.psgdk_rms_norm_mx_backward(*b) == 1, (i, v)
    wb = C.c_size_t()
    assert lib.psgdk_rms_norm_mx_backward_work_bytes(4, 16385, C.byref(wb)) == 2 and lib.psgdk_rms_norm_mx_backward_work_bytes(4, 0, C.byref(wb)) == 1


def test_python_refuses_cpu_tensors_and_bad_arguments():
    import psgd_torch_amd as p
    E = p._lib.PsgdkError
    x = torch.zeros(4, 64)
    t = p.MxTensor(torch.zeros(4, 128, dtype=torch.uint8), torch.zeros(4, 8, dtype=torch.uint8), (4, 64), "fp4")
    for call in (lambda: p.mx_quantize(x), lambda: p.mx_dequantize(t), lambda: p.mx_matmul(t, t), lambda: p.rms_norm_mx(x, x[0]),
                 lambda: p.rms_norm_mx_backward(x, x, x[0], x[:, 0]), lambda: p.MxWeight(x), lambda: p.mx_quantize([1.0]), lambda: p.mx_matmul(x, x),
                 lambda: p.mx_linear(x, x), lambda: p.refresh_mx_weights([x])):
        with pytest.raises(E):
            call()
    codes, scales = torch.zeros(4, 128, dtype=torch.uint8), torch.zeros(4, 8, dtype=torch.uint8)
    for bad in ((codes[:3], scales, (4, 64), "fp4"), (codes, scales, (4, 257), "fp4"), (codes, scales, (4, 64), "fp8"), (codes, scales, (4, 64), "int4"),
                (codes.float(), scales, (4, 64), "fp4"), (codes, scales[:, :7], (4, 64), "fp4"), (codes, scales, (-1, 64), "fp4"),
                (torch.zeros(4, 256, dtype=torch.uint8)[:, ::2], scales, (4, 64), "fp4"), (torch.zeros(4 * 128 + 1, dtype=torch.uint8)[1:].view(4, 128), scales, (4, 64), "fp4")):
        with pytest.raises(E):
            p.MxTensor(*bad)


def test_keep_mx_takes_this_optimizers_weights_only():
    import psgd_torch_amd as p
    w = torch.nn.Parameter(torch.zeros(4, 64))
    opt = p.KWNS4([w])
    with pytest.raises(TypeError):
        opt.keep_mx([w])
    other = object.__new__(p.MxWeight)
    other.param = torch.nn.Parameter(torch.zeros(2, 2))
    with pytest.raises(ValueError):
        opt.keep_mx([other])
    mine = object.__new__(p.MxWeight)
    mine.param = w
    opt.keep_mx([mine])
    opt.keep_mx([mine])
    assert opt._mx_weights == [mine]


def test_oracle_rounding():
    """Every value of a table is a fixed point, every midpoint goes to the even code, everything else to the nearer neighbour."""
    for fmt in ("fp4", "fp8"):
        t = O.table(fmt)
        top = t[-1]
        mids = (t[1:] + t[:-1]) / 2
        for v, want in [(a, a) for a in t.tolist()] + [(m, t[i] if i % 2 == 0 else t[i + 1]) for i, m in enumerate(mids.tolist())]:
            x = torch.zeros(1, 32, dtype=torch.float64)
            x[0, 0], x[0, 1], x[0, 2] = top, v, -v
            q = O.rounded(x, fmt)
            assert q[0, 1] == want and q[0, 2] == -want, (fmt, v)
    assert O.scale_exponent(6.0, "fp4") == 0 and O.scale_exponent(6.0000001, "fp4") == 1 and O.scale_exponent(448.0, "fp8") == 0
    x = torch.full((1, 32), 1.0)
    x[0, 5] = math.inf
    assert torch.isnan(O.rounded(x, "fp4")).all()


def _kernels():
    """{kernel: its instructions} of the library's gfx950 code objects."""
    import os
    import re
    import subprocess
    import tempfile
    from psgd_torch_amd import _lib
    llvm = "/opt/rocm/lib/llvm/bin"
    out = {}
    with tempfile.TemporaryDirectory() as tmp:
        fat = os.path.join(tmp, "fat")
        subprocess.run([f"{llvm}/llvm-objcopy", "-O", "binary", "--only-section=.hip_fatbin", _lib.LIB_PATH, fat], check=True)
        data = open(fat, "rb").read()
        magic = b"__CLANG_OFFLOAD_BUNDLE__"
        starts = [m.start() for m in re.finditer(magic, data)]
        for i, a in enumerate(starts):
            part, co = os.path.join(tmp, f"b{i}"), os.path.join(tmp, f"c{i}")
            open(part, "wb").write(data[a:starts[i + 1] if i + 1 < len(starts) else len(data)])
            subprocess.run([f"{llvm}/clang-offload-bundler", "--unbundle", "--type=o", f"--input={part}", "--targets=hipv4-amdgcn-amd-amdhsa--gfx950", f"--output={co}"],
                           check=True, capture_output=True)
            text = subprocess.run([f"{llvm}/llvm-objdump", "-d", "--no-show-raw-insn", "--no-leading-addr", co], check=True, capture_output=True, text=True).stdout
            for f in re.split(r"\n(?=<)", text):
                m = re.match(r"<([^>]+)>:", f)
                if m:
                    out[m.group(1)] = [line.split("//")[0].strip() for line in f.split("\n")[1:]]
    return out


def test_main_loops_of_the_large_tiles(lib):
    """The large tile's products are inline assembly on accumulators that the compiler must not touch while they are in flight: between the first and the last
    matrix instruction nothing may read, move or spill an accumulation register, nor go to scratch; behind the last one come the waits."""
    found = 0
    for name, code in _kernels().items():
        if "mx_tile_gemm_kernel" not in name or "Li256ELi256E" not in name:
            continue
        found += 1
        mfma = [i for i, c in enumerate(code) if c.startswith("v_mfma")]
        assert len(mfma) == 128, (name, len(mfma))
        for c in code[mfma[0]:mfma[-1]]:
            assert not c.startswith(("v_accvgpr", "scratch_")), (name, c)
            assert c.startswith("v_mfma") or not any(op.startswith(("a[", "a0", "a1", "a2")) for op in c.replace(",", " ").split()[1:]), (name, c)
        behind = code[mfma[-1] + 1:]
        waits = [i for i, c in enumerate(behind) if c.startswith("s_nop 15")][:2]
        assert len(waits) == 2 and all(c.startswith("s_") for c in behind[:waits[1]]), name
        loop = [i for i, c in enumerate(behind[:waits[0]]) if c.startswith("s_cbranch")]
        assert len(loop) == 1 and not any(c.startswith("s_branch") for c in behind[:waits[1]]), name      # the loop's own end, then straight on
    assert found == 4, found


def test_copies_and_pickles_have_addresses_of_their_own():
    import copy
    import io

    import psgd_torch_amd as p
    one = p.MxTensor.empty(4, 300, "fp8", "cpu")
    one.codes.random_(0, 256)
    one.scales.random_(0, 255)
    two = p.MxTensor(one.codes.clone(), one.scales.clone(), (4, 300), "fp8")
    for t in (one, two):
        file = io.BytesIO()
        torch.save(t, file)
        file.seek(0)
        for c in (copy.deepcopy(t), torch.load(file, weights_only=False)):
            assert (c.shape, c.fmt, c.device) == (t.shape, t.fmt, t.device)
            assert torch.equal(c.codes, t.codes) and torch.equal(c.scales, t.scales)
            assert c._ptrs == (c.codes.data_ptr(), c.scales.data_ptr()) and not set(c._ptrs) & set(t._ptrs)
        c = copy.copy(t)                                     # the same memory, held by the copy too
        assert c._ptrs == t._ptrs == (c.codes.data_ptr(), c.scales.data_ptr())


def test_more_threads_than_a_launch_can_have_are_refused(lib):
    # (2^32 threads; addresses are never reached)
    t = _arg(rows=1 << 28)
    assert lib.psgdk_mx_quantize(1, C.byref(t), 0, 4, None) == 2
    t = _arg(rows=1 << 30, cols=128 * 8, ld=1 << 10, codes=None, scales=None, codes_t=8192, scales_t=8192)
    assert lib.psgdk_mx_quantize(1, C.byref(t), 1, 4, None) == 2
    assert lib.psgdk_mx_dequantize(4096, 4096, 1 << 28, 64, 4, 8192, 0, None) == 2
    ok = [4096, None, 4096, 1, 1 << 27, 64, 0, 1e-5, 8, None, 8192, 8192, 8192, None, None, None]
    assert lib.psgdk_rms_norm_mx(*ok) == 2
    ok[4], ok[5] = 1 << 25, 4096
    assert lib.psgdk_rms_norm_mx(*ok) == 2
    assert lib.psgdk_mx_matmul(4096, 4096, 1 << 30, 4, 4096, 4096, 1 << 12, 4, 256, 8192, 0, 65536, 1 << 60, None) == 2


def test_plan_query(lib):
    """psgdk_test_mx_plan: which kernel a product takes, and its refusals."""
    def plan(*a):
        out = [C.c_int(-1) for _ in range(4)]
        return lib.psgdk_test_mx_plan(*a, *[C.byref(v) for v in out]), tuple(v.value for v in out)
    assert plan(3, 1000, 512, 4, 8, 0) == (0, (16, 0, 2, 0)) and plan(33, 100, 512, 8, 8, 1) == (0, (48, 0, 2, 1))
    assert plan(8192, 8192, 8192, 4, 4, 0) == (0, (256, 256, 1, 0)) and plan(300, 300, 300, 8, 4, 1) == (0, (128, 128, 1, 1))
    assert plan(50, 16500, 600, 8, 4, 0) == (0, (64, 128, 1, 0))
    for bad in ((0, 1, 1, 4, 4, 0), (1, 0, 1, 4, 4, 0), (1, 1, -1, 4, 4, 0), (1, 1, 1, 5, 4, 0), (1, 1, 1, 4, 5, 0), (1, 1, 1, 4, 4, 3), (1 << 31, 1, 1, 4, 4, 0)):
        assert plan(*bad)[0] == 1
    assert lib.psgdk_test_mx_plan(1, 1, 1, 4, 4, 0, None, None, None, None) == 1


def test_quantize_refuses_before_it_launches(lib):
    """One tensor too large for a launch behind 32 others, which fill a launch of their own: refused as a whole."""
    from psgd_torch_amd import _lib
    for kw in (dict(), dict(codes=None, scales=None, codes_t=8192, scales_t=8192)):
        ts = (_lib.MxTensorArg * 33)(*[_arg(**kw) for _ in range(32)], _arg(rows=1 << 30, cols=1024, ld=1 << 10, **kw))
        assert lib.psgdk_mx_quantize(33, ts, 1, 4, None) == 2


def test_negated_views_are_resolved():
    """The imaginary part of a conjugated tensor has memory of the other sign, contiguous where it has one column or one element: kernels read memory."""
    from psgd_torch_amd import mx

    def memory(t):
        return [C.c_float.from_address(t.data_ptr() + 4 * i * t.stride(0)).value for i in range(t.shape[0])]
    z = torch.complex(torch.zeros(5, 1), torch.arange(1.0, 6.0)[:, None]).conj()
    x = z.imag
    assert x.is_neg() and x[:, 0].tolist() == [-1.0, -2.0, -3.0, -4.0, -5.0] and memory(x) == [1.0, 2.0, 3.0, 4.0, 5.0]
    assert memory(mx._rows("x", x)) == memory(mx._flat(x)) == x[:, 0].tolist()
    one = z[:1].imag
    assert one.is_neg() and one.is_contiguous() and memory(mx._flat(one)) == [-1.0]
    plain = torch.ones(3, 4)
    assert mx._flat(plain) is plain and mx._rows("x", plain) is plain
