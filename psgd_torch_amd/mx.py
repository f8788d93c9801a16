"""Microscaled (MX) numbers next to the optimizer: the low-precision products of the layers whose weights KWNS4 updates, and the norm before them.

    mx_quantize, mx_dequantize                 rounding to 4 or 8 bits with a scale per 32 neighbours, and back
    mx_matmul                                  A B^T of two MX matrices on the scaled matrix instructions, fp32 sums
    rms_norm_mx, rms_norm_mx_backward          residual addition + root-mean-square norm ending in MX blocks; its gradients
    MxWeight, mx_linear, mx_norm_linear        a weight kept in MX form in both directions, and differentiable layers on it
    refresh_mx_weights, KWNS4.keep_mx          the kept forms renewed from the parameters, by hand or at the end of every optimizer step

The format (include/psgdk.h): 32 neighbours along the contracted axis share a scale 2^e (byte e + 127); an element is e2m1 ("fp4") or e4m3 ("fp8").
e is the smallest integer that keeps the block's largest magnitude inside the element's range (6 or 448), so nothing saturates; a block with an
infinity or a NaN reads as NaN.  Rows are stored in multiples of 256 elements.

Everything computes through libpsgdk.so on the current stream of the tensors' device; there is no CPU fallback.  No call keeps or reuses memory of its
own: outputs and workspaces come from torch's allocator, so calls on different streams, in captured graphs and on several devices do not meet.
A CUDA graph of a backward pass must not be captured while another autograd graph over the same leaves is alive (torch binds a leaf's gradient
accumulation to the stream it first ran on, and a capture that has to wait for that stream fails): free earlier losses first, or use
torch.autograd.grad inside the capture.
"""
from __future__ import annotations

import ctypes as C
import functools
from typing import List, Optional, Sequence, Tuple

import torch

from . import _lib as L

_FMT = {"fp4": 4, "fp8": 8}
_DTYPE = {torch.bfloat16: L.BF16, torch.float32: L.F32, torch.float16: L.F16}
_PAD = 256          # elements a stored row is a multiple of
_BLOCK = 32
_NONE = (None, None)
NORM_MAX_COLS = 16384


def _bad(msg):
    return L.PsgdkError(L.PSGDK_ERR_INVALID, msg)


def _fmt(fmt) -> int:
    if fmt not in _FMT:
        raise _bad(f'MX format {fmt!r}: "fp4" (e2m1) or "fp8" (e4m3)')
    return _FMT[fmt]


def _dtype(what, dt) -> int:
    if dt not in _DTYPE:
        raise _bad(f"{what} has dtype {dt}: bfloat16, float16 or float32")
    return _DTYPE[dt]


def _tensor(what, t, device=None):
    if not isinstance(t, torch.Tensor):
        raise _bad(f"{what} is not a tensor")
    if not t.is_cuda:
        raise _bad(f"{what} lives on {t.device}: MX operators need tensors on a ROCm device; there is no CPU fallback")
    if device is not None and t.device != device:
        raise _bad(f"{what} lives on {t.device}, the others on {device}")


def _rows(what, x) -> torch.Tensor:
    """x as a matrix of rows with contiguous elements (a view where the strides allow it, a copy otherwise)."""
    if x.dim() == 0:
        raise _bad(f"{what} has no dimensions: MX blocks run along the last one")
    if x.dim() != 2:
        n = 1
        for d in x.shape[:-1]:
            n *= d
        x = x.reshape(n, x.shape[-1])
    if x.shape[1] > 1 and x.stride(1) != 1 or x.shape[0] > 1 and x.stride(0) < x.shape[1]:
        x = x.contiguous()
    return _flat(x) if x.shape[1] == 1 else x


def _flat(t) -> torch.Tensor:
    """t with memory that is what it reads as.  The imaginary part of a conjugated tensor is a view of memory with the other sign and with gaps, which
    contiguous() resolves; where one element a row or one at all is left there are no gaps, and it does not."""
    return t.resolve_neg() if t.is_neg() else t


def _ld(x) -> int:
    return x.stride(0) if x.shape[0] > 1 else max(x.shape[1], 1)


def _ptr(t) -> Optional[int]:
    return None if t is None else t.data_ptr()


# (the calls below cost microseconds on the device at the smallest sizes: the host side avoids objects it does not need)
_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice          # (a tensor on the device is at hand: CUDA is initialised)


def _launch(what, device, fn, *args):
    """fn(*args, current stream of `device`) with that device current."""
    i = device.index
    if i == _current_device():
        rc = fn(*args, _raw_stream(i))
    else:
        with torch.cuda.device(i):
            rc = fn(*args, _raw_stream(i))
    if rc:
        L.check(rc, what)


@functools.lru_cache(maxsize=4096)
def _work_bytes(name, *sizes) -> int:
    """The library's answer for these sizes (it depends on nothing else)."""
    wb = C.c_size_t()
    L.check(getattr(L.lib(), name)(*sizes, C.byref(wb)), name)
    return wb.value


class MxTensor:
    """A rows x cols matrix in MX form, blocks along its rows.  codes: uint8 (rows, pad(cols) * bits / 8), in 4 bits the even element in the low half
    of its byte; scales: uint8 (rows, pad(cols) / 32), 2^(byte - 127), 255 for NaN; pad: the next multiple of 256.  Elements behind `cols` are zero
    codes under finite scales (they take part in products).  Holds no autograd history."""

    __slots__ = ("shape", "fmt", "device", "_codes", "_scales", "_buffer", "_at", "_ptrs")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, shape: Tuple[int, int], fmt: str):
        bits = _fmt(fmt)
        rows, cols = shape
        if rows < 0 or cols < 0:
            raise _bad(f"MxTensor shape {tuple(shape)}")
        wide = -(-cols // _PAD) * _PAD
        for what, t, n in (("codes", codes, wide * bits // 8), ("scales", scales, wide // _BLOCK)):
            if not isinstance(t, torch.Tensor) or t.dtype is not torch.uint8 or t.shape != (rows, n) or not t.is_contiguous():
                raise _bad(f"MxTensor {what}: a contiguous uint8 tensor of shape {(rows, n)} for a {rows} x {cols} matrix in {fmt}")
        device = codes.device
        if device != scales.device:
            raise _bad(f"MxTensor codes live on {device}, scales on {scales.device}")
        ptrs = codes.data_ptr(), scales.data_ptr()
        if ptrs[0] % 16 or ptrs[1] % 8:
            raise _bad("MxTensor codes need 16-byte, scales 8-byte alignment")
        self.shape, self.fmt, self.device = (rows, cols), fmt, device
        self._codes, self._scales, self._buffer, self._at, self._ptrs = codes, scales, None, 0, ptrs

    @classmethod
    def empty(cls, rows: int, cols: int, fmt: str, device) -> "MxTensor":
        """A new one in one piece of memory; codes and scales become tensors (views of it) when somebody asks for them."""
        wide = -(-cols // _PAD) * _PAD
        n, m = rows * (wide * _fmt(fmt) // 8), rows * (wide // _BLOCK)          # (a stored row of codes is a multiple of 128 bytes)
        t = object.__new__(cls)
        t._buffer = torch.empty(n + m, dtype=torch.uint8, device=device)
        base = t._buffer.data_ptr()
        t.shape, t.fmt, t.device, t._codes, t._scales, t._at, t._ptrs = (rows, cols), fmt, t._buffer.device, None, None, n, (base, base + n)
        return t

    @property
    def codes(self) -> torch.Tensor:
        if self._codes is None:
            self._codes = self._buffer[:self._at].view(self.shape[0], -(-self.shape[1] // _PAD) * _PAD * _FMT[self.fmt] // 8)
        return self._codes

    @property
    def scales(self) -> torch.Tensor:
        if self._scales is None:
            self._scales = self._buffer[self._at:].view(self.shape[0], -(-self.shape[1] // _PAD) * _PAD // _BLOCK)
        return self._scales

    def __reduce__(self):
        """Copies and pickles go through the constructor: the addresses belong to this object's memory."""
        return MxTensor, (self.codes, self.scales, self.shape, self.fmt)

    def _memory(self) -> List[torch.Tensor]:
        """The tensors that hold it (autograd saves these, and sees by them whether it was written again)."""
        return [self._codes, self._scales] if self._buffer is None else [self._buffer]

    def _form(self):
        """What _of needs besides the memory."""
        return self.shape, self.fmt, self._at, 2 if self._buffer is None else 1

    @classmethod
    def _of(cls, form, memory) -> "MxTensor":
        """The matrix that had this _form(), in the tensors that its _memory() has become."""
        shape, fmt, at, n = form
        if n == 2:
            return cls(*memory, shape, fmt)
        t = object.__new__(cls)
        t._buffer, = memory
        base = t._buffer.data_ptr()
        t.shape, t.fmt, t.device, t._codes, t._scales, t._at, t._ptrs = shape, fmt, t._buffer.device, None, None, at, (base, base + at)
        return t

    def dequantize(self, dtype=torch.bfloat16) -> torch.Tensor:
        return mx_dequantize(self, dtype)

    def __repr__(self):
        return f"MxTensor({self.shape[0]} x {self.shape[1]}, {self.fmt}, {self.device})"


def _mx(what, t, device=None) -> MxTensor:
    if not isinstance(t, MxTensor):
        raise _bad(f"{what} is not an MxTensor")
    if t.device.type != "cuda":
        raise _bad(f"{what} lives on {t.device}: MX operators need tensors on a ROCm device; there is no CPU fallback")
    if device is not None and t.device != device:
        raise _bad(f"{what} lives on {t.device}, the others on {device}")
    return t


# ---------------------------------------------------------------------------------------------------------------------------- rounding

def _quantize(items, fmt, device):
    """items: [(x (2-D), noise or None, MxTensor of x or None, MxTensor of x transposed or None)] of one dtype, all with the same outputs."""
    jobs = (L.MxTensorArg * len(items))(*[
        (x.data_ptr(), None if noise is None else noise.data_ptr(), *(_NONE if r is None else r._ptrs), *(_NONE if c is None else c._ptrs),
         x.shape[0], x.shape[1], _ld(x))
        for x, noise, r, c in items])
    _launch("mx_quantize", device, L.lib().psgdk_mx_quantize, len(items), jobs, _DTYPE[items[0][0].dtype], _FMT[fmt])


def _rounded(x, fmt, rows, cols, noise=None):
    """(MxTensor of x or None, MxTensor of x transposed or None) of a checked tensor."""
    n, k = x.shape
    r = MxTensor.empty(n, k, fmt, x.device) if rows else None
    c = MxTensor.empty(k, n, fmt, x.device) if cols else None
    _quantize([(x, noise, r, c)], fmt, x.device)
    return r, c


def mx_quantize(x: torch.Tensor, fmt: str = "fp4", *, which: str = "rows", noise: Optional[torch.Tensor] = None):
    """x (..., K) in bf16, fp16 or fp32 -> MX form.  which: "rows" -- x as an (R x K) matrix, blocks along K; "cols" -- its transpose (K x R), blocks
    along R; "both" -- the pair, from one reading of x.  Rounds to nearest, ties to even; with `noise` (uint8, x's shape, uniform bytes; "fp4" only)
    stochastically: up iff frac + (noise + 1/2) / 256 >= 1, the same byte for both directions.  The result carries no gradient."""
    _tensor("x", x)
    _dtype("x", x.dtype)
    _fmt(fmt)
    if which not in ("rows", "cols", "both"):
        raise _bad(f'which={which!r}: "rows", "cols" or "both"')
    shape = x.shape
    x = _rows("x", x.detach() if x.requires_grad else x)
    if noise is not None:
        if fmt != "fp4":
            raise _bad("stochastic rounding is for fp4: an 8-bit element is rounded to nearest")
        _tensor("noise", noise, x.device)
        if noise.dtype != torch.uint8 or noise.shape != shape:
            raise _bad(f"noise: uint8 of x's shape {tuple(shape)}, got {noise.dtype} {tuple(noise.shape)}")
        noise = noise.contiguous()
    r, c = _rounded(x, fmt, which != "cols", which != "rows", noise)
    return (r, c) if which == "both" else r if c is None else c


def mx_dequantize(t: MxTensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values t stands for (bf16 and fp32 hold them exactly within their range)."""
    _mx("t", t)
    code = _dtype("out", dtype)
    out = torch.empty(t.shape, dtype=dtype, device=t.device)
    _launch("mx_dequantize", out.device, L.lib().psgdk_mx_dequantize, *t._ptrs, *t.shape, _FMT[t.fmt], out.data_ptr(), code)
    return out


# ---------------------------------------------------------------------------------------------------------------------------- products

def mx_matmul(a: MxTensor, b: MxTensor, *, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """A B^T (M x N) of a (M x K) and b (N x K), either in either format; fp32 sums, rounded once to out_dtype.  The same inputs give the same bits:
    a long contraction with few outputs is split, and the parts are added in a fixed order.
    With an fp8 operand and a 16-bit output the scaled matrix instruction drops the bits of a product below 2^-13 of the largest one in its block of 32.
    For normally distributed operands that is 2e-5 of the results, a hundredth of a bf16 output's rounding; where the large products of a block cancel, what
    is left may be off by up to 32 2^-13 of the largest.  An fp32 output has fp32 sums throughout: at half the rate with an fp8 operand (elements
    below 2^-126 count as zero there), at the full rate with two fp4 operands."""
    _mx("a", a)
    _mx("b", b, a.device)
    if a.shape[1] != b.shape[1]:
        raise _bad(f"mx_matmul: a is {a.shape[0]} x {a.shape[1]}, b is {b.shape[0]} x {b.shape[1]}: both are contracted along their rows")
    return _matmul(a, b, out_dtype, _dtype("out", out_dtype))


def _matmul(a, b, out_dtype, code):
    (m, k), n = a.shape, b.shape[0]
    device = a.device
    out = torch.empty((m, n), dtype=out_dtype, device=device)
    wb = _work_bytes("psgdk_mx_matmul_work_bytes", m, n, k, _FMT[a.fmt], _FMT[b.fmt], code)
    work = torch.empty(wb, dtype=torch.uint8, device=device) if wb else None
    _launch("mx_matmul", device, L.lib().psgdk_mx_matmul, *a._ptrs, m, _FMT[a.fmt], *b._ptrs, n, _FMT[b.fmt], k, out.data_ptr(), code, work.data_ptr() if wb else None, wb)
    return out


# ---------------------------------------------------------------------------------------------------------------------------- norm

def _norm_args(x, gain, residual, name="x", other="residual"):
    _tensor(name, x)
    _dtype(name, x.dtype)
    if x.dim() == 0 or x.shape[-1] == 0:
        raise _bad(f"{name} of shape {tuple(x.shape)}: the norm needs at least one column")
    if x.shape[-1] > NORM_MAX_COLS:
        raise L.PsgdkError(L.PSGDK_ERR_UNSUPPORTED, f"rms_norm_mx: {x.shape[-1]} columns, at most {NORM_MAX_COLS} (a row stays in registers)")
    _tensor("gain", gain, x.device)
    _dtype("gain", gain.dtype)
    if gain.shape != x.shape[-1:]:
        raise _bad(f"gain of shape {tuple(gain.shape)} for rows of {x.shape[-1]}")
    if residual is not None:
        _tensor(other, residual, x.device)
        if residual.shape != x.shape or residual.dtype != x.dtype:
            raise _bad(f"{other} is {residual.dtype} {tuple(residual.shape)}, {name} is {x.dtype} {tuple(x.shape)}")


def rms_norm_mx(x: torch.Tensor, gain: torch.Tensor, residual: Optional[torch.Tensor] = None, *, eps: float = 1e-5, fmt: str = "fp8",
                which: str = "rows"):
    """s = x + residual (rounded to x's dtype; without a residual s is x), inv = (mean of s^2 + eps)^-1/2 of every row in fp32, y = s inv gain.
    Returns (y in MX form as mx_quantize's `which` says, s, inv).  The squares are summed in 64 bits, inv is the fp32 number nearest to the exact one, y is
    rounded once, from fp32.  At most 16384 columns.  Not differentiable by itself (rms_norm_mx_backward has the gradients, mx_norm_linear is the
    differentiable layer)."""
    _norm_args(x, gain, residual)
    if torch.is_grad_enabled() and (x.requires_grad or gain.requires_grad or residual is not None and residual.requires_grad):
        raise _bad("rms_norm_mx does not record gradients: use mx_norm_linear, or call it under torch.no_grad()")
    _fmt(fmt)
    if which not in ("rows", "cols", "both"):
        raise _bad(f'which={which!r}: "rows", "cols" or "both"')
    if not 0.0 <= eps < float("inf"):
        raise _bad(f"eps={eps}")
    r, c, s, inv = _norm(x, gain, residual, eps, fmt, which != "cols", which != "rows")
    return (r, c) if which == "both" else r if c is None else c, s, inv


def _norm(x, gain, residual, eps, fmt, rows, cols):
    """(y or None, y transposed or None, s, inv) of checked arguments."""
    d = x.shape[-1]
    x, gain = x.contiguous(), gain.contiguous()
    if d == 1:
        x, gain = _flat(x), _flat(gain)
    n = x.numel() // d
    device = x.device
    if residual is None:
        s, res = x, None
    else:
        residual = residual.contiguous()
        if d == 1:
            residual = _flat(residual)
        s, res = torch.empty_like(x), residual.data_ptr()
    inv = torch.empty(n, dtype=torch.float32, device=device)
    r = MxTensor.empty(n, d, fmt, device) if rows else None
    c = MxTensor.empty(d, n, fmt, device) if cols else None
    _launch("rms_norm_mx", device, L.lib().psgdk_rms_norm_mx, x.data_ptr(), res, gain.data_ptr(), _DTYPE[gain.dtype], n, d, _DTYPE[x.dtype], eps, _FMT[fmt],
            s.data_ptr(), inv.data_ptr(), *(r._ptrs if rows else _NONE), *(c._ptrs if cols else _NONE))
    return r, c, s, inv


def rms_norm_mx_backward(dy: torch.Tensor, s: torch.Tensor, gain: torch.Tensor, inv: torch.Tensor, *, ds: Optional[torch.Tensor] = None):
    """(dx, dgain) of rms_norm_mx at the s and inv it returned, the rounding of y taken as the identity: with u = s inv,
    dx = inv (dy gain - u mean(dy gain u)) + ds -- the gradient of x and of the residual -- and dgain = the sum over rows of dy u (fp32, the same
    bits every run).  dy: s's dtype or fp32.  ds: the gradient that reaches s by its other uses.  The results carry no gradient: in grad mode a dy, s, inv or ds
    that requires one is refused; gain may be a parameter."""
    _norm_args(s, gain, ds, "s", "ds")
    _tensor("dy", dy, s.device)
    _tensor("inv", inv, s.device)
    if dy.shape != s.shape or dy.dtype not in (s.dtype, torch.float32):
        raise _bad(f"dy is {dy.dtype} {tuple(dy.shape)}, s is {s.dtype} {tuple(s.shape)}: the same shape, the same dtype or float32")
    d = s.shape[-1]
    n = s.numel() // d
    if inv.dtype != torch.float32 or inv.numel() != n:
        raise _bad(f"inv: {n} values in float32, got {inv.dtype} {tuple(inv.shape)}")
    if torch.is_grad_enabled() and (dy.requires_grad or s.requires_grad or inv.requires_grad or ds is not None and ds.requires_grad):
        raise _bad("rms_norm_mx_backward does not record gradients (there is no second backward pass): call it under torch.no_grad(), or on detached tensors")
    return _norm_backward(dy, s, gain, inv, ds)


def _norm_backward(dy, s, gain, inv, ds):
    dy, s, gain, inv = dy.contiguous(), s.contiguous(), gain.contiguous(), inv.contiguous()
    if ds is not None:
        ds = ds.contiguous()
    d = s.shape[-1]
    n = s.numel() // d
    if d == 1 or n == 1:
        dy, s, gain, inv, ds = _flat(dy), _flat(s), _flat(gain), _flat(inv), None if ds is None else _flat(ds)
    device = s.device
    dx = torch.empty_like(s)
    dgain = torch.empty(d, dtype=torch.float32, device=device)
    wb = _work_bytes("psgdk_rms_norm_mx_backward_work_bytes", n, d)
    work = torch.empty(max(wb, 4), dtype=torch.uint8, device=device)
    _launch("rms_norm_mx_backward", device, L.lib().psgdk_rms_norm_mx_backward, dy.data_ptr(), _DTYPE[dy.dtype], s.data_ptr(), gain.data_ptr(), _DTYPE[gain.dtype],
            inv.data_ptr(), None if ds is None else ds.data_ptr(), n, d, _DTYPE[s.dtype], dx.data_ptr(), dgain.data_ptr(), work.data_ptr(), wb)
    return dx, dgain


# ---------------------------------------------------------------------------------------------------------------------------- layers

class MxWeight:
    """The MX forms of a 2-D parameter (N x K): `rows` (blocks along K: the forward product) and `cols` (the transpose, blocks along N: the gradient of
    the layer's input).  They are rounded once here and renewed by refresh() -- KWNS4.keep_mx does that after every step.  `rows` / `cols` may be
    handed over instead: such a form keeps its contents until the first refresh, and only what is missing is rounded here.  backward=False keeps the
    forward form only (and `cols` where it is handed over)."""

    def __init__(self, param: torch.Tensor, fmt: str = "fp4", *, backward: bool = True, rows: Optional[MxTensor] = None, cols: Optional[MxTensor] = None):
        _tensor("param", param)
        _dtype("param", param.dtype)
        if param.dim() != 2:
            raise _bad(f"MxWeight holds a matrix, got shape {tuple(param.shape)}")
        if type(param) not in (torch.Tensor, torch.nn.Parameter):
            raise _bad(f"MxWeight holds a plain tensor or parameter, got {type(param).__name__}")
        n, k = param.shape
        for what, t, shape in (("rows", rows, (n, k)), ("cols", cols, (k, n))):
            if t is not None and _mx(what, t, param.device).shape != shape:
                raise _bad(f"MxWeight {what} is {t.shape[0]} x {t.shape[1]}, expected {shape[0]} x {shape[1]}")
        _fmt(fmt)
        if rows is not None and cols is not None and cols.fmt != rows.fmt:
            raise _bad(f"MxWeight rows are {rows.fmt}, cols {cols.fmt}")
        self.param = param
        self.fmt = rows.fmt if rows is not None else cols.fmt if cols is not None else fmt
        need_rows, need_cols = rows is None, cols is None and backward
        if need_rows or need_cols:
            r, c = _rounded(_rows("param", param.detach()), self.fmt, need_rows, need_cols)
            rows, cols = rows if rows is not None else r, cols if cols is not None else c
        self.rows, self.cols = rows, cols

    def refresh(self):
        refresh_mx_weights([self])


@torch.no_grad()
def refresh_mx_weights(weights: Sequence[MxWeight]) -> None:
    """Rounds the parameters of `weights` again into the memory of their MX forms, one launch for up to 32 of them: what KWNS4 does at the end of a step for
    the weights it keeps.  An autograd graph that was recorded before and still needs the old forms refuses its backward pass, as for any tensor
    that was modified in place."""
    groups = {}
    for w in weights:
        if not isinstance(w, MxWeight):
            raise _bad(f"{type(w).__name__} is not an MxWeight")
        p = w.param.detach()
        _tensor("param", p, w.rows.device)
        _dtype("param", p.dtype)
        if tuple(p.shape) != w.rows.shape:
            raise _bad(f"the parameter is {tuple(p.shape)} now, its MxWeight {w.rows.shape}")
        groups.setdefault((p.device, p.dtype, w.fmt, w.cols is not None), []).append((_rows("param", p), None, w.rows, w.cols))
    for (device, _, fmt, both), items in groups.items():
        _quantize(items, fmt, device)
        for _, _, r, c in items:
            torch.autograd.graph.increment_version([t for q in (r, c) if q is not None for t in q._memory()])


def _weight_args(x, weight, fmt, grad_fmt):
    if not isinstance(weight, MxWeight):
        raise _bad(f"weight is a {type(weight).__name__}, not an MxWeight")
    _tensor("x", x, weight.rows.device)
    _dtype("x", x.dtype)
    _fmt(fmt)
    _fmt(grad_fmt)
    if x.dim() == 0 or x.shape[-1] != weight.rows.shape[1]:
        raise _bad(f"x of shape {tuple(x.shape)} against a weight of {weight.rows.shape}")


def _need_cols(weight):
    if weight.cols is None:
        raise _bad("the input of this layer needs a gradient: MxWeight(..., backward=True) keeps the form that its product reads")


def _tracked(*ts):
    """The tensors as autograd is to see them: without gradient mode none of them needs one (a custom function is told of requires_grad alone)."""
    return ts if torch.is_grad_enabled() else tuple(None if t is None else t.detach() for t in ts)


def _product_grads(ctx, saved, dout, need_x, need_w, x_dtype):
    """(gradient of the product's input in x_dtype, of the weight) from dout; saved: what _keep saved behind `more`."""
    dr, dc = _rounded(_rows("gradient", dout), ctx.grad_fmt, need_x, need_w)
    dx = dw = None
    if need_x:
        n = ctx.cols[3]
        dx = _matmul(dr, MxTensor._of(ctx.cols, saved[:n]), x_dtype, _DTYPE[x_dtype])
        saved = saved[n:]
    if need_w:
        dw = _matmul(dc, MxTensor._of(ctx.act, saved), ctx.weight_dtype, _DTYPE[ctx.weight_dtype])
    return dx, dw


def _keep(ctx, weight, param, act, need_x, need_w, grad_fmt, *more):
    """What the backward pass needs.  The memory of the MX forms is saved as tensors and ctx holds no form itself: autograd refuses what was written
    again, frees the activations once they are used, and hands them to whoever packs saved tensors (checkpoints, offloading)."""
    memory = []
    if need_x:
        _need_cols(weight)
        ctx.cols = weight.cols._form()
        memory += weight.cols._memory()
    if need_w:
        ctx.act = act._form()
        memory += act._memory()
    ctx.save_for_backward(*more, *memory)
    ctx.weight_dtype, ctx.grad_fmt = param.dtype, grad_fmt


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, param, weight, fmt, grad_fmt):
        need_x, need_w = ctx.needs_input_grad[:2]
        xr, xc = _rounded(_rows("x", x), fmt, True, need_w)
        out = _matmul(xr, weight.rows, x.dtype, _DTYPE[x.dtype])
        _keep(ctx, weight, param, xc, need_x, need_w, grad_fmt)
        ctx.x_shape, ctx.x_dtype = x.shape, x.dtype
        return out if x.dim() == 2 else out.view(*x.shape[:-1], weight.rows.shape[0])

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        need_x, need_w = ctx.needs_input_grad[:2]
        dx, dw = _product_grads(ctx, ctx.saved_tensors, dout, need_x, need_w, ctx.x_dtype)      # (raises where a kept form was renewed since)
        return (dx.view(ctx.x_shape) if need_x else None), dw, None, None, None


class _NormLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, gain, param, weight, eps, fmt, grad_fmt):
        need_s = ctx.needs_input_grad[0] or ctx.needs_input_grad[1]
        need_g, need_w = ctx.needs_input_grad[2:4]
        yr, yc, s, inv = _norm(x, gain, residual, eps, fmt, True, need_w)
        out = _matmul(yr, weight.rows, x.dtype, _DTYPE[x.dtype])
        _keep(ctx, weight, param, yc, need_s or need_g, need_w, grad_fmt, s, inv, gain)
        ctx.set_materialize_grads(False)
        if residual is not None and not need_s:
            ctx.mark_non_differentiable(s)
        out = out if x.dim() == 2 else out.view(*x.shape[:-1], weight.rows.shape[0])
        return out if residual is None else (out, s)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, ds=None):
        need_s = ctx.needs_input_grad[0] or ctx.needs_input_grad[1]
        need_g, need_w = ctx.needs_input_grad[2:4]
        need_y = need_s or need_g
        s, inv, gain, *saved = ctx.saved_tensors
        dx = dg = dw = None
        if dout is not None:
            # (the gradient of y stays in fp32 between the two kernels: one rounding, at dx)
            dy, dw = _product_grads(ctx, saved, dout, need_y, need_w, torch.float32)
            if need_y:
                dx, dg = _norm_backward(dy.view(s.shape), s, gain, inv, ds)
                dg = dg.to(gain.dtype)
        elif need_s:
            dx = ds
        need = ctx.needs_input_grad
        return (dx if need[0] else None), (dx if need[1] else None), (dg if need_g else None), dw, None, None, None, None


def mx_linear(x: torch.Tensor, weight: MxWeight, *, fmt: str = "fp8", grad_fmt: str = "fp8") -> torch.Tensor:
    """x W^T in x's dtype: x is rounded to `fmt`, W is the weight's kept form.  Backward: dx = MX(dY) W and dW = MX(dY^T) MX(x^T)^T with dY rounded to
    `grad_fmt` along the contracted axis of each (roundings count as the identity); dW has the parameter's dtype."""
    _weight_args(x, weight, fmt, grad_fmt)
    x, param = _tracked(x, weight.param)
    return _Linear.apply(x, param, weight, fmt, grad_fmt)


def mx_norm_linear(x: torch.Tensor, gain: torch.Tensor, weight: MxWeight, residual: Optional[torch.Tensor] = None, *, eps: float = 1e-5,
                   fmt: str = "fp8", grad_fmt: str = "fp8"):
    """(rms_norm(x + residual) W^T, s): the residual's addition, the norm that ends in MX blocks and the product that reads them, differentiable in x,
    residual, gain and the weight's parameter.  s = x + residual is the next residual (x itself without one)."""
    _weight_args(x, weight, fmt, grad_fmt)
    _norm_args(x, gain, residual)
    x, residual, gain, param = _tracked(x, residual, gain, weight.param)
    if not 0.0 <= eps < float("inf"):
        raise _bad(f"eps={eps}")
    out = _NormLinear.apply(x, residual, gain, param, weight, eps, fmt, grad_fmt)
    return (out, x) if residual is None else out
