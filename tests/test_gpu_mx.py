"""The microscaled operators on the GPU against their definition in 64 bits (mx_oracle.py): rounding bit for bit, products and norms within bounds
that follow from fp32 arithmetic."""
import math

import pytest
import torch

import mx_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
EPS24 = 2.0 ** -24          # half a step of fp32
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}      # half a step, relative
SIZES = [(1, 1), (1, 32), (2, 31), (3, 33), (31, 7), (33, 64), (129, 100), (128, 256), (300, 257), (257, 1000), (5, 2049)]


@pytest.fixture(scope="module")
def p():
    import psgd_torch_amd
    return psgd_torch_amd


def _inputs(shape, dt, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * torch.exp(2 * torch.randn(shape[0], 1, generator=g))
    return x.to(dt)


def _same(q, want, what):
    codes, scales = want
    assert torch.equal(q.scales.cpu(), scales), f"{what}: scales differ"
    assert torch.equal(q.codes.cpu(), codes), f"{what}: codes differ"


# ---- rounding ----------------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("shape", SIZES)
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("fmt", ["fp4", "fp8"])
def test_quantize(p, shape, dt, fmt):
    x = _inputs(shape, dt, 1)
    xd = x.to(DEV)
    rows, cols = O.quantize(x, fmt), O.quantize(x.t(), fmt)
    _same(p.mx_quantize(xd, fmt), rows, "rows")
    _same(p.mx_quantize(xd, fmt, which="cols"), cols, "cols")
    r, c = p.mx_quantize(xd, fmt, which="both")
    _same(r, rows, "rows of both")
    _same(c, cols, "cols of both")
    for out in DTYPES:
        want = O.rounded(x, fmt)
        got = p.mx_dequantize(r, out).cpu()
        assert torch.equal(got, want.to(out)), out


@pytest.mark.parametrize("shape", SIZES)
@pytest.mark.parametrize("dt", DTYPES)
def test_quantize_stochastic(p, shape, dt):
    x = _inputs(shape, dt, 2)
    u = torch.randint(0, 256, shape, dtype=torch.uint8, generator=torch.Generator().manual_seed(3))
    r, c = p.mx_quantize(x.to(DEV), "fp4", which="both", noise=u.to(DEV))
    _same(r, O.quantize(x, "fp4", u), "rows")
    _same(c, O.quantize(x.t(), "fp4", u.t()), "cols")
    _same(p.mx_quantize(x.to(DEV), "fp4", noise=u.to(DEV)), O.quantize(x, "fp4", u), "rows only")


def _special(dt):
    fi = torch.finfo(dt)
    x = torch.zeros(40, 96, dtype=torch.float64)
    x[0] = torch.linspace(-6, 6, 96)
    x[1, :32] = fi.max
    x[1, 40] = -fi.max
    x[2, ::3] = fi.smallest_normal
    x[2, 1] = fi.smallest_normal / 4                 # subnormal
    x[3] = fi.smallest_normal / 8
    x[4, 5], x[4, 40] = math.inf, 1.0
    x[5, 64], x[5, 3] = math.nan, 2.0
    x[6] = -0.0
    x[7, 0], x[7, 1] = 6.0, 6.0 / 4096               # far below the block's largest
    x[8, 0], x[8, 1:32] = 448.0, 2.0 ** -9           # the smallest e4m3 at scale 1
    x[9, 0], x[9, 1:32] = 448.0, 2.0 ** -10          # half of it: to even, zero
    x[10] = fi.tiny * 3
    x[11, 7] = -math.inf
    x[12:40, 70] = 1.0
    x[30, 70] = math.nan                             # a column block
    return x.to(dt)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("fmt", ["fp4", "fp8"])
def test_quantize_special_values(p, dt, fmt):
    x = _special(dt)
    r, c = p.mx_quantize(x.to(DEV), fmt, which="both")
    _same(r, O.quantize(x, fmt), "rows")
    _same(c, O.quantize(x.t(), fmt), "cols")
    _same(p.mx_quantize(x.to(DEV), fmt), O.quantize(x, fmt), "rows only")
    got, want = p.mx_dequantize(r, torch.float32).cpu(), O.rounded(x, fmt)
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got.nan_to_num(0), want.float().nan_to_num(0))
    if fmt == "fp4":
        u = torch.full(x.shape, 200, dtype=torch.uint8)
        _same(p.mx_quantize(x.to(DEV), fmt, noise=u.to(DEV)), O.quantize(x, fmt, u), "stochastic")


def test_quantize_every_bf16(p):
    """Every finite bf16 next to a neighbour that sets the scale."""
    bits = torch.arange(0, 1 << 16, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    x = bits[torch.isfinite(bits)]
    x = x[:len(x) // 32 * 32].view(-1, 32)
    y = x.clone().t().contiguous().view(-1, 32)      # neighbours of very different sizes
    for fmt in ("fp4", "fp8"):
        for v in (x, y):
            _same(p.mx_quantize(v.to(DEV), fmt), O.quantize(v, fmt), fmt)


@pytest.mark.parametrize("dt", DTYPES)
def test_quantize_strides_and_shapes(p, dt):
    base = _inputs((37, 150), dt, 5)
    for x in (base[:, :100], base[:, 1:90], base[3:, 5:6], base.t(), base[::2], base[:, ::3], base[:1].expand(5, 150), base[:30].reshape(5, 6, 150)[:, 1:4], base[4],
              base[:30].reshape(2, 15, 150).transpose(0, 1)):
        xd = base.to(DEV).as_strided(x.size(), x.stride(), x.storage_offset())
        flat = x.reshape(-1, x.shape[-1])
        r, c = p.mx_quantize(xd, "fp4", which="both")
        _same(r, O.quantize(flat, "fp4"), tuple(x.shape))
        _same(c, O.quantize(flat.t(), "fp4"), tuple(x.shape))


def test_empty(p):
    for shape in ((0, 5), (5, 0), (0, 0), (0,), (3, 0, 4)):
        x = torch.zeros(shape, dtype=torch.bfloat16, device=DEV)
        r, c = p.mx_quantize(x, "fp8", which="both")
        k = shape[-1]
        n = x.numel() // k if k else math.prod(shape[:-1])
        assert r.shape == (n, k) and c.shape == (k, n)
        assert p.mx_dequantize(r).shape == (n, k)
    a, b = (p.mx_quantize(torch.ones(s, device=DEV)) for s in ((3, 0), (4, 0)))
    assert torch.equal(p.mx_matmul(a, b).cpu(), torch.zeros(3, 4, dtype=torch.bfloat16))
    a, b = (p.mx_quantize(torch.ones(s, device=DEV)) for s in ((0, 9), (4, 9)))
    assert p.mx_matmul(a, b).shape == (0, 4) and p.mx_matmul(b, a).shape == (4, 0)
    x, g = torch.ones(0, 8, device=DEV), torch.ones(8, device=DEV)
    y, s, inv = p.rms_norm_mx(x, g, x)
    assert y.shape == (0, 8) and s.shape == (0, 8) and inv.shape == (0,)
    dx, dg = p.rms_norm_mx_backward(x, s, g, inv)
    assert dx.shape == (0, 8) and torch.equal(dg.cpu(), torch.zeros(8))


# ---- products ----------------------------------------------------------------------------------------------------------------------------

def _operand(p, rows, k, fmt, seed, scale=1.0):
    x = _inputs((rows, k), torch.float32, seed) * scale
    return p.mx_quantize(x.to(DEV), fmt), O.rounded(x, fmt)


def _product_bound(a, b, out_dtype, c, fast):
    """fp32 sums: every product of two elements is exact (8 significant bits at most), so the error is that of at most K / 32 + 32 additions, each off
    by less than a step (2^-23) of a partial sum that |A| |B| bounds; then the output's rounding.  `fast` (an 8-bit operand and a 16-bit
    output: the scaled instruction): every product is off by less than 2^-13 of 2^(ea + eb), the largest exponents it meets, which the rows' largest elements bound."""
    k = a.shape[1]
    bound = (k / 32 + 32) * 2.0 ** -23 * (a.abs() @ b.abs().t().contiguous()) + HALF[out_dtype] * 1.01 * c.abs() + torch.finfo(out_dtype).smallest_normal * 2.0 ** -8
    if fast:
        bound = bound + k * 2.0 ** -13 * a.abs().amax(1)[:, None] * b.abs().amax(1)[None]
    return bound


def _check_product(got, a, b, c, fast):
    err = (got.to(c.device).double() - c).abs()
    bound = _product_bound(a, b, got.dtype, c, fast)
    assert bool((err <= bound).all()), (got.dtype, float((err / bound).max()))
    if fast and c.numel() >= 1000:
        # signs are random, so the dropped bits do not add up: in the 2-norm the error is that of one product, 2^-13 of the largest one an instruction
        # adds -- for normally distributed operands less than 12 times their root mean square -- against the products' own size
        rel = float(err.norm() / c.norm())
        assert rel <= HALF[got.dtype] + 12 * 2.0 ** -13, rel


PRODUCTS = [(1, 1, 1), (1, 16, 32), (1, 100, 1000), (2, 17, 255), (16, 33, 256), (17, 64, 257), (33, 130, 512), (64, 300, 129), (65, 63, 300), (65, 129, 2049),
            (128, 128, 4096), (200, 77, 700), (257, 513, 520), (1, 20000, 300), (50, 16500, 64), (4, 5, 6000)]


@pytest.mark.parametrize("m,n,k", PRODUCTS)
@pytest.mark.parametrize("fa", ["fp4", "fp8"])
@pytest.mark.parametrize("fb", ["fp4", "fp8"])
def test_matmul(p, m, n, k, fa, fb):
    (qa, a), (qb, b) = _operand(p, m, k, fa, 11), _operand(p, n, k, fb, 12)
    want = a @ b.t().contiguous()
    eight = "fp8" in (fa, fb)
    for dt in (torch.float32, torch.bfloat16):
        got = p.mx_matmul(qa, qb, out_dtype=dt)
        assert got.dtype == dt and got.shape == (m, n)
        _check_product(got, a, b, want, eight and dt != torch.float32)


def test_matmul_half_output(p):
    (qa, a), (qb, b) = _operand(p, 70, 200, "fp8", 13), _operand(p, 90, 200, "fp4", 14, 0.01)
    want = a @ b.t().contiguous()
    got = p.mx_matmul(qa, qb, out_dtype=torch.float16).cpu().double()
    ok = want.abs() < 60000
    assert bool(((got - want).abs() <= _product_bound(a, b, torch.float16, want, True))[ok].all())


@pytest.mark.parametrize("m,n", [(3, 40), (300, 520)])
def test_matmul_keeps_nan_to_its_rows(p, m, n):
    x, w = _inputs((m, 300), torch.float32, 15), _inputs((n, 300), torch.float32, 16)
    x[1, 290] = math.nan
    w[7, 0] = math.inf
    want = torch.zeros(m, n, dtype=torch.bool)
    want[1] = True
    want[:, 7] = True
    for fa, fb in (("fp8", "fp4"), ("fp4", "fp8"), ("fp8", "fp8"), ("fp4", "fp4")):
        for dt in (torch.float32, torch.bfloat16):
            got = p.mx_matmul(p.mx_quantize(x.to(DEV), fa), p.mx_quantize(w.to(DEV), fb), out_dtype=dt).cpu()
            assert torch.equal(torch.isnan(got), want), (fa, fb, dt)


@pytest.mark.parametrize("m,n,k", [(1, 4096, 1024), (33, 1000, 768), (300, 300, 3000), (128, 128, 16384), (2304, 2100, 600)])
def test_matmul_same_bits_every_run(p, m, n, k):
    (qa, _), (qb, _) = _operand(p, m, k, "fp8", 17), _operand(p, n, k, "fp4", 18)
    first = p.mx_matmul(qa, qb, out_dtype=torch.float32)
    for _ in range(3):
        assert torch.equal(p.mx_matmul(qa, qb, out_dtype=torch.float32), first)


def test_matmul_tiles_agree_with_a_row_at_a_time(p):
    """Large tiles, ragged in both directions, against the few-rows kernel and fp64."""
    m, n, k = 4100, 4099, 1100
    for fa, fb in (("fp4", "fp4"), ("fp8", "fp4"), ("fp4", "fp8"), ("fp8", "fp8")):
        g = torch.Generator(device=DEV).manual_seed(19)
        qa, qb = (p.mx_quantize(torch.randn(r, k, generator=g, device=DEV), f) for r, f in ((m, fa), (n, fb)))
        a, b = p.mx_dequantize(qa, torch.float32).double(), p.mx_dequantize(qb, torch.float32).double()
        want = a @ b.t().contiguous()
        _check_product(p.mx_matmul(qa, qb, out_dtype=torch.float32), a, b, want, False)
        _check_product(p.mx_matmul(qa, qb), a, b, want, "fp8" in (fa, fb))


def test_matmul_refuses(p):
    E = p._lib.PsgdkError
    a = p.mx_quantize(torch.ones(4, 64, device=DEV))
    for bad in (lambda: p.mx_matmul(a, p.mx_quantize(torch.ones(4, 65, device=DEV))), lambda: p.mx_matmul(a, a, out_dtype=torch.float64), lambda: p.mx_matmul(a, a.codes),
                lambda: p.mx_quantize(torch.ones(4, 4, device=DEV, dtype=torch.float64)), lambda: p.mx_quantize(torch.ones((), device=DEV)),
                lambda: p.mx_quantize(torch.ones(4, 4, device=DEV), "fp6"), lambda: p.mx_quantize(torch.ones(4, 4, device=DEV), which="columns"),
                lambda: p.mx_quantize(torch.ones(4, 4, device=DEV), "fp8", noise=torch.zeros(4, 4, dtype=torch.uint8, device=DEV)),
                lambda: p.mx_quantize(torch.ones(4, 4, device=DEV), noise=torch.zeros(4, 5, dtype=torch.uint8, device=DEV)),
                lambda: p.mx_quantize(torch.ones(4, 4, device=DEV), noise=torch.zeros(4, 4, device=DEV)),
                lambda: p.mx_quantize(torch.ones(4, 4, device=DEV), noise=torch.zeros(4, 4, dtype=torch.uint8)), lambda: p.mx_dequantize(a, torch.int8)):
        with pytest.raises(E):
            bad()


# ---- norm --------------------------------------------------------------------------------------------------------------------------------

NORMS = [(1, 1), (1, 32), (3, 33), (5, 100), (7, 512), (4, 513), (130, 768), (3, 1024), (2, 2049), (6, 4096), (2, 5000), (3, 16384)]


def _check_norm_codes(q, y, fmt, cols, rel):
    """Codes of y known to a relative error `rel`: the scale is that of the block's largest magnitude give or take it, every value within half a step of its
    scale (plus the error) of y."""
    r = y.shape[0]
    val = O.dequantize(q.codes.cpu(), q.scales.cpu(), cols, fmt)
    wide = torch.zeros(r, -(-cols // 32) * 32, dtype=torch.float64)
    wide[:, :cols] = y
    amax = wide.view(r, -1, 32).abs().amax(-1)
    s = q.scales.cpu()[:, :amax.shape[1]].double() - 127
    lo = torch.tensor([[O.scale_exponent(v * (1 - rel), fmt) for v in row] for row in amax.tolist()])
    hi = torch.tensor([[O.scale_exponent(v * (1 + rel), fmt) for v in row] for row in amax.tolist()])
    assert bool(((s >= lo) & (s <= hi)).all()), "scale"
    scale = torch.exp2(s).repeat_interleave(32, 1)[:, :cols]
    a = y.abs() / scale * (1 + rel)
    t = O.table(fmt)
    # half of the wider step around a value: to the next code above the one at or below it
    i = (torch.bucketize(a, t, right=True) - 1).clamp(max=len(t) - 2)
    half = (t[i + 1] - t[i]) / 2 * scale
    assert bool(((val - y).abs() <= half + rel * y.abs() + 1e-300).all()), "codes"


@pytest.mark.parametrize("rows,cols", NORMS)
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("fmt,res", [("fp8", True), ("fp4", False)])
def test_norm(p, rows, cols, dt, fmt, res):
    g = torch.Generator().manual_seed(21)
    x, r = torch.randn(rows, cols, generator=g).to(dt), torch.randn(rows, cols, generator=g).to(dt) if res else None
    gain = (1 + 0.3 * torch.randn(cols, generator=g)).to(torch.float32 if res else dt)
    s, inv, y = O.norm(x, gain, r, 1e-5)
    (yr, yc), gs, ginv = p.rms_norm_mx(x.to(DEV), gain.to(DEV), None if r is None else r.to(DEV), fmt=fmt, which="both")
    assert torch.equal(gs.cpu(), s)
    # the sum of squares: at most 8 * 8 + 12 additions in a chain, every term rounded once (all positive: relative errors); its square root halves
    # that; division, root, reciprocal and eps half a step each
    rel = (76 + 1) / 2 * EPS24 + 4 * EPS24
    assert bool(((ginv.cpu().double() - inv).abs() <= rel * inv).all())
    _check_norm_codes(yr, y, fmt, cols, rel + 2 * EPS24)
    _check_norm_codes(yc, y.t().contiguous(), fmt, rows, rel + 2 * EPS24)
    y2, s2, inv2 = p.rms_norm_mx(x.to(DEV), gain.to(DEV), None if r is None else r.to(DEV), fmt=fmt)
    assert torch.equal(y2.codes, yr.codes) and torch.equal(y2.scales, yr.scales) and torch.equal(inv2, ginv) and torch.equal(s2, gs)
    y3, _, inv3 = p.rms_norm_mx(x.to(DEV), gain.to(DEV), None if r is None else r.to(DEV), fmt=fmt, which="cols")
    assert torch.equal(y3.codes, yc.codes) and torch.equal(y3.scales, yc.scales) and torch.equal(inv3, ginv)


def test_norm_rows_do_not_meet(p):
    """A zero row, one with an infinity and one with a NaN leave the others as they are."""
    x = _inputs((9, 700), torch.bfloat16, 22)
    gain = torch.ones(700)
    clean = p.rms_norm_mx(x.to(DEV), gain.to(DEV))[0]
    x[2], x[4, 3], x[6, 699] = 0, math.inf, math.nan
    y, s, inv = p.rms_norm_mx(x.to(DEV), gain.to(DEV), fmt="fp8")
    v = p.mx_dequantize(y).cpu()
    assert torch.equal(v[2], torch.zeros(700, dtype=torch.bfloat16))
    assert torch.isnan(v[6]).all() and torch.isnan(v[4, :32]).all() and torch.equal(v[4, 32:], torch.zeros(668, dtype=torch.bfloat16))
    keep = [0, 1, 3, 5, 7, 8]
    assert torch.equal(y.codes[keep], clean.codes[keep])


@pytest.mark.parametrize("rows,cols", NORMS + [(700, 96), (2100, 520), (600, 4100)])
@pytest.mark.parametrize("dt,dyt", [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float16, torch.float16), (torch.float32, torch.float32)])
@pytest.mark.parametrize("skip", [True, False])
def test_norm_backward(p, rows, cols, dt, dyt, skip):
    g = torch.Generator().manual_seed(23)
    s, dy = torch.randn(rows, cols, generator=g).to(dt), torch.randn(rows, cols, generator=g).to(dyt)
    ds = torch.randn(rows, cols, generator=g).to(dt) if skip else None
    gain = 1 + 0.3 * torch.randn(cols, generator=g)
    inv = (1 / torch.sqrt(s.float().square().mean(-1) + 1e-5))
    dx, dg = O.norm_backward(dy, s, gain, inv, ds)
    gx, gg = p.rms_norm_mx_backward(dy.to(DEV), s.to(DEV), gain.to(DEV), inv.to(DEV), ds=None if ds is None else ds.to(DEV))
    assert gx.dtype == dt and gg.dtype == torch.float32
    # the mean: three roundings a term, at most 8 * 8 + 12 additions, one division; then four products and two additions of terms of these sizes
    u, dyg = s.double() * inv.double()[:, None], dy.double() * gain.double()
    mean_abs = (dyg * u).abs().mean(-1, keepdim=True)
    size = inv.double()[:, None] * (dyg.abs() + u.abs() * mean_abs) + (0 if ds is None else ds.double().abs())
    bound = 84 * EPS24 * size + HALF[dt] * 1.01 * dx.abs() + torch.finfo(dt).smallest_normal
    err = (gx.cpu().double() - dx).abs()
    assert bool((err <= bound).all()), float((err / bound).max())
    # a column: two roundings a term; a wave adds at most rows / lines (+ 1) of them, then at most lines / 4 + 8 shares
    lines = min(512, -(-rows // 4) if cols <= 2048 else rows)
    bound = (2 + rows / lines + 1 + lines / 4 + 8) * EPS24 * (dy.double() * u).abs().sum(0) + 1e-37
    err = (gg.cpu().double() - dg).abs()
    assert bool((err <= bound).all()), float((err / bound).max())
    again = p.rms_norm_mx_backward(dy.to(DEV), s.to(DEV), gain.to(DEV), inv.to(DEV), ds=None if ds is None else ds.to(DEV))
    assert torch.equal(again[0], gx) and torch.equal(again[1], gg)


def test_norm_backward_against_differences(p):
    """The gradient's formula itself, against central differences of the norm in 64 bits."""
    g = torch.Generator().manual_seed(24)
    x, gain, dy, ds = (torch.randn(s, generator=g, dtype=torch.float64) for s in ((3, 40), (40,), (3, 40), (3, 40)))

    def f(x, gain):
        return float(((x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-5) * gain) * dy).sum() + (x * ds).sum())
    h = 1e-6
    nx, ng = torch.zeros_like(x), torch.zeros_like(gain)
    for i in range(3):
        for j in range(40):
            e = torch.zeros_like(x)
            e[i, j] = h
            nx[i, j] = (f(x + e, gain) - f(x - e, gain)) / (2 * h)
    for j in range(40):
        e = torch.zeros_like(gain)
        e[j] = h
        ng[j] = (f(x, gain + e) - f(x, gain - e)) / (2 * h)
    inv = 1 / torch.sqrt(x.square().mean(-1) + 1e-5)
    ox, og = O.norm_backward(dy, x, gain, inv, ds)
    # differences: h^2 of the third derivative, and the rounding of f (about 100) by 2^-52 / h
    assert torch.allclose(ox, nx, rtol=0, atol=1e-7) and torch.allclose(og, ng, rtol=0, atol=1e-7)
    f32 = [t.float().to(DEV) for t in (dy, x, gain, inv, ds)]
    gx, gg = p.rms_norm_mx_backward(*f32[:4], ds=f32[4])
    assert float((gx.cpu().double() - nx).abs().max()) < 1e-5 and float((gg.cpu().double() - ng).abs().max()) < 1e-5


def test_norm_refuses(p):
    E = p._lib.PsgdkError
    x, g = torch.ones(4, 64, device=DEV), torch.ones(64, device=DEV)
    inv = torch.ones(4, device=DEV)
    for bad in (lambda: p.rms_norm_mx(x, g[:63]), lambda: p.rms_norm_mx(x, g, x[:3]), lambda: p.rms_norm_mx(x, g, x.half()), lambda: p.rms_norm_mx(x, g, eps=-1.0),
                lambda: p.rms_norm_mx(x, g, eps=math.nan), lambda: p.rms_norm_mx(x, g, fmt="fp6"), lambda: p.rms_norm_mx(x, g.cpu()), lambda: p.rms_norm_mx(x, g, which="row"),
                lambda: p.rms_norm_mx(torch.ones(2, 16385, device=DEV), torch.ones(16385, device=DEV)), lambda: p.rms_norm_mx(x.requires_grad_(), g),
                lambda: p.rms_norm_mx(torch.ones(3, 0, device=DEV), torch.ones(0, device=DEV)), lambda: p.rms_norm_mx_backward(x, x, g, inv[:3]),
                lambda: p.rms_norm_mx_backward(x.half(), x, g, inv), lambda: p.rms_norm_mx_backward(x[:2], x, g, inv)):
        with pytest.raises(E):
            bad()


# ---- layers and the optimizer ------------------------------------------------------------------------------------------------------------

def _layer_reference(x, res, gain, w, dout, ds, fmt, gfmt, wfmt, eps=1e-5):
    """The layer in 64 bits, with y and the weight rounded as the definition says."""
    s, inv, y = O.norm(x, gain, res, eps)
    yr, yc = O.rounded(y, fmt), O.rounded(y.t(), fmt)
    out = yr @ O.rounded(w, wfmt).t()
    dy = O.rounded(dout, gfmt) @ O.rounded(w.t(), wfmt).t()
    dw = O.rounded(dout.t(), gfmt) @ yc.t()
    dx, dg = O.norm_backward(dy, s, gain, inv, ds)
    return out, s, dx, dg, dw


@pytest.mark.parametrize("t,k,n", [(1, 32, 32), (5, 100, 70), (130, 256, 96), (300, 520, 300)])
@pytest.mark.parametrize("dt,fmt,wfmt", [(torch.bfloat16, "fp8", "fp4"), (torch.float16, "fp4", "fp4"), (torch.float32, "fp8", "fp8")])
def test_norm_linear(p, t, k, n, dt, fmt, wfmt):
    g = torch.Generator().manual_seed(31)
    x, res, ds = (torch.randn(t, k, generator=g).to(dt) for _ in range(3))
    dout = (0.1 * torch.randn(t, n, generator=g)).to(dt)
    gain, w = 1 + 0.1 * torch.randn(k, generator=g), torch.randn(n, k, generator=g) / math.sqrt(k)
    out, s, dx, dg, dw = _layer_reference(x, res, gain, w, dout, ds, fmt, fmt, wfmt)
    leaves = [v.to(DEV).requires_grad_() for v in (x, res, gain, w)]
    weight = p.MxWeight(leaves[3], wfmt)
    go, gs = p.mx_norm_linear(leaves[0], leaves[2], weight, leaves[1], fmt=fmt, grad_fmt=fmt)
    assert go.dtype == dt and torch.equal(gs.cpu(), s)
    gx, gr, gg, gw = torch.autograd.grad((go, gs), leaves, (dout.to(DEV), ds.to(DEV)))
    assert torch.equal(gx, gr) and gw.dtype == torch.float32 and gg.dtype == torch.float32
    # An element of y within fp32's error (2^-18 relative, test_norm) of a rounding border may go the other way: one step of e2m1 (at most half the value)
    # or e4m3 (an eighth).  That concerns about one element in 2^18 / 2^3, here a handful at most; in the 2-norm of an output it is bounded by
    # step * sqrt(share) = 0.5 * sqrt(2^-15) < 3e-3 of the result's own size.  The rest is the outputs' rounding.
    for got, want, h in ((go, out, HALF[dt]), (gx, dx, HALF[dt]), (gg, dg, 2.0 ** -20), (gw, dw, 2.0 ** -20)):
        rel = float((got.detach().cpu().double() - want).norm() / want.norm().clamp(min=1e-30))
        # and 12 * 2^-13 (test_matmul) for the products' dropped bits
        assert rel <= h + 3e-3 + 12 * 2.0 ** -13, rel


def test_norm_linear_without_residual_and_partial_gradients(p):
    g = torch.Generator().manual_seed(32)
    x, w = torch.randn(2, 9, 64, generator=g).to(DEV), torch.randn(40, 64, generator=g).to(DEV)
    gain = torch.ones(64, device=DEV)
    full = [v.clone().requires_grad_() for v in (x, gain, w)]
    out, s = p.mx_norm_linear(full[0], full[1], p.MxWeight(full[2]))
    assert s is full[0] and out.shape == (2, 9, 40)
    want = torch.autograd.grad(out.sum() + (s * 2).sum(), full)
    for i in range(3):
        leaves = [v.clone().requires_grad_(j == i) for j, v in enumerate((x, gain, w))]
        out, s = p.mx_norm_linear(leaves[0], leaves[1], p.MxWeight(leaves[2]))
        (got,) = torch.autograd.grad(out.sum() + (s * 2).sum(), [leaves[i]])
        assert torch.equal(got, want[i]), i
    res = x.clone().requires_grad_()
    out, s = p.mx_norm_linear(x, gain, p.MxWeight(w), res)
    (only,) = torch.autograd.grad(s.sum(), [res])                      # the product's output unused
    assert torch.equal(only, torch.ones_like(only))
    with torch.no_grad():
        out, s = p.mx_norm_linear(x, gain, p.MxWeight(torch.nn.Parameter(w)), res)
    assert not out.requires_grad and not s.requires_grad


def test_linear(p):
    g = torch.Generator().manual_seed(33)
    for lead in ((), (7,), (3, 5)):
        x, w = torch.randn(*lead, 72, generator=g).to(torch.bfloat16), torch.randn(50, 72, generator=g)
        dout = torch.randn(*lead, 50, generator=g).to(torch.bfloat16)
        x2, d2 = x.reshape(-1, 72), dout.reshape(-1, 50)
        out = O.rounded(x2, "fp8") @ O.rounded(w, "fp4").t()
        dx = O.rounded(d2, "fp8") @ O.rounded(w.t(), "fp4").t()
        dw = O.rounded(d2.t(), "fp8") @ O.rounded(x2.t(), "fp8").t()
        xg, wg = x.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
        weight = p.MxWeight(wg)
        go = p.mx_linear(xg, weight)
        gx, gw = torch.autograd.grad(go, (xg, wg), dout.to(DEV))
        assert go.shape == (*lead, 50) and gx.shape == x.shape
        for got, want, h in ((go, out, 2.0 ** -8), (gx, dx, 2.0 ** -8), (gw, dw, 2.0 ** -20)):
            got = got.detach().cpu().double().reshape(want.shape)
            # roundings to the formats are exact here (inputs are given): fp32 sums and the output's rounding are all
            # (K 2^-13 of the rows' largest elements, as _product_bound, with K <= 72 and operands of at most 6 and 1 root mean squares)
            assert bool(((got - want).abs() <= h * 1.01 * want.abs() + 72 * 2.0 ** -13 * want.abs().max()).all())
            assert float((got - want).norm() / want.norm()) <= h + 12 * 2.0 ** -13


def test_linear_gradient_is_the_products(p):
    """Where inputs lie on the formats' grids the roundings are the identity, and the layer's gradients are those of a plain product -- also by
    differences (the output is linear in x and in w, so that a difference of any size on the grid is exact)."""
    g = torch.Generator().manual_seed(34)
    x = torch.randint(-2, 3, (4, 64), generator=g).float()
    w = torch.randint(-2, 3, (8, 64), generator=g).float()
    d = torch.randint(-2, 3, (4, 8), generator=g).float()
    xg, wg = x.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
    out = p.mx_linear(xg, p.MxWeight(wg))
    gx, gw = torch.autograd.grad(out, (xg, wg), d.to(DEV))
    assert torch.equal(out.detach().cpu(), x @ w.t()) and torch.equal(gx.cpu(), d @ w) and torch.equal(gw.cpu(), d.t() @ x)
    e = torch.zeros_like(x)
    e[2, 5] = 1.0
    loss = [float((p.mx_linear((x + f * e).to(DEV), p.MxWeight(w.to(DEV))).cpu() * d).sum()) for f in (1, -1)]
    assert (loss[0] - loss[1]) / 2 == float(gx[2, 5])


def test_linear_refuses(p):
    E = p._lib.PsgdkError
    w = torch.nn.Parameter(torch.randn(8, 64, device=DEV))
    x = torch.randn(4, 64, device=DEV)
    weight = p.MxWeight(w, backward=False)
    assert p.mx_linear(x, weight).shape == (4, 8)
    for bad in (lambda: p.mx_linear(x[:, :63], weight), lambda: p.mx_linear(x.double(), weight), lambda: p.mx_linear(x, w), lambda: p.mx_linear(x, weight, fmt="fp6"),
                lambda: p.mx_linear(x.clone().requires_grad_(), weight), lambda: p.MxWeight(w[0]), lambda: p.MxWeight(w, rows=p.mx_quantize(x)),
                lambda: p.MxWeight(w, "fp3")):
        with pytest.raises(E):
            bad()


def test_refresh(p):
    """One call over many weights of different sizes, types and formats; a graph recorded before refuses its backward pass."""
    g = torch.Generator().manual_seed(35)
    ws = [torch.nn.Parameter(torch.randn(3 + i, 40 + 7 * i, generator=g).to(torch.bfloat16 if i % 3 == 0 else torch.float32).to(DEV)) for i in range(70)]
    mx = [p.MxWeight(w, "fp8" if i % 5 == 0 else "fp4", backward=i % 4 != 0) for i, w in enumerate(ws)]
    x = torch.randn(2, ws[1].shape[1], device=DEV, requires_grad=True)
    out = p.mx_linear(x, mx[1])
    with torch.no_grad():
        for w in ws:
            w.mul_(-1.7).add_(0.1)
    ptr = mx[0].rows.codes.data_ptr()
    p.refresh_mx_weights(mx)
    assert mx[0].rows.codes.data_ptr() == ptr
    for w, q in zip(ws, mx):
        _same(q.rows, O.quantize(w.detach().cpu(), q.fmt), "rows")
        if q.cols is not None:
            _same(q.cols, O.quantize(w.detach().cpu().t(), q.fmt), "cols")
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()
    ws[5].data = torch.randn(2, 2, device=DEV)
    with pytest.raises(p._lib.PsgdkError):
        p.refresh_mx_weights(mx)
    p.refresh_mx_weights([])


def _block(p, ws, gains, x):
    """Two pre-norm layers of a residual stream, as a model would stack them."""
    s = x
    h, s = p.mx_norm_linear(x, gains[0], ws[0])
    h = p.mx_linear(torch.nn.functional.gelu(h), ws[1])
    h2, s = p.mx_norm_linear(h, gains[1], ws[2], s)
    h2 = p.mx_linear(torch.nn.functional.gelu(h2), ws[3])
    return s + h2


def test_training_with_kwns4(p):
    """Forward, backward and optimizer step together: KWNS4 renews the kept weights at the end of every step."""
    torch.manual_seed(0)
    d = 96
    params = [torch.nn.Parameter(torch.randn(o, i, device=DEV) / math.sqrt(i)) for o, i in ((4 * d, d), (d, 4 * d), (4 * d, d), (d, 4 * d))]
    gains = [torch.nn.Parameter(torch.ones(d, device=DEV)) for _ in range(2)]
    ws = [p.MxWeight(w) for w in params]
    opt = p.KWNS4(params + gains, lr_params=1e-3, preconditioner_dtype=torch.float32, seed=3)
    opt.keep_mx(ws)
    for _ in range(4):
        x, y = torch.randn(64, d, device=DEV), torch.randn(64, d, device=DEV)
        opt.zero_grad(set_to_none=True)
        loss = (_block(p, ws, gains, x) - y).square().mean()
        loss.backward()
        for q in params + gains:
            assert bool(torch.isfinite(q.grad).all()) and q.grad.shape == q.shape
        before = [w.detach().clone() for w in params]
        opt.step()
        for w, b, m in zip(params, before, ws):
            assert not torch.equal(w.detach(), b)
            _same(m.rows, O.quantize(w.detach().cpu(), "fp4"), "rows")
            _same(m.cols, O.quantize(w.detach().cpu().t(), "fp4"), "cols")


def test_layers_on_no_tokens(p):
    w, gain = torch.randn(40, 64, device=DEV, requires_grad=True), torch.ones(64, device=DEV, requires_grad=True)
    x = torch.zeros(0, 64, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    out, s = p.mx_norm_linear(x, gain, p.MxWeight(w), x)
    gx, gg, gw = torch.autograd.grad((out.float().sum() + s.float().sum()), (x, gain, w))
    assert out.shape == (0, 40) and gx.shape == (0, 64) and not gg.any() and not gw.any() and gw.shape == w.shape
    (gw,) = torch.autograd.grad(p.mx_linear(x, p.MxWeight(w)).float().sum(), w)
    assert not gw.any()


def test_one_tensor_as_input_and_residual(p):
    """s = 2 x: both paths' gradients add up; the graph is walked twice."""
    g = torch.Generator().manual_seed(36)
    x, w, gain = torch.randn(6, 64, generator=g), torch.randn(32, 64, generator=g), torch.ones(64)
    d = torch.randn(6, 32, generator=g)
    _, _, dx, _, dw = _layer_reference(x, x, gain, w, d, None, "fp8", "fp8", "fp4")
    xg, wg = x.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
    out, _ = p.mx_norm_linear(xg, gain.to(DEV), p.MxWeight(wg), xg)
    for _ in range(2):
        gx, gw = torch.autograd.grad(out, (xg, wg), d.to(DEV), retain_graph=True)
        assert float((gx.cpu().double() - 2 * dx).norm() / dx.norm()) < 3e-3 and float((gw.cpu().double() - dw).norm() / dw.norm()) < 5e-3


# ---- streams, graphs, size ---------------------------------------------------------------------------------------------------------------

def test_another_stream(p):
    x = torch.randn(300, 700, device=DEV)
    w = p.mx_quantize(torch.randn(200, 700, device=DEV), "fp4")
    want = p.mx_matmul(p.mx_quantize(x, "fp8"), w)
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        y = x * 2
        got = p.mx_matmul(p.mx_quantize(y * 0.5, "fp8"), w)
    st.synchronize()
    assert torch.equal(got, want)


def test_two_streams_at_once(p):
    """The same operators on two streams, interleaved: each has its own outputs and workspaces."""
    sets = []
    for seed, (m, n, k) in ((1, (300, 200, 5000)), (2, (700, 130, 3000))):
        g = torch.Generator(device=DEV).manual_seed(seed)
        sets.append((torch.randn(m, k, generator=g, device=DEV), p.mx_quantize(torch.randn(n, k, generator=g, device=DEV)), torch.ones(k, device=DEV)))

    def run(x, w, gain):
        y, s, inv = p.rms_norm_mx(x, gain, x, which="both")
        return p.mx_matmul(y[0], w, out_dtype=torch.float32), p.mx_dequantize(y[1]), *p.rms_norm_mx_backward(x, s, gain, inv)
    want = [run(*t) for t in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(run(*sets[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for r in got[i]:
            for a, b in zip(r, want[i]):
                assert torch.equal(a, b)


def test_layer_captured_with_its_backward(p):
    """Forward and backward of the differentiable layer in a graph (torch.autograd.grad inside the capture), the weight renewed between replays."""
    g = torch.Generator(device=DEV).manual_seed(4)
    x, res, dout = (torch.randn(130, n, generator=g, device=DEV).to(torch.bfloat16) for n in (96, 96, 70))
    w = torch.nn.Parameter(torch.randn(70, 96, generator=g, device=DEV))
    gain = torch.ones(96, device=DEV)
    weight = p.MxWeight(w)

    def run():
        leaves = [x.detach().requires_grad_(), res.detach().requires_grad_(), gain.detach().requires_grad_()]
        out, s = p.mx_norm_linear(leaves[0], leaves[2], weight, leaves[1])
        return out.detach(), s.detach(), *torch.autograd.grad(out, [*leaves, w], dout)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = run()
    for i in range(4):
        with torch.no_grad():
            w.add_(0.1 * torch.randn_like(w))
            x.copy_(torch.randn_like(x))
        weight.refresh()
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in outs]
        for a, b in zip(kept, run()):
            assert torch.equal(a, b), i


def test_graph_replays(p):
    """Two graphs captured one after the other and replayed in turn, with eager work between: each has workspaces of its own."""
    def run(x, w, res, gain):
        y, s, inv = p.rms_norm_mx(x, gain, res, which="both")
        out = p.mx_matmul(y[0], w, out_dtype=torch.float32)
        d = p.mx_quantize(out, "fp4", which="both")
        dw = p.mx_matmul(d[1], y[1], out_dtype=torch.float32)                   # few outputs, split contraction
        dx, dg = p.rms_norm_mx_backward(s, s, gain, inv, ds=res)
        return [out, dw, dx, dg, s]
    sets = []
    for seed, (t, k, n) in ((1, (1100, 96, 70)), (2, (600, 200, 130))):
        g = torch.Generator(device=DEV).manual_seed(seed)
        x, res = (torch.randn(t, k, generator=g, device=DEV) for _ in range(2))
        w = p.mx_quantize(torch.randn(n, k, generator=g, device=DEV))
        gain = torch.ones(k, device=DEV)
        run(x, w, res, gain)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = run(x, w, res, gain)
        sets.append((graph, outs, x, w, res, gain))
    for i in range(4):
        for graph, outs, x, w, res, gain in sets:
            x.copy_(torch.randn_like(x))
            graph.replay()
            want = run(x, w, res, gain)
            torch.cuda.synchronize()
            for a, b in zip(outs, want):
                assert torch.equal(a, b), i


def test_offsets_past_32_bits(p):
    """Tensors of more than 2^32 elements (and bytes): the last rows are what the same rows are by themselves."""
    rows, k = (1 << 20) + 3, 4096 + 5
    x = torch.zeros(rows, k, dtype=torch.bfloat16, device=DEV)
    tail = torch.randn(130, k, device=DEV).to(torch.bfloat16)
    x[-130:] = tail
    x[7, 9] = 3.0
    q = p.mx_quantize(x, "fp8")
    t = p.mx_quantize(tail, "fp8")
    assert torch.equal(q.codes[-130:], t.codes) and torch.equal(q.scales[-130:], t.scales)
    assert float(p.mx_dequantize(p.MxTensor(q.codes[7:8], q.scales[7:8], (1, k), "fp8"))[0, 9]) == 3.0
    del x
    w = p.mx_quantize(torch.randn(20, k, device=DEV), "fp4")
    big, small = p.mx_matmul(q, w, out_dtype=torch.float32), p.mx_matmul(t, w, out_dtype=torch.float32)
    assert torch.equal(big[:7].cpu(), torch.zeros(7, 20))
    assert bool(((big[-130:] - small).abs() <= 1e-5 * small.abs().max()).all())
    big = p.mx_matmul(w, q, out_dtype=torch.float32)                            # the long operand second, few rows first
    assert bool(((big[:, -130:] - small.t()).abs() <= 1e-5 * small.abs().max()).all())


def _layers(p, seed, t=300, k=512, n=520):
    g = torch.Generator().manual_seed(seed)
    x, res = (torch.randn(t, k, generator=g).to(DEV, torch.bfloat16).requires_grad_() for _ in range(2))
    gain = (1 + 0.1 * torch.randn(k, generator=g)).to(DEV).requires_grad_()
    w, v = (p.MxWeight(torch.nn.Parameter(0.05 * torch.randn(*s, generator=g).to(DEV)), "fp4") for s in ((n, k), (k, n)))

    def run(x, res, gain):
        y, s = p.mx_norm_linear(x, gain, w, res)
        return p.mx_linear(y, v) + s
    return run, (x, res, gain), (w, v)


def test_activations_are_freed_by_the_backward_pass(p):
    run, leaves, ws = _layers(p, 50, t=4096)
    grads = lambda out: torch.autograd.grad(out.float().square().sum(), (*leaves, *(w.param for w in ws)))      # noqa: E731
    grads(run(*leaves))
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    out = run(*leaves)
    held = torch.cuda.memory_allocated() - before
    got = grads(out)
    del got
    left = torch.cuda.memory_allocated() - before
    # held: the output, s, the activations of both layers (fp8, 1 byte an element and more); left, with the graph's nodes alive: the output, in 2 bytes
    assert out.grad_fn is not None and held > left and left <= 2 * out.numel() + 4096, (held, left)
    with pytest.raises(RuntimeError):
        grads(out)


@pytest.mark.parametrize("way", ["checkpoint", "offload"])
def test_saved_tensors_may_be_packed(p, way):
    from torch.utils.checkpoint import checkpoint
    run, leaves, ws = _layers(p, 51)
    wrt = (*leaves, *(w.param for w in ws))
    want = torch.autograd.grad(run(*leaves).float().square().sum(), wrt)
    if way == "checkpoint":
        got = torch.autograd.grad(checkpoint(run, *leaves, use_reentrant=False).float().square().sum(), wrt)
    else:
        with torch.autograd.graph.save_on_cpu():
            out = run(*leaves)
        for w in ws:                                                   # (what was packed is what counts)
            with torch.no_grad():
                w.param.mul_(2)
            w.refresh()
        got = torch.autograd.grad(out.float().square().sum(), wrt)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_s_needs_a_gradient_only_through_its_terms(p):
    run, (x, res, gain), (w, _) = _layers(p, 52)
    y, s = p.mx_norm_linear(x.detach(), gain, w, res.detach())
    assert y.requires_grad and not s.requires_grad
    y.float().sum().backward()
    assert gain.grad is not None and w.param.grad is not None
    y, s = p.mx_norm_linear(x.detach(), gain, w, res)
    assert y.requires_grad and s.requires_grad


def test_layers_under_a_deep_copied_module(p):
    import copy
    run, leaves, (w, _) = _layers(p, 53)
    x = leaves[0].detach()
    want = p.mx_linear(x, w).detach()
    c = copy.deepcopy(w)
    with torch.no_grad():
        w.param.zero_()
    w.refresh()
    assert torch.equal(p.mx_linear(x, c), want) and not p.mx_linear(x, w).any()
    c.refresh()
    assert torch.equal(p.mx_linear(x, c), want)


# ---- the norm's sums ---------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("rows,cols", [(2049, 520), (1500, 768), (700, 2100), (300, 4096), (70, 16384)])
@pytest.mark.parametrize("dt", DTYPES)
def test_norm_inv_is_the_nearest(p, rows, cols, dt):
    """Squares and their sum are held in 64 bits: inv is off by its own rounding alone, half a step of fp32 (and 2^-40, far above what 16384 additions in 64
    bits can amount to).  y is then off by inv's rounding and its own, in either form, whatever the number of rows."""
    g = torch.Generator().manual_seed(61)
    x, r = (torch.randn(rows, cols, generator=g).to(dt) for _ in range(2))
    gain = 1 + 0.3 * torch.randn(cols, generator=g)
    s, inv, y = O.norm(x, gain, r, 1e-5)
    (yr, yc), gs, ginv = p.rms_norm_mx(x.to(DEV), gain.to(DEV), r.to(DEV), which="both")
    assert torch.equal(gs.cpu(), s)
    assert bool(((ginv.cpu().double() - inv).abs() <= (EPS24 + 2.0 ** -40) * inv).all())
    _check_norm_codes(yr, y, "fp8", cols, 2.01 * EPS24)
    _check_norm_codes(yc, y.t().contiguous(), "fp8", rows, 2.01 * EPS24)


def test_norm_of_very_large_and_very_small_rows(p):
    """Sums of squares far outside fp32's range: the rows are normalised like any other."""
    g = torch.Generator().manual_seed(62)
    x = torch.randn(6, 700, generator=g) * torch.tensor([1e25, 1e-25, 1.0, 1e36, 1e-30, 1e19])[:, None]
    gain = torch.ones(700)
    for dt in (torch.float32, torch.bfloat16):
        s, inv, y = O.norm(x.to(dt), gain, None, 0.0)
        (yr, yc), _, ginv = p.rms_norm_mx(x.to(dt).to(DEV), gain.to(DEV), eps=0.0, which="both")
        # (the smallest number here, 1e-36, is normal)
        assert bool(((ginv.cpu().double() - inv).abs() <= (EPS24 + 2.0 ** -40) * inv).all())
        _check_norm_codes(yr, y, "fp8", 700, 2.01 * EPS24)
        _check_norm_codes(yc, y.t().contiguous(), "fp8", 6, 2.01 * EPS24)


# ---- products, kernel by kernel ----------------------------------------------------------------------------------------------------------

FMT = {"fp4": 4, "fp8": 8}
PAIRS = [("fp4", "fp4"), ("fp4", "fp8"), ("fp8", "fp4"), ("fp8", "fp8")]


def _plan(p, m, n, k, fa, fb, dt):
    """(tile rows, tile columns, splits of K, WIDE) that the library chooses; 0 columns: the few-rows kernel."""
    import ctypes as C
    from psgd_torch_amd import _lib
    out = [C.c_int() for _ in range(4)]
    assert _lib.lib().psgdk_test_mx_plan(m, n, k, FMT[fa], FMT[fb], p.mx._DTYPE[dt], *[C.byref(v) for v in out]) == 0
    return tuple(v.value for v in out)


def _device_operand(p, rows, k, fmt, seed, scales=None):
    """(MX form, its values in 64 bits on the device) of normally distributed numbers; scales: a factor for each block of 32 (rows x blocks)."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(rows, k, generator=g, device=DEV)
    if scales is not None:
        x = x * scales.to(DEV).repeat_interleave(32, 1)[:, :k]
    q = p.mx_quantize(x, fmt)
    return q, p.mx_dequantize(q, torch.float32).double()


def _product_into_guarded(p, qa, qb, dt):
    """mx_matmul by the C call into the middle of a larger buffer: what lies before and behind the output stays as it was."""
    import ctypes as C
    from psgd_torch_amd import _lib
    (m, k), n, lib, code = qa.shape, qb.shape[0], _lib.lib(), p.mx._DTYPE[dt]
    guard = 1 << 16
    buf = torch.full((m * n + 2 * guard,), 77.0, dtype=dt, device=DEV)
    out = buf[guard:guard + m * n].view(m, n)
    wb = C.c_size_t()
    assert lib.psgdk_mx_matmul_work_bytes(m, n, k, FMT[qa.fmt], FMT[qb.fmt], code, C.byref(wb)) == 0
    work = torch.empty(max(wb.value, 16), dtype=torch.uint8, device=DEV)
    rc = lib.psgdk_mx_matmul(*qa._ptrs, m, FMT[qa.fmt], *qb._ptrs, n, FMT[qb.fmt], k, out.data_ptr(), code, work.data_ptr(), wb.value,
                             torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    assert bool((buf[:guard] == 77).all()) and bool((buf[guard + m * n:] == 77).all())
    return out


def _check_kernel(p, m, n, k, fa, fb, dt, tile, splits=None):
    plan = _plan(p, m, n, k, fa, fb, dt)
    assert plan[:2] == tile and (splits is None or plan[2] == splits), (m, n, k, fa, fb, dt, plan)
    (qa, a), (qb, b) = _device_operand(p, m, k, fa, 71), _device_operand(p, n, k, fb, 72)
    want = a @ b.t().contiguous()
    got = _product_into_guarded(p, qa, qb, dt)
    _check_product(got, a, b, want, "fp8" in (fa, fb) and dt != torch.float32)
    assert torch.equal(p.mx_matmul(qa, qb, out_dtype=dt), got)                    # the same bits, whatever lies around the output
    # the first rows by themselves, through the few-rows kernel
    few = p.MxTensor(qa.codes[:3], qa.scales[:3], (3, k), fa)
    assert _plan(p, 3, n, k, fa, fb, dt)[1] == 0
    _check_product(p.mx_matmul(few, qb, out_dtype=dt), a[:3], b, want[:3], "fp8" in (fa, fb) and dt != torch.float32)


# ragged in M and N (an odd output pitch, the last tile's columns stored one by one), K past a multiple of 256: 3, 5, 9 and 10 blocks, of which scales come in fours
LARGE = [(4090, 4095, 2500, fa, fb, dt) for fa, fb in PAIRS for dt in (torch.bfloat16, torch.float16)] + \
        [(4090, 4095, 2500, "fp4", "fp4", torch.float32)] + \
        [(3900, 4091, 2049, fa, fb, torch.bfloat16) for fa, fb in PAIRS] + [(4090, 4095, 700, fa, fb, torch.bfloat16) for fa, fb in PAIRS[1:]] + \
        [(4095, 4090, 1300, fa, fb, torch.bfloat16) for fa, fb in PAIRS[1:]]


@pytest.mark.parametrize("m,n,k,fa,fb,dt", LARGE)
def test_matmul_tiles_of_256(p, m, n, k, fa, fb, dt):
    _check_kernel(p, m, n, k, fa, fb, dt, (256, 256), 1)


@pytest.mark.parametrize("fa,fb", PAIRS[1:])
def test_matmul_tiles_of_256_split(p, fa, fb):
    _check_kernel(p, 4345, 139, 33900, fa, fb, torch.bfloat16, (256, 256), 8)


@pytest.mark.parametrize("fa,fb", PAIRS)
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,n,k,splits", [(33, 50001, 200, 1), (50, 16500, 600, 1), (5, 50257, 1100, 1), (64, 33001, 513, 1), (17, 40001, 520, 1), (64, 4099, 4000, None),
                                          (33, 2001, 5900, 8)])
def test_matmul_tiles_of_64(p, m, n, k, splits, fa, fb, dt):
    _check_kernel(p, m, n, k, fa, fb, dt, (64, 128), splits)


def _block_maxima(a, b):
    """The sum over K's blocks of 32 of the largest product of each, for every element of A B^T (M x N, 64 bits)."""
    k = -(-a.shape[1] // 32) * 32
    a, b = (torch.nn.functional.pad(v.abs(), (0, k - v.shape[1])) for v in (a, b))
    out = torch.zeros(a.shape[0], b.shape[0], dtype=torch.float64, device=a.device)
    for i in range(0, k, 32):
        out += (a[:, None, i:i + 32] * b[None, :, i:i + 32]).amax(-1)
    return out


@pytest.mark.parametrize("spread", [2, 8, 13, 20, 30])
@pytest.mark.parametrize("m,n,k", [(3, 40, 128), (3, 40, 1000), (50, 300, 1000), (300, 300, 1024)])
@pytest.mark.parametrize("fa,fb", PAIRS)
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
def test_matmul_of_blocks_far_apart(p, m, n, k, fa, fb, dt, spread):
    """Scales within a row up to 2^spread apart on either side.  Sums are fp32 sums of the blocks (_product_bound); an 8-bit operand and a 16-bit output
    add what the scaled instruction drops: of each of a block's 32 products less than 2^-13 of the largest one of that block."""
    g = torch.Generator().manual_seed(73)
    sa, sb = (torch.exp2((torch.rand(r, -(-k // 32), generator=g) * (spread + 1)).floor()) for r in (m, n))
    (qa, a), (qb, b) = _device_operand(p, m, k, fa, 74, sa), _device_operand(p, n, k, fb, 75, sb * 2.0 ** -spread)
    want = a @ b.t().contiguous()
    if dt == torch.float16:
        (qa, a), (qb, b) = _device_operand(p, m, k, fa, 74, sa * 2.0 ** -spread), _device_operand(p, n, k, fb, 75, sb * 2.0 ** -spread)
        want = a @ b.t().contiguous()
        assert float(want.abs().max()) < 60000
    got = p.mx_matmul(qa, qb, out_dtype=dt)
    bound = _product_bound(a, b, dt, want, False)
    if "fp8" in (fa, fb) and dt != torch.float32:
        bound = bound + 32 * 2.0 ** -13 * _block_maxima(a, b)
    err = (got.double() - want).abs()
    assert bool((err <= bound).all()), float((err / bound).max())


def test_matmul_sums_of_two_4_bit_operands_are_fp32_sums(p):
    """What one instruction adds (128 elements) with two 4-bit operands: a large pair that cancels within its block leaves a later block's small product as
    it is, whatever its size; where the small one has to share a partial sum with a large one, it is kept while 2^gap + 1 has 24 bits (an fp32 sum can
    promise no more, in whatever order it adds)."""
    for gap in range(0, 45):
        for i, j, l, most in ((0, 1, 32, 99), (3, 31, 96, 99), (64, 70, 0, 23), (0, 64, 32, 23), (32, 96, 64, 23)):
            x = torch.zeros(2, 128)
            x[:, i], x[:, j], x[:, l] = 2.0 ** gap, -2.0 ** gap, 1.0
            a, b = p.mx_quantize(x.to(DEV)), p.mx_quantize(torch.ones(20, 128, device=DEV))
            assert torch.equal(p.mx_dequantize(a, torch.float32).cpu(), x)
            got = p.mx_matmul(a, b, out_dtype=torch.float32).cpu()
            if gap <= most:
                assert torch.equal(got, torch.ones(2, 20)), (gap, i, j, l)
            else:
                assert bool(((got == 0) | (got == 1)).all()), (gap, i, j, l)


def test_matmul_bits_dropped_with_an_8_bit_operand(p):
    """One large product, its negative in the next 128 elements, a small one beside the first: with a 16-bit output what lies below 2^-13 of the largest of
    the block is dropped, with a 32-bit output nothing is."""
    for fa, fb in PAIRS[1:]:
        for e in range(8, -10, -1):
            x = torch.zeros(1, 256)
            x[0, 0], x[0, 3], x[0, 128] = 256.0, 2.0 ** e, -256.0
            one = torch.ones(20, 256)
            a, b = (p.mx_quantize(v.to(DEV), f) for v, f in (((x, fa), (one, fb)) if fa == "fp8" else ((one[:1], fa), (x.expand(20, 256), fb))))
            assert bool((p.mx_matmul(a, b, out_dtype=torch.float32) == 2.0 ** e).all())
            got = p.mx_matmul(a, b)
            assert bool(((got.float() - 2.0 ** e).abs() <= 256 * 2.0 ** -13).all())


# ---- what a caller may hand over, and what is refused ------------------------------------------------------------------------------------

def test_weight_forms_handed_over_are_kept(p):
    """A form that is handed over keeps its contents and its memory; what is missing is rounded from the parameter; a refresh renews both."""
    g = torch.Generator().manual_seed(81)
    w, other = (torch.randn(40, 72, generator=g) for _ in range(2))
    param = torch.nn.Parameter(w.to(DEV))
    for fmt in ("fp4", "fp8"):
        own = [O.quantize(v, fmt) for v in (w, w.t())]
        theirs = [O.quantize(v, fmt) for v in (other, other.t())]
        for have_rows, have_cols, backward in ((True, False, True), (False, True, True), (True, True, True), (True, False, False), (False, True, False), (False, False, False)):
            r, c = p.mx_quantize(other.to(DEV), fmt, which="both")
            r, c = r if have_rows else None, c if have_cols else None
            weight = p.MxWeight(param, fmt, backward=backward, rows=r, cols=c)
            assert (r is None or weight.rows is r) and (c is None or weight.cols is c) and weight.fmt == fmt
            _same(weight.rows, theirs[0] if have_rows else own[0], "rows")
            assert (weight.cols is not None) == (have_cols or backward)
            if weight.cols is not None:
                _same(weight.cols, theirs[1] if have_cols else own[1], "cols")
                x = torch.randn(3, 72, device=DEV, requires_grad=True)
                (gx,) = torch.autograd.grad(p.mx_linear(x, weight).sum(), x)
                assert gx.shape == x.shape
            weight.refresh()
            _same(weight.rows, own[0], "rows, refreshed")
            if weight.cols is not None:
                _same(weight.cols, own[1], "cols, refreshed")
    r, c = p.mx_quantize(other.to(DEV), "fp8", which="both")
    assert p.MxWeight(param, rows=r).fmt == p.MxWeight(param, cols=c).fmt == "fp8"               # the given form's, for both
    _same(p.MxWeight(param, cols=c).rows, O.quantize(w, "fp8"), "rows")
    with pytest.raises(p._lib.PsgdkError):
        p.MxWeight(param, rows=r, cols=p.mx_quantize(other.to(DEV), "fp4", which="cols"))


def test_norm_backward_names_what_it_refuses(p):
    E = p._lib.PsgdkError
    s, g, inv = torch.ones(4, 64, device=DEV), torch.ones(64, device=DEV), torch.ones(4, device=DEV)
    for call, words in ((lambda: p.rms_norm_mx_backward(s, s, g, inv, ds=s[:3]), "ds is .*, s is "), (lambda: p.rms_norm_mx_backward(s, s, g, inv, ds=s.half()), "ds is .*, s is "),
                        (lambda: p.rms_norm_mx_backward(s, s, g, inv, ds=s.cpu()), "ds lives on "), (lambda: p.rms_norm_mx_backward(s, s.cpu(), g, inv), "s lives on "),
                        (lambda: p.rms_norm_mx_backward(s, s.double(), g, inv), "s has dtype "), (lambda: p.rms_norm_mx_backward(s, s[:, :0], g[:0], inv), "s of shape "),
                        (lambda: p.rms_norm_mx(s, g, s[:3]), "residual is .*, x is ")):
        with pytest.raises(E, match=words):
            call()


def test_norm_backward_refuses_to_drop_gradients(p):
    E = p._lib.PsgdkError
    dy, s, ds = (torch.randn(4, 64, device=DEV) for _ in range(3))
    inv, gain = torch.ones(4, device=DEV), torch.nn.Parameter(torch.ones(64, device=DEV))
    want = p.rms_norm_mx_backward(dy, s, gain, inv, ds=ds)                        # a parameter as the gain is what a program has
    assert not want[0].requires_grad and not want[1].requires_grad
    for i in range(4):
        a = [t.clone().requires_grad_(j == i) for j, t in enumerate((dy, s, inv, ds))]
        with pytest.raises(E, match="does not record gradients"):
            p.rms_norm_mx_backward(a[0], a[1], gain, a[2], ds=a[3])
        with torch.no_grad():
            got = p.rms_norm_mx_backward(a[0], a[1], gain, a[2], ds=a[3])
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("shape", [(5, 1), (1, 1), (3, 7), (1, 40)])
def test_negated_views(p, shape):
    """Imaginary parts of conjugated tensors: views whose memory has the other sign."""
    g = torch.Generator().manual_seed(82)
    x, r, gain = (torch.randn(s, generator=g).to(DEV) for s in (shape, shape, shape[1:]))
    neg = lambda t: torch.complex(torch.zeros_like(t), -t).conj().imag      # noqa: E731  (reads as t)
    assert neg(x).is_neg() and torch.equal(neg(x), x)
    a, b = p.mx_quantize(neg(x), which="both"), p.mx_quantize(x, which="both")
    assert all(torch.equal(i.codes, j.codes) and torch.equal(i.scales, j.scales) for i, j in zip(a, b))
    ya, sa, ia = p.rms_norm_mx(neg(x), neg(gain), neg(r))
    yb, sb, ib = p.rms_norm_mx(x, gain, r)
    assert torch.equal(ya.codes, yb.codes) and torch.equal(sa, sb) and torch.equal(ia, ib)
    da, db = p.rms_norm_mx_backward(neg(x), neg(sb), neg(gain), neg(ib), ds=neg(r)), p.rms_norm_mx_backward(x, sb, gain, ib, ds=r)
    assert torch.equal(da[0], db[0]) and torch.equal(da[1], db[1])
