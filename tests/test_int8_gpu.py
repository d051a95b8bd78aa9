"""8-bit rows and their products on the GPU against the definition in 64 bits: sizes from one element to long rows, odd ones, strides, halves of joint
rows, rows of zeros, infinities and NaN."""
import pytest
import torch

from levanter_b200.ops import int8 as I
from levanter_b200.ops import lib
from levanter_b200.utils.activation import ActivationFunctionEnum as Act

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
STEP = {BF: 2.0 ** -8, F32: 2.0 ** -24}  # most that one rounding moves a value, relative to it


def rand(*shape, seed=0, std=1.0, dtype=BF):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


def whole(y, factor=None):
    """Whole numbers and scales of ``factor * y`` in 64 bits."""
    y = y.double()
    top = y.abs().amax(-1, keepdim=True)
    most = top if factor is None else top * factor
    live = most >= I.TINY
    return torch.where(live, (127 * y / top).round(), 0.0), torch.where(live, most / 127, 0.0).squeeze(-1)


def check_rows(rows, y, factor=None, slack=0.0):
    """``slack``: how far, relative to itself, an element of ``y`` may be from the kernel's, so that near a tie either whole number is right."""
    q, s = whole(y, factor)
    got = rows.values.double()
    off = (got - q).abs()
    if slack == 0.0:
        assert torch.equal(got, q)
    else:
        exact = 127 * y.double() / y.double().abs().amax(-1, keepdim=True)
        # whole numbers one apart only where the quotient is within its own error (its element's and the largest one's) of the border
        near = ((exact - exact.floor() - 0.5).abs() <= 127 * 2 * slack)
        assert off.max() <= 1 and bool((near | (off == 0)).all())
    # fp32 scale: the norm's factor (a sum over the row, a root), the largest element, a product and a quotient
    assert ((rows.scale.double() - s).abs() <= (slack + 2.0 ** -20) * s).all()


SIZES = [(1, 1), (3, 7), (5, 8), (2, 255), (9, 256), (4, 513), (7, 1000), (130, 1024), (3, 1025), (5, 2048), (2, 4096), (3, 5001), (2, 8192), (2, 14336), (3, 16385),
         (1, 32768), (2, 40001)]


@pytest.mark.parametrize("rows,cols", SIZES)
@pytest.mark.parametrize("dtype", [BF, F32])
def test_quantize_rows(rows, cols, dtype):
    x = rand(rows, cols, seed=rows * 7 + cols, dtype=dtype)
    x[0, cols // 2] = x[0].abs().max() / 2  # half of the largest value: a tie
    check_rows(I.quantize_rows(x), x, slack=0.0 if dtype == BF else 2.0 ** -23)


def test_quantize_rows_with_strides_and_more_dimensions():
    wide = rand(6, 5, 700, seed=3)
    for x in (wide[:, :, 3:500], wide[::2, 1:3], wide.transpose(0, 1), wide[:, :, ::2], wide[0, 0], rand(1, 300).expand(4, 300)):
        rows = I.quantize_rows(x)
        assert rows.shape == x.shape and rows.scale.shape == x.shape[:-1]
        check_rows(rows, x)


def test_rows_of_zeros_tiny_values_infinities_and_nan():
    x = rand(8, 600, seed=4, dtype=F32)
    x[0] = 0
    x[1] *= 1e-33
    x[2, 5] = float("inf")
    x[3, 7] = float("nan")
    x[4] *= 1e30
    x[5] = 0
    x[5, 9] = -3.0
    x[6, 0] = -float("inf")
    for dtype in (F32, BF):
        rows = I.quantize_rows(x.to(dtype))
        assert rows.scale[0] == 0 and rows.scale[1] == 0 and not rows.values[:2].any()
        assert rows.scale[[2, 3, 6]].isnan().all() and not rows.values[[2, 3, 6]].any()
        assert rows.values[5, 9] == -127 and rows.values[5].abs().sum() == 127
        check_rows(I.Int8Rows(rows.values[4:6], rows.scale[4:6]), x[4:6].to(dtype), slack=0.0 if dtype == BF else 2.0 ** -23)
        back = rows.dequantize(F32)
        assert back[[2, 3, 6]].isnan().all() and not back[:2].any()
    empty = I.quantize_rows(rand(0, 64))
    assert empty.shape == (0, 64) and empty.dequantize().shape == (0, 64)


@pytest.mark.parametrize("cols", [64, 1000, 4096, 9007])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_rows_of_the_largest_numbers(cols, dtype):
    m = torch.finfo(dtype).max  # as masks have it
    x = (rand(3, cols, seed=6, dtype=F32).clamp(-1, 1) * m).to(dtype).clamp(-m, m)
    x[:, :7] = torch.tensor([m, m / 2, -m / 2, m / 4, -m, m / 127 * 3, 1.0], dtype=dtype)
    x[1] = -m
    x[2, 7:] = torch.arange(cols - 7, device="cuda").remainder(254).sub(127).double().add(0.5).mul(m).div(127).to(dtype)  # close to ties
    rows = I.quantize_rows(x)
    check_rows(rows, x, slack=0.0 if dtype == BF else 2.0 ** -23)
    back = rows.dequantize(F32)
    assert bool(back.isfinite().all()) and bool(((back[:, 4].double() + m).abs() <= 2.0 ** -22 * m).all())


@pytest.mark.parametrize("rows,cols", SIZES)
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("residual", [False, True])
def test_rms_norm_int8(rows, cols, dtype, residual):
    x, w = rand(rows, cols, seed=cols, dtype=dtype), (1 + rand(cols, seed=1, std=0.1, dtype=F32)).to(BF if cols % 2 else F32)
    r = rand(rows, cols, seed=2, dtype=dtype) if residual else None
    got, h = I.rms_norm_int8(x, w, 1e-5, residual=r)
    want = x if r is None else (x.float() + r.float()).to(dtype)
    assert (h is None) == (r is None) and (h is None or torch.equal(h, want))
    d = want.double()
    exact = dtype == BF and w.dtype == BF  # the product of two bf16 numbers is exact in fp32
    check_rows(got, d * w.double(), (d.square().mean(-1, keepdim=True) + 1e-5).rsqrt(), slack=0.0 if exact else 2.0 ** -22)


def test_rms_norm_int8_offset_no_weight_and_tiny_rows():
    x = rand(5, 700, seed=8)
    x[1] = 0
    d = x.double()
    f = (d.square().mean(-1, keepdim=True) + 1e-6).rsqrt()
    check_rows(I.rms_norm_int8(x, None)[0], d, f)
    w = rand(700, seed=9, std=0.1)
    check_rows(I.rms_norm_int8(x, w, w_offset=1.0)[0], d * (w.double() + 1.0), f, slack=2.0 ** -22)
    x[2, 3] = float("nan")
    x[3, 4] = float("inf")
    rows, _ = I.rms_norm_int8(x, w)
    assert rows.scale[[2, 3]].isnan().all() and not rows.scale[[0, 1, 4]].isnan().any()


@pytest.mark.parametrize("rows,cols", [(1500, 64), (3, 1000), (700, 4096), (700, 8208), (5, 4095), (700, 11007), (400, 14335), (2, 40001)])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("eps", [1e-5, 0.0])
def test_norms_whose_squares_leave_the_range_of_fp32(rows, cols, dtype, residual, eps):
    """Among ordinary rows, whose bits do not depend on them."""
    x, w = rand(rows, cols, seed=cols, dtype=dtype).clamp(-4, 4), (1 + rand(cols, seed=1, std=0.1, dtype=F32)).to(dtype)
    r = rand(rows, cols, seed=2, dtype=dtype).clamp(-4, 4) if residual else None
    first = I.rms_norm_int8(x, w, eps, residual=r)[0]
    sizes = torch.ones(rows, device="cuda")
    sizes[1::7], sizes[2::7] = 1e20, 3e37
    if eps == 0.0:
        sizes[3::7], sizes[4::7] = 1e-22, 1e-30
    x = (x.float() * sizes[:, None]).to(dtype)
    r = None if r is None else (r.float() * sizes[:, None]).to(dtype)
    x[0, cols // 2] = float("inf")
    got, h = I.rms_norm_int8(x, w, eps, residual=r)
    want = x if r is None else (x.float() + r.float()).to(dtype)
    assert h is None or torch.equal(h, want)
    assert got.scale[0].isnan() and not got.values[0].any()
    same = sizes == 1
    same[0] = False
    assert torch.equal(got.values[same], first.values[same]) and torch.equal(got.scale[same], first.scale[same])
    d = want[1:].double()
    check_rows(I.Int8Rows(got.values[1:], got.scale[1:]), d * w.double(), (d.square().mean(-1, keepdim=True) + eps).rsqrt(), slack=0.0 if dtype == BF else 2.0 ** -22)


@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (5, 500), (2, 4096), (3, 5001), (2, 14336), (1, 40001)])
@pytest.mark.parametrize("act", ["silu", "gelu_new", "gelu", "relu", "quick_gelu"])
def test_gated_activation_int8(rows, cols, act):
    y = rand(rows, 2 * cols, seed=cols, std=3.0)
    got = I.gated_activation_int8(y[:, :cols], y[:, cols:], Act(act))
    g, u = y.double().chunk(2, -1)
    # the exponential's argument is rounded (|g| <= 20: 20 * 2^-23), the exponential, the quotient and the product each by 2^-22 at most; where 1 + tanh
    # or 1 + erf cancels (g < 0), what is lost counts against 1 and not against the little that is left
    want = Act(act).to_fn()(g) * u
    top = want.abs().amax(-1, keepdim=True)
    if act in ("gelu_new", "gelu"):
        q, s = whole(want)
        assert (got.values.double() - 127 * want / top.clamp(min=I.TINY)).abs().max() <= 0.5 + 127 * 2.0 ** -18
        assert ((got.scale.double() - s).abs() <= 2.0 ** -18 * s).all()
    else:
        check_rows(got, want, slack=2.0 ** -18)


def test_gated_activation_int8_of_fp32_rows_and_other_gates():
    from levanter_b200.ops.glu import ClampedGlu

    g, u = rand(3, 333, seed=1, dtype=F32), rand(3, 333, seed=2, dtype=F32)
    check_rows(I.gated_activation_int8(g, u, Act.silu), torch.nn.functional.silu(g.double()) * u.double(), slack=2.0 ** -18)
    g, u = g.to(BF), u.to(BF)
    check_rows(I.gated_activation_int8(g, u, ClampedGlu(7.0)), ClampedGlu(7.0)(g, u))
    check_rows(I.gated_activation_int8(g, u, Act.tanh), torch.tanh(g) * u)


@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (5, 512), (700, 1000)])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_dequantize(rows, cols, dtype):
    held = I.quantize_rows(rand(rows, cols, seed=5))
    assert torch.equal(held.dequantize(dtype), (held.values.float() * held.scale[:, None]).to(dtype))
    part = I.Int8Rows(held.values[:, cols // 2:], held.scale)  # rows that start anywhere
    assert torch.equal(part.dequantize(dtype), (part.values.float() * part.scale[:, None]).to(dtype))


@pytest.mark.parametrize("cols", [12, 17, 333, 4095, 4097])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_dequantize_of_rows_that_start_and_end_anywhere(cols, dtype):
    values = torch.randint(-128, 128, (37, cols + 40), device="cuda", dtype=torch.int8)
    scale = torch.rand(37, device="cuda")
    for first in (0, 1, 2, 3, 6, 16):
        for ld in (cols, cols + 3, cols + 24):
            part = values.flatten()[first:].as_strided((37, cols), (ld, 1), first)
            assert torch.equal(I.Int8Rows(part, scale).dequantize(dtype), (part.float() * scale[:, None]).to(dtype))


# ------------------------------------------------------------------------------------------------ products
def int8(rows, cols, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    v = torch.randint(-128, 128, (rows, cols), generator=g, device="cuda", dtype=torch.int32).to(torch.int8)
    return I.Int8Rows(v, torch.rand(rows, generator=g, device="cuda") + 0.5)


def check_product(rows, weight, bias=None, residual=None, out_dtype=BF, **form):
    y = I._product(rows, weight, bias, residual, out_dtype, **form)
    lib.check_status()
    sums = rows.values.double() @ weight.values.double().t()
    want = sums * rows.scale.double()[..., None] * weight.scale.double()
    size = want.abs()
    for t in (bias, residual):
        if t is not None:
            want, size = want + t.double(), size + t.double().abs()
    # fp32: the sum of whole numbers and two scales rounded once each, two additions; then the rounding of the result
    tol = 5 * 2.0 ** -24 * size + STEP[out_dtype] * want.abs()
    assert y.dtype == out_dtype and y.shape == want.shape and bool(((y.double() - want).abs() <= tol).all())


FORMS = [(1, 1, 1), (1, 16, 16), (2, 33, 100), (3, 17, 64), (7, 130, 513), (8, 256, 1000), (9, 300, 2048), (16, 64, 4096), (16, 5, 14336)]


@pytest.mark.parametrize("M,N,K", FORMS)
def test_product_of_few_rows(M, N, K):
    check_product(int8(M, K, 1), int8(N, K, 2), form=1)
    check_product(int8(M, K, 3), int8(N, K, 4), rand(N), rand(M, N), F32, form=1)


@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (5, 130, 100), (16, 128, 128), (17, 129, 1000), (33, 300, 640), (64, 257, 2048), (100, 128, 4096), (129, 384, 1111),
                                   (256, 200, 768), (300, 130, 513), (513, 64, 256)])
@pytest.mark.parametrize("splits", [1, 2, 3, 5, 8])
def test_product_of_some_rows(M, N, K, splits):
    check_product(int8(M, K, 1), int8(N, K, 2), form=2, splits=splits)
    check_product(int8(M, K, 3), int8(N, K, 4), rand(N, dtype=F32), rand(M, N, dtype=F32), F32, form=2, splits=splits, stages=2)


@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (5, 130, 100), (256, 256, 128), (257, 300, 1000), (300, 513, 640), (1000, 777, 1111), (2048, 4096, 512)])
def test_product_of_many_rows(M, N, K):
    check_product(int8(M, K, 1), int8(N, K, 2), form=3)
    check_product(int8(M, K, 3), int8(N, K, 4), rand(N, dtype=F32), rand(M, N), F32, form=3)
    check_product(int8(M, K, 5), int8(N, K, 6), rand(N), rand(M, N, dtype=F32), BF, form=3)


def test_product_of_the_largest_sums():
    """-128 times -128 over the longest rows: the sum is 2^31 - 16384."""
    K = I.MAX_COLS
    for form, M in ((1, 3), (2, 20), (3, 20)):
        v = torch.full((M, K), -128, dtype=torch.int8, device="cuda")
        w = torch.full((5, K), -128, dtype=torch.int8, device="cuda")
        y = I._product(I.Int8Rows(v, torch.ones(M, device="cuda")), I.Int8Rows(w, torch.ones(5, device="cuda")), out_dtype=F32, form=form)
        assert bool((y == float(2 ** 31 - 16384)).all())


@pytest.mark.parametrize("M,form", [(5, dict(form=1)), (13, dict(form=1)), (20, dict(form=2, splits=1)), (20, dict(form=2, splits=3)), (300, dict(form=2, splits=1)),
                                    (300, dict(form=3))])
@pytest.mark.parametrize("N", [64, 61])
def test_product_of_the_largest_numbers(M, form, N):
    """Scales as rows of up to 3e38 have them, beside ordinary ones whose results are the same bits without such neighbours."""
    a, b = int8(M, 512, 1), int8(N, 512, 2)
    a = I.Int8Rows(a.values.abs().clamp(min=0), a.scale.clone())
    b = I.Int8Rows(b.values.abs().clamp(min=0), (0.5 + b.scale) * torch.logspace(-20, 12, N, base=10.0, device="cuda"))  # sums of some 2^21
    ordinary = {dtype: I._product(a, b, rand(N), rand(M, N), dtype, **form) for dtype in (BF, F32)}
    a.scale[::2] = (0.5 + a.scale[::2]) * torch.logspace(15, 35, len(a.scale[::2]), base=10.0, device="cuda")
    a.scale[0], b.scale[5] = I.MOST_SCALE, 0.0
    want = (a.values.double() @ b.values.double().t()) * a.scale.double()[:, None] * b.scale.double()
    for dtype in (BF, F32):
        got = I._product(a, b, rand(N), rand(M, N), dtype, **form)
        assert torch.equal(torch.cat([got[1::2, :5], got[1::2, 6:]], 1), torch.cat([ordinary[dtype][1::2, :5], ordinary[dtype][1::2, 6:]], 1))
        w = want + rand(N).double() + rand(M, N).double()
        size = want.abs() + rand(N).double().abs() + rand(M, N).double().abs()
        fits = w.abs() < 0.99 * torch.finfo(dtype).max
        # two scales, two additions and the result rounded once each
        assert not got[w.abs() > 1.01 * torch.finfo(dtype).max].isfinite().any()
        assert bool(((got.double() - w).abs() <= 5 * 2.0 ** -24 * size + STEP[dtype] * w.abs())[fits].all()) and int((~fits).sum()) > 0
        assert got[:, 5].isfinite().all()
    lib.check_status()


def test_product_of_views():
    """Rows with strides, rows that start anywhere, more dimensions, transposed biases and residuals."""
    a, b = int8(40, 1000, 1), int8(70, 1000, 2)
    check_product(I.Int8Rows(a.values[::2, 16:400], a.scale[::2]), I.Int8Rows(b.values[:, 16:400], b.scale))
    check_product(I.Int8Rows(a.values[:, 3:502], a.scale), I.Int8Rows(b.values[:, 3:502], b.scale))
    check_product(I.Int8Rows(a.values.view(4, 10, 1000), a.scale.view(4, 10)), b, residual=rand(10, 4, 70).transpose(0, 1))
    check_product(I.Int8Rows(a.values.t().contiguous().t(), a.scale), b, bias=rand(70, 2)[:, 0], residual=rand(40, 100)[:, 7:77])
    one = I.Int8Rows(a.values[0], a.scale[0])
    assert torch.equal(I.int8_product(one, b), I.int8_product(I.Int8Rows(a.values[:1], a.scale[:1]), b)[0])
    assert I.int8_product(I.Int8Rows(a.values[:0], a.scale[:0]), b).shape == (0, 70)
    assert I.int8_product(a, I.Int8Rows(b.values[:0], b.scale[:0])).shape == (40, 0)


def test_bytes_behind_a_row_do_not_count():
    """A view's rows end inside 16 bytes whose rest belongs to others."""
    for M, form in ((4, 1), (20, 2), (20, 3)):
        a, b = int8(M, 512, 1), int8(33, 512, 2)
        for cols in (1, 63, 65, 129, 500):
            check_product(I.Int8Rows(a.values[:, :cols], a.scale), I.Int8Rows(b.values[:, :cols], b.scale), form=form)


def test_nan_rows_stay_where_they_are():
    x = rand(20, 256)
    x[3, 4] = float("nan")
    w = I.quantize_rows(rand(40, 256, seed=2))
    y = I.int8_product(I.quantize_rows(x), w)
    assert y[3].isnan().all() and int(y.isnan().sum()) == 40


# ------------------------------------------------------------------------------------------------ layers in training
def held(x):
    q, s = whole(x)
    return q * s[..., None]


@pytest.mark.parametrize("shape,outs,bias", [((1, 64), [8], False), ((5, 7, 768), [256, 1000, 8], False), ((3, 200), [16, 24], True), ((2100, 1024), [512, 528], False), ((4100, 64), [256, 72], False),
                                             ((999, 768), [2304], True), ((2, 3, 1040), [64, 8, 16, 24], False), ((130, 544), [16, 8, 8, 8, 8, 16], False)])
def test_linear_many_and_its_gradients(shape, outs, bias):
    x = rand(*shape, seed=1).requires_grad_()
    ws = [rand(n, shape[-1], seed=2 + n, std=0.05).requires_grad_() for n in outs]
    bs = [rand(n, seed=3 + n).requires_grad_() for n in outs] if bias else None
    ys = I.int8_linear_many(x, ws, bs)
    dys = [rand(*y.shape, seed=7 + i) for i, y in enumerate(ys)]
    grads = torch.autograd.grad(ys, [x, *ws, *(bs or [])], dys)
    lib.check_status()
    xd, wd, gd = held(x.detach()), [held(w.detach()) for w in ws], [g.double() for g in dys]
    dx = torch.zeros_like(xd)
    size = torch.zeros_like(xd)
    for i, (y, w, g) in enumerate(zip(ys, wd, gd)):
        want = xd @ w.t() + (bs[i].double() if bias else 0.0)
        assert y.shape == want.shape and bool(((y.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -21 * (xd.abs() @ w.abs().t() + 1)).all())
        dx += g @ w
        size += g.abs() @ w.abs()
        dw, mag = g.flatten(0, -2).t() @ xd.flatten(0, -2), g.flatten(0, -2).abs().t() @ xd.flatten(0, -2).abs()
        # operands rounded to bf16 (2^-8 of every product at most), sums in fp32, one rounding of the result
        assert bool(((grads[1 + i].double() - dw).abs() <= 2.0 ** -8 * dw.abs() + 1.01 * 2.0 ** -8 * mag).all())
        if bias:
            db = g.flatten(0, -2).sum(0)
            assert bool(((grads[1 + len(outs) + i].double() - db).abs() <= 2.0 ** -8 * db.abs() + 2.0 ** -18 * g.flatten(0, -2).abs().sum(0)).all())
    assert bool(((grads[0].double() - dx).abs() <= 2.0 ** -8 * dx.abs() + 1.01 * 2.0 ** -8 * size).all())
    # and not only at worst: roundings of either sign average out
    assert (grads[0].double() - dx).norm() <= 2.0 ** -8 * dx.norm()


def test_gradient_against_differences():
    """The loss is linear in what the rows stand for, so the difference between two inputs whose rows are exact is the gradient times their difference."""
    g = torch.Generator(device="cuda").manual_seed(3)
    q = torch.randint(-63, 64, (6, 64), generator=g, device="cuda").float()
    q[:, 0] = 127  # the scale of every row is 2^-6, before and after
    x = (q * 2.0 ** -6).to(BF)
    w = (torch.randint(-63, 64, (32, 64), generator=g, device="cuda").float() * 2.0 ** -6).to(BF)
    w[:, 0] = 127 * 2.0 ** -6
    c = torch.randint(-4, 5, (6, 32), generator=g, device="cuda").to(BF)
    xr, wr = x.clone().requires_grad_(), w.clone().requires_grad_()
    gx, gw = torch.autograd.grad((I.int8_linear(xr, wr).float() * c.float()).sum(), [xr, wr])
    with torch.no_grad():
        rows, wrows = I.quantize_rows(x), I.quantize_rows(w)
        f = lambda a, b: (I.int8_product(I.quantize_rows(a), I.quantize_rows(b), out_dtype=F32).double() * c.double()).sum()  # noqa: E731
        assert torch.equal(rows.dequantize(), x) and torch.equal(wrows.dequantize(), w)
        for i, j in ((0, 5), (3, 63), (5, 17)):
            step = torch.zeros_like(x)
            step[i, j] = 2.0 ** -6
            assert abs((f(x + step, w) - f(x, w)).item() - gx[i, j].double().item() * 2.0 ** -6) <= 2.0 ** -8 * abs(gx[i, j].item()) * 2.0 ** -6
        for i, j in ((0, 5), (31, 63), (7, 17)):
            step = torch.zeros_like(w)
            step[i, j] = 2.0 ** -6
            assert abs((f(x, w + step) - f(x, w)).item() - gw[i, j].double().item() * 2.0 ** -6) <= 2.0 ** -8 * abs(gw[i, j].item()) * 2.0 ** -6


def test_what_is_kept_is_in_8_bits():
    x, w = rand(4000, 4096).requires_grad_(), rand(1024, 4096, seed=2).requires_grad_()
    I.int8_linear(x, w)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    y = I.int8_linear(x, w)
    kept = torch.cuda.memory_allocated() - before - y.numel() * 2
    assert kept <= 1.05 * (x.numel() + w.numel())
    del y


def test_gradients_of_some():
    x, ws = rand(64, 1024).requires_grad_(), [rand(32, 1024, seed=2 + i).requires_grad_() for i in range(3)]
    y0, y1, y2 = I.int8_linear_many(x, ws)
    gx, g1 = torch.autograd.grad(y1.sum(), [x, ws[1]], retain_graph=True)
    want = torch.autograd.grad(I.int8_linear(x, ws[1]).sum(), [x, ws[1]])
    assert torch.equal(gx, want[0]) and torch.equal(g1, want[1])
    assert torch.autograd.grad(y0.sum(), [ws[1]], retain_graph=True, allow_unused=True)[0] is None
    frozen = [w.detach() for w in ws]
    (gx,) = torch.autograd.grad(sum(y.float().sum() for y in I.int8_linear_many(x, frozen)), [x])
    assert gx.shape == x.shape
    ys = I.int8_linear_many(x.detach(), ws)
    assert all(g.shape == w.shape for g, w in zip(torch.autograd.grad(sum(y.float().sum() for y in ys), ws), ws))


def test_main_grad_receives_the_weight_gradient():
    x, w = rand(64, 512).requires_grad_(), rand(32, 512, seed=2).requires_grad_()
    want = torch.autograd.grad(I.int8_linear(x, w).sum(), [w])[0]
    w.main_grad = torch.ones(32, 512, device="cuda")
    I.int8_linear(x, w).sum().backward()
    assert w.grad is None and bool(((w.main_grad - 1 - want.float()).abs() <= 2.0 ** -8 * want.float().abs() + 2.0 ** -22).all())


def test_one_weight_twice_and_results_written_in_place():
    x, w = rand(64, 512).requires_grad_(), rand(32, 512, seed=2).requires_grad_()
    a, b = I.int8_linear_many(x, [w, w])
    assert torch.equal(a, b)
    a.mul_(2.0)  # its neighbour stays as it is
    assert torch.equal(a, 2 * b)
    dy = rand(64, 32, seed=3)
    gx, gw = torch.autograd.grad([a, b], [x, w], [dy, dy])
    wx, ww = torch.autograd.grad(I.int8_linear(x, w), [x, w], dy)
    # three times the gradient, of which each part was rounded (2^-8), the larger one being twice as large, and their sum once
    assert bool(((gw.double() - 3 * ww.double()).abs() <= 3 * 2.0 ** -8 * 3 * ww.double().abs()).all())
    size = dy.double().abs() @ held(w.detach()).abs() * 3
    assert bool(((gx.double() - 3 * wx.double()).abs() <= 2.0 ** -8 * (gx.double().abs() + 3 * wx.double().abs()) + 2.02 * 2.0 ** -8 * size).all())


def test_gradients_that_are_broadcast_or_lie_anywhere():
    x, w = rand(4, 16, 512).requires_grad_(), rand(40, 512, seed=2).requires_grad_()
    wide = rand(4, 16, 83, seed=3)
    for dy in (torch.ones(1, 1, 1, dtype=BF, device="cuda").expand(4, 16, 40), rand(4, 1, 40, seed=4).expand(4, 16, 40), wide[:, :, 3:43], wide[:, :, 1:81:2],
               rand(16, 4, 40, seed=5).transpose(0, 1)):
        for got, want in zip(torch.autograd.grad(I.int8_linear(x, w), [x, w], dy), torch.autograd.grad(I.int8_linear(x, w), [x, w], dy.contiguous())):
            assert torch.equal(got, want)


def training_pass(x, ws, dys):
    return torch.autograd.grad(I.int8_linear_many(x, ws), [x, *ws], dys)


def test_training_is_captured_and_replayed():
    """Two graphs over the same weights, replayed in turn on new inputs."""
    ws = [rand(n, 1024, seed=n, std=0.05).requires_grad_() for n in (512, 64)]
    sets = [(rand(n, 1024, seed=n).requires_grad_(), [rand(n, w.shape[0], seed=n + w.shape[0]) for w in ws]) for n in (70, 2100)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for x, dys in sets:
            training_pass(x, ws, dys)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for x, dys in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(training_pass(x, ws, dys))
        graphs.append(g)
    for turn in range(2):
        for x, _ in sets:
            with torch.no_grad():
                x.copy_(rand(*x.shape, seed=50 + turn))
        with torch.no_grad():
            ws[0].copy_(rand(512, 1024, seed=60 + turn, std=0.05))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for out, (x, dys) in zip(outs, sets):
            assert all(torch.equal(a, b) for a, b in zip(out, training_pass(x, ws, dys)))
    lib.check_status()


def test_training_from_two_threads():
    import threading

    sets = [(rand(n, 1024, seed=n).requires_grad_(), [rand(m, 1024, seed=m, std=0.05).requires_grad_() for m in (512, 64)]) for n in (70, 2100)]
    dys = [[rand(x.shape[0], w.shape[0], seed=4) for w in ws] for x, ws in sets]
    want = [training_pass(*s, d) for s, d in zip(sets, dys)]
    torch.cuda.synchronize()
    got = [None, None]

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(10):
                got[i] = training_pass(*sets[i], dys[i])
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w))


def test_sizes_without_a_kernel_take_the_library():
    x, w = rand(6, 100).requires_grad_(), rand(13, 100, seed=2).requires_grad_()
    y = I.int8_linear(x, w)
    want = held(x.detach()) @ held(w.detach()).t()
    assert bool(((y.double() - want).abs() <= 2.0 ** -6 * (held(x.detach()).abs() @ held(w.detach()).abs().t())).all())
    y.sum().backward()
    assert x.grad.shape == x.shape and w.grad.shape == w.shape


# ------------------------------------------------------------------------------------------------ together
def half_layer(x, r, w, gu, down, act=Act.silu):
    rows, h = I.rms_norm_int8(x, w, 1e-5, residual=r)
    y = I.int8_product(rows, gu)
    ff = y.shape[-1] // 2
    return I.int8_product(I.gated_activation_int8(y[..., :ff], y[..., ff:], act), down, residual=h)


def half_layer_operands(rows, cols, ff, seed=0):
    return (rand(rows, cols, seed=seed), rand(rows, cols, seed=seed + 1, std=0.5), (1 + rand(cols, seed=seed + 2, std=0.1)).to(BF),
            I.quantize_rows(rand(2 * ff, cols, seed=seed + 3, std=0.05)), I.quantize_rows(rand(cols, ff, seed=seed + 4, std=0.05)))


@pytest.mark.parametrize("rows,cols,ff", [(1, 256, 512), (7, 1024, 768), (64, 520, 1000), (300, 1024, 2048)])
def test_feed_forward_half(rows, cols, ff):
    x, r, w, gu, down = half_layer_operands(rows, cols, ff)
    got = half_layer(x, r, w, gu, down)
    h = (x.float() + r.float()).to(BF).double()
    q, s = whole(h * w.double(), (h.square().mean(-1, keepdim=True) + 1e-5).rsqrt())
    y = ((q * s[:, None]) @ (gu.values.double() * gu.scale.double()[:, None]).t()).to(BF).double()
    g, u = y.chunk(2, -1)
    mid = torch.nn.functional.silu(g) * u
    want = held(mid) @ (down.values.double() * down.scale.double()[:, None]).t() + h
    # One bf16 rounding of y may fall the other way and move a row's scale by 2^-8, and with it every rounding of that row to 8 bits: then two
    # quantisations of the same row differ, each by up to half a step of max |mid| / 127 per element, of random signs.
    step = mid.abs().amax(-1, keepdim=True) / 127
    noise = step.squeeze(-1) / 6 ** 0.5 * (down.dequantize(F32).double().square().sum(-1).max() ** 0.5)
    assert bool(((got.double() - want).abs() <= 2.0 ** -8 * want.abs() + 6 * noise[:, None] + 2.0 ** -8 * mid.abs().amax(-1, keepdim=True)).all())
    # and in the mean such rows are few
    assert (got.double() - want).norm() <= 2.0 ** -7 * want.norm()


def test_captured_and_replayed():
    """Two graphs of the same sizes, replayed in turn on new inputs: no workspace is shared between them."""
    sets = [half_layer_operands(33, 1024, 768, seed=10 * i) for i in range(2)]
    graphs, outs = [], []
    for ops in sets:
        half_layer(*ops)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(half_layer(*ops))
        graphs.append(g)
    for turn in range(3):
        for i, ops in enumerate(sets):
            ops[0].copy_(rand(33, 1024, seed=100 * turn + i))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for out, ops in zip(outs, sets):
            assert torch.equal(out, half_layer(*ops))


def test_on_other_streams_and_from_two_threads():
    import threading

    sets = [half_layer_operands(n, 1024, 768, seed=n) for n in (5, 200)]
    want = [half_layer(*ops) for ops in sets]
    torch.cuda.synchronize()
    got = [None, None]

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got[i] = half_layer(*sets[i])
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    lib.check_status()


def test_calls_through_ctypes_give_the_same(monkeypatch):
    """Where Python's headers are missing the library is called without the module that launches faster."""
    ops = half_layer_operands(9, 1024, 768)
    want, rows = half_layer(*ops), I.quantize_rows(ops[0])
    monkeypatch.setattr(lib, "_launcher", lambda: None)
    monkeypatch.setattr(lib, "_quick", {})
    monkeypatch.setattr(I, "_f", {})
    assert torch.equal(half_layer(*ops), want) and torch.equal(I.quantize_rows(ops[0]).values, rows.values) and torch.equal(rows.dequantize(F32), rows.values * rows.scale[:, None])


def test_a_single_row_without_a_leading_dimension():
    x, w, bias = rand(333), I.quantize_rows(rand(7, 333, seed=2)), rand(7, seed=3)
    for row in (I.quantize_rows(x), I.Int8Rows(I.quantize_rows(rand(2, 700, seed=4)).values[1, 9:342], torch.tensor(0.5, device="cuda"))):
        want = (row.values.double() @ w.values.double().t()) * row.scale.double() * w.scale.double() + bias.double()
        got = I.int8_product(row, w, bias, out_dtype=F32)
        # a product of three numbers and a sum: one rounding each
        assert got.shape == (7,) and bool(((got.double() - want).abs() <= 2.0 ** -22 * (want.abs() + 2 * bias.double().abs())).all())
        assert torch.equal(row.dequantize(F32), row.values * row.scale)


def test_inputs_are_left_as_they_are_and_results_are_new():
    x, r, w, gu, down = half_layer_operands(9, 512, 256)
    before = [t.clone() for t in (x, r, w, gu.values, gu.scale, down.values, down.scale)]
    a = half_layer(x, r, w, gu, down)
    b = half_layer(x, r, w, gu, down)
    assert torch.equal(a, b) and a.data_ptr() != b.data_ptr()
    assert all(torch.equal(t, u) for t, u in zip((x, r, w, gu.values, gu.scale, down.values, down.scale), before))
    assert torch.equal(half_layer(x, x, w, gu, down), half_layer(x, x.clone(), w, gu, down))  # the same rows twice


def test_offsets_beyond_32_bits():
    """More than 2^32 bytes of rows: the last ones are as right as the first."""
    rows, cols = 1100000, 4096
    x = torch.zeros(rows, cols, dtype=BF, device="cuda")
    tail = rand(3, cols)
    x[-3:] = tail
    got = I.quantize_rows(x)
    assert torch.equal(got.values[-3:], I.quantize_rows(tail).values) and not got.values[:1000].any() and not got.scale[:-3].any()
    back = got.dequantize()
    assert torch.equal(back[-3:], I.quantize_rows(tail).dequantize()) and not back[-5].any()
    del x, back
    y = I.int8_product(got, I.quantize_rows(rand(8, cols, seed=5)), out_dtype=F32)
    assert torch.equal(y[-3:], I.int8_product(I.quantize_rows(tail), I.quantize_rows(rand(8, cols, seed=5)), out_dtype=F32)) and not y[:-3].any()


# ------------------------------------------------------------------------------------------------ models
def serving_llama(**kw):
    from levanter_b200.models.llama import LlamaConfig
    from levanter_b200.quantization import QuantizationConfig, quantize_for_serving

    cfg = dict(seq_len=256, hidden_dim=256, intermediate_dim=512, num_layers=2, num_heads=4, num_kv_heads=2, gradient_checkpointing=False)
    model = LlamaConfig(**{**cfg, **kw}).build(512, seed=0, device="cuda", dtype=BF).eval()
    return quantize_for_serving(model, QuantizationConfig(int8=True))


def engine_of(model, graph=False):
    from levanter_b200.data.passthrough_tokenizer import PassthroughTokenizer
    from levanter_b200.inference.engine import InferenceEngine, InferenceEngineConfig
    from levanter_b200.quantization import QuantizationConfig

    return InferenceEngine.from_model_with_config(model, PassthroughTokenizer(512), InferenceEngineConfig(
        max_pages=64, max_seqs=4, page_size=16, max_pages_per_seq=16, use_cuda_graph=graph, quantization=QuantizationConfig(int8=True)))


def requests():
    from levanter_b200.inference.engine import Request
    from levanter_b200.inference.jit_scheduler import SeqDecodingParams

    return [Request(prompt_tokens=list(range(5 + i, 40 + 3 * i)), request_id=i, decode_params=SeqDecodingParams(35 + 2 * i + 20, None, 0.0, i), n_generations=1)
            for i in range(3)]


@pytest.mark.parametrize("kw", [dict(), dict(use_bias=True), dict(hybrid_norm=True)])
def test_llama_serves_what_it_computes_without_a_cache(kw):
    from levanter_b200.layers.attention import AttentionMask

    model = serving_llama(**kw)
    with torch.no_grad():
        engine = engine_of(model)
        out = engine.generate(requests()).tokens
        for r, tokens in zip(requests(), out):
            seq = torch.tensor([list(r.prompt_tokens) + [int(t) for t in tokens]], dtype=torch.int32, device="cuda")
            logits = torch.nn.functional.linear(model.activations(seq, AttentionMask.causal()), model.get_lm_head())[0].float()
            n = len(r.prompt_tokens)
            for i, t in enumerate(tokens):
                row = logits[n - 1 + i]
                # the two ways differ by the attention kernels' roundings, which can move every rounding to 8 bits behind them: two layers of
                # four quantisers with steps of some 4 / 127 of a standard deviation, 0.9 % each, 5 % in all at most
                assert row[int(t)] >= row.max() - 2 * 0.05 * row.norm() / row.numel() ** 0.5 * 4


def test_engine_with_graphs_gives_the_same_tokens():
    with torch.no_grad():
        plain = engine_of(serving_llama()).generate(requests()).tokens
        graph = engine_of(serving_llama(), graph=True).generate(requests()).tokens
    assert [list(map(int, t)) for t in plain] == [list(map(int, t)) for t in graph]


def test_joint_projections_give_what_each_gives():
    model = serving_llama()
    layer = model.transformer.layers[0]
    x = rand(5, 256)
    with torch.no_grad():
        apart = [m(x) for m in (layer.self_attn.q_proj, layer.self_attn.k_proj, layer.self_attn.v_proj)]
        h = layer.mlp(x, residual=x)
        model.initial_cache(8, 16)
        joint = layer.self_attn._fused_int8()
        assert joint is not None
        y = I.int8_product(I.quantize_rows(x), *joint)
        assert torch.equal(y[:, :512], torch.cat(apart, 1)) and torch.equal(layer.mlp(x, residual=x), h)
        assert layer.mlp._rows.get([layer.mlp.gate_proj.weight, layer.mlp.up_proj.weight], build=False) is not None


def test_training_step_of_a_model_in_int8():
    from levanter_b200.models.llama import LlamaConfig
    from levanter_b200.models.lm_model import LmExample, compute_next_token_loss
    from levanter_b200.quantization import QuantizationConfig, quantize_linear_layers

    cfg = LlamaConfig(seq_len=128, hidden_dim=256, intermediate_dim=512, num_layers=2, num_heads=4, num_kv_heads=2, gradient_checkpointing=False)
    plain, model = (cfg.build(512, seed=0, device="cuda", dtype=BF) for _ in range(2))
    quantize_linear_layers(model, QuantizationConfig(int8=True))
    ex = LmExample.causal(torch.randint(0, 512, (2, 128), device="cuda", dtype=torch.int32))
    for m in (plain, model):
        compute_next_token_loss(m, ex).backward()
    for (n, p), q in zip(model.named_parameters(), plain.named_parameters()):
        q = q[1]
        # eight quantisers of 0.9 % on the way through two layers and back, and as much again from the weights
        assert (p.grad.float() - q.grad.float()).norm() <= 0.15 * q.grad.float().norm() + 1e-6, n
    lib.check_status()


@pytest.mark.parametrize("cols", [40, 1000, 4096])
def test_norms_of_zeros_without_an_eps(cols):
    for x, w in ((torch.zeros(3, cols, dtype=BF, device="cuda"), None), (rand(3, cols), torch.zeros(cols, device="cuda"))):
        for rows in (I.rms_norm_int8(x, w, 0.0)[0], I.rms_norm_int8(x.cpu(), None if w is None else w.cpu(), 0.0)[0]):
            assert not rows.values.any() and not rows.scale.any()


@pytest.mark.parametrize("shape,outs,bias", [((6, 100), [13], True), ((64, 1000), [301], False), ((3, 7, 77), [5, 1, 130], False), ((1, 1), [1], False), ((2500, 331), [129, 7], True),
                                             ((301, 515), [260, 300], False), ((5000, 40), [203, 51], False), ((129, 1111), [641], False), ((33, 17), [9, 8, 7, 6, 5, 4], True)])
def test_sizes_that_are_no_multiples_of_8(shape, outs, bias):
    """The products round once, as int8_product does; the gradients' operands are rounded to bf16, as at any other size."""
    x, ws = rand(*shape).requires_grad_(), [rand(n, shape[-1], seed=2 + n).requires_grad_() for n in outs]
    bs = [rand(n, seed=3).requires_grad_() for n in outs] if bias else None
    ys = I.int8_linear_many(x, ws, bs)
    dys = [rand(*y.shape, seed=4 + i) for i, y in enumerate(ys)]
    grads = torch.autograd.grad(ys, [x, *ws, *(bs or [])], dys)
    lib.check_status()
    rows = I.quantize_rows(x.detach())
    dx = size = 0
    for i, (y, w, d) in enumerate(zip(ys, ws, dys)):
        assert torch.equal(y, I.int8_product(rows, I.quantize_rows(w.detach()), bs[i].detach() if bias else None))
        xh, wh, d = held(x.detach()).flatten(0, -2), held(w.detach()), d.double().flatten(0, -2)
        dx, size = dx + d @ wh, size + d.abs() @ wh.abs()
        want, mag = d.t() @ xh, d.abs().t() @ xh.abs()
        assert grads[1 + i].dtype == BF and bool(((grads[1 + i].double() - want).abs() <= 2.0 ** -8 * want.abs() + 1.01 * 2.0 ** -8 * mag).all())
        if bias:
            assert bool(((grads[1 + len(outs) + i].double() - d.sum(0)).abs() <= 2.0 ** -8 * d.sum(0).abs() + 2.0 ** -18 * d.abs().sum(0)).all())
    got = grads[0].double().flatten(0, -2)
    assert grads[0].dtype == BF and bool(((got - dx).abs() <= 2.0 ** -8 * dx.abs() + 1.01 * 2.0 ** -8 * size).all())
    some = torch.autograd.grad(I.int8_linear_many(x, ws, bs)[-1], [x, ws[-1]], dys[-1])
    alone = torch.autograd.grad(I.int8_linear(x, ws[-1], bs[-1] if bias else None), [x, ws[-1]], dys[-1])
    assert torch.equal(some[0], alone[0]) and torch.equal(some[1], alone[1])


def test_gradients_of_sums_over_rows():
    """Such output gradients are one row, read again and again."""
    x, w = rand(70, 512).requires_grad_(), rand(40, 512, seed=2).requires_grad_()
    v = rand(40, seed=3)
    got = torch.autograd.grad(I.int8_linear(x, w).sum(0), [x, w], v)
    want = torch.autograd.grad(I.int8_linear(x, w), [x, w], v.expand(70, 40).contiguous())
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_fp32_streams_get_results_that_were_not_rounded_to_bf16():
    from levanter_b200.models.llama import LlamaMlp
    from levanter_b200.quantization import QuantizationConfig, quantize_for_serving

    x, stream = rand(37, 256), rand(37, 256, seed=1, dtype=F32)
    mlp = quantize_for_serving(LlamaMlp(256, 512, Act.silu, init_std=0.2).to("cuda", BF).eval(), QuantizationConfig(int8=True, targets=["down_proj"]))
    with torch.no_grad():
        rows = I.quantize_rows(mlp._inner(x))
        want = (rows.values.double() @ mlp.down_proj.weight.double().t()) * rows.scale.double()[:, None] * mlp.down_proj.weight_scale.double()
        # a sum, two scales and an addition, rounded once each
        assert bool(((mlp.forward_fp32(x).double() - want).abs() <= 3 * 2.0 ** -24 * want.abs()).all())
        got = mlp.add_to_stream(stream.clone(), x).double()
        assert bool(((got - want - stream.double()).abs() <= 4 * 2.0 ** -24 * (want.abs() + stream.double().abs())).all())


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("hidden,ff,shared,experts", [(64, 32, 96, 8), (72, 24, 40, 10), (128, 16, 22, 9)])
def test_a_shared_expert_in_8_bits_leaves_the_others_on_their_kernels(gated, hidden, ff, shared, experts, monkeypatch):
    from levanter_b200.layers.experts import GroupedSoftmaxMoe
    from levanter_b200.ops import moe
    from levanter_b200.quantization import QuantizationConfig, quantize_for_serving

    torch.manual_seed(3)
    block = GroupedSoftmaxMoe(hidden, ff, experts, 2, shared_intermediate=shared, shared_gated=gated, init_std=0.2).to("cuda", BF).eval()
    alone = GroupedSoftmaxMoe(hidden, ff, experts, 2).to("cuda", BF).eval()
    alone.load_state_dict({k: v for k, v in block.state_dict().items() if not k.startswith("shared")})
    quantize_for_serving(block, QuantizationConfig(int8=True))
    x, h = rand(21, hidden, seed=1, dtype=F32), rand(21, hidden, seed=2)
    monkeypatch.setattr(moe, "expert_outputs", None)  # what runs where the kernels do not
    with torch.no_grad():
        part = block.shared.forward_fp32(h)
        if gated:
            part = part * torch.sigmoid(h.float() @ block.shared_gate.weight.float().t())
        base = alone.add_to_stream(x.clone(), h)
        want = base.double() + part.double()
        got = block.add_to_stream(x.clone(), h)
        # the routing weights and the gate from sums of some hundred products in fp32, in another order
        tol = 200 * 2.0 ** -24 * (x.abs() + (base - x).abs() + part.abs() + 1)
        assert bool(((got.double() - want).abs() <= tol).all())
        replayed, g = x.clone(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            block.add_to_stream(replayed, h)
        g.replay()
        assert torch.equal(replayed, got)


def test_tangents_are_refused():
    import torch.autograd.forward_ad as ad

    x, w = rand(4, 64), I.quantize_rows(rand(64, 64, seed=2))
    rows = I.quantize_rows(x)
    with torch.no_grad(), ad.dual_level():
        d = ad.make_dual(x, rand(4, 64, seed=3))
        for call in (lambda: I.quantize_rows(d), lambda: I.rms_norm_int8(x, None, residual=d), lambda: I.gated_activation_int8(x, d, Act.silu),
                     lambda: I.int8_product(rows, w, residual=d), lambda: I.int8_linear(d, rand(8, 64))):
            with pytest.raises((RuntimeError, NotImplementedError)):
                call()


def test_weights_that_moved_are_read_where_they_lie():
    m = I.Int8ServingLinear(torch.randn(40, 100), None).cuda()
    assert m.weight.stride() == (112, 1) and m.weight_scale.is_cuda
    x = rand(5, 100)
    with torch.no_grad():
        m(x)
        before = torch.cuda.memory_stats()["allocation.all.allocated"]
        m(x)
        assert torch.cuda.memory_stats()["allocation.all.allocated"] - before == 3  # values and scales of the rows, the result


def test_converted_weights_are_not_kept():
    """Of fp32 weights the forward pass makes bf16 copies, of which the backward pass needs nothing."""
    lin = I.Int8Linear(torch.nn.Parameter(rand(4096, 2048, dtype=F32, std=0.05)), None)
    x, dy = rand(64, 2048).requires_grad_(), rand(64, 4096, seed=3)
    lin(x)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    y = lin(x)
    assert torch.cuda.memory_allocated() - before <= y.nbytes + 1.05 * (x.numel() + lin.weight.numel())
    y.backward(dy)
    want = torch.autograd.grad(I.int8_linear(x, lin.weight.detach().to(BF).requires_grad_()), [x], dy)[0]
    assert lin.weight.grad.dtype == F32 and torch.equal(x.grad, want)
    grad, lin.weight.grad = lin.weight.grad, None
    y = lin(x)
    lin.weight.main_grad = torch.zeros(4096, 2048, device="cuda")  # named after the forward pass
    y.backward(dy)
    assert lin.weight.grad is None and bool(((lin.weight.main_grad - grad).abs() <= 2.0 ** -8 * grad.abs() + 2.0 ** -22).all())


# Blocks that go on to a second and a third row: the next row's reads under way, two sets of partial results.  Aligned rows of 8208 to 12288 columns run on two blocks per SM;
# rows that start anywhere have forms for 512, 768 and 1024 threads and one that reads twice; up to 512 columns a warp has a row.
MANY = [(1500, 8208), (1500, 11008), (1500, 12288), (3000, 4096), (1000, 14336), (3000, 528), (3000, 4095), (1500, 8191), (1500, 11007), (1000, 14335), (12000, 256), (9000, 511)]


@pytest.mark.parametrize("rows,cols", MANY)
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("dtype,wtype", [(BF, BF), (BF, F32), (F32, F32)])
def test_norms_of_many_rows(rows, cols, residual, dtype, wtype):
    x, w = rand(rows, cols, seed=cols, dtype=dtype) * torch.logspace(-2, 2, rows, device="cuda")[:, None].to(dtype), (1 + rand(cols, seed=1, std=0.1, dtype=F32)).to(wtype)
    r = rand(rows, cols, seed=2, dtype=dtype) if residual else None
    got, h = I.rms_norm_int8(x, w, 1e-5, residual=r)
    want = x if r is None else (x.float() + r.float()).to(dtype)
    assert h is None or torch.equal(h, want)
    d = want.double()
    check_rows(got, d * w.double(), (d.square().mean(-1, keepdim=True) + 1e-5).rsqrt(), slack=0.0 if dtype == wtype == BF else 2.0 ** -22)


@pytest.mark.parametrize("rows,cols", MANY)
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("joint", [False, True])
def test_gated_activations_of_many_rows(rows, cols, dtype, joint):
    y = rand(rows, 2 * cols, seed=cols, std=3.0, dtype=dtype)
    g, u = (y[:, :cols], y[:, cols:]) if joint else (y[:, :cols].contiguous(), y[:, cols:].contiguous())
    u.mul_(torch.logspace(-2, 2, rows, device="cuda")[:, None])
    check_rows(I.gated_activation_int8(g, u, Act.silu), torch.nn.functional.silu(g.double()) * u.double(), slack=2.0 ** -18)


@pytest.mark.parametrize("rows,cols", MANY)
@pytest.mark.parametrize("dtype", [BF, F32])
def test_quantize_many_rows_and_back(rows, cols, dtype):
    x = rand(rows, cols, seed=cols, dtype=dtype) * torch.logspace(-2, 2, rows, device="cuda")[:, None].to(dtype)
    held_rows = I.quantize_rows(x)
    check_rows(held_rows, x, slack=0.0 if dtype == BF else 2.0 ** -23)
    assert torch.equal(held_rows.dequantize(dtype), (held_rows.values.float() * held_rows.scale[:, None]).to(dtype))


@pytest.mark.parametrize("M", [1, 16, 33, 64, 65])
@pytest.mark.parametrize("N", [6144, 7168, 8699, 9216])
@pytest.mark.parametrize("K", [2048, 4096])
def test_products_on_both_sides_of_the_lines_of_the_rule(M, N, K):
    check_product(int8(M, K, 1), int8(N, K, 2), rand(N), rand(M, N))


@pytest.mark.parametrize("outs,cols", [(40, 100), (40, 96), (13, 77)])
def test_gradient_buffers_of_any_size_and_those_that_start_anywhere(outs, cols):
    """A buffer whose rows would be written 16 bytes at a time has to start on 16 bytes; others may start anywhere."""
    x, w, dy = rand(70, cols).requires_grad_(), rand(outs, cols, seed=2).requires_grad_(), rand(70, outs, seed=3)
    want = torch.autograd.grad(I.int8_linear(x, w), [w], dy)[0]
    flat = torch.zeros(outs * cols + 16, device="cuda")
    for first in (4, 1):
        flat.zero_()
        w.main_grad = flat[first:first + outs * cols].view(outs, cols)
        if first == 1 and cols % 4 == 0:
            with pytest.raises(ValueError, match="16 bytes"):
                I.int8_linear(x, w).backward(dy)
            continue
        I.int8_linear(x, w).backward(dy)
        lib.check_status()
        assert w.grad is None and bool(((w.main_grad - want.float()).abs() <= 2.0 ** -8 * want.float().abs() + 2.0 ** -22).all())
        assert not flat[:first].any() and not flat[first + outs * cols:].any()
