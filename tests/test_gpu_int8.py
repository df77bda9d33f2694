"""GPU tests of the products on 8-bit integers against their definitions in float64: codes and sums are exact, what
is left are a few fp32 roundings and the one to the output's type."""
import numpy as np
import pytest

from instantcua_amd import engine as eng
from instantcua_amd import int8

pytestmark = pytest.mark.gpu
NP = {int8.F32: np.float32, int8.F16: np.float16}
dev = eng.DeviceBuffer.from_array
EPS = 1e-6


def quantised(x, norm=None, eps=EPS):
    """(codes, scales) of the definition."""
    t = x.astype(np.float64)
    r = np.ones(len(t))
    if norm is not None:
        r = 1 / np.sqrt((t * t).mean(-1) + eps)
        t = t * norm.astype(np.float64)
    top = np.abs(t).max(-1)
    return np.rint(t * 127 / np.where(top > 0, top, 1)[:, None]).astype(np.int8), top * r / 127


def run_quantize(x, norm=None, type=int8.F32, gap=0, eps=EPS):
    """Rows with a gap of `gap` values behind them (NaN in x, 77 in the codes)."""
    rows, cols = x.shape
    wide = np.full((rows, cols + gap), np.nan, NP[type])
    wide[:, :cols] = x
    codes = dev(np.full((rows, cols + 2 * gap), 77, np.int8))
    scales = dev(np.full(rows + 3, 5, np.float32))
    int8.quantize(dev(wide), codes, scales, rows, cols, norm=None if norm is None else dev(norm), eps=eps, type=type,
                  x_stride=cols + gap, codes_stride=cols + 2 * gap)
    got = codes.to_array(np.int8, (rows, cols + 2 * gap))
    s = scales.to_array(np.float32, rows + 3)
    assert (got[:, cols:] == 77).all() and (s[rows:] == 5).all()
    return got[:, :cols], s[:rows]


@pytest.mark.parametrize("type", [int8.F32, int8.F16])
@pytest.mark.parametrize("with_norm", [False, True])
@pytest.mark.parametrize("rows,cols,gap", [(1, 16, 0), (1, 2048, 8), (3, 48, 16), (7, 1040, 0), (33, 6144, 8),
                                           (5, 8208, 24), (2, 1 << 17, 0), (700, 2048, 0)])
def test_quantize(type, with_norm, rows, cols, gap):
    rng = np.random.default_rng(rows * 7 + cols)
    x = rng.standard_normal((rows, cols)) * 10.0 ** rng.uniform(-2, 2, (rows, 1))
    x[:, 5::37] *= 4
    x = x.astype(NP[type])
    norm = (1 + 0.3 * rng.standard_normal(cols)).astype(np.float32) if with_norm else None
    codes, scales = run_quantize(x, norm, type, gap)
    want, s = quantised(x, norm)
    assert np.array_equal(codes, want)
    # Sums in another order (64 bits, 2^-53 a term), then one rounding to fp32.
    assert (np.abs(scales - s) <= s * 2.0 ** -23).all()


@pytest.mark.parametrize("type", [int8.F32, int8.F16])
def test_quantize_ties_and_sizes(type):
    """Values half way between two codes go to the even one; rows of any magnitude, of zeros and of one value."""
    k = np.arange(-126, 127)
    x = np.zeros((9, 512), NP[type])
    x[0, :253] = (k + 0.5) * 0.25  # the largest of the row is 127 * 0.25
    x[0, 253] = 127 * 0.25
    x[1, :253] = k + 0.5
    x[1, 300] = -127
    x[2] = 3
    x[4] = -np.finfo(NP[type]).tiny
    x[5, 17] = np.finfo(NP[type]).max
    x[6, :4] = np.finfo(NP[type]).smallest_subnormal * np.arange(4)
    x[7] = np.linspace(-1, 1, 512) * float(np.finfo(NP[type]).max)
    x[8, 0] = 1
    codes, scales = run_quantize(x, type=type)
    want, s = quantised(x)
    assert np.array_equal(codes, want)
    assert (codes[3] == 0).all() and scales[3] == 0
    tiny = 2.0 ** -150  # half of fp32's smallest step
    assert (np.abs(scales - s) <= s * 2.0 ** -24 + tiny).all()


@pytest.mark.parametrize("cols", [2048, 2064, 6160, 16384, 16400])
@pytest.mark.parametrize("with_norm", [False, True])
@pytest.mark.parametrize("size", [0, -61, 62, -100])
def test_quantize_next_to_ties(cols, with_norm, size):
    """Quotients some fp32 steps from half way between two codes, on both sides: closer than fp32 arithmetic tells."""
    rng = np.random.default_rng(cols)
    half = (np.arange(cols) % 127 - 63 + 0.5).astype(np.float32)
    x = half * (1 + rng.integers(-3, 4, (4, cols)) * 2.0 ** -23).astype(np.float32)
    norm = np.ones(cols, np.float32)
    if with_norm:
        norm = np.ldexp(np.float32(1), rng.integers(-3, 4, cols)).astype(np.float32)
        norm[::3] *= np.float32(1 + 2.0 ** -23)
    x = (x / norm * 2.0 ** size).astype(np.float32)
    x[:, 7] = 127 * 2.0 ** size / norm[7]
    codes, _ = run_quantize(x, norm if with_norm else None)
    assert np.array_equal(codes, quantised(x, norm if with_norm else None)[0])


def test_quantize_rows_that_are_no_numbers():
    rng = np.random.default_rng(3)
    x = rng.standard_normal((6, 256)).astype(np.float32)
    norm = np.ones(256, np.float32)
    x[1, 255], x[2, 0], x[4, 100] = np.nan, np.inf, -np.inf
    for w in (None, norm):
        codes, scales = run_quantize(x, w)
        fine = [0, 3, 5]
        want, s = quantised(x[fine], w)
        assert np.array_equal(codes[fine], want) and (np.abs(scales[fine] - s) <= s * 2.0 ** -23).all()
        assert (codes[[1, 2, 4]] == 0).all() and np.isnan(scales[[1, 2, 4]]).all()
    # Squares beyond fp32, a sum that eps alone keeps from zero, and a norm of zeros.
    x[0], x[1], x[2] = 1e30, 0, 1e-30
    codes, scales = run_quantize(x[:3], norm)
    assert (codes[0] == 127).all() and abs(scales[0] * 127 - 1) < 2.0 ** -22
    assert (codes[1] == 0).all() and scales[1] == 0
    assert (codes[2] == 127).all() and abs(scales[2] * 127 / 1e-27 - 1) < 2.0 ** -22
    codes, scales = run_quantize(x[:3], 0 * norm)
    assert (codes == 0).all() and (scales == 0).all()


def product(x, sx, w, sw, add=None, gated=False):
    """(y, how far fp32 may be from it) of exact sums: a product has the roundings of the sum, of two scales' products
    and of the addition, 2^-24 each.  Gate: an error of g (3 roundings) counts by at most 1 + |g|, the exponential is
    2^-22 (1 + |g|) off, three further operations; below fp32's normal range 2^-126 of up."""
    acc = x.astype(np.float64) @ w.astype(np.float64).T
    y = acc * sx.astype(np.float64)[:, None] * sw.astype(np.float64)
    if not gated:
        tol = 3 * 2.0 ** -24 * np.abs(y)
        if add is not None:
            y = y + add
            tol += 2.0 ** -24 * np.abs(y)
        return y, tol + 2.0 ** -149
    n = len(sw) // 2
    g, u = y[:, :n], y[:, n:]
    with np.errstate(over="ignore"):
        y = g / (1 + np.exp(-g)) * u
    return y, (3 * (2 + np.abs(g)) + 4 * (1 + np.abs(g)) + 4) * 2.0 ** -24 * np.abs(y) + 2.0 ** -126 * (1 + np.abs(u))


def check(got, want, tol, type):
    if type == int8.F16:
        with np.errstate(over="ignore"):
            far = np.abs(want) > 65519
        assert np.isinf(got[np.abs(want) > 65521]).all()
        got, want, tol = got[~far], want[~far], tol[~far]
        tol = tol + 2.0 ** -11 * np.abs(want) + 2.0 ** -25
    assert got.shape == want.shape and np.isfinite(got).all()
    over = np.abs(got.astype(np.float64) - want) - tol
    assert (over <= 0).all(), (np.unravel_index(over.argmax(), over.shape) if over.ndim > 1 else int(over.argmax()), float(over.max()))


def operands(rng, m, n, k, gated=False, low=-127):
    x = rng.integers(low, 128, (m, k)).astype(np.int8)
    w = rng.integers(low, 128, (n * (1 + gated), k)).astype(np.int8)
    sx = (rng.uniform(0.5, 2, m) * 1.5 * 3 / 127).astype(np.float32)
    sw = (rng.uniform(0.5, 2, n * (1 + gated)) * 0.02 / 74 * (2048 / k) ** 0.5).astype(np.float32)
    return x, sx, w, sw


def run_matmul(x, sx, w, sw, add=None, gated=False, type=int8.F32, gap=0, in_place=False):
    """Rows with gaps behind them; y's hold 7."""
    m, k = x.shape
    n = len(w) // (1 + gated)

    def wide(a, fill, more):
        y = np.full((a.shape[0], a.shape[1] + more), fill, a.dtype)
        y[:, :a.shape[1]] = a
        return dev(y)

    ys = n + gap
    y = wide(add.astype(np.float32), 7, gap) if in_place else dev(np.full((m, ys), 7, NP[type]))
    extra = {} if add is None else {"add": y if in_place else wide(add.astype(np.float32), np.nan, gap + 1),
                                    "add_stride": ys if in_place else n + gap + 1}
    need = int8.matmul_work(m, n, k, gated=gated)
    work = dev(np.full(need, 0xFF, np.uint8)) if need else None
    int8.matmul(wide(x, 99, 16 * gap), dev(sx), wide(w, -99, 32 * gap), dev(sw), y, m, n, k, gated=gated, type=type,
                x_stride=k + 16 * gap, w_stride=k + 32 * gap, y_stride=ys, work=work, **extra)
    got = y.to_array(NP[type], (m, ys))
    assert (got[:, n:] == 7).all()
    return got[:, :n]


SHAPES = [
    # rows, channels, depth, gap
    (1, 1, 16, 0), (1, 31, 48, 1), (1, 4096, 2048, 0), (2, 33, 128, 3), (3, 65, 144, 0), (8, 500, 2048, 0),
    (8, 96, 6144, 1), (15, 127, 1040, 0), (16, 64, 272, 5), (17, 129, 256, 0), (31, 260, 400, 0), (33, 1000, 2064, 1),
    (64, 128, 6144, 0), (65, 63, 4096, 0), (100, 257, 112, 0), (127, 255, 384, 2), (128, 256, 2048, 0),
    (129, 513, 528, 0), (200, 2048, 2048, 0), (257, 300, 1024, 1), (400, 777, 240, 0), (1000, 96, 512, 0),
    (1111, 1300, 640, 0), (2048, 2050, 256, 0), (4, 3, 1 << 17, 0), (130, 2, 20000, 0),
    # With those before, every tile of the products: whole ones, ragged ones, ends of 16 to 112 codes.
    (36, 1478, 400, 1), (24, 2050, 1040, 0), (150, 17, 688, 0), (2, 9193, 1040, 1), (200, 2050, 2064, 0), (33, 8284, 1040, 0),
    (250, 2050, 2064, 3), (3, 16659, 2480, 0), (66, 17549, 144, 1), (512, 4096, 272, 0), (1030, 6150, 400, 0), (131, 35815, 80, 0),
    (1024, 6144, 256, 0), (67, 839, 144, 0), (130, 17037, 112, 1), (300, 6100, 336, 0),
]


@pytest.mark.parametrize("type", [int8.F32, int8.F16])
@pytest.mark.parametrize("form", ["plain", "add", "gated"])
@pytest.mark.parametrize("m,n,k,gap", SHAPES)
def test_matmul(type, form, m, n, k, gap):
    rng = np.random.default_rng(m * 31 + n * 7 + k)
    gated = form == "gated"
    x, sx, w, sw = operands(rng, m, n, k, gated)
    add = rng.standard_normal((m, n)).astype(np.float32) if form == "add" else None
    got = run_matmul(x, sx, w, sw, add, gated, type, gap)
    want, tol = product(x, sx, w, sw, add, gated)
    check(got, want, tol, type)


@pytest.mark.parametrize("form,m,n,k,gap", [("add", 4090, 2040, 6160, 1), ("gated", 2040, 2040, 6160, 0), ("plain", 3970, 1800, 8192, 0)])
def test_deep_products_that_fill_the_gpu(form, m, n, k, gap):
    test_matmul(int8.F32, form, m, n, k, gap)


@pytest.mark.parametrize("m,n,k,gap", [(1, 100, 256, 0), (40, 130, 512, 3), (300, 520, 1024, 0)])
def test_matmul_adds_in_place(m, n, k, gap):
    rng = np.random.default_rng(m)
    x, sx, w, sw = operands(rng, m, n, k)
    add = rng.standard_normal((m, n)).astype(np.float32)
    got = run_matmul(x, sx, w, sw, add, gap=gap, in_place=True)
    want, tol = product(x, sx, w, sw, add)
    check(got, want, tol, int8.F32)


@pytest.mark.parametrize("m", [1, 20, 150])
@pytest.mark.parametrize("gated", [False, True])
def test_sums_are_exact_at_their_largest(m, gated):
    """2^17 products of 127 and 127 of one sign, and one less: sums next to 2^31 that fp32 does not hold apart, so the
    difference of two channels shows them.  Scales of 1 and 2^-31, gates of 31 or so pass the up through."""
    k, n = 1 << 17, 6
    x = np.full((m, k), 127, np.int8)
    w = np.full((n * (1 + gated), k), 127, np.int8)
    w[1], w[2, ::2], w[3, -1], w[4, 0], w[5, 5::2] = -127, -127, 126, 126, -127
    sx = np.full(m, 1, np.float32)
    sw = np.full(len(w), 2.0 ** -31, np.float32)
    got = run_matmul(x, sx, w, sw, gated=gated)
    want, tol = product(x, sx, w, sw, gated=gated)
    check(got, want, tol, int8.F32)
    if not gated:
        assert got[0, 2] == 0 and (got == got[:1]).all()


@pytest.mark.parametrize("m", [2, 140])
def test_scales_that_are_no_numbers_and_far_apart(m):
    rng = np.random.default_rng(m)
    for gated in (False, True):
        x, sx, w, sw = operands(rng, m, 40, 256, gated)
        sx[1] = np.nan
        got = run_matmul(x, sx, w, sw, gated=gated)
        assert np.isnan(got[1]).all()
        rest = np.arange(m) != 1
        want, tol = product(x[rest], sx[rest], w, sw, gated=gated)
        check(got[rest], want, tol, int8.F32)
    x, sx, w, sw = operands(rng, m, 40, 256)
    sx[0], sx[1] = 1e-30, 1e30
    sw[:5], sw[5:9] = 1e-12, 1e3  # products of the scales below fp32's normal range: the sum's comes first
    got = run_matmul(x, sx, w, sw)
    want, tol = product(x, sx, w, sw)
    check(got, want, tol + 2.0 ** -126 * 2.0 ** -23, int8.F32)


def test_fp16_outputs_beyond_its_range_are_infinite():
    rng = np.random.default_rng(9)
    x, sx, w, sw = operands(rng, 40, 70, 512)
    sw *= 1e6
    got = run_matmul(x, sx, w, sw, type=int8.F16)
    want, tol = product(x, sx, w, sw)
    check(got, want, tol, int8.F16)
    assert np.isinf(got).any() and not np.isnan(got).any()


def test_gates_far_from_zero():
    """Gates of -200 .. 200: exponentials beyond fp32 leave zeros, none that is no number."""
    x = np.full((3, 16), 1, np.int8)
    n = 101
    w = np.zeros((2 * n, 16), np.int8)
    w[:n, 0] = np.arange(n) - 50
    w[n:] = 1
    sx, sw = np.full(3, 1, np.float32), np.full(2 * n, 4, np.float32)
    got = run_matmul(x, sx, w, sw, gated=True)
    want, tol = product(x, sx, w, sw, gated=True)
    check(got, want, tol, int8.F32)


def test_matrices_are_quantised_by_their_channels():
    """A matrix and tokens through both calls: the product of what the codes stand for."""
    rng = np.random.default_rng(11)
    W, X = rng.standard_normal((300, 512)).astype(np.float32), rng.standard_normal((50, 512)).astype(np.float32)
    wc, ws = run_quantize(W)
    xc, xs = run_quantize(X)
    got = run_matmul(xc, xs, wc, ws)
    want, tol = product(xc, xs, wc, ws)
    check(got, want, tol, int8.F32)
    # Codes are off by half a step of about 3.3 / 127 at most, spread evenly: each of the two operands adds 0.0075 of
    # the products' rms; together 0.011.
    rms = np.sqrt(((got - X.astype(np.float64) @ W.astype(np.float64).T) ** 2).mean() / 512)
    assert rms < 0.02


def test_as_many_rows_as_a_call_takes():
    """2^24 rows of 16 values, and as many of a product with two channels, looked at in places."""
    rows = 1 << 24
    look = np.r_[0:70, (1 << 20) - 3:(1 << 20) + 3, (1 << 23) - 1:(1 << 23) + 1, rows - 70:rows]
    rng = np.random.default_rng(1)
    x = np.tile(rng.standard_normal((1 << 12, 16)).astype(np.float16), (1 << 12, 1))
    x[look] = rng.standard_normal((len(look), 16)).astype(np.float16)
    codes, scales = dev(np.full((rows, 16), 77, np.int8)), dev(np.full(rows, 5, np.float32))
    int8.quantize(dev(x), codes, scales, rows, 16, type=int8.F16)
    want, s = quantised(x[look])
    c, sx = codes.to_array(np.int8, (rows, 16)), scales.to_array(np.float32, rows)
    assert np.array_equal(c[look], want) and (np.abs(sx[look] - s) <= s * 2.0 ** -24).all()
    w, sw = rng.integers(-127, 128, (2, 16)).astype(np.int8), np.ones(2, np.float32)
    y = dev(np.full((rows, 2), 7, np.float32))
    int8.matmul(codes, scales, dev(w), dev(sw), y, rows, 2, 16)
    want, tol = product(c[look], sx[look], w, sw)
    check(y.to_array(np.float32, (rows, 2))[look], want, tol, int8.F32)
