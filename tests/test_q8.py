"""8-bit rows (th_q8): rows, weights, norms and activations in 8 bits, their
products, and what is refused.

A row's integers are decided in 64 bits, so here they are compared for
equality with the definition's (numpy, float64), and so are products, whose
sums are exact and whose two roundings numpy repeats. What is not exact: a
scale of the norm, whose sum of squares has another order in 64 bits
(n * 2^-53 of it), which can round to the next f32: one step, 2^-23; and
integers of silu(gate) * up and of the norm whose quotient lies within 1e-9 of
a border (the exponential, the sum and four operations are each off by a few
2^-53, times 127), of which the inputs here have none.
"""

from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from titania_amd import HipError, InvalidArgument, Tensor, _lib
from titania_amd.synth import bf16_to_f32, f32_to_bf16

EPS = 1e-6
gpu = pytest.mark.gpu


def rows64(v, scale64=None):
    """The integers and scales of rows v (float64); scale64: A / 127 where it is not the rows' own."""
    v = np.atleast_2d(np.asarray(v, np.float64))
    with np.errstate(all="ignore"):
        top = np.max(np.abs(v), axis=1)
        s = (top / 127 if scale64 is None else scale64).astype(np.float32)
        bad = ~np.isfinite(v).all(axis=1) | ~np.isfinite(s)
        q = np.rint(v * 127 / top[:, None])
    q[bad | (s == 0)] = 0
    s[bad] = np.nan
    return q.astype(np.int8), s


def far_from_borders(v):
    """Whether no quotient of rows v lies within 1e-9 of a border."""
    v = np.atleast_2d(v)
    with np.errstate(all="ignore"):
        t = np.abs(v * 127 / np.max(np.abs(v), axis=1)[:, None])
        return not np.any(np.abs(t - np.floor(t) - 0.5) < 1e-9)


def product32(wq, ws, xq, xs):
    """out[t][r] in the order of the definition: the exact sum to f32, times x's scale, times w's."""
    total = xq.astype(np.float64) @ wq.astype(np.float64).T  # exact: every partial sum is below 2^53
    with np.errstate(all="ignore"):
        return total.astype(np.float32) * xs[:, None] * ws[None, :]


def norm64(x, gain, eps=EPS):
    """v up to its positive factor (x g, exact), and A / 127."""
    x64 = x.astype(np.float64)
    with np.errstate(all="ignore"):
        p = x64 * bf16_to_f32(gain).astype(np.float64)
        return p, np.max(np.abs(p), axis=1) / np.sqrt(np.mean(x64 * x64, axis=1) + np.float64(np.float32(eps))) / 127


def silu64(g, u):
    g = g.astype(np.float64)
    with np.errstate(all="ignore"):
        return g / (1 + np.exp(-g)) * u.astype(np.float64)


def buf(hip, a):
    b = hip.alloc(np.asarray(a).size)
    hip.write(b, a)
    return b


def q8(hip, values, scales):
    q = hip.alloc_q8(*values.shape)
    hip.write_q8(q, values, scales)
    return q


def same(a, b):
    """Equal bits, any NaN as any other."""
    return np.array_equal(a, b, equal_nan=True) and np.array_equal(np.signbit(a[~np.isnan(a)]), np.signbit(b[~np.isnan(b)]))


def near(got, want):
    """Scales that are one f32 step apart at most."""
    both = np.isfinite(want)
    return np.array_equal(np.isnan(got), np.isnan(want)) and np.all(
        np.abs(got[both].astype(np.float64) - want[both]) <= 2.0**-23 * np.abs(want[both]) + 2.0**-149)


# Columns about the 16, 64, 128 and 256 that kernels step by, and more than any holds of a row at once.
COLS = [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 256, 260, 512, 520, 1024, 1101, 1500, 2000, 2050, 2560, 4096,
        4100, 5001, 6000, 6148, 8190, 9728, 10244, 12300, 16388, 20011, 20482, 24000, 28000, 28675, 33001, 40000, 41000, 131071]
SIZES = [(3 if c < 20000 else 2, c) for c in COLS] + [(1, 2560), (1, 9728), (16, 512), (17, 512), (33, 130), (300, 96), (520, 8200),
    (260, 13000), (260, 18000)]


@gpu
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 17), (16, 64), (17, 65), (50, 1101), (33, 128)])
def test_write_and_read(hip, rows, cols):
    r = np.random.default_rng(rows + cols)
    v, s = r.integers(-128, 128, (rows, cols), dtype=np.int8), r.standard_normal(rows).astype(np.float32)
    q = q8(hip, v, s)
    assert q.shape == (rows, cols)
    got, scales = hip.read_q8(q)
    assert np.array_equal(got, v) and np.array_equal(scales, s)
    out = hip.alloc(rows * cols)
    hip.dequantize_q8(out, q)
    assert np.array_equal(hip.read(out).reshape(rows, cols), v.astype(np.float32) * s[:, None])


@gpu
def test_write_and_read_in_pieces(hip):
    """More integers (71 MB) than the block that they go through holds."""
    r = np.random.default_rng(9)
    v, s = r.integers(-128, 128, (7001, 10101), dtype=np.int8), r.standard_normal(7001).astype(np.float32)
    q = q8(hip, v, s)
    got, scales = hip.read_q8(q)
    assert np.array_equal(got, v) and np.array_equal(scales, s)


@gpu
def test_allocated_rows_are_zero(hip):
    q = hip.alloc_q8(5, 100)
    v, s = hip.read_q8(q)
    assert not v.any() and not s.any()
    out = hip.alloc(500)
    hip.dequantize_q8(out, q)
    assert not hip.read(out).any()


@gpu
@pytest.mark.parametrize("rows,cols", SIZES)
def test_quantize(hip, rows, cols):
    x = np.random.default_rng(cols).standard_normal((rows, cols)).astype(np.float32)
    x *= np.float32(10.0) ** np.arange(-1, rows - 1, dtype=np.float32)[:, None] if rows < 20 else np.float32(1)
    b, q, out = buf(hip, x), hip.alloc_q8(rows, cols), hip.alloc(rows * cols)
    hip.quantize_q8(q, b)
    want_q, want_s = rows64(x)
    v, s = hip.read_q8(q)
    assert np.array_equal(v, want_q) and np.array_equal(s, want_s)
    hip.dequantize_q8(out, q)
    got = hip.read(out).reshape(rows, cols)
    assert np.array_equal(got, want_q.astype(np.float32) * want_s[:, None])
    # Half a step, and what the scale's own rounding and the product's add.
    assert np.all(np.abs(got - x.astype(np.float64)) <= want_s[:, None] * (0.5 + 127 * 2.0**-23))


@gpu
def test_more_rows_than_a_launch_takes(hip):
    rows, cols = (1 << 21) + 300, 3
    x = np.random.default_rng(14).standard_normal((rows, cols)).astype(np.float32)
    q, out = hip.alloc_q8(rows, cols), hip.alloc(rows * cols)
    hip.quantize_q8(q, buf(hip, x))
    want_q, want_s = rows64(x)
    v, s = hip.read_q8(q)
    assert np.array_equal(v, want_q) and np.array_equal(s, want_s)
    hip.dequantize_q8(out, q)
    assert np.array_equal(hip.read(out).reshape(rows, cols), want_q.astype(np.float32) * want_s[:, None])


def special_rows(cols, seed=3):
    """Rows that the definition treats on their own, each beside ordinary ones."""
    x = np.random.default_rng(seed).standard_normal((14, cols)).astype(np.float32)
    x[1] = 0
    x[2] = -0.0
    x[3, cols // 2] = np.nan
    x[4, cols - 1] = np.inf
    x[5, 0] = -np.inf
    x[6] *= np.float32(1e-42)                      # subnormal values, scale subnormal
    x[7] = np.where(np.arange(cols) % 2, 3e-45, 0)  # scale rounds to zero
    x[8] = np.clip(x[8], -3, 3) * np.float32(1.1e38)  # near f32's largest
    x[9] = np.float32(0.5) * (np.arange(cols) % 255 - 127)   # borders: 127 v / A whole and halves
    x[9, 0] = 63.5 if cols > 1 else x[9, 0]
    x[10] = (np.arange(cols) % 509 - 254) * np.float32(2.0**-9)
    x[11] = -7.25
    x[12, cols // 3] = 1e30                       # one value beside which the rest is nothing
    return x


@gpu
@pytest.mark.parametrize("cols", [96, 1101, 2560, 9728, 12000])
def test_quantize_special_rows(hip, cols):
    x = special_rows(cols)
    b, q, out = buf(hip, x), hip.alloc_q8(*x.shape), hip.alloc(x.size)
    hip.quantize_q8(q, b)
    want_q, want_s = rows64(x)
    v, s = hip.read_q8(q)
    assert same(s, want_s)
    for i in range(len(x)):
        assert np.array_equal(v[i], want_q[i]), f"row {i}"
    hip.dequantize_q8(out, q)
    got = hip.read(out).reshape(x.shape)
    assert np.isnan(got[3:6]).all() and np.isfinite(np.delete(got, [3, 4, 5], axis=0)).all()
    assert np.array_equal(hip.read(b).view(np.uint32), x.reshape(-1).view(np.uint32)), "x stays as it was"


@gpu
@pytest.mark.parametrize("rows,cols", [(1, 1), (5, 64), (17, 1101), (300, 130), (24, 9728), (3, 20000)])
def test_quantize_weight(hip, rows, cols):
    bits = f32_to_bf16(np.random.default_rng(rows).standard_normal(rows * cols).astype(np.float32) * np.float32(0.02))
    if rows > 4:
        bits = bits.reshape(rows, cols)
        bits[1] = 0
        bits[2, cols // 2] = 0x7fc0  # NaN
        bits[3, 0] = 0xff80          # -inf
    q = hip.alloc_q8(rows, cols)
    hip.quantize_weight_q8(q, hip.upload(Tensor((rows, cols), bits)))
    want_q, want_s = rows64(bf16_to_f32(bits.reshape(-1)).reshape(rows, cols))
    v, s = hip.read_q8(q)
    assert np.array_equal(v, want_q) and same(s, want_s)


@gpu
@pytest.mark.parametrize("residual", [True, False])
@pytest.mark.parametrize("rows,cols", SIZES)
def test_add_rmsnorm(hip, rows, cols, residual):
    r = np.random.default_rng(rows * 7 + cols)
    x, y = (r.standard_normal((rows, cols)).astype(np.float32) for _ in range(2))
    gain = f32_to_bf16((1 + 0.1 * r.standard_normal(cols)).astype(np.float32))
    bx, by, q = buf(hip, x), buf(hip, y) if residual else None, hip.alloc_q8(rows, cols)
    hip.add_rmsnorm_q8(bx, by, q, hip.upload(Tensor((cols,), gain)), EPS)
    want = x + y if residual else x
    assert np.array_equal(hip.read(bx).reshape(rows, cols), want)
    p, scale = norm64(want, gain)
    want_q, want_s = rows64(p, scale)
    v, s = hip.read_q8(q)
    assert far_from_borders(p) and np.array_equal(v, want_q) and near(s, want_s)
    if residual:
        assert np.array_equal(hip.read(by).reshape(rows, cols), y)


@gpu
@pytest.mark.parametrize("cols", [96, 1101, 2560, 5001, 12000, 30000, 50000])
def test_add_rmsnorm_special_rows(hip, cols):
    x = special_rows(cols)
    y = np.zeros((20, cols), np.float32)  # longer than x: the rest is not looked at
    y[14:] = np.nan
    y[13, cols // 2] = np.inf
    x[8] *= np.float32(0.9)
    y[8] = x[8]                           # sums past f32: infinities
    gain = f32_to_bf16((1 + 0.1 * np.random.default_rng(5).standard_normal(cols)).astype(np.float32))
    bx, by, q = buf(hip, x), buf(hip, y), hip.alloc_q8(*x.shape)
    hip.add_rmsnorm_q8(bx, by, q, hip.upload(Tensor((cols,), gain)), EPS)
    with np.errstate(all="ignore"):
        want = x + y[:14]
    assert same(hip.read(bx).reshape(x.shape), want)
    p, scale = norm64(want, gain)
    want_q, want_s = rows64(p, scale)
    assert np.isnan(want_s[[3, 4, 5, 8, 13]]).all()
    v, s = hip.read_q8(q)
    assert near(s, want_s)
    for i in range(len(x)):
        assert np.array_equal(v[i], want_q[i]), f"row {i}"


@gpu
def test_add_rmsnorm_of_zero_rows_and_eps(hip):
    x = np.zeros((2, 200), np.float32)
    x[1] = np.random.default_rng(1).standard_normal(200) * 1e-20
    gain = np.full(200, 0x3f80, np.uint16)
    for eps in (0.0, 1e-6):
        bx, q = buf(hip, x), hip.alloc_q8(2, 200)
        hip.add_rmsnorm_q8(bx, None, q, hip.upload(Tensor((200,), gain)), eps)
        v, s = hip.read_q8(q)
        p, scale = norm64(x, gain, eps)
        assert s[0] == 0 and not v[0].any()
        assert np.array_equal(v[1], rows64(p)[0][1]) and near(s[1:], scale[1:].astype(np.float32))


@gpu
@pytest.mark.parametrize("rows,cols", SIZES)
def test_silu_mul(hip, rows, cols):
    r = np.random.default_rng(rows * 5 + cols)
    g, u = (2 * r.standard_normal((rows, cols)).astype(np.float32) for _ in range(2))
    bg, bu, q = buf(hip, g), buf(hip, u), hip.alloc_q8(rows, cols)
    hip.silu_mul_q8(q, bg, bu)
    want = silu64(g, u)
    want_q, want_s = rows64(want)
    v, s = hip.read_q8(q)
    assert far_from_borders(want) and np.array_equal(v, want_q) and near(s, want_s)
    assert np.array_equal(hip.read(bg).reshape(g.shape), g) and np.array_equal(hip.read(bu).reshape(g.shape), u)


@gpu
@pytest.mark.parametrize("cols", [96, 1101, 2560, 5001, 9728, 12000, 30000, 50000])
def test_silu_mul_special_rows(hip, cols):
    g = special_rows(cols)
    u = np.random.default_rng(6).standard_normal(g.shape).astype(np.float32)
    u[9:11] = 1
    g[0, :8] = [-1000, -200, -104, -88, 88, 200, 1000, 0]  # where f32's exponential overflows or vanishes
    g[11], u[11] = -700, 1e-30  # 64 bits hold it, f32 does not
    g[13], u[13] = 1e25, 1e25   # past f32, and A / 127 too
    g[12], u[12] = 3e37, 20     # past f32, A / 127 is not
    u[1, 0] = np.inf            # 0 * inf
    bg, bu, q = buf(hip, g), buf(hip, u), hip.alloc_q8(*g.shape)
    hip.silu_mul_q8(q, bg, bu)
    want_q, want_s = rows64(silu64(g, u))
    assert np.isnan(want_s[[1, 3, 4, 5, 13]]).all() and np.isfinite(want_s[12]) and want_s[11] == 0
    v, s = hip.read_q8(q)
    assert near(s, want_s)
    for i in range(len(g)):
        assert np.array_equal(v[i], want_q[i]), f"row {i}"


@gpu
@pytest.mark.parametrize("cols", [96, 1101, 9728, 20011])
def test_silu_mul_of_subnormal_gates(hip, cols):
    """Gates below f32's normal numbers with large ups: silu(gate) in f32 has few bits left, the product does not show it."""
    r = np.random.default_rng(13)
    g = (r.integers(1, 2000, (4, cols)) * 2.0**-149).astype(np.float32)
    u = (r.standard_normal((4, cols)) * 1e37).astype(np.float32)
    u[1], u[2] = u[1] * np.float32(1e-15), u[2] * np.float32(1e-30)
    g[3, ::2] = r.standard_normal(g[3, ::2].shape)
    q = hip.alloc_q8(4, cols)
    hip.silu_mul_q8(q, buf(hip, g), buf(hip, u))
    want_q, want_s = rows64(silu64(g, u))
    v, s = hip.read_q8(q)
    assert near(s, want_s) and np.array_equal(v, want_q)


def repeated(hip, a, rows):
    """A buffer of `rows` rows, those of a again and again."""
    b, have, total = hip.alloc(rows * a.shape[1]), a.size, rows * a.shape[1]
    first = buf(hip, a)
    hip.copy(b, 0, first, 0, have)
    while have < total:
        n = min(have, total - have)
        hip.copy(b, have, b, 0, n)
        have += n
    return b


@gpu
@pytest.mark.parametrize("cols", [200, 512, 1000, 1500, 2000, 2560, 4096, 5001, 6000, 8190, 9728, 12000, 16000, 20011, 24000, 28000,
                                  32000, 40000, 50000])
def test_more_than_the_caches_hold(hip, cols):
    """Inputs of 128 MB and more are read another way."""
    r = np.random.default_rng(cols)
    x, y = (r.standard_normal((19, cols)).astype(np.float32) for _ in range(2))
    gain = f32_to_bf16((1 + 0.1 * r.standard_normal(cols)).astype(np.float32))
    rows = (1 << 25) // cols + 1
    half = rows // 2 + 1  # of two inputs each

    def check(q, v, scale64=None):
        want_q, want_s = rows64(v, scale64)
        got, s = hip.read_q8(q)
        again = np.arange(len(s)) % 19
        assert np.array_equal(got, want_q[again]) and near(s, want_s[again])

    q, x0 = hip.alloc_q8(rows, cols), repeated(hip, x, rows)
    hip.quantize_q8(q, x0)
    check(q, x)
    hip.add_rmsnorm_q8(x0, None, q, hip.upload(Tensor((cols,), gain)), EPS)
    check(q, *norm64(x, gain))
    hip.resize_q8(q, half)
    x1, y1 = repeated(hip, x, half), repeated(hip, y, half)
    hip.silu_mul_q8(q, x1, y1)
    assert far_from_borders(silu64(x, y))  # the others' values are exact, ties among them
    check(q, silu64(x, y))
    hip.add_rmsnorm_q8(x1, y1, q, hip.upload(Tensor((cols,), gain)), EPS)
    check(q, *norm64(x + y, gain))
    assert np.array_equal(hip.read(x1).reshape(half, cols), (x + y)[np.arange(half) % 19])


@gpu
def test_silu_mul_of_one_buffer(hip):
    g = np.random.default_rng(2).standard_normal((4, 300)).astype(np.float32)
    b, q = buf(hip, g), hip.alloc_q8(4, 300)
    hip.silu_mul_q8(q, b, b)
    want_q, _ = rows64(silu64(g, g))
    assert np.array_equal(hip.read_q8(q)[0], want_q)


@gpu
@pytest.mark.parametrize("cols", [757, 1500, 2560, 4096, 5001, 6000, 8000, 9728, 12000, 16000, 20011, 24000, 28000, 32000, 40000])
def test_values_next_to_borders(hip, cols):
    """Quotients of k + 1/2 exactly, and one f32 step to either side, with a
    largest value that 127 does not divide: 32 bits would not tell them apart."""
    top = np.float32(1.7)
    k = np.arange(-126, 126)
    mid = ((k + 0.5) * np.float64(top) / 127).astype(np.float32)
    x = np.concatenate([[top], mid, np.nextafter(mid, np.float32(9)), np.nextafter(mid, np.float32(-9))]).astype(np.float32)
    x = np.resize(x, cols)
    b, q = buf(hip, x), hip.alloc_q8(1, x.size)
    hip.quantize_q8(q, b)
    assert np.array_equal(hip.read_q8(q)[0], rows64(x)[0])
    gain = np.full(x.size, 0x3f80, np.uint16)
    hip.add_rmsnorm_q8(b, None, q, hip.upload(Tensor((x.size,), gain)), EPS)
    assert np.array_equal(hip.read_q8(q)[0], rows64(x)[0])
    hip.write(b, x / 2)
    hip.add_rmsnorm_q8(b, buf(hip, x / 2), q, hip.upload(Tensor((x.size,), gain)), EPS)
    assert np.array_equal(hip.read_q8(q)[0], rows64(x)[0])


# Tokens and rows about 16, 32, 64, 128 and 256, columns about 64 and 128, and the layers' own.
PRODUCTS = [(1, 1, 1), (1, 16, 64), (1, 17, 65), (2, 3, 127), (15, 15, 128), (16, 16, 129), (17, 33, 192), (31, 63, 256),
            (33, 65, 320), (63, 127, 100), (65, 129, 1101), (50, 1003, 1101), (127, 255, 384), (129, 257, 640),
            (255, 130, 1000), (257, 300, 513), (300, 1000, 70), (513, 511, 260), (1, 1024, 2048), (1, 9728, 2560),
            (4, 2560, 9728), (11, 4096, 2560), (64, 2560, 9728), (512, 1030, 2560), (1, 5, 131071), (40, 20, 131071),
            (1000, 16, 128), (3, 20000, 33), (700, 2050, 200),
            # Each variant that a product can take, whole and with K split.
            # (Four tall tiles with K split have theirs beside the list of variants.)
            (17, 515, 2500), (17, 3001, 2500), (33, 3001, 60), (70, 3001, 60), (17, 3001, 60), (131, 3001, 60),
            (50, 1037, 16000), (131, 7001, 60), (33, 3001, 16000), (700, 7001, 60), (2000, 1037, 60),
            (70, 3001, 16000), (515, 7001, 60), (4100, 130, 9000), (700, 7001, 130), (131, 7001, 9000),
            (8192, 1037, 60), (131, 7001, 16000), (1300, 7001, 60), (1550, 7001, 60), (1030, 12000, 600),
            (6000, 3001, 60)]


@gpu
@pytest.mark.parametrize("n,rows,cols", PRODUCTS)
def test_matmul(hip, n, rows, cols):
    r = np.random.default_rng(n + rows + cols)
    xq, wq = (r.integers(-128, 128, (m, cols), dtype=np.int8) for m in (n, rows))
    xs, ws = (r.random(m).astype(np.float32) + np.float32(0.01) for m in (n, rows))
    out = buf(hip, np.full(n * rows + 64, -5.0))  # the tail stays as it is
    hip.resize(out, n * rows)
    hip.matmul_q8(out, q8(hip, wq, ws), q8(hip, xq, xs))
    got = hip.read(out).reshape(n, rows)
    want = product32(wq, ws, xq, xs)
    bad = np.argwhere(got != want)
    assert not len(bad), f"{len(bad)} of {got.size} differ, first at {bad[0]}: {got[tuple(bad[0])]} for {want[tuple(bad[0])]}"
    hip.resize(out, n * rows + 64)
    assert np.all(hip.read(out)[n * rows:] == -5.0)


@gpu
@pytest.mark.parametrize("n", [1, 40, 300])
def test_matmul_largest_sums(hip, n):
    """Every product 128 * 128, at the most columns: 2^31 - 2^14."""
    cols, rows = 131071, 20
    out = hip.alloc(n * rows)
    one = np.ones(max(n, rows), np.float32)
    hip.matmul_q8(out, q8(hip, np.full((rows, cols), -128, np.int8), one[:rows]),
                  q8(hip, np.full((n, cols), -128, np.int8), one[:n]))
    assert np.all(hip.read(out) == np.float32(131071 * 16384))


@gpu
@pytest.mark.parametrize("n", [1, 20, 200])
def test_matmul_of_special_scales(hip, n):
    r = np.random.default_rng(n)
    rows, cols = 70, 300
    xq, wq = (r.integers(-127, 128, (m, cols), dtype=np.int8) for m in (n, rows))
    xs, ws = np.ones(n, np.float32), np.ones(rows, np.float32)
    xs[0], ws[1], ws[2], ws[3], ws[4], ws[5] = np.float32(1e-38), np.nan, np.inf, 0, -2, np.float32(1e-40)
    if n > 2:
        xs[1], xs[2] = np.nan, 0
    out = hip.alloc(n * rows)
    hip.matmul_q8(out, q8(hip, wq, ws), q8(hip, xq, xs))
    assert same(hip.read(out).reshape(n, rows), product32(wq, ws, xq, xs))


@gpu
def test_offsets_past_32_bits(hip):
    """Rows of 4.4 GB, f32 values of 17.6: those behind 2^32 elements are as good as the first."""
    rows, cols = 110000, 40000
    look = [0, 1, 53687, 53688, 107374, 107375, rows - 1]  # about 2^31 and 2^32 values, and the last
    r = np.random.default_rng(21)
    aq, bq = (r.integers(-127, 128, (m, 128), dtype=np.int8) for m in (rows, cols))
    sa, sb = (r.random(m).astype(np.float32) + np.float32(0.5) for m in (rows, cols))
    a, b, x, one = q8(hip, aq, sa), q8(hip, bq, sb), hip.alloc(rows * cols), hip.alloc(cols)

    def row(i):
        hip.copy(one, 0, x, i * cols, cols)
        return hip.read(one)

    hip.matmul_q8(x, b, a)
    v = product32(bq, sb, aq[look], sa[look])
    assert np.array_equal(np.stack([row(i) for i in look]), v)

    q = hip.alloc_q8(rows, cols)
    hip.quantize_q8(q, x)
    want_q, want_s = rows64(v)
    for n in (3, 40, 200):  # columns of it, picked by tokens of one 1 each
        at = r.permutation(cols)[:n]
        at[:2] = 0, cols - 1
        pick = np.zeros((n, cols), np.int8)
        pick[np.arange(n), at] = 1
        out = hip.alloc(n * rows)
        hip.matmul_q8(out, q, q8(hip, pick, np.ones(n, np.float32)))
        assert np.array_equal(hip.read(out).reshape(n, rows)[:, look], (want_q[:, at].astype(np.float32) * want_s[:, None]).T)
        hip.matmul_q8(out, q8(hip, pick, np.ones(n, np.float32)), q)
        assert np.array_equal(hip.read(out).reshape(rows, n)[look], want_q[:, at].astype(np.float32) * want_s[:, None])

    gain = f32_to_bf16((1 + 0.1 * r.standard_normal(cols)).astype(np.float32))
    for quantize, values in ((lambda: hip.silu_mul_q8(q, x, x), silu64(v, v)),
                             (lambda: hip.add_rmsnorm_q8(x, None, q, hip.upload(Tensor((cols,), gain)), EPS), None)):
        quantize()
        if values is None:
            assert np.array_equal(np.stack([row(i) for i in look]), v)
            values, scales = norm64(v, gain)
            want_q, scales = rows64(values, scales)
        else:
            want_q, scales = rows64(values)
        assert far_from_borders(values)
        hip.dequantize_q8(x, q)
        got = np.stack([row(i) for i in look])
        s = np.abs(got).max(axis=1) / np.float32(127)  # 127 is among a row's integers: two roundings, and the norm's step
        assert np.all(np.abs(s - scales) <= 2.0**-22 * scales)
        assert np.array_equal(np.rint(got / s[:, None]).astype(np.int8), want_q)
        hip.matmul_q8(x, b, a)


@gpu
def test_rows_with_themselves(hip):
    v = np.random.default_rng(8).integers(-127, 128, (40, 200), dtype=np.int8)
    s = np.linspace(0.1, 2, 40).astype(np.float32)
    q, out = q8(hip, v, s), hip.alloc(1600)
    hip.matmul_q8(out, q, q)
    assert np.array_equal(hip.read(out).reshape(40, 40), product32(v, s, v, s))


@gpu
def test_fewer_rows_than_allocated(hip):
    """A batch's handle serves smaller batches; what lies behind them is neither used nor changed."""
    r = np.random.default_rng(4)
    cols = 130
    v, s = r.integers(-127, 128, (40, cols), dtype=np.int8), r.random(40).astype(np.float32)
    s[5:] = np.nan
    q, w = q8(hip, v, s), q8(hip, v[:30], np.ones(30, np.float32))
    hip.resize_q8(q, 5)
    out = hip.alloc(150)
    hip.matmul_q8(out, w, q)
    assert np.array_equal(hip.read(out).reshape(5, 30), product32(v[:30], np.ones(30, np.float32), v[:5], s[:5]))
    x = r.standard_normal((3, cols)).astype(np.float32)
    hip.resize_q8(q, 3)
    hip.quantize_q8(q, buf(hip, x))
    hip.resize_q8(q, 40)
    got, scales = hip.read_q8(q)
    assert np.array_equal(got[:3], rows64(x)[0]) and np.array_equal(got[3:], v[3:])
    assert np.array_equal(scales[3:], s[3:], equal_nan=True)
    hip.resize_q8(q, 0)
    empty = hip.alloc(0)
    hip.matmul_q8(empty, w, q)
    hip.quantize_q8(q, empty)
    hip.dequantize_q8(empty, q)
    hip.silu_mul_q8(q, empty, empty)
    assert hip.read_q8(q)[0].shape == (0, cols)


class Mlp:
    """The MLP half of a layer (model/model.rs:132-143) over 8-bit rows, then
    the next layer's norm and its q projection: x += y; h = rmsnorm(x);
    y = down . (silu(gate . h) * (up . h)); x += y; q = wq . rmsnorm(x)."""

    def __init__(self, hip, n, hidden, inter, heads):
        r = np.random.default_rng(n + hidden)
        self.hip, self.n, self.hidden, self.inter, self.heads = hip, n, hidden, inter, heads
        self.x, self.y = (r.standard_normal((n, hidden)).astype(np.float32) for _ in range(2))
        self.w = {k: f32_to_bf16(r.standard_normal(s).astype(np.float32).reshape(-1) * np.float32(0.05)).reshape(s)
                  for k, s in {"gate": (inter, hidden), "up": (inter, hidden), "down": (hidden, inter),
                               "q": (heads, hidden)}.items()}
        self.gain = f32_to_bf16((1 + 0.1 * r.standard_normal((2, hidden))).astype(np.float32).reshape(-1)).reshape(2, hidden)
        self.q8 = {}
        for k, w in self.w.items():
            self.q8[k] = hip.alloc_q8(*w.shape)
            hip.quantize_weight_q8(self.q8[k], hip.upload(Tensor(w.shape, w)))
        self.gains = [hip.upload(Tensor((hidden,), g)) for g in self.gain]
        self.bx, self.by = hip.alloc(n * hidden), hip.alloc(n * hidden)
        self.bg, self.bu, self.bq = hip.alloc(n * inter), hip.alloc(n * inter), hip.alloc(n * heads)
        self.h, self.a = hip.alloc_q8(n, hidden), hip.alloc_q8(n, inter)

    def load(self):
        self.hip.write(self.bx, self.x)
        self.hip.write(self.by, self.y)

    def calls(self):
        h = self.hip
        h.add_rmsnorm_q8(self.bx, self.by, self.h, self.gains[0], EPS)
        h.matmul_q8(self.bg, self.q8["gate"], self.h)
        h.matmul_q8(self.bu, self.q8["up"], self.h)
        h.silu_mul_q8(self.a, self.bg, self.bu)
        h.matmul_q8(self.by, self.q8["down"], self.a)
        h.add_rmsnorm_q8(self.bx, self.by, self.h, self.gains[1], EPS)
        h.matmul_q8(self.bq, self.q8["q"], self.h)

    def results(self):
        return self.hip.read(self.bx).reshape(self.n, -1), self.hip.read(self.bq).reshape(self.n, -1)

    def want(self):
        w = {k: rows64(bf16_to_f32(v.reshape(-1)).reshape(v.shape)) for k, v in self.w.items()}

        def norm(x, gain):
            p, scale = norm64(x, gain)
            return rows64(p, scale)

        x = self.x + self.y
        h = norm(x, self.gain[0])
        a = rows64(silu64(product32(*w["gate"], *h), product32(*w["up"], *h)))
        x = x + product32(*w["down"], *a)
        return x, product32(*w["q"], *norm(x, self.gain[1]))


MLPS = [(1, 1024, 2304, 512), (9, 512, 1536, 700), (70, 512, 1536, 512), (150, 333, 1001, 90)]


def check_mlp(m, got, want):
    """The steps repeat the definition's, but a scale may be one f32 step off
    (2^-23), which moves the following quotients by 127 * 2^-22 and with that
    an integer in some 30000 to its neighbour: one step of the row, 1/127 of
    its largest. A sum of `inter` products of which k moved is off by at most
    k / 127 of the largest activation times the largest weight; k is 0 or 1
    here, a few at most. Against the values' own size (norm-wise) that is
    under 1e-3, where 8 bits themselves cost 1e-2."""
    for name, g, w in zip(("x", "q"), got, want):
        off = np.linalg.norm(g.astype(np.float64) - w) / np.linalg.norm(w.astype(np.float64))
        assert off < 1e-3, (name, off)


@gpu
@pytest.mark.parametrize("n,hidden,inter,heads", MLPS)
def test_run_of_a_layer(hip, n, hidden, inter, heads):
    m = Mlp(hip, n, hidden, inter, heads)
    m.load()
    m.calls()
    got = m.results()
    check_mlp(m, got, m.want())
    # And 8 bits are near the layer in the weights' and activations' own types.
    f = {k: bf16_to_f32(v.reshape(-1)).reshape(v.shape).astype(np.float64) for k, v in m.w.items()}

    def norm(x, gain):
        return x / np.sqrt(np.mean(x * x, axis=1, keepdims=True) + EPS) * bf16_to_f32(gain)

    x = (m.x + m.y).astype(np.float64)
    h = norm(x, m.gain[0])
    g = h @ f["gate"].T
    x = x + (g / (1 + np.exp(-g)) * (h @ f["up"].T)) @ f["down"].T
    # Each 8-bit row is off by step / sqrt(12), steps of A / 127 with A at most
    # 5 of the row's own size (10 for the activations' products): 0.012 and
    # 0.023; three products in a row of two such factors each stay below 0.1.
    assert np.linalg.norm(got[0] - x) / np.linalg.norm(x) < 0.1


@gpu
@pytest.mark.parametrize("n,hidden,inter,heads", MLPS)
def test_captured_run_replays(hip, n, hidden, inter, heads):
    """Two graphs of the run, which share the device's memory for partial
    sums, replayed in turn with eager work between: each the eager bits."""
    a, b = Mlp(hip, n, hidden, inter, heads), Mlp(hip, n + 1, hidden, inter, heads)
    want = []
    for m in (a, b):
        m.load()
        m.calls()
        want.append(m.results())
    graphs = []
    for m in (a, b):
        hip.graph_begin()
        try:
            m.calls()
        finally:
            graphs.append(hip.graph_end())
    for replay in range(3):
        for m in (a, b):
            m.load()
        for g in graphs:
            g.launch()
        for m, w in zip((a, b), want):
            for g, e in zip(m.results(), w):
                assert np.array_equal(g, e), f"replay {replay}"
        a.load()
        a.calls()
        hip.synchronize()
    for g in graphs:
        g.free()


@gpu
def test_capture_refuses_copies_and_allocations(hip):
    q = hip.alloc_q8(2, 64)
    hip.graph_begin()
    try:
        for call in (lambda: hip.alloc_q8(2, 64), lambda: hip.read_q8(q),
                     lambda: hip.write_q8(q, np.zeros((2, 64), np.int8), np.zeros(2)), lambda: q.free()):
            with pytest.raises(Exception, match="captur"):
                call()
    finally:
        graph = hip.graph_end()
    hip.write_q8(q, np.ones((2, 64), np.int8), np.ones(2))
    assert hip.read_q8(q)[0].all()
    graph.free()


@gpu
def test_graphs_share_the_block_of_sums(hip):
    """Two captured products that split K (their sums go through one block of
    the device's), replayed in turn with an eager one between."""
    r = np.random.default_rng(12)
    runs = []
    for n, rows, cols in ((70, 3001, 16000), (131, 2050, 16000)):
        xq, wq = (r.integers(-127, 128, (m, cols), dtype=np.int8) for m in (n, rows))
        xs, ws = (r.random(m).astype(np.float32) for m in (n, rows))
        runs.append((hip.alloc(n * rows), q8(hip, wq, ws), q8(hip, xq, xs), product32(wq, ws, xq, xs).reshape(-1)))
    graphs = []
    for out, w, x, _ in runs:
        hip.graph_begin()
        try:
            hip.matmul_q8(out, w, x)
        finally:
            graphs.append(hip.graph_end())
    for replay in range(3):
        for out, *_ in runs:
            hip.write(out, np.zeros(len(out), np.float32))
        for g in graphs:
            g.launch()
        assert all(np.array_equal(hip.read(out), want) for out, _, _, want in runs), f"replay {replay}"
        hip.matmul_q8(*runs[replay % 2][:3])
    for g in graphs:
        g.free()


@gpu
def test_allocation_that_fails_leaves_no_error(hip):
    """4 TB are not there; the next launch does not report it."""
    with pytest.raises(HipError) as e:
        hip.alloc_q8(1 << 25, 131071)
    assert e.value.code == _lib.TH_ERR_NOMEM
    x = np.arange(64, dtype=np.float32)
    q = hip.alloc_q8(1, 64)
    hip.quantize_q8(q, buf(hip, x))
    assert np.array_equal(hip.read_q8(q)[0], rows64(x)[0])


@gpu
def test_refusals_on_the_device(hip):
    q, x = hip.alloc_q8(2, 64), hip.alloc(128)
    for call in (lambda: hip.alloc_q8(2, 0), lambda: hip.alloc_q8(1, 131072), lambda: hip.alloc_q8((1 << 25) + 1, 1),
                 lambda: hip.resize_q8(q, 3),
                 lambda: hip.quantize_q8(q, hip.alloc(64)), lambda: hip.dequantize_q8(hip.alloc(64), q),
                 lambda: hip.silu_mul_q8(q, x, hip.alloc(64)), lambda: hip.matmul_q8(x, hip.alloc_q8(2, 65), q),
                 lambda: hip.add_rmsnorm_q8(x, x, q, hip.upload(Tensor((64,), np.zeros(64, np.uint16))), EPS)):
        with pytest.raises(InvalidArgument):
            call()
    with pytest.raises(TypeError):
        hip.write_q8(q, np.zeros((2, 64)), np.zeros(2))
    with pytest.raises(ValueError):
        hip.write_q8(q, np.zeros((2, 64), np.int8), np.zeros(3))


# ---- refusals without a GPU: handles made here, which no call may get past ----

class _Buffer(C.Structure):
    _fields_ = [("ptr", C.c_void_p), ("len", C.c_size_t), ("cap", C.c_size_t)]


class _Weight(C.Structure):
    _fields_ = [("ptr", C.c_void_p), ("ndim", C.c_size_t), ("shape", C.c_size_t * 2), ("numel", C.c_size_t)]


class _Q8(C.Structure):
    _fields_ = [("ptr", C.c_void_p), ("scale", C.c_void_p), ("rows", C.c_size_t), ("cap", C.c_size_t),
                ("cols", C.c_size_t), ("ordinal", C.c_int)]


DEV = C.create_string_buffer(8192)  # a device of zeros: GPU 0, not capturing


def _b(n, at=0x1000):
    return C.byref(_Buffer(at, n, n))


def _q(rows, cols, ordinal=0):
    return C.byref(_Q8(0x1000, 0x2000, rows, rows, cols, ordinal))


def _w(*shape):
    return C.byref(_Weight(0x1000, len(shape), (C.c_size_t * 2)(*shape), int(np.prod(shape))))


OUT = C.c_void_p()
REFUSED = {
    "alloc: no columns": lambda l: l.th_q8_alloc(DEV, 4, 0, C.byref(OUT)),
    "alloc: sums past 32 bits": lambda l: l.th_q8_alloc(DEV, 4, 131072, C.byref(OUT)),
    "alloc: too many rows": lambda l: l.th_q8_alloc(DEV, (1 << 25) + 1, 64, C.byref(OUT)),
    "alloc: rows past 64 bits": lambda l: l.th_q8_alloc(DEV, 1 << 62, 64, C.byref(OUT)),
    "alloc: no output": lambda l: l.th_q8_alloc(DEV, 4, 64, None),
    "alloc: no device": lambda l: l.th_q8_alloc(None, 4, 64, C.byref(OUT)),
    "shape: null": lambda l: l.th_q8_shape(None, None, None),
    "resize: more than allocated": lambda l: l.th_q8_resize(DEV, _q(4, 64), 5),
    "resize: null": lambda l: l.th_q8_resize(DEV, None, 5),
    "read: null output": lambda l: l.th_q8_read(DEV, _q(4, 64), None, None),
    "write: null data": lambda l: l.th_q8_write(DEV, _q(4, 64), None, None),
    "read: another GPU": lambda l: l.th_q8_read(DEV, _q(4, 64, 1), C.byref(OUT), C.byref(OUT)),
    "quantize: fewer": lambda l: l.th_quantize_q8(DEV, _q(4, 64), _b(255)),
    "quantize: more": lambda l: l.th_quantize_q8(DEV, _q(4, 64), _b(320)),
    "quantize: null": lambda l: l.th_quantize_q8(DEV, _q(4, 64), None),
    "quantize: another GPU": lambda l: l.th_quantize_q8(DEV, _q(4, 64, 1), _b(256)),
    "weight: transposed": lambda l: l.th_quantize_weight_q8(DEV, _q(4, 64), _w(64, 4)),
    "weight: a vector": lambda l: l.th_quantize_weight_q8(DEV, _q(1, 64), _w(64)),
    "weight: null": lambda l: l.th_quantize_weight_q8(DEV, _q(1, 64), None),
    "dequantize: another length": lambda l: l.th_dequantize_q8(DEV, _b(255), _q(4, 64)),
    "dequantize: another GPU": lambda l: l.th_dequantize_q8(DEV, _b(256), _q(4, 64, 1)),
    "norm: gains": lambda l: l.th_add_rmsnorm_q8(DEV, _b(256), _b(256, 0x9000), _q(4, 64), _w(65), 1e-6),
    "norm: x": lambda l: l.th_add_rmsnorm_q8(DEV, _b(255), None, _q(4, 64), _w(64), 1e-6),
    "norm: y too short": lambda l: l.th_add_rmsnorm_q8(DEV, _b(256), _b(255, 0x9000), _q(4, 64), _w(64), 1e-6),
    "norm: y is x": lambda l: l.th_add_rmsnorm_q8(DEV, _b(256), _b(256), _q(4, 64), _w(64), 1e-6),
    "norm: null": lambda l: l.th_add_rmsnorm_q8(DEV, _b(256), None, None, _w(64), 1e-6),
    "norm: another GPU": lambda l: l.th_add_rmsnorm_q8(DEV, _b(256), None, _q(4, 64, 1), _w(64), 1e-6),
    "silu: gate": lambda l: l.th_silu_mul_q8(DEV, _q(4, 64), _b(255), _b(256)),
    "silu: up": lambda l: l.th_silu_mul_q8(DEV, _q(4, 64), _b(256), _b(320)),
    "silu: null": lambda l: l.th_silu_mul_q8(DEV, _q(4, 64), _b(256), None),
    "silu: another GPU": lambda l: l.th_silu_mul_q8(DEV, _q(4, 64, 1), _b(256), _b(256)),
    "matmul: columns": lambda l: l.th_matmul_q8(DEV, _b(32), _q(8, 64), _q(4, 65)),
    "matmul: out": lambda l: l.th_matmul_q8(DEV, _b(33), _q(8, 64), _q(4, 64)),
    "matmul: null": lambda l: l.th_matmul_q8(DEV, _b(32), _q(8, 64), None),
    "matmul: weights on another GPU": lambda l: l.th_matmul_q8(DEV, _b(32), _q(8, 64, 1), _q(4, 64)),
    "matmul: rows on another GPU": lambda l: l.th_matmul_q8(DEV, _b(32), _q(8, 64), _q(4, 64, 1)),
}


@pytest.mark.parametrize("name", list(REFUSED))
def test_refusals(name):
    lib = _lib.lib()
    assert REFUSED[name](lib) == _lib.TH_ERR_INVALID
    assert lib.th_last_error()


def test_free_of_nothing():
    _lib.lib().th_q8_free(DEV, None)
    _lib.lib().th_q8_free(None, None)
