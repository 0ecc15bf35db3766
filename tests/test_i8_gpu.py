"""8-bit rows with one scale each through the C ABI, against 64-bit numpy.

Tolerances, by arithmetic: a scale is one FP32 rounding of a 64-bit value
(2^-24 of it; 2^-23 where the 64-bit value itself lies next to a border);
codes are the nearest integers of value / scale, so |value / scale - code| <=
1/2, plus 1e-9 for the 64-bit arithmetic on either side; a product is an
exact integer (one rounding to FP32), times two scales (two roundings), plus
a residual (one): 3 * 2^-24 of the product and 2^-24 of the sum, 1% more for
their compounding.
"""
import numpy as np
import pytest

from sharpinference_amd import native

pytestmark = pytest.mark.gpu

EPS24 = 2.0 ** -24


def _rows(rng, rows, n):
    """Rows of different sizes, some with outliers."""
    x = rng.standard_normal((rows, n)) * np.exp(rng.uniform(-6, 6, (rows, 1)))
    x[::3, rng.integers(0, n)] *= 50
    return x.astype(np.float32)


def _check_codes(y, codes, scale):
    """y [rows, n] in 64 bits."""
    top = np.abs(y).max(1)
    want = top / 127
    assert np.all(np.abs(scale.astype(np.float64) - want) <= 2.0 ** -23 * want + 1e-45)
    live = scale > 0
    assert np.all(codes[~live] == 0)
    t = y[live] / scale[live].astype(np.float64)[:, None]
    assert np.all(np.abs(t - codes[live]) <= 0.5 + 1e-9)
    assert np.all(np.abs(codes.astype(int)) <= 127)


def _guarded(hip, nbytes, fill=0x5A):
    """A buffer with 64 spare bytes behind it."""
    return hip.to_device(np.full(nbytes + 64, fill, np.uint8))


def _spare_untouched(buf, nbytes, fill=0x5A):
    assert np.all(buf.readback(np.uint8, 64, nbytes) == fill)


SHAPES = [(1, 1), (1, 2048), (3, 17), (5, 64), (2, 5001), (1030, 130), (1025, 2048), (4, 8192), (2, 8193), (3, 16384),
          (2, 33000), (1, 70001)]


@pytest.mark.parametrize("rows,n", SHAPES)
@pytest.mark.parametrize("residual", [False, True])
def test_norm_codes(hip, rows, n, residual):
    rng = np.random.default_rng(rows * 7919 + n)
    h, r = _rows(rng, rows, n), rng.standard_normal((rows, n)).astype(np.float32)
    w = (1 + 0.2 * rng.standard_normal(n)).astype(np.float32)
    dh, dr, dw = hip.to_device(h), hip.to_device(r), hip.to_device(w)
    up, q, s = _guarded(hip, h.nbytes), _guarded(hip, rows * n), _guarded(hip, rows * 4)
    hip.residual_rms_norm_i8(dh.ptr, dr.ptr if residual else 0, dw.ptr, up.ptr if residual else 0, q.ptr, s.ptr, rows, n,
                             1e-5)
    u = h + r if residual else h
    if residual:
        assert np.array_equal(up.readback(np.float32, rows * n).reshape(rows, n), u)
    codes, scale = q.readback(np.int8, rows * n).reshape(rows, n), s.readback(np.float32, rows)
    u64 = u.astype(np.float64)
    y = u64 / np.sqrt((u64 * u64).mean(1, keepdims=True) + float(np.float32(1e-5))) * w.astype(np.float64)
    _check_codes(y, codes, scale)
    for b, nb in ((up, h.nbytes), (q, rows * n), (s, rows * 4)):
        _spare_untouched(b, nb)


@pytest.mark.parametrize("rows,n", [(1024, 3), (1500, 2), (1024, 255), (1100, 256), (1030, 1003), (1024, 1024), (2, 4097),
                                    (1, 6002), (2, 8190), (3, 16385)])
@pytest.mark.parametrize("shift", [0, 1, 2])
@pytest.mark.parametrize("fmt", [None, native.F32, native.F16, native.BF16])
def test_rows_of_any_length_at_any_address(hip, fmt, rows, n, shift):
    """Ends inside a four, one place of the type off its alignment; None: the norm with a residual."""
    rng = np.random.default_rng(rows * n + shift)
    x = (_rows(rng, rows, n) / 50).astype(np.float32)
    size = 2 if fmt in (native.F16, native.BF16) else 4
    raw = x.astype(np.float16) if fmt == native.F16 else (x.view(np.uint32) >> 16).astype(np.uint16) if fmt == native.BF16 else x
    exact = (raw.astype(np.uint32) << 16).view(np.float32).astype(np.float64) if fmt == native.BF16 else raw.astype(np.float64)

    def at(a, step):
        b = hip.alloc(a.nbytes + 64)
        b.upload(np.ascontiguousarray(a), step * shift)
        return b, b.ptr + step * shift
    held, dx = at(raw, size)
    q, s = hip.to_device(np.full(rows * n + 64, 0x5A, np.uint8)), hip.alloc(rows * 4)
    if fmt is None:
        r, w = rng.standard_normal((rows, n)).astype(np.float32), (1 + 0.2 * rng.standard_normal(n)).astype(np.float32)
        (hr, dr), (hw, dw) = at(r, 4), at(w, 4)
        up = hip.to_device(np.full(rows * n * 4 + 64, 0x5A, np.uint8))
        hip.residual_rms_norm_i8(dx, dr, dw, up.ptr + 4 * shift, q.ptr + shift, s.ptr, rows, n, 1e-5)
        u = x + r
        assert np.array_equal(up.readback(np.float32, rows * n, 4 * shift).reshape(rows, n), u)
        assert np.all(up.readback(np.uint8, 64 - 4 * shift, rows * n * 4 + 4 * shift) == 0x5A)
        u = u.astype(np.float64)
        exact = u / np.sqrt((u * u).mean(1, keepdims=True) + float(np.float32(1e-5))) * w.astype(np.float64)
    else:
        hip.quantize_i8(fmt, dx, q.ptr + shift, s.ptr, rows, n)
    codes, scale = q.readback(np.int8, rows * n, shift).reshape(rows, n), s.readback(np.float32, rows)
    _check_codes(exact, codes, scale)
    assert np.all(q.readback(np.uint8, 64 - shift, rows * n + shift) == 0x5A)
    back = hip.to_device(np.full(rows * n * 4 + 64, 0x5A, np.uint8))
    hip.dequant_i8(q.ptr + shift, s.ptr, back.ptr + 4 * shift, rows, n)
    assert np.array_equal(back.readback(np.float32, rows * n, 4 * shift).reshape(rows, n), codes * scale[:, None])
    assert np.all(back.readback(np.uint8, 64 - 4 * shift, rows * n * 4 + 4 * shift) == 0x5A)


def test_norm_codes_at_odd_addresses(hip):
    rng = np.random.default_rng(5)
    rows, n = 3, 1024
    h, w = _rows(rng, rows, n), (1 + 0.2 * rng.standard_normal(n)).astype(np.float32)
    outs = []
    for shift in (0, 1):
        dh, dw = hip.alloc(h.nbytes + 16), hip.alloc(w.nbytes + 16)
        dh.upload(h, 4 * shift)
        dw.upload(w, 4 * shift)
        q, s = hip.alloc(rows * n + 16), hip.alloc(rows * 4 + 16)
        hip.residual_rms_norm_i8(dh.ptr + 4 * shift, 0, dw.ptr + 4 * shift, 0, q.ptr + shift, s.ptr + 4 * shift, rows, n,
                                 1e-5)
        outs.append((q.readback(np.int8, rows * n, shift), s.readback(np.float32, rows, 4 * shift)))
    assert np.array_equal(outs[0][0], outs[1][0]) and np.array_equal(outs[0][1], outs[1][1])


@pytest.mark.parametrize("n", [64, 2048, 9000])
def test_norm_special_rows(hip, n):
    """Zeros, infinities, NaN, the largest and the smallest values."""
    rng = np.random.default_rng(n)
    h = rng.standard_normal((7, n)).astype(np.float32)
    h[0] = 0
    h[1, n // 2] = np.inf
    h[2, n - 1] = np.nan
    h[3] *= np.float32(1e38) / np.abs(h[3]).max()
    h[4] = (np.sign(h[4]) * 1e-40).astype(np.float32)
    h[5] = 0
    h[5, 3] = -1e-45
    w = np.ones(n, np.float32)
    dh, dw = hip.to_device(h), hip.to_device(w)
    for eps in (0.0, 1e-5):
        q, s, back = hip.alloc(7 * n), hip.alloc(28), hip.alloc(28 * n)
        hip.residual_rms_norm_i8(dh.ptr, 0, dw.ptr, 0, q.ptr, s.ptr, 7, n, eps)
        codes, scale = q.readback(np.int8).reshape(7, n), s.readback(np.float32)
        assert scale[0] == 0 and np.isnan(scale[1]) and np.isnan(scale[2]) and np.all(codes[:3] == 0)
        h64 = h[3:].astype(np.float64)
        y = h64 / np.sqrt((h64 * h64).mean(1, keepdims=True) + float(np.float32(eps)))
        t = np.zeros_like(y)
        live = scale[3:] > 0
        t[live] = np.clip(y[live] / scale[3:][live].astype(np.float64)[:, None], -127, 127)
        assert np.all(np.abs(t - codes[3:]) <= 0.5 + 1e-9)
        hip.dequant_i8(q.ptr, s.ptr, back.ptr, 7, n)
        v = back.readback(np.float32).reshape(7, n)
        assert np.all(v[0] == 0) and np.all(np.isnan(v[1:3])) and np.array_equal(v[3:], codes[3:] * scale[3:, None])


@pytest.mark.parametrize("fmt", [None, native.F32, native.F16, native.BF16])
@pytest.mark.parametrize("rows,n", [(1000, 255), (1100, 256), (2, 4097), (1, 9001)])
def test_codes_between_two_steps(hip, fmt, rows, n):
    """Whole numbers over a whole scale: many quotients are halves exactly, and go to the even
    code.  (None: the norm of rows of -1 and 1 with such weights, whose mean square is 1.)"""
    rng = np.random.default_rng(n)
    # 127 times the scale has to be exact in the format, and every half of it
    most = {native.F16: 8, native.BF16: 1}.get(fmt, 16000)
    step = rng.integers(1, most + 1, 1 if fmt is None else rows) * 2.0
    half = rng.integers(-253, 254, (len(step), n))
    half[:, n // 2] = 254
    x = half * (step[:, None] / 2)
    want = np.rint(half / 2).astype(np.int8)                   # (ties to even)
    codes, scale = hip.alloc(rows * n), hip.alloc(rows * 4)
    if fmt is None:
        signs = rng.choice([-1.0, 1.0], (rows, n)).astype(np.float32)
        hip.residual_rms_norm_i8(hip.to_device(signs).ptr, 0, hip.to_device(x[0].astype(np.float32)).ptr, 0, codes.ptr,
                                 scale.ptr, rows, n, 0.0)
        step, want = np.repeat(step, rows), (want * signs).astype(np.int8)
    else:
        raw = x.astype({native.F32: np.float32, native.F16: np.float16, native.BF16: np.float32}[fmt])
        assert np.array_equal(raw.astype(np.float64), x)
        if fmt == native.BF16:
            assert not np.any(raw.view(np.uint32) & 0xFFFF)
            raw = (raw.view(np.uint32) >> 16).astype(np.uint16)
        hip.quantize_i8(fmt, hip.to_device(raw).ptr, codes.ptr, scale.ptr, rows, n)
    assert np.array_equal(scale.readback(np.float32), step.astype(np.float32))
    assert np.array_equal(codes.readback(np.int8).reshape(rows, n), want)


@pytest.mark.parametrize("fmt", [native.F32, native.F16, native.BF16])
@pytest.mark.parametrize("rows,n", [(1, 16), (3, 33), (1024, 96), (2, 8192), (1, 40000)])
def test_quantize_and_back(hip, fmt, rows, n):
    rng = np.random.default_rng(rows + n)
    x = (_rows(rng, rows, n) / 50).astype(np.float32)
    if fmt == native.F16:
        x = x.astype(np.float16)
        raw, exact = x, x.astype(np.float64)
    elif fmt == native.BF16:
        raw = (x.view(np.uint32) >> 16).astype(np.uint16)
        exact = (raw.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    else:
        raw, exact = x, x.astype(np.float64)
    dx = hip.to_device(raw)
    q, s, back = _guarded(hip, rows * n), _guarded(hip, rows * 4), _guarded(hip, rows * n * 4)
    hip.quantize_i8(fmt, dx.ptr, q.ptr, s.ptr, rows, n)
    codes, scale = q.readback(np.int8, rows * n).reshape(rows, n), s.readback(np.float32, rows)
    _check_codes(exact, codes, scale)
    hip.dequant_i8(q.ptr, s.ptr, back.ptr, rows, n)
    assert np.array_equal(back.readback(np.float32, rows * n).reshape(rows, n), codes * scale[:, None])
    for b, nb in ((q, rows * n), (s, rows * 4), (back, rows * n * 4)):
        _spare_untouched(b, nb)


def _gemm(hip, x, xs, w, ws, residual=None, in_place=False):
    m, cols = x.shape
    rows = w.shape[0]
    bufs = [hip.to_device(a) for a in (x, xs, w, ws)]
    y = _guarded(hip, m * rows * 4)
    dr = 0
    if residual is not None:
        if in_place:
            y.upload(residual)
            dr = y.ptr
        else:
            dr = hip.to_device(residual).ptr
    hip.gemm_i8(*[b.ptr for b in bufs], y.ptr, m, rows, cols, dr)
    out = y.readback(np.float32, m * rows).reshape(m, rows)
    _spare_untouched(y, m * rows * 4)
    return out


def _check_gemm(y, x, xs, w, ws, residual=None):
    dot = x.astype(np.float64) @ w.astype(np.float64).T          # exact: below 2^53
    p = dot * xs.astype(np.float64)[:, None] * ws.astype(np.float64)
    t = p if residual is None else p + residual.astype(np.float64)
    assert np.all(np.abs(y - t) <= 1.01 * EPS24 * (3 * np.abs(p) + (0 if residual is None else np.abs(t))))


GEMMS = [(1, 1, 16), (1, 64, 16), (1, 333, 2048), (2, 17, 48), (3, 1000, 4096), (8, 96, 1040), (15, 40, 144),
         (16, 256, 512), (17, 128, 8192), (31, 500, 1008), (33, 257, 272), (40, 5000, 1024), (64, 64, 64),
         (65, 130, 4112), (100, 1024, 128), (128, 300, 16384), (129, 129, 2064), (200, 260, 656), (257, 513, 1024),
         (300, 4100, 256), (512, 512, 512), (700, 1031, 2192), (1025, 2050, 96)]


@pytest.mark.parametrize("m,rows,cols", GEMMS)
@pytest.mark.parametrize("residual", [None, "apart", "in place"])
def test_gemm(hip, m, rows, cols, residual):
    rng = np.random.default_rng(m * 31 + rows * 7 + cols)
    x, w = (rng.integers(-128, 128, s, dtype=np.int8) for s in ((m, cols), (rows, cols)))
    xs, ws = (np.exp(rng.uniform(-8, 2, n)).astype(np.float32) for n in (m, rows))
    r = None if residual is None else (rng.standard_normal((m, rows)) * 100).astype(np.float32)
    _check_gemm(_gemm(hip, x, xs, w, ws, r, residual == "in place"), x, xs, w, ws, r)


def test_gemm_largest_sums(hip):
    """All codes at their ends: sums up to 2^14 * 65536."""
    for m, rows in ((1, 40), (70, 70), (300, 300)):
        x, w = np.full((m, 65536), -128, np.int8), np.full((rows, 65536), -128, np.int8)
        x[::2] = 127
        one = np.ones(max(m, rows), np.float32)
        _check_gemm(_gemm(hip, x, one[:m], w, one[:rows]), x, one[:m], w, one[:rows])


def test_gemm_rows_without_scale(hip):
    """A row quantized from something infinite gives NaN outputs, its neighbours none."""
    rng = np.random.default_rng(3)
    for m in (2, 40, 140):
        x, w = (rng.integers(-127, 128, (n, 256), dtype=np.int8) for n in (m, 150))
        xs, ws = np.ones(m, np.float32), np.ones(150, np.float32)
        xs[1], ws[7] = np.nan, 0
        y = _gemm(hip, x, xs, w, ws)
        assert np.all(np.isnan(y[1])) and np.all(y[0:1, 7] == 0)
        keep = np.arange(m) != 1
        _check_gemm(y[keep], x[keep], xs[keep], w, ws)


def test_rows_of_one_batch_do_not_depend_on_it(hip):
    """A token's codes and products are the same bits alone and among others."""
    rng = np.random.default_rng(9)
    n, rows = 1024, 320
    h, w = rng.standard_normal((600, n)).astype(np.float32), np.ones(n, np.float32)
    q8 = rng.integers(-127, 128, (rows, n), dtype=np.int8)
    dw, dq, ds = hip.to_device(w), hip.to_device(q8), hip.to_device(np.full(rows, 0.01, np.float32))
    found = []
    for count in (600, 90, 20, 1):
        dh = hip.to_device(h[:count])
        q, s, y = hip.alloc(count * n), hip.alloc(count * 4), hip.alloc(count * rows * 4)
        hip.residual_rms_norm_i8(dh.ptr, 0, dw.ptr, 0, q.ptr, s.ptr, count, n, 1e-6)
        hip.gemm_i8(q.ptr, s.ptr, dq.ptr, ds.ptr, y.ptr, count, rows, n)
        found.append((q.readback(np.int8, n), s.readback(np.float32, 1), y.readback(np.float32, rows)))
    for other in found[1:]:
        assert all(np.array_equal(a, b) for a, b in zip(found[0], other))


def test_plans_replay(hip):
    """Recorded, replayed with new contents, eager work in between."""
    rng = np.random.default_rng(11)
    m, n, rows = 37, 512, 190
    w = rng.integers(-127, 128, (rows, n), dtype=np.int8)
    dw, dws = hip.to_device(w), hip.to_device(np.full(rows, 0.01, np.float32))
    dh, dr, dg = hip.alloc(m * n * 4), hip.alloc(m * n * 4), hip.to_device(np.ones(n, np.float32))
    bufs = [[hip.alloc(m * n * 4), hip.alloc(m * n), hip.alloc(m * 4), hip.alloc(m * rows * 4)] for _ in range(2)]

    def body(b):
        hip.residual_rms_norm_i8(dh.ptr, dr.ptr, dg.ptr, b[0].ptr, b[1].ptr, b[2].ptr, m, n, 1e-5)
        hip.gemm_i8(b[1].ptr, b[2].ptr, dw.ptr, dws.ptr, b[3].ptr, m, rows, n)
    plan = hip.record(lambda: body(bufs[0]))
    for turn in range(4):
        dh.upload(rng.standard_normal((m, n)).astype(np.float32))
        dr.upload(rng.standard_normal((m, n)).astype(np.float32))
        plan.launch()
        body(bufs[1])
        a, b = ([x.readback() for x in bs] for bs in bufs)
        assert all(np.array_equal(p, q) for p, q in zip(a, b))
    plan.destroy()


def test_refusals(hip):
    b = hip.alloc(1 << 16)
    p = b.ptr

    def refused(status, call, *args):
        with pytest.raises(native.HipError) as e:
            call(*args)
        assert e.value.status == status, str(e.value)

    arg, uns = native.ERR_ARGUMENT, native.ERR_UNSUPPORTED
    norm = hip.residual_rms_norm_i8
    h, r, w, u, q, s = (p + 4096 * i for i in range(6))
    norm(h, r, w, u, q, s, 2, 64, 1e-5)
    for bad in ((0, r, w, u, q, s, 2, 64, 1e-5), (h, 0, w, u, q, s, 2, 64, 1e-5), (h, r, w, 0, q, s, 2, 64, 1e-5),
                (h, r, 0, u, q, s, 2, 64, 1e-5), (h, r, w, u, 0, s, 2, 64, 1e-5), (h, r, w, u, q, 0, 2, 64, 1e-5),
                (h, r, w, u, q, s, 0, 64, 1e-5), (h, r, w, u, q, s, 2, 0, 1e-5), (h, r, w, u, q, s, (1 << 21) + 1, 64, 1e-5),
                (h, r, w, u, q, s, 2, (1 << 20) + 1, 1e-5), (h, r, w, u, q, s, 2, 64, -1.0),
                (h, r, w, u, q, s, 2, 64, float("nan")), (h, r, w, h, q, s, 2, 64, 1e-5), (h, r, w, u, u + 4, s, 2, 64, 1e-5),
                (h + 2, r, w, u, q, s, 2, 64, 1e-5), (h, r, w, u, q, w, 2, 64, 1e-5)):
        refused(arg, norm, *bad)
    hip.quantize_i8(native.F16, h, q, s, 2, 64)
    refused(uns, hip.quantize_i8, native.Q4_0, h, q, s, 2, 64)
    for bad in ((native.F32, 0, q, s, 2, 64), (native.F16, h + 1, q, s, 2, 64), (native.F32, h, h + 8, s, 2, 64),
                (native.BF16, h, q, s, 2, -1)):
        refused(arg, hip.quantize_i8, *bad)
    for bad in ((0, s, u, 2, 64), (q, s, q, 2, 64), (q, s, u + 2, 2, 64), (q, s, u, 0, 64)):
        refused(arg, hip.dequant_i8, *bad)
    x, xs, w, ws, y = h, r, w, u, q
    hip.gemm_i8(x, xs, w, ws, y, 2, 8, 64)
    hip.gemm_i8(x, xs, w, ws, y, 2, 8, 64, y)
    for bad in ((x, xs, w, ws, y, 2, 8, 60), (x, xs, w, ws, y, 2, 8, 0), (x, xs, w, ws, y, 2, 8, 65552),
                (x, xs, w, ws, y, 0, 8, 64), (x, xs, w, ws, y, 2, 0, 64), (x + 8, xs, w, ws, y, 2, 8, 64),
                (x, xs, w + 4, ws, y, 2, 8, 64), (x, 0, w, ws, y, 2, 8, 64), (x, xs, w, 0, y, 2, 8, 64),
                (x, xs, w, ws, 0, 2, 8, 64), (x, xs, w, ws, x, 2, 8, 64), (x, xs, w, ws, y, 2, 8, 64, y + 4)):
        refused(arg, hip.gemm_i8, *bad)
