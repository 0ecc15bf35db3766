"""The paged cache of many sequences through the C ABI: append with rotary
embedding, rows read back, causal attention, against 64-bit numpy.

Tolerances, by arithmetic.  Append: queries and FP16 / 4-bit rows are one
rounding of 64-bit values, so they equal the reference's bits.  Attention:
with h = 2^-11 (half an FP16 step), a score is a sum of products of a query
value and a cached value, each rounded once, so it is off by at most 2 h x
slack, slack = sum |q| |k| / sqrt(d); weights then by a factor exp(+-2 h
slack) in numerator and denominator, and once h for their own rounding and
once h for the value's: |error| <= (exp(4 h slack) - 1 + 2 h) * (weighted
mean of |v|), plus half a step of the output, plus 1e-5 of the mean for FP32
sums and exponentials.  Over a whole output the roundings average out: its
norm is off by no more than half a step of the output and 6 h.  Outputs of
F16 and F32 come of two-term operands: h = 2^-18 stands for their 2^-22, the
terms' floor of 2^-25 and FP32 sums of up to 128 products.
"""
import itertools

import numpy as np
import pytest

from sharpinference_amd import native
from tests import paged_reference as ref

F32, F16, BF16, Q4 = native.F32, native.F16, native.BF16, native.Q4_0
gpu = pytest.mark.gpu
SENTINEL = 0x7B


@pytest.mark.parametrize("fmt,page,head,want", [(F16, 16, 64, 2048), (F16, 256, 128, 65536), (Q4, 16, 64, 576),
                                                (Q4, 64, 128, 4608)])
def test_page_bytes(fmt, page, head, want):
    assert native.paged_page_bytes(fmt, page, head) == want


def test_sizes_refused_without_a_device():
    for bad, status in (((native.F32, 16, 64), native.ERR_UNSUPPORTED), ((F16, 16, 96), native.ERR_UNSUPPORTED),
                        ((F16, 24, 64), native.ERR_ARGUMENT), ((F16, 8, 64), native.ERR_ARGUMENT),
                        ((Q4, 512, 64), native.ERR_ARGUMENT)):
        with pytest.raises(native.HipError) as e:
            native.paged_page_bytes(*bad)
        assert e.value.status == status
    assert native.paged_attention_workspace_bytes(24, 8, 128) > 0
    for bad, status in (((24, 8, 256), native.ERR_UNSUPPORTED), ((7, 2, 64), native.ERR_ARGUMENT),
                        ((34, 2, 64), native.ERR_ARGUMENT), ((0, 2, 64), native.ERR_ARGUMENT),
                        ((4, 0, 64), native.ERR_ARGUMENT)):
        with pytest.raises(native.HipError) as e:
            native.paged_attention_workspace_bytes(*bad)
        assert e.value.status == status
    lib = native.lib()
    for name in ("si_hip_paged_kv_append", "si_hip_paged_attention"):
        assert getattr(lib, name)(None, None) == native.ERR_ARGUMENT
    assert lib.si_hip_paged_kv_read(None, None, None, None, None) == native.ERR_ARGUMENT
    for call in (lambda: lib.si_hip_gemm_i8(None, None, None, None, None, None, 1, 1, 16, None),
                 lambda: lib.si_hip_quantize_i8(None, F16, None, None, None, 1, 1),
                 lambda: lib.si_hip_dequant_i8(None, None, None, None, 1, 1),
                 lambda: lib.si_hip_residual_rms_norm_i8(None, None, None, None, None, None, None, 1, 1, 0.0)):
        assert call() == native.ERR_ARGUMENT


class Setup:
    """Pools, tables and a batch: `seqs` is a list of (new rows, length)."""

    def __init__(self, hip, fmt, head, kv, page, seqs, seed=0, spare_rows=2, extra_pages=2):
        self.hip, self.fmt, self.d, self.kv, self.ps, self.seqs = hip, fmt, head, kv, page, seqs
        rng = self.rng = np.random.default_rng(seed)
        held = [-(-max(l, 0) // page) for _, l in seqs]
        self.pages = max(1, sum(held) + extra_pages)
        order = rng.permutation(self.pages)
        # what lies behind a sequence's end in the table is not looked at
        self.table = rng.choice(np.array([-1, 2 ** 31 - 1, -2 ** 31, 12345678]), (len(seqs), max(max(held), 1) + 1))
        self.table = self.table.astype(np.int32)
        at = 0
        for s, n in enumerate(held):
            self.table[s, :n] = order[at:at + n]
            at += n
        self.starts = np.concatenate([[0], np.cumsum([n for n, _ in seqs])]).astype(np.int32)
        self.lengths = np.array([l for _, l in seqs], np.int32)
        self.used = int(self.starts[-1])
        self.rows = max(1, self.used + spare_rows)
        self.most = max(1, max(n for n, _ in seqs))
        self.k = ref.Pool(fmt, self.pages, kv, page, head, rng)
        self.v = ref.Pool(fmt, self.pages, kv, page, head, rng)

    def fill(self, sigma_k=1.0, sigma_v=1.0):
        """Random rows at every place that a sequence holds; what is left stays stale."""
        for s, (_, length) in enumerate(self.seqs):
            for p in range(max(0, length)):
                page = int(self.table[s, p // self.ps])
                for pool, sigma in ((self.k, sigma_k), (self.v, sigma_v)):
                    pool.store(page, p % self.ps, (sigma * self.rng.standard_normal((self.kv, self.d))).astype(np.float32))
        return self

    def upload(self):
        up = self.hip.to_device
        self.dev = [up(self.table), up(self.starts), up(self.lengths), up(self.k.raw), up(self.v.raw)]
        t, st, ln, k, v = (b.ptr for b in self.dev)
        self.batch = native.PagedBatch(t, st, ln, len(self.seqs), self.table.shape[1], self.rows, self.most)
        self.cache = native.PagedCache(k, v, self.pages, self.ps, self.kv, self.d, self.fmt)
        return self

    def rows_of(self, s, upto):
        """[positions, kv, d] keys and values of sequence s."""
        get = lambda pool: np.stack([pool.load(int(self.table[s, p // self.ps]), p % self.ps) for p in range(upto)]) \
            if upto > 0 else np.zeros((0, self.kv, self.d))
        return get(self.k), get(self.v)


# ---- append and read -----------------------------------------------------------------------

APPENDS = [
    # fmt, head, heads, kv, page, rotary, [(new, length)]
    (Q4, 128, 3, 1, 16, 96, [(1, 1)]),
    (Q4, 64, 8, 8, 32, 64, [(5, 5), (0, 7), (1, 40), (33, 65)]),
    (F16, 128, 24, 8, 64, 128, [(1, 64), (1, 65), (1, 1), (0, 0), (130, 200)]),
    (F16, 64, 5, 1, 16, 0, [(17, 17)]),
    (Q4, 128, 16, 2, 128, 2, [(3, 129), (2, 128)]),
    (Q4, 64, 3, 3, 256, 42, [(7, 300)]),
    (Q4, 64, 48, 3, 64, 22, [(2, 70001), (1, 64)]),
]


def _append(hip, st, heads, rotary, qkv, freq, scale, query=None):
    query = query or hip.to_device(np.full(st.rows * heads * st.d * 4, SENTINEL, np.uint8))
    dq, df = hip.to_device(qkv), hip.to_device(freq if freq.size else np.zeros(1, np.float32))
    hip.paged_kv_append(native.PagedAppendArgs(st.batch, st.cache, dq.ptr, df.ptr, query.ptr, heads, rotary, scale))
    return query


def _expect_append(st, heads, rotary, qkv, freq, scale):
    """The pools and queries as they have to be afterwards."""
    q = np.full((st.rows, heads * st.d), SENTINEL * 0x01010101, np.uint32).view(np.float32)
    for t in range(st.rows):
        s, p, page = ref.place(st.table, st.starts, st.lengths, st.ps, st.pages, t)
        if page is None:
            continue
        x = qkv[t].reshape(-1, st.d)
        turned = ref.rotate(x[:heads + st.kv], p, freq, rotary, scale)
        q[t] = turned[:heads].reshape(-1)
        st.k.store(page, p % st.ps, turned[heads:])
        st.v.store(page, p % st.ps, x[heads + st.kv:])
    return q


def _same(a, b):
    return np.array_equal(a.view(np.uint8), b.view(np.uint8))


@gpu
@pytest.mark.parametrize("fmt,head,heads,kv,page,rotary,seqs", APPENDS)
def test_append_and_read(hip, fmt, head, heads, kv, page, rotary, seqs):
    st = Setup(hip, fmt, head, kv, page, seqs, seed=len(seqs)).upload()
    qkv = st.rng.standard_normal((st.rows, (heads + 2 * kv) * head)).astype(np.float32)
    qkv[0, heads * head:heads * head + 32] = 0                       # a block of zeros
    qkv[0, -32:] = 2.0 ** -8                                         # equals: the first one's sign
    qkv[0, -1] = -2.0 ** -8
    freq = (10000.0 ** (-2.0 * np.arange(rotary // 2) / max(rotary, 1))).astype(np.float32)
    query = _append(hip, st, heads, rotary, qkv, freq, 1.19)
    want = _expect_append(st, heads, rotary, qkv, freq, 1.19)
    got = query.readback(np.float32).reshape(want.shape)
    assert _same(got, want)
    for b, pool in zip(st.dev[3:], (st.k, st.v)):
        assert np.array_equal(b.readback(np.uint8), pool.raw.reshape(-1))
    # and back as values: the batch's rows alone are written
    keys, vals = (hip.to_device(np.full(st.rows * kv * head * 4, SENTINEL, np.uint8)) for _ in range(2))
    hip.paged_kv_read(st.batch, st.cache, keys.ptr, vals.ptr)
    for b, pool in ((keys, st.k), (vals, st.v)):
        rows = b.readback(np.float32).reshape(st.rows, kv, head)
        for t in range(st.rows):
            _, p, page_at = ref.place(st.table, st.starts, st.lengths, st.ps, st.pages, t)
            if page_at is None:
                assert np.all(rows[t].view(np.uint8) == SENTINEL)
            else:
                assert np.array_equal(rows[t], pool.load(page_at, p % st.ps).astype(np.float32))


@gpu
@pytest.mark.parametrize("fmt,head,rotary", [(Q4, 128, 96), (F16, 64, 64), (Q4, 64, 6)])
def test_append_and_read_at_any_word(hip, fmt, head, rotary):
    """Rows that begin at any multiple of four bytes."""
    heads, kv = 3, 1
    st = Setup(hip, fmt, head, kv, 16, [(5, 20), (1, 3)], seed=rotary).upload()
    qkv = st.rng.standard_normal((st.rows, (heads + 2 * kv) * head)).astype(np.float32)
    freq = (0.4 ** np.arange(rotary // 2)).astype(np.float32)
    want = _expect_append(st, heads, rotary, qkv, freq, 1.0)
    for off in (1, 2, 3):
        dq = hip.to_device(np.concatenate([np.zeros(off, np.float32), qkv.reshape(-1)]))
        df = hip.to_device(np.concatenate([np.zeros(off, np.float32), freq]))
        query, keys = (hip.to_device(np.full((st.rows * n * head + off) * 4, SENTINEL, np.uint8)) for n in (heads, kv))
        vals = hip.to_device(np.zeros(st.rows * kv * head + off, np.float32))
        hip.paged_kv_append(native.PagedAppendArgs(st.batch, st.cache, dq.ptr + 4 * off, df.ptr + 4 * off,
                                                   query.ptr + 4 * off, heads, rotary, 1.0))
        assert _same(query.readback(np.float32)[off:].reshape(want.shape), want)
        for b, pool in zip(st.dev[3:], (st.k, st.v)):
            assert np.array_equal(b.readback(np.uint8), pool.raw.reshape(-1))
        hip.paged_kv_read(st.batch, st.cache, keys.ptr + 4 * off, vals.ptr + 4 * off)
        rows = keys.readback(np.float32)[off:].reshape(st.rows, kv, head)
        for t in range(st.used):
            _, p, page = ref.place(st.table, st.starts, st.lengths, 16, st.pages, t)
            assert np.array_equal(rows[t], st.k.load(page, p % 16).astype(np.float32))


@gpu
def test_append_many_rows(hip):
    """Enough rows for whole rows a workgroup, and more sequences than threads."""
    seqs = [(2, 2 + 3 * (i % 5)) for i in range(300)]
    st = Setup(hip, Q4, 64, 2, 16, seqs, seed=4).upload()
    qkv = st.rng.standard_normal((st.rows, 8 * 64)).astype(np.float32)
    freq = (0.3 ** np.arange(16)).astype(np.float32)
    query = _append(hip, st, 4, 32, qkv, freq, 1.0)
    want = _expect_append(st, 4, 32, qkv, freq, 1.0)
    assert _same(query.readback(np.float32).reshape(want.shape), want)
    assert np.array_equal(st.dev[3].readback(np.uint8), st.k.raw.reshape(-1))
    assert np.array_equal(st.dev[4].readback(np.uint8), st.v.raw.reshape(-1))


@gpu
@pytest.mark.parametrize("fmt", [F16, Q4])
def test_append_special_values(hip, fmt):
    """What FP16 cannot hold: infinities (FP16 pages), NaN blocks (4-bit pages)."""
    st = Setup(hip, fmt, 128, 1, 16, [(6, 6)], spare_rows=0).upload()
    qkv = st.rng.standard_normal((6, 3 * 128)).astype(np.float32)
    qkv[0, 300], qkv[1, 301], qkv[2, 302] = np.inf, np.nan, -70000
    qkv[3, 256:288] = 65504
    qkv[4, 256:288] *= 1e-8
    qkv[5, 256:288] *= 1e-5
    _append(hip, st, 1, 0, qkv, np.zeros(0, np.float32), 1.0)
    _expect_append(st, 1, 0, qkv, np.zeros(0, np.float32), 1.0)
    keys, vals = hip.alloc(6 * 512), hip.alloc(6 * 512)
    hip.paged_kv_read(st.batch, st.cache, keys.ptr, vals.ptr)
    got = vals.readback(np.float32).reshape(6, 128)
    want = np.stack([st.v.load(int(st.table[0, 0]), p)[0] for p in range(6)]).astype(np.float32)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(got[~np.isnan(got)], want[~np.isnan(want)])
    if fmt == Q4:
        assert np.all(np.isnan(got[0, 32:64])) and np.all(np.isnan(got[1, 32:64])) and np.all(np.isnan(got[2, 32:64]))
        assert np.all(np.isfinite(got[3:])) and np.all(got[3, :32] == 65504)


@gpu
def test_append_rows_without_a_place(hip):
    """Positions before 0 or behind the table, pages outside the pool: nothing is written."""
    st = Setup(hip, Q4, 64, 2, 16, [(3, 2), (2, 20), (2, 40), (2, 5)], seed=8)
    st.lengths[1] = 16 * st.table.shape[1] + 1          # its last row lies behind the table
    st.table[1, :] = st.table[1, 0]
    st.table[2, 2] = st.pages                           # rows 38, 39
    st.table[3, 0] = -1
    st.upload()
    qkv = st.rng.standard_normal((st.rows, 6 * 64)).astype(np.float32)
    freq = np.ones(4, np.float32)
    query = _append(hip, st, 2, 8, qkv, freq, 1.0)
    want = _expect_append(st, 2, 8, qkv, freq, 1.0)
    assert _same(query.readback(np.float32).reshape(want.shape), want)
    assert np.array_equal(st.dev[3].readback(np.uint8), st.k.raw.reshape(-1))
    keys, vals = (hip.to_device(np.zeros(st.rows * 128, np.float32)) for _ in range(2))
    hip.paged_kv_read(st.batch, st.cache, keys.ptr, vals.ptr)
    rows = keys.readback(np.float32).reshape(st.rows, 128)
    lost = [t for t in range(st.used) if ref.place(st.table, st.starts, st.lengths, 16, st.pages, t)[2] is None]
    assert lost == [0, 4, 5, 6, 7, 8] and np.all(np.isnan(rows[lost])) and np.all(rows[st.used:] == 0)
    assert np.all(np.isfinite(rows[[1, 2, 3]]))


# ---- attention -------------------------------------------------------------------------------

def _attend(hip, st, heads, q, out_fmt=BF16, ws_fill=0xFF):
    """Output [rows, heads, d] in 64 bits; the workspace starts with NaN in it."""
    wide = out_fmt == F32
    nbytes = st.rows * heads * st.d * (4 if wide else 2)
    out = hip.to_device(np.full(nbytes + 64, SENTINEL, np.uint8))
    dq = hip.to_device(q)
    size = native.paged_attention_workspace_bytes(heads, st.kv, st.d)
    ws = hip.alloc(size + 64)
    hip.fill_u32(ws.ptr, ws_fill * 0x01010101, size // 4 + 16)
    hip.paged_attention(native.PagedAttentionArgs(st.batch, st.cache, dq.ptr, out.ptr, ws.ptr, heads, out_fmt))
    assert np.all(ws.readback(np.uint8, 64, size) == ws_fill)
    raw = out.readback(np.uint8)
    assert np.all(raw[nbytes:] == SENTINEL)
    u = raw[:nbytes].view(np.uint32 if wide else np.uint16).reshape(st.rows, heads, st.d)
    assert np.all(u[st.used:] == SENTINEL * (0x01010101 if wide else 0x0101)), "rows behind the last sequence"
    if wide:
        return u.view(np.float32).astype(np.float64)
    if out_fmt == F16:
        return u.view(np.float16).astype(np.float64)
    return (u.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def _check_rows(st, heads, q, got, out_fmt, rows=None):
    half_out = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}[out_fmt]
    # (FP16 outputs among the subnormals have a step of their own)
    floor = 2.0 ** -25 if out_fmt == F16 else 0.0
    h = 2.0 ** -11 if out_fmt == BF16 else 2.0 ** -18
    err2 = norm2 = 0.0
    for s, (new, length) in enumerate(st.seqs):
        if rows is not None and not set(rows) & set(range(st.starts[s], st.starts[s + 1])):
            continue
        keys, values = st.rows_of(s, length)
        for i in range(new):
            t = st.starts[s] + i
            if rows is not None and t not in rows:
                continue
            want, mag, slack = ref.attention(q[t].reshape(heads, st.d), keys, values, length - new + i + 1)
            bound = (np.expm1(4 * h * slack)[:, None] + 2 * h + 1e-5) * mag * (1 + half_out) + half_out * np.abs(want) + floor
            assert np.all(np.abs(got[t] - want) <= bound), (s, i, np.max(np.abs(got[t] - want) / (bound + 1e-300)))
            err2 += np.sum((got[t] - want) ** 2)
            norm2 += np.sum(want ** 2)
    assert np.sqrt(err2) <= (half_out + 6 * h) * np.sqrt(norm2) + 1e-12


ATTENDS = [
    # head, heads, kv, page, [(new, length)]
    (128, 1, 1, 16, [(1, 1)]),
    (128, 24, 8, 64, [(1, 1), (1, 63), (1, 64), (1, 65), (1, 200), (0, 30), (1, 16)]),
    (64, 32, 4, 16, [(3, 3), (5, 300), (1, 129), (2, 17)]),
    (64, 16, 1, 32, [(1, 257), (1, 31)]),
    (128, 7, 7, 128, [(2, 130), (9, 9), (17, 33)]),
    (128, 6, 2, 256, [(40, 40), (33, 290), (1, 5)]),
    (64, 10, 2, 64, [(100, 100), (1, 1), (70, 200), (0, 0)]),
    (128, 16, 2, 32, [(150, 150), (1, 700), (130, 400)]),
    (128, 3, 1, 64, [(5, 3), (2, 0), (4, 4), (20, 7)]),          # more rows than positions: the first see nothing
    (64, 4, 4, 16, [(1, 1500)]),
    (128, 8, 2, 16, [(1, 2100), (3, 1000)]),
    (64, 12, 4, 128, [(300, 555)]),
]


@gpu
@pytest.mark.parametrize("head,heads,kv,page,seqs", ATTENDS)
@pytest.mark.parametrize("fmt,out_fmt", [(Q4, BF16), (F16, F16), (Q4, F32), (F16, BF16)])
def test_attention(hip, fmt, out_fmt, head, heads, kv, page, seqs):
    st = Setup(hip, fmt, head, kv, page, seqs, seed=heads).fill().upload()
    q = st.rng.standard_normal((st.rows, heads * head)).astype(np.float32)
    got = _attend(hip, st, heads, q, out_fmt)
    _check_rows(st, heads, q, got, out_fmt)
    for s, (new, length) in enumerate(seqs):
        for i in range(max(0, new - length)):
            assert np.all(got[st.starts[s] + i] == 0)


@gpu
@pytest.mark.parametrize("fmt", [F16, Q4])
def test_attention_sharp_and_flat(hip, fmt):
    """Scores that differ by hundreds, and scores that are all equal; large and tiny values."""
    for qs, vs in ((60.0, 1.0), (0.0, 1.0), (1.0, 3000.0), (1.0, 2e-4)):
        st = Setup(hip, fmt, 128, 2, 64, [(1, 333), (20, 150)], seed=3).fill(1.0, vs).upload()
        q = (qs * st.rng.standard_normal((st.rows, 6 * 128))).astype(np.float32)
        # (scores of hundreds are off by more than the weights' own size: only the element bound holds them)
        got = _attend(hip, st, 6, q, BF16)
        if qs < 50:
            _check_rows(st, 6, q, got, BF16)
        else:
            assert np.all(np.isfinite(got[:st.used]))
            for s, (new, length) in enumerate(st.seqs):
                keys, values = st.rows_of(s, length)
                for i in range(new):
                    t, n = st.starts[s] + i, length - new + i + 1
                    want, mag, slack = ref.attention(q[t].reshape(6, 128), keys, values, n)
                    bound = np.minimum(np.expm1(4 * 2.0 ** -11 * slack), 2 * 1e3)[:, None] * mag + 2.0 ** -8 * np.abs(want) + 2e-3 * mag
                    assert np.all(np.abs(got[t] - want) <= bound)


@gpu
@pytest.mark.parametrize("course", ["flat", "rising", "falling"])
@pytest.mark.parametrize("sign", [-1, 1])
@pytest.mark.parametrize("fmt,out_fmt", [(F16, F32), (Q4, BF16)])
def test_attention_far_from_zero(hip, fmt, out_fmt, sign, course):
    """Scores around -300 or 300, all alike or on their way there: what they are
    taken relative to starts far from 0, or moves many times."""
    d, heads, kv = 128, 6, 2
    st = Setup(hip, fmt, d, kv, 32, [(1, 333), (5, 200), (90, 333), (150, 150)], seed=27)
    flips = st.rng.choice([-1.0, 1.0], d)
    for s, (_, length) in enumerate(st.seqs):
        for p in range(length):
            part = {"flat": 1.0, "rising": p / length, "falling": 1 - p / length}[course]
            k = 2 * part * flips + 0.1 * st.rng.standard_normal((kv, d))
            page = int(st.table[s, p // 32])
            st.k.store(page, p % 32, k.astype(np.float32))
            st.v.store(page, p % 32, st.rng.standard_normal((kv, d)).astype(np.float32))
    st.upload()
    q = (sign * 13.3 * np.tile(flips, heads) + 0.5 * st.rng.standard_normal((st.rows, heads * d))).astype(np.float32)
    got = _attend(hip, st, heads, q, out_fmt)
    # (scores of hundreds: the element bound alone, as their roundings do not average out over few weights)
    h, half_out = (2.0 ** -11, 2.0 ** -8) if out_fmt == BF16 else (2.0 ** -18, 2.0 ** -24)
    for s, (new, length) in enumerate(st.seqs):
        keys, values = st.rows_of(s, length)
        for i in range(new):
            t = st.starts[s] + i
            want, mag, slack = ref.attention(q[t].reshape(heads, d), keys, values, length - new + i + 1)
            bound = (np.expm1(4 * h * slack)[:, None] + 2 * h + 1e-5) * mag * (1 + half_out) + half_out * np.abs(want)
            assert np.all(np.abs(got[t] - want) <= bound), (s, i, np.max(np.abs(got[t] - want) / bound))


COURSES = ["flat", "rising", "falling", "steps"]


def _exact_operands(hip, fmt, course, sign):
    """A batch whose operands are exact in FP16: scores around +-300 (in units of log 2), all alike
    or on their way there.  Queries times log2(e) / sqrt(d) are +-1 or +-1/2, to FP32's two
    roundings; three quarters of a key are a multiple of 1/64 whose sign follows the query's, the
    last one small random multiples of 1/64; values are whole."""
    d, heads, kv, page = 128, 6, 2, 32
    st = Setup(hip, fmt, d, kv, page, [(1, 333), (5, 200), (90, 333), (150, 150)], seed=53)
    rng = st.rng
    flips = rng.choice([-1, 1], d)
    for s, (_, length) in enumerate(st.seqs):
        for p in range(length):
            share = {"flat": 1.0, "rising": p / length, "falling": 1 - p / length, "steps": 0.5 + 0.05 * (p // 23 % 10)}[course]
            codes = np.tile(flips, (kv, 1))
            codes[:, 96:] = rng.integers(-7, 8, (kv, 32))
            scales = np.full(4, round(200 * share) / 64.0)       # 96 products of up to 3.125: 300
            scales[3] = 1 / 64
            values = rng.integers(-7, 8, (kv, d))
            at, slot = int(st.table[s, p // page]), p % page
            for pool, c, b in ((st.k, codes, scales), (st.v, values, np.ones(4))):
                if fmt == F16:
                    pool.values_view()[at, :, slot] = c * np.repeat(b, 32)
                    continue
                pool.nibble_view()[at, :, slot] = (c + 8)[:, 0::2] | (c + 8)[:, 1::2] << 4
                for h, i in itertools.product(range(kv), range(4)):
                    pool.put_scale(at, h, i, slot, b[i])
    q = np.tile(sign * flips, (st.rows, heads, 1)).astype(np.float64)
    q[:, :, 96:] = rng.choice([-1, -0.5, 0.5, 1], (st.rows, heads, 32))
    return st, heads, (q * np.sqrt(d) * np.log(2)).astype(np.float32).reshape(st.rows, -1)


def _exact_rows(st, heads, q, out_fmt, rescaled=True):
    """(want, bound) of all rows.  What is left of the errors where the operands are exact: the
    query's two FP32 roundings and a score's (2^-22 of sum |q| |k| / sqrt(d)), in numerator and
    sum; the weights' half step of FP16 (2^-22 in two terms), twice; FP32 sums of chains of less
    than 100; the output's half step.  Not `rescaled`: as if sums and accumulators stayed as they
    are when a later unit of 64 positions brings a larger maximum."""
    half_out, weight = (2.0 ** -8, 2.0 ** -11) if out_fmt == BF16 else (2.0 ** -24, 2.0 ** -22)
    wants, bounds = np.zeros((st.used, heads, st.d)), np.zeros((st.used, heads, st.d))
    for s, (new, length) in enumerate(st.seqs):
        keys, values = st.rows_of(s, length)
        for i in range(new):
            t, n = st.starts[s] + i, length - new + i + 1
            x = q[t].reshape(heads, st.d)
            want, mag, slack = ref.attention(x, keys, values, n)
            rel = np.expm1(2 * 2.0 ** -22 * slack)[:, None] + 2 * weight + 100 * 2.0 ** -24
            bounds[t] = rel * mag * (1 + half_out) + half_out * np.abs(want)
            if not rescaled:
                for h in range(heads):
                    score = keys[:n, h * st.kv // heads] @ x[h].astype(np.float64) / np.sqrt(st.d)
                    top = np.maximum.accumulate([score[u:u + 64].max() for u in range(0, n, 64)])
                    p = np.exp(score - np.repeat(top, 64)[:n])
                    want[h] = p @ values[:n, h * st.kv // heads] / p.sum()
            wants[t] = want
    return wants, bounds


@pytest.mark.parametrize("course", COURSES)
@pytest.mark.parametrize("sign", [-1, 1])
def test_bounds_of_exact_operands_hold_what_they_say(course, sign):
    """The bound of the next test passes neither zeros nor outputs whose rescaling was left out."""
    st, heads, q = _exact_operands(None, Q4, course, sign)
    want, bound = _exact_rows(st, heads, q, BF16)
    assert np.mean(np.abs(want) <= bound) < 0.02
    if (course, sign) in (("steps", 1), ("rising", 1), ("falling", -1)):      # maxima that grow a lot
        wrong = _exact_rows(st, heads, q, BF16, rescaled=False)[0]
        for s, (new, length) in enumerate(st.seqs):
            rows = slice(st.starts[s + 1] - 1, st.starts[s + 1])      # its last row: sees every unit
            assert np.mean(np.abs(wrong[rows] - want[rows]) > bound[rows]) > 0.1


@gpu
@pytest.mark.parametrize("course", COURSES)
@pytest.mark.parametrize("sign", [-1, 1])
@pytest.mark.parametrize("fmt,out_fmt", [(Q4, BF16), (F16, BF16), (F16, F32), (Q4, F32)])
def test_attention_of_exact_operands(hip, fmt, out_fmt, sign, course):
    """Scores far from 0 whose reference starts there or moves many times, within a few steps of the output."""
    st, heads, q = _exact_operands(hip, fmt, course, sign)
    st.upload()
    want, bound = _exact_rows(st, heads, q, out_fmt)
    off = np.abs(_attend(hip, st, heads, q, out_fmt)[:st.used] - want)
    assert np.all(off <= bound), np.max(off / bound)
    # over the whole output the roundings average out
    half_out, weight = (2.0 ** -8, 2.0 ** -11) if out_fmt == BF16 else (2.0 ** -24, 2.0 ** -18)
    assert np.linalg.norm(off) <= (half_out + 6 * weight) * np.linalg.norm(want)


@gpu
@pytest.mark.parametrize("new,at,count", [(1, 0, 1), (1, 0, 64), (1, -1, 64), (9, 4321, 64), (100, 0, 1), (100, 0, 32),
                                          (100, -1, 32)])
@pytest.mark.parametrize("fmt,out_fmt", [(Q4, BF16), (F16, BF16), (F16, F32), (Q4, F32)])
@pytest.mark.parametrize("head", [64, 128])
def test_weights_far_below_the_largest(hip, fmt, out_fmt, head, new, at, count):
    """One position far above 40000 alike ones, which hold a share of the sum all the
    same; one sequence, cut into short runs, and many (of the same pages), whose runs are long.

    Every operand is exact in FP16: the query times log2(e) / sqrt(d) is a number
    of at most ten bits (to FP32's two roundings), keys are 0 or 1 and values whole.
    What is left are the weights: half an FP16 step of themselves (twice, in
    numerator and sum; 2^-22 in two terms) and half FP16's smallest step, which
    is at most 2^-32 of the row's largest (2^-38 in two terms); FP32 sums; and the
    output's.  An FP32 sum is off by half a step, 2^-24 of the sum, for each addition
    that it is a chain of: at most 625 units' weights and as many joined runs, and in an
    accumulator 625 units' products, four each (of 16 positions) for one, two or three
    pairs of terms.
    """
    heads, kv, length, page = 16, 8, 40000 + new, 256
    st = Setup(hip, fmt, head, kv, page, [(new, length)], seed=43, spare_rows=0)
    columns = np.arange(head) % 13 - 6
    top = at if at >= 0 else length - new                  # seen by all rows
    top_page, slot = int(st.table[0, top // page]), top % page
    for pool, rest, one in ((st.k, np.zeros(head, np.int64), np.ones(head, np.int64)),
                            (st.v, columns, np.zeros(head, np.int64))):
        if fmt == F16:
            pool.values_view()[:], pool.values_view()[top_page, :, slot] = rest, one
        else:
            pool.raw[:, :, page * head // 2:] = np.tile(np.frombuffer(np.float16(1).tobytes(), np.uint8), page * head // 32)
            pool.nibble_view()[:] = (rest + 8)[0::2] | (rest + 8)[1::2] << 4
            pool.nibble_view()[top_page, :, slot] = (one + 8)[0::2] | (one + 8)[1::2] << 4
    st.seqs, st.table, st.lengths = st.seqs * count, np.repeat(st.table, count, 0), np.repeat(st.lengths, count)
    st.starts = (new * np.arange(count + 1)).astype(np.int32)
    st.used = st.rows = new * count
    st.upload()
    half_out, weight, floor = (2.0 ** -8, 2.0 ** -11, 2.0 ** -32) if out_fmt == BF16 else (2.0 ** -24, 2.0 ** -22, 2.0 ** -38)
    chain = 2 * 625 + 625 * 4 * (1 if out_fmt == BF16 else 3 if fmt == Q4 else 2)
    others = np.tile(length - new + np.arange(new), count)
    for far in (14.03125, 20.03125, 22.6875, 25.1875):      # in units of log 2
        q = np.full((st.rows, heads * head), far / head * np.sqrt(head) * np.log(2), np.float32)
        w = np.exp(-q[0, 0].astype(np.float64) * np.sqrt(head))
        share = others * w / (1 + others * w)
        want = share[:, None, None] * columns
        rel = np.expm1(far * 2.0 ** -21) + 2 * weight + chain * 2.0 ** -24
        bound = rel * np.abs(want) + (2 * floor * others / (1 + others * w))[:, None, None] * np.abs(columns)
        bound = bound * (1 + half_out) + half_out * np.abs(want)
        off = np.abs(_attend(hip, st, heads, q, out_fmt) - want)
        worst = float(np.max((off / share[:, None, None])[..., columns != 0] / np.abs(columns[columns != 0])))
        inside = bool(np.all(off <= bound))
        assert inside, (far, worst)


@gpu
@pytest.mark.parametrize("new", [1, 100])
@pytest.mark.parametrize("fmt,out_fmt", [(Q4, BF16), (F16, BF16), (F16, F32), (Q4, F32)])
def test_scores_with_coarse_steps(hip, fmt, out_fmt, new):
    """Scores of 2^25 to 2^28, whose FP32 steps are 2 to 16: what lies a little below the
    largest rounds to it, or to a whole step further down.  Two positions of the same
    key share the sum, all else is nothing beside them: their values' mean (whole and
    half numbers), 2^-20 for exponentials, the reciprocal and its product."""
    head, heads, length, page = 64, 2, 300 + new, 64
    st = Setup(hip, fmt, head, 1, page, [(new, length)], seed=47, spare_rows=0)
    for p in (37, 290):
        assert p < length - new
    values = np.stack([np.arange(head) % 15 - 7, np.arange(head) % 11 - 5])
    half_out = 2.0 ** -8 if out_fmt == BF16 else 2.0 ** -24
    for size, odd in itertools.product((64, 128, 256, 512), (1, 3, 5, 7)):
        key = np.ones(head, np.int64)
        key[63] = odd
        for pool, rows, scale in ((st.k, [key, key], size), (st.v, values, 1)):
            if fmt == F16:
                pool.values_view()[:] = 0
            else:
                pool.nibble_view()[:] = 0x88
                pool.raw[:, :, page * head // 2:] = np.tile(np.frombuffer(np.float16(scale).tobytes(), np.uint8), page * head // 32)
            for p, row in zip((37, 290), rows):
                at = int(st.table[0, p // page]), slice(None), p % page
                if fmt == F16:
                    pool.values_view()[at] = row * scale
                else:
                    pool.nibble_view()[at] = (row + 8)[0::2] | (row + 8)[1::2] << 4
        st.upload()
        t = np.full(head, 8192.0)
        t[63] = 2.0 ** -5
        q = np.tile((t * np.sqrt(head) * np.log(2)).astype(np.float32), (st.rows, heads))
        got = _attend(hip, st, heads, q, out_fmt)
        want = values.mean(0)
        off = np.abs(got - want)
        assert np.all(off <= (2.0 ** -20 + half_out * (1 + 2.0 ** -20)) * np.abs(want)), (size, odd)


@gpu
@pytest.mark.parametrize("fmt,out_fmt", [(Q4, BF16), (F16, F32)])
@pytest.mark.parametrize("head,heads,kv,page,seqs", [
    (64, 16, 16, 16, [(70 + i, 70 + i + 41 * (i % 3)) for i in range(16)]),     # as many tiles as workgroups
    (64, 32, 16, 32, [(65, 900), (33, 64), (1, 500), (260, 300), (65, 65), (40, 1000)] * 2),
    (128, 6, 2, 64, [(90, 3001)]),                                              # one tile in many parts
    (128, 5, 1, 16, [(120, 130), (1, 2000), (13, 1500)]),
])
def test_attention_shared_out(hip, fmt, out_fmt, head, heads, kv, page, seqs):
    """Tiles that several workgroups share, borders anywhere, decode beside prompts."""
    st = Setup(hip, fmt, head, kv, page, seqs, seed=len(seqs)).fill().upload()
    q = st.rng.standard_normal((st.rows, heads * head)).astype(np.float32)
    got = _attend(hip, st, heads, q, out_fmt)
    pick = st.rng.choice(st.used, min(st.used, 160), replace=False)
    _check_rows(st, heads, q, got, out_fmt, set(int(t) for t in pick))
    assert np.all(np.isfinite(got[:st.used]))


@gpu
@pytest.mark.parametrize("new,length", [(1, 70), (6, 70), (40, 150), (200, 333)])
@pytest.mark.parametrize("fmt", [F16, Q4])
def test_hidden_positions_change_nothing(hip, fmt, new, length):
    """Stale rows of any bytes behind the end, and later positions that hold NaN."""
    heads = 4
    outs = []
    for turn in range(2):
        st = Setup(hip, fmt, 128, 2, 64, [(new, length), (new, length)], seed=21).fill()
        q = st.rng.standard_normal((st.rows, heads * 128)).astype(np.float32)
        if turn:
            # NaN from the middle of the new rows on: rows before it are the same bits as without
            hole = length - new + new // 2
            for p in range(hole, length):
                for pool in (st.k, st.v):
                    page = int(st.table[0, p // 64])
                    if fmt == F16:
                        pool.raw.view(np.float16).reshape(pool.pages, 2, 64, 128)[page, :, p % 64] = np.nan
                    else:
                        for h, b in itertools.product(range(2), range(4)):
                            pool.put_scale(page, h, b, p % 64, np.nan)
        st.upload()
        outs.append(_attend(hip, st, heads, q, BF16))
    before = new // 2
    assert np.array_equal(outs[0][:before], outs[1][:before])
    assert np.all(np.isnan(outs[1][before:new])) and np.all(np.isfinite(outs[0][:2 * new]))
    assert np.array_equal(outs[0][new:2 * new], outs[1][new:2 * new])


@gpu
@pytest.mark.parametrize("fmt", [F16, Q4])
@pytest.mark.parametrize("new", [1, 3, 90])
def test_values_that_are_not_finite(hip, fmt, new):
    """An infinite value that a row sees makes the row's values NaN or infinite, the other sequence's not."""
    st = Setup(hip, fmt, 64, 1, 16, [(new, 200), (new, 100)], seed=2).fill()
    page = int(st.table[0, 1])
    if fmt == F16:
        st.v.raw.view(np.float16).reshape(st.pages, 1, 16, 64)[page, 0, 3, 40] = np.inf
    else:
        st.v.put_scale(page, 0, 1, 3, np.inf)
    st.upload()
    q = st.rng.standard_normal((st.rows, 2 * 64)).astype(np.float32)
    got = _attend(hip, st, 2, q, F16)
    assert np.all(~np.isfinite(got[:new, :, 40])) and np.all(np.isfinite(got[new:2 * new]))


@gpu
@pytest.mark.parametrize("out_fmt", [BF16, F32])
@pytest.mark.parametrize("head", [64, 128])
@pytest.mark.parametrize("value", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("new", [1, 3, 90])
def test_keys_that_are_not_finite(hip, out_fmt, head, value, new):
    """A row that sees an infinite or NaN key is NaN whichever way its score goes, in units that
    every row sees as in those that only some do; the other rows and sequences are right."""
    seqs = [(new, 300)] * 5 + [(new, 90)]
    st = Setup(hip, F16, head, 1, 16, seqs, seed=49).fill()
    # positions in the first unit, in the last one, the last that the first row sees, one that only the last row sees
    holes = [3, 300 - new, 300 - new - 1, 299]
    for s, p in enumerate(holes):
        st.k.values_view()[int(st.table[s, p // 16]), 0, p % 16, 5] = value
    # and behind the end: seen by none
    st.k.values_view()[int(st.table[4, 300 // 16]), 0, 300 % 16] = value
    st.upload()
    q = st.rng.standard_normal((st.rows, 2 * head)).astype(np.float32)
    q[:, 5], q[:, head + 5] = np.abs(q[:, 5]) + 0.1, -np.abs(q[:, head + 5]) - 0.1       # scores of both signs
    got = _attend(hip, st, 2, q, out_fmt)
    bad = [t for s, p in enumerate(holes) for t in range(st.starts[s] + max(0, p - (300 - new)), st.starts[s + 1])]
    assert np.all(np.isnan(got[bad]))
    _check_rows(st, 2, q, got, out_fmt, set(range(st.used)) - set(bad)) if new > 1 else \
        _check_rows(st, 2, q, got, out_fmt, {4, 5})


@gpu
@pytest.mark.parametrize("fmt,out_fmt", [(Q4, BF16), (F16, BF16), (F16, F32), (Q4, F32)])
@pytest.mark.parametrize("head,limit", [(64, 363000.0), (128, 513000.0)])
@pytest.mark.parametrize("new", [1, 90])
def test_queries_beyond_fp16(hip, fmt, out_fmt, head, limit, new):
    """A query that passes FP16 once it is scaled makes its head's row NaN, whatever the keys'
    signs; just below that it counts, and a row that sees nothing stays 0."""
    seqs = [(new, 200), (new, new), (1, 0)]
    st = Setup(hip, fmt, head, 1, 16, seqs, seed=51).fill()
    key = -np.ones((1, head), np.float32)                   # scores of one sign
    for s, (_, length) in enumerate(seqs):
        for p in range(length):
            st.k.store(int(st.table[s, p // 16]), p % 16, key)
    st.upload()
    for value, nan in ((limit, False), (-limit, False), (1.01 * limit, True), (-1.01 * limit, True), (1e30, True),
                       (np.inf, True), (-np.inf, True), (np.nan, True)):
        q = np.zeros((st.rows, 2 * head), np.float32)
        q[:, 7] = value
        got = _attend(hip, st, 2, q, out_fmt)
        assert np.all(np.isnan(got[:2 * new, 0])) if nan else np.all(np.isfinite(got[:2 * new, 0]))
        assert np.all(np.isfinite(got[:2 * new, 1])) and np.all(got[2 * new] == 0)


@gpu
def test_pages_outside_the_pool(hip):
    """A row that sees a bad page is NaN, earlier rows and other sequences are right."""
    st = Setup(hip, Q4, 128, 2, 16, [(40, 100), (2, 50), (1, 20), (30, 300), (1, 64)], seed=6).fill()
    st.upload()
    q = st.rng.standard_normal((st.rows, 4 * 128)).astype(np.float32)
    table = st.table.copy()
    table[0, 5] = st.pages                     # positions 80..95
    table[1, 0] = -5                           # all rows of the sequence
    table[3, 17] = 2 ** 31 - 1                 # positions 272..287
    st.dev[0].upload(table)
    got = _attend(hip, st, 4, q)
    bad = [t for t in range(20, 40)] + [40, 41] + [43 + i for i in range(2, 30)]
    good = [t for t in range(st.used) if t not in bad]
    assert np.all(np.isnan(got[bad])) and np.all(np.isfinite(got[good]))
    _check_rows(st, 4, q, got, BF16, good)


@gpu
def test_sequences_that_do_not_fit(hip):
    """Lengths and row counts that break their bounds give NaN rows; malformed starts write nothing."""
    st = Setup(hip, F16, 64, 1, 16, [(2, 10), (2, 10), (3, 10), (1, 10)], seed=6, spare_rows=3).fill()
    st.lengths[0], st.lengths[1] = -3, 16 * st.table.shape[1] + 1
    st.most = 2
    st.upload()
    q = st.rng.standard_normal((st.rows, 64)).astype(np.float32)
    got = _attend(hip, st, 1, q)
    assert np.all(np.isnan(got[:7])) and np.all(np.isfinite(got[7]))
    st.dev[1].upload(np.array([0, -4, 2, 2 ** 31 - 1, 8], np.int32))
    st.dev[2].upload(np.full(4, 10, np.int32))
    u = _attend_raw(hip, st, 1, q)
    assert np.all(u[6:8] == SENTINEL * 0x0101)


@gpu
@pytest.mark.parametrize("fmt,out_fmt", [(Q4, BF16), (F16, F16), (Q4, F32)])
@pytest.mark.parametrize("head,more", [(128, []), (64, []), (128, [(60, 100)]), (64, [(43, 43)]), (128, [(33, 70)] * 9)])
def test_attention_between_few_and_many(hip, fmt, out_fmt, head, more):
    """Sequences of 48 to 128 packed rows, alone, beside one of more, and in a larger batch."""
    seqs = [(22, 300), (40, 40), (1, 9), (16, 130), (42, 501), (21, 21)] + more
    st = Setup(hip, fmt, head, 2, 64, seqs, seed=35).fill().upload()
    q = st.rng.standard_normal((st.rows, 6 * head)).astype(np.float32)
    _check_rows(st, 6, q, _attend(hip, st, 6, q, out_fmt), out_fmt)


@gpu
@pytest.mark.parametrize("most", [1, 3, 90])
@pytest.mark.parametrize("out_fmt", [BF16, F32])
def test_more_rows_than_said(hip, most, out_fmt):
    """Sequences of more rows than max_rows are NaN, however many they are; the others are right."""
    st = Setup(hip, Q4, 128, 2, 16, [(1, 40), (100, 300), (1, 20), (4, 4), (200, 150)], seed=31).fill()
    st.most = most
    st.upload()
    q = st.rng.standard_normal((st.rows, 4 * 128)).astype(np.float32)
    got = _attend(hip, st, 4, q, out_fmt)
    good = [t for s, (new, _) in enumerate(st.seqs) if new <= most for t in range(st.starts[s], st.starts[s + 1])]
    bad = [t for t in range(st.used) if t not in good]
    assert np.all(np.isnan(got[bad])) and len(bad) == {1: 304, 3: 304, 90: 300}[most]
    _check_rows(st, 4, q, got, out_fmt, good)


@gpu
@pytest.mark.parametrize("head,heads,kv,seqs", [
    (64, 1, 1, [(4096, 500)]),                             # sixteen tiles in eight parts each, fourteen of them see nothing
    (64, 4, 2, [(900, 130), (1, 70), (700, 0)]),
    (128, 3, 1, [(1000, 1000), (1000, 64), (1000, 63)]),
])
@pytest.mark.parametrize("fmt,out_fmt", [(Q4, BF16), (F16, F32)])
def test_prompts_with_more_rows_than_positions(hip, fmt, out_fmt, head, heads, kv, seqs):
    """Whole tiles of rows far before position 0, shared between workgroups: 0, and the rows behind them are right."""
    st = Setup(hip, fmt, head, kv, 16, seqs, seed=41).fill().upload()
    q = st.rng.standard_normal((st.rows, heads * head)).astype(np.float32)
    got = _attend(hip, st, heads, q, out_fmt)
    for s, (new, length) in enumerate(seqs):
        assert np.all(got[st.starts[s]:st.starts[s] + max(0, new - length)] == 0)
    seen = [t for s, (new, length) in enumerate(seqs) for t in range(st.starts[s] + max(0, new - length), st.starts[s + 1])]
    pick = set(int(t) for t in st.rng.choice(seen, min(len(seen), 300), replace=False))
    _check_rows(st, heads, q, got, out_fmt, pick)


def _attend_raw(hip, st, heads, q):
    out = hip.to_device(np.full(st.rows * heads * st.d * 2, SENTINEL, np.uint8))
    ws = hip.alloc(native.paged_attention_workspace_bytes(heads, st.kv, st.d))
    hip.paged_attention(native.PagedAttentionArgs(st.batch, st.cache, hip.to_device(q).ptr, out.ptr, ws.ptr, heads, BF16))
    return out.readback(np.uint16).reshape(st.rows, -1)


@gpu
def test_many_sequences(hip):
    """More sequences than lanes, most of them without a row."""
    seqs = [((i % 3) % 2 * (1 + i % 4), 5 + (i * 37) % 90) for i in range(200)]
    st = Setup(hip, F16, 64, 2, 16, seqs, seed=12).fill().upload()
    q = st.rng.standard_normal((st.rows, 4 * 64)).astype(np.float32)
    _check_rows(st, 4, q, _attend(hip, st, 4, q, F16), F16)


@gpu
def test_repeats_and_batches_agree(hip):
    """The same call twice gives the same bits."""
    st = Setup(hip, Q4, 128, 2, 64, [(1, 900), (1, 40), (60, 500)], seed=14).fill().upload()
    q = st.rng.standard_normal((st.rows, 6 * 128)).astype(np.float32)
    first = _attend(hip, st, 6, q)
    for fill in (0x00, 0x3C):
        assert np.array_equal(first[:st.used], _attend(hip, st, 6, q, ws_fill=fill)[:st.used])


@gpu
def test_plan_serves_growing_sequences(hip):
    """Append and attention recorded once, replayed while lengths grow and rows move; eager calls in between."""
    heads, kv, d = 4, 2, 64
    st = Setup(hip, Q4, d, kv, 16, [(1, 60), (1, 5), (1, 33)], seed=15, extra_pages=12).fill()
    table = np.full((3, 8), -1, np.int32)
    table[:, :st.table.shape[1]] = st.table[:, :8]
    free = [p for p in range(st.pages) if p not in {int(st.table[s, i]) for s, (_, l) in enumerate(st.seqs)
                                                    for i in range(-(-l // 16))}]
    for s, (_, l) in enumerate(st.seqs):
        table[s, -(-l // 16)] = free[s]
    st.table = table
    st.upload()
    width = (heads + 2 * kv) * d
    freq = (0.5 ** np.arange(32)).astype(np.float32)
    dqkv, dfreq = hip.alloc(st.rows * width * 4), hip.to_device(freq)
    query = hip.to_device(np.zeros(st.rows * heads * d, np.float32))
    out = hip.to_device(np.zeros(st.rows * heads * d, np.uint16))
    ws = hip.alloc(native.paged_attention_workspace_bytes(heads, kv, d))
    app = native.PagedAppendArgs(st.batch, st.cache, dqkv.ptr, dfreq.ptr, query.ptr, heads, d, 1.0)
    att = native.PagedAttentionArgs(st.batch, st.cache, query.ptr, out.ptr, ws.ptr, heads, BF16)

    def body():
        hip.paged_kv_append(app)
        hip.paged_attention(att)
    plan = hip.record(body)
    for turn in range(4):
        st.lengths = st.lengths + (1 if turn else 0)
        st.seqs = [(1, int(l)) for l in st.lengths]
        st.dev[2].upload(st.lengths)
        qkv = st.rng.standard_normal((st.rows, width)).astype(np.float32)
        dqkv.upload(qkv)
        plan.launch()
        q = _expect_append(st, heads, d, qkv, freq, 1.0)
        q[st.used:] = 0
        assert _same(query.readback(np.float32).reshape(q.shape), q)
        u = out.readback(np.uint16).reshape(st.rows, heads, d)
        _check_rows(st, heads, q, (u.astype(np.uint32) << 16).view(np.float32).astype(np.float64), BF16)
        body()
        assert np.array_equal(u, out.readback(np.uint16).reshape(u.shape))
    plan.destroy()


@gpu
@pytest.mark.parametrize("fmt,out_fmt", [(Q4, BF16), (F16, F32)])
def test_plan_serves_changing_batches(hip, fmt, out_fmt):
    """One recorded call over batches whose rows move between prompts, drafts and single
    tokens; eager calls in between, the workspace never cleared."""
    heads, kv, d = 6, 2, 128
    st = Setup(hip, fmt, d, kv, 32, [(100, 420), (100, 420), (1, 420)], seed=37, spare_rows=0).fill().upload()
    out = hip.alloc(st.rows * heads * d * (4 if out_fmt == F32 else 2))
    ws = hip.alloc(native.paged_attention_workspace_bytes(heads, kv, d))
    q = st.rng.standard_normal((st.rows, heads * d)).astype(np.float32)
    dq = hip.to_device(q)
    att = native.PagedAttentionArgs(st.batch, st.cache, dq.ptr, out.ptr, ws.ptr, heads, out_fmt)
    # (twice: a plan of more than four kernels is a graph)
    plan = hip.record(lambda: [hip.paged_attention(att) for _ in range(2)])
    for seqs in ([(100, 420), (90, 90), (1, 33)], [(1, 400), (1, 7), (1, 64)], [(30, 30), (3, 420), (70, 300)],
                 [(0, 5), (100, 100), (0, 0)], [(1, 1), (40, 411), (100, 420)]):
        st.seqs = seqs
        st.starts = np.concatenate([[0], np.cumsum([n for n, _ in seqs])]).astype(np.int32)
        st.used = int(st.starts[-1])
        st.dev[1].upload(st.starts)
        st.dev[2].upload(np.array([l for _, l in seqs], np.int32))
        raws = []
        for call in (plan.launch, lambda: hip.paged_attention(att), plan.launch):
            hip.fill_u32(out.ptr, 0xFFFFFFFF, out.nbytes // 4)
            call()
            raws.append(out.readback(np.uint32 if out_fmt == F32 else np.uint16).reshape(st.rows, heads, d))
        assert all(np.array_equal(raws[0], r) for r in raws[1:])
        assert np.all(raws[0][st.used:] == raws[0].dtype.type(-1 & 0xFFFFFFFF if out_fmt == F32 else 0xFFFF))
        got = raws[0].view(np.float32) if out_fmt == F32 else (raws[0].astype(np.uint32) << 16).view(np.float32)
        _check_rows(st, heads, q, got.astype(np.float64), out_fmt)
    plan.destroy()


@gpu
def test_two_contexts_on_one_cache(hip):
    """Another context's stream, workspaces of their own."""
    st = Setup(hip, F16, 128, 2, 32, [(1, 500), (30, 200)], seed=16).fill().upload()
    q = st.rng.standard_normal((st.rows, 4 * 128)).astype(np.float32)
    want = _attend(hip, st, 4, q)
    with native.HipContext(0) as other:
        dq = hip.to_device(q)
        outs = [hip.to_device(np.zeros(st.rows * 4 * 128, np.uint16)) for _ in range(2)]
        wss = [hip.alloc(native.paged_attention_workspace_bytes(4, 2, 128)) for _ in range(2)]
        for _ in range(3):
            for ctx, o, w in zip((hip, other), outs, wss):
                ctx.paged_attention(native.PagedAttentionArgs(st.batch, st.cache, dq.ptr, o.ptr, w.ptr, 4, BF16))
        other.sync()
        for o in outs:
            u = o.readback(np.uint16).reshape(st.rows, 4, 128)[:st.used]
            assert np.array_equal((u.astype(np.uint32) << 16).view(np.float32).astype(np.float64), want[:st.used])


@gpu
@pytest.mark.parametrize("fmt", [F16, Q4])
def test_pages_far_into_a_pool(hip, fmt):
    """Pages more than 4 GiB into their pools: append, read, attention of few and of many rows."""
    heads, kv, d = 4, 2, 128
    st = Setup(hip, fmt, d, kv, 256, [(1, 300), (40, 270), (3, 5)], seed=33).fill().upload()
    page = kv * native.paged_page_bytes(fmt, 256, d)
    shift = 2 ** 32 // page + 3
    pools = [hip.alloc((shift + st.pages) * page) for _ in range(2)]
    for b, pool in zip(pools, (st.k, st.v)):
        b.upload(pool.raw, shift * page)
    held = (st.table >= 0) & (st.table < st.pages)
    st.dev[0].upload(np.where(held, st.table + shift, st.table).astype(np.int32))
    st.cache = native.PagedCache(pools[0].ptr, pools[1].ptr, shift + st.pages, 256, kv, d, fmt)
    qkv = st.rng.standard_normal((st.rows, (heads + 2 * kv) * d)).astype(np.float32)
    freq = (0.7 ** np.arange(d // 2)).astype(np.float32)
    query = _append(hip, st, heads, d, qkv, freq, 1.0)
    want = _expect_append(st, heads, d, qkv, freq, 1.0)
    q = query.readback(np.float32).reshape(want.shape)
    assert _same(q, want)
    for b, pool in zip(pools, (st.k, st.v)):
        assert np.array_equal(b.readback(np.uint8, pool.raw.size, shift * page), pool.raw.reshape(-1))
    keys, vals = (hip.alloc(st.rows * kv * d * 4) for _ in range(2))
    hip.paged_kv_read(st.batch, st.cache, keys.ptr, vals.ptr)
    rows = vals.readback(np.float32).reshape(st.rows, kv, d)
    for t in range(st.used):
        _, p, at = ref.place(st.table, st.starts, st.lengths, 256, st.pages, t)
        assert np.array_equal(rows[t], st.v.load(at, p % 256).astype(np.float32))
    _check_rows(st, heads, q, _attend(hip, st, heads, q, BF16), BF16)


# ---- an attention block of a step ------------------------------------------------------------

@gpu
def test_attention_block_of_a_step(hip):
    """Norm into 8 bits, qkv product, append, attention, 8 bits, output
    product with the residual, in one plan, against 64 bits along the same
    path (codes of the 64-bit path: two paths' codes differ where a value
    lies next to a border, by one step, 1/127 of a row's largest value, so the
    block's own contribution agrees to 2%)."""
    heads, kv, d, hidden = 8, 2, 64, 512
    st = Setup(hip, Q4, d, kv, 32, [(1, 90), (1, 7), (12, 40), (1, 33)], seed=17).fill().upload()
    rng, width = st.rng, (heads + 2 * kv) * d
    h, r = (rng.standard_normal((st.rows, hidden)).astype(np.float32) for _ in range(2))
    g = (1 + 0.1 * rng.standard_normal(hidden)).astype(np.float32)
    wq, wo = ((rng.standard_normal(s) * s[1] ** -0.5).astype(np.float32) for s in ((width, hidden), (hidden, heads * d)))
    freq = (10000.0 ** (-np.arange(d // 2) / (d // 2))).astype(np.float32)
    up = hip.to_device
    dh, dr, dg, dfreq = up(h), up(r), up(g), up(freq)
    alloc = hip.alloc
    weights = []
    for w in (wq, wo):
        c, s = alloc(w.size), alloc(w.shape[0] * 4)
        hip.quantize_i8(native.F32, up(w).ptr, c.ptr, s.ptr, *w.shape)
        weights.append((c, s, c.readback(np.int8).reshape(w.shape).astype(np.float64) *
                        s.readback(np.float32).astype(np.float64)[:, None]))
    T = st.rows
    u, q8, s8, qkv = alloc(h.nbytes), alloc(h.size), alloc(T * 4), alloc(T * width * 4)
    query, out = up(np.zeros(T * heads * d, np.float32)), up(np.zeros(T * heads * d, np.uint16))
    o8, os8, y = alloc(T * heads * d), alloc(T * 4), alloc(h.nbytes)
    ws = alloc(native.paged_attention_workspace_bytes(heads, kv, d))

    def body():
        hip.residual_rms_norm_i8(dh.ptr, dr.ptr, dg.ptr, u.ptr, q8.ptr, s8.ptr, T, hidden, 1e-5)
        hip.gemm_i8(q8.ptr, s8.ptr, weights[0][0].ptr, weights[0][1].ptr, qkv.ptr, T, width, hidden)
        hip.paged_kv_append(native.PagedAppendArgs(st.batch, st.cache, qkv.ptr, dfreq.ptr, query.ptr, heads, d, 1.0))
        hip.paged_attention(native.PagedAttentionArgs(st.batch, st.cache, query.ptr, out.ptr, ws.ptr, heads, BF16))
        hip.quantize_i8(BF16, out.ptr, o8.ptr, os8.ptr, T, heads * d)
        hip.gemm_i8(o8.ptr, os8.ptr, weights[1][0].ptr, weights[1][1].ptr, y.ptr, T, hidden, heads * d, u.ptr)
    plan = hip.record(body)
    for _ in range(2):
        plan.launch()
    got = y.readback(np.float32).reshape(h.shape).astype(np.float64)
    plan.destroy()

    def codes(v):
        step = np.abs(v).max(1, keepdims=True) / 127
        return np.rint(v / np.where(step == 0, 1, step)) * step
    x = (h + r).astype(np.float64)
    v = codes(x / np.sqrt((x * x).mean(1, keepdims=True) + 1e-5) * g) @ weights[0][2].T
    q = _expect_append(st, heads, d, v.astype(np.float32), freq, 1.0)
    attn = np.zeros((T, heads * d))
    for s, (new, length) in enumerate(st.seqs):
        keys, values = st.rows_of(s, length)
        for i in range(new):
            t = st.starts[s] + i
            attn[t] = ref.attention(q[t].reshape(heads, d), keys, values, length - new + i + 1)[0].reshape(-1)
    part = (codes(attn) @ weights[1][2].T)[:st.used]
    assert np.linalg.norm(got[:st.used] - x[:st.used] - part) <= 0.02 * np.linalg.norm(part)


# ---- refusals -----------------------------------------------------------------------------------

@gpu
def test_refusals(hip):
    st = Setup(hip, Q4, 128, 2, 16, [(2, 20)], seed=1, spare_rows=0).fill().upload()
    before = st.dev[3].readback(np.uint8)
    heads = 4
    qkv, freq = hip.alloc(st.rows * 8 * 128 * 4), hip.alloc(512)
    query, out = hip.alloc(st.rows * heads * 128 * 4), hip.alloc(st.rows * heads * 128 * 2)
    ws = hip.alloc(native.paged_attention_workspace_bytes(heads, 2, 128))

    def with_(base, **change):
        new = type(base).from_buffer_copy(base)
        for k, v in change.items():
            setattr(new, k, v)
        return new

    def refused(status, call, *args):
        with pytest.raises(native.HipError) as e:
            call(*args)
        assert e.value.status == status, str(e.value)

    arg, uns = native.ERR_ARGUMENT, native.ERR_UNSUPPORTED
    batches = [(arg, with_(st.batch, **c)) for c in (
        {"page_table": None}, {"row_starts": None}, {"lengths": None}, {"sequences": 0}, {"sequences": 4097},
        {"max_pages": 0}, {"max_pages": 1 << 27}, {"rows": 0}, {"rows": (1 << 20) + 1}, {"max_rows": 0}, {"max_rows": 3})]
    caches = [(s, with_(st.cache, **c)) for s, c in (
        (arg, {"key_pages": None}), (arg, {"value_pages": None}), (arg, {"key_pages": st.cache.key_pages + 8}),
        (arg, {"pages": 0}), (arg, {"pages": 1 << 31}), (arg, {"page_size": 48}), (arg, {"page_size": 8}),
        (arg, {"page_size": 512}), (arg, {"kv_heads": 0}), (arg, {"kv_heads": 257}), (uns, {"head_size": 96}),
        (uns, {"cache_format": native.F32}), (uns, {"cache_format": native.Q8_0}))]
    app = native.PagedAppendArgs(st.batch, st.cache, qkv.ptr, freq.ptr, query.ptr, heads, 128, 1.0)
    att = native.PagedAttentionArgs(st.batch, st.cache, query.ptr, out.ptr, ws.ptr, heads, BF16)
    for status, b in batches:
        refused(status, hip.paged_kv_append, with_(app, batch=b))
        refused(status, hip.paged_attention, with_(att, batch=b))
        refused(status, hip.paged_kv_read, b, st.cache, query.ptr, out.ptr)
    for status, c in caches:
        refused(status, hip.paged_kv_append, with_(app, cache=c))
        refused(status, hip.paged_attention, with_(att, cache=c))
        refused(status, hip.paged_kv_read, st.batch, c, query.ptr, out.ptr)
    for c in ({"qkv": None}, {"query": None}, {"frequencies": None}, {"query_heads": 0}, {"query_heads": 3},
              {"query_heads": 34}, {"rotary_size": 130}, {"rotary_size": 7}, {"rotary_size": -2},
              {"rope_scale": float("inf")}, {"query": qkv.ptr}, {"query": st.cache.key_pages},
              {"qkv": st.cache.value_pages}):
        refused(arg, hip.paged_kv_append, with_(app, **c))
    same = with_(st.cache, value_pages=st.cache.key_pages)
    refused(arg, hip.paged_kv_append, with_(app, cache=same))
    for c in ({"query": None}, {"output": None}, {"workspace": None}, {"query": query.ptr + 4}, {"output": out.ptr + 2},
              {"workspace": ws.ptr + 4}, {"query_heads": 0}, {"query_heads": 5}, {"query_heads": 34},
              {"output": query.ptr}, {"output": st.cache.key_pages}, {"workspace": out.ptr}):
        refused(arg, hip.paged_attention, with_(att, **c))
    refused(uns, hip.paged_attention, with_(att, output_format=native.Q8_0))
    for keys, vals in ((0, out.ptr), (query.ptr, 0), (query.ptr, query.ptr), (st.cache.key_pages, query.ptr)):
        refused(arg, hip.paged_kv_read, st.batch, st.cache, keys, vals)
    assert np.array_equal(before, st.dev[3].readback(np.uint8))
