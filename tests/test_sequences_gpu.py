"""The operators over many sequences at once (rows normalised and mixed, the time-mix scan, beam
selection, slot moves) through the C ABI, against 64-bit numpy with bounds that count roundings
(tests/sequences_reference.py)."""
import numpy as np
import pytest

from tests import sequences_reference as ref
from sharpinference_amd import native

pytestmark = pytest.mark.gpu

FORMATS = [native.F32, native.F16, native.BF16]
FILL = 0x5A


def _guarded(hip, nbytes):
    """A filled buffer with 64 spare bytes behind it."""
    return hip.to_device(np.full(int(nbytes) + 64, FILL, np.uint8))


def _spare_untouched(buf, nbytes):
    assert np.all(buf.readback(np.uint8, 64, int(nbytes)) == FILL)


def _i32(hip, x):
    return hip.to_device(np.asarray(x, np.int32))


def _batch(hip, starts, source, to, slots, rows, max_rows=None):
    """(RowBatch, what it points at)."""
    held = [_i32(hip, starts), _i32(hip, source), _i32(hip, to)]
    most = max_rows or max(1, max(np.diff(starts)))
    return native.RowBatch(*[h.ptr for h in held], len(source), slots, rows, min(most, rows)), held


def _lay(rng, counts, tail=0):
    """starts, from, to of sequences with these row counts in shuffled slots; every third is new."""
    n = len(counts)
    starts = np.concatenate([[0], np.cumsum(counts)])
    order = rng.permutation(2 * n + 1)
    source, to = order[:n].copy(), order[n:2 * n].copy()
    source[2::3] = -1
    return starts, source, to, 2 * n + 1, int(starts[-1]) + tail


def _near(got, want, bound):
    """Within the bound; NaN and infinities in the same places."""
    finite = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)) or np.all(~np.isfinite(got) == ~finite)
    off = np.abs(got[finite] - want[finite])
    limit = np.broadcast_to(bound, want.shape)[finite]
    worst = np.max(off / np.maximum(limit, 1e-300)) if off.size else 0.0
    assert worst <= 1.0, f"{worst} times the bound"


# ---- rows normalised and mixed -------------------------------------------------------------------

def _mix_inputs(rng, rows, n, mixes, residual, slots):
    f = lambda *s: rng.standard_normal(s).astype(np.float32)
    x = f(rows, n) * np.exp(rng.uniform(-3, 3, (rows, 1))).astype(np.float32) + np.float32(0.3)
    return dict(x=x, residual=f(rows, n) if residual else None, weight=1 + 0.2 * f(n), bias=0.2 * f(n),
                mix=rng.random((mixes, n)).astype(np.float32), state=f(slots, n))


def _run_mix(hip, inp, starts, source, to, slots, fmt, eps=1e-5, shift=0, max_rows=None):
    rows, n = inp["x"].shape
    mixes = len(inp["mix"])
    dev = {}
    for k, v in inp.items():
        if v is None or v.size == 0:
            dev[k] = 0
            continue
        b = hip.alloc(v.nbytes + 64)
        b.upload(v, 4 * shift)
        dev[k] = b
    at = lambda k: dev[k].ptr + 4 * shift if dev[k] else 0
    batch, held = _batch(hip, starts, source, to, slots, rows, max_rows)
    size = ref.SIZE[fmt]
    out_bytes = max(mixes, 1) * rows * n * size
    up, out = _guarded(hip, rows * n * 4 + 4 * shift), _guarded(hip, out_bytes + size * shift)
    hip.layernorm_mix_rows(native.LayernormMixRowsArgs(
        batch, at("x"), at("residual"), at("weight"), at("bias"), at("mix"), at("state"),
        up.ptr + 4 * shift if inp["residual"] is not None else 0, out.ptr + size * shift, n, mixes, fmt, eps))
    got = out.readback(np.uint8, out_bytes, size * shift)
    _spare_untouched(up, rows * n * 4 + 4 * shift)
    _spare_untouched(out, out_bytes + size * shift)
    updated = up.readback(np.float32, rows * n, 4 * shift).reshape(rows, n)
    state = dev["state"].readback(np.float32, slots * n, 4 * shift).reshape(slots, n) if dev["state"] else None
    for b in [up, out, *held, *[v for v in dev.values() if v]]:
        b.free()
    return updated, got, state


def _check_mix(hip, inp, starts, source, to, slots, fmt, **more):
    rows, n = inp["x"].shape
    mixes = max(1, len(inp["mix"]))
    updated, raw, state = _run_mix(hip, inp, starts, source, to, slots, fmt, **more)
    u, out, bound, held, held_off, live = ref.mix_rows(inp["x"], inp["residual"], inp["weight"], inp["bias"], inp["mix"],
                                                       inp["state"], starts, source, to, more.get("eps", 1e-5))
    got = ref.values(raw, fmt).reshape(mixes, rows, n)
    _near(got[:, live], out[:, live], bound[:, live] + ref.STEP[fmt] * np.abs(out[:, live]) + ref.TINY[fmt])
    assert np.all(raw.reshape(mixes, rows, -1)[:, ~live] == FILL)
    if inp["residual"] is not None:
        assert np.array_equal(updated[live], u[live])
        assert np.all(updated[~live].view(np.uint8) == FILL)
    if len(inp["mix"]):
        _near(state.astype(np.float64), held, held_off)


@pytest.mark.parametrize("n,mixes,fmt", [(1, 1, native.F32), (3, 2, native.BF16), (64, 6, native.F16), (2047, 6, native.BF16),
                                         (2048, 6, native.BF16), (2052, 1, native.F32), (4096, 1, native.BF16),
                                         (8191, 2, native.F16), (8192, 8, native.BF16), (1000, 0, native.BF16)])
@pytest.mark.parametrize("counts", [[1], [5, 1, 1, 40, 0, 2], [0, 0, 9]])
def test_mix_rows(hip, n, mixes, fmt, counts):
    rng = np.random.default_rng(n * 31 + mixes + len(counts))
    starts, source, to, slots, rows = _lay(rng, counts, tail=3)
    inp = _mix_inputs(rng, rows, n, mixes, len(counts) > 1, slots)
    _check_mix(hip, inp, starts, source, to, slots, fmt)


@pytest.mark.parametrize("n,mixes", [(7, 2), (8, 1), (9, 2), (15, 6), (511, 1), (515, 6), (1000, 6), (1027, 3), (2051, 1), (4099, 6),
                                     (5003, 6), (6144, 2), (6145, 1)])
def test_mix_rows_widths(hip, n, mixes):
    """Widths over which threads and values do not come out even, sequences that stay in their slots."""
    rng = np.random.default_rng(n)
    starts, source, to, slots, rows = _lay(rng, [1, 1, 6, 1, 2, 1])
    inp = _mix_inputs(rng, rows, n, mixes, n % 2 == 0, slots)
    for fmt in (native.BF16, native.F32):
        _check_mix(hip, inp, starts, to, to, slots, fmt)


@pytest.mark.parametrize("rows,sequences,n", [(1500, 1, 300), (4100, 3, 64), (5000, 4096, 36), (1030, 1030, 256)])
def test_mix_rows_many(hip, rows, sequences, n):
    """More rows than a workgroup takes in one run; as many sequences as a call takes."""
    rng = np.random.default_rng(rows)
    cuts = np.sort(rng.choice(np.arange(1, rows), sequences - 1, replace=sequences > rows // 2)) if sequences > 1 else []
    if sequences == rows:
        cuts = np.arange(1, rows)
    counts = np.diff(np.concatenate([[0], cuts, [rows]])).astype(int)
    starts, source, to, slots, rows = _lay(rng, counts, tail=1)
    _check_mix(hip, _mix_inputs(rng, rows, n, 2, True, slots), starts, source, to, slots, native.BF16)


@pytest.mark.parametrize("shift", [1, 2, 3])
@pytest.mark.parametrize("n", [64, 2500])
def test_mix_rows_at_any_address(hip, shift, n):
    rng = np.random.default_rng(shift)
    starts, source, to, slots, rows = _lay(rng, [7, 2])
    for fmt in FORMATS:
        _check_mix(hip, _mix_inputs(rng, rows, n, 3, True, slots), starts, source, to, slots, fmt, shift=shift)


def test_mix_rows_slots(hip):
    """From and to the same slot, one slot for several, no slot, slots that are none; rows before the first sequence and
    starts that fall."""
    rng = np.random.default_rng(8)
    n, slots = 128, 5
    inp = _mix_inputs(rng, 20, n, 2, False, slots)
    _check_mix(hip, inp, [3, 6, 7, 12, 12, 15], [2, 0, 0, 1, -1], [2, 3, -1, 4, 1], slots, native.F32)
    _check_mix(hip, inp, [0, 4, 9], [5, 1], [0, 99], slots, native.F32)   # 5 is no slot: its first row is NaN
    _check_mix(hip, inp, [0, 4, 9], [-7, 1], [3, -2], slots, native.F32)
    _, raw, state = _run_mix(hip, inp, [0, 4, 2, 25], [1, 2, 3], [0, 0, 0], slots, native.F32)
    want = ref.mix_rows(inp["x"], None, inp["weight"], inp["bias"], inp["mix"], inp["state"], [0, 4], [1], [0], 1e-5)
    got = ref.values(raw, native.F32).reshape(2, 20, n)
    _near(got[:, :2], want[1][:, :2], want[2][:, :2])   # (rows 2 and 3 lie in a sequence that leaves the batch, too)


def test_mix_rows_special_values(hip):
    """Constant rows, huge and tiny values; NaN and infinity stay in their row and the one behind it."""
    rng = np.random.default_rng(9)
    starts, source, to, slots, rows = _lay(rng, [12, 3])
    inp = _mix_inputs(rng, rows, 256, 2, False, slots)
    inp["x"][1] = 3.0
    inp["x"][3] *= np.float32(1e15)
    inp["x"][5] = rng.standard_normal(256).astype(np.float32) * np.float32(1e-15)
    _check_mix(hip, inp, starts, source, to, slots, native.F32)
    clean, raw, _ = _run_mix(hip, inp, starts, source, to, slots, native.F32)
    inp["x"][7, 9] = np.nan
    inp["x"][13, 0] = np.inf
    _, bad, _ = _run_mix(hip, inp, starts, source, to, slots, native.F32)
    a, b = (ref.values(x, native.F32).reshape(2, rows, -1) for x in (raw, bad))
    touched = [7, 8, 13, 14]
    keep = [i for i in range(rows) if i not in touched]
    assert np.array_equal(a[:, keep], b[:, keep])
    assert np.isnan(b[:, touched]).all()


# ---- the time-mix scan -----------------------------------------------------------------------------

def _wkv_inputs(rng, rows, heads, first, slots, decay=(-7, 1)):
    c = heads * ref.HEAD
    f = lambda *s: rng.standard_normal(s).astype(np.float32)
    inp = dict(r=f(rows, c), k=f(rows, c), v=f(rows, c), w_lora=0.5 * f(rows, c), a_lora=0.5 * f(rows, c),
               gate=2 * rng.random((rows, c)).astype(np.float32), v_lora=None if first else 0.5 * f(rows, c),
               w0=np.tile(np.linspace(*decay, ref.HEAD), heads).astype(np.float32) + 0.3 * f(c), a0=f(c),
               v0=None if first else f(c), k_k=1 + 0.1 * f(c), k_a=rng.random(c).astype(np.float32), r_k=0.1 * f(c),
               lnx_weight=1 + 0.1 * f(c), lnx_bias=0.1 * f(c), v_first=f(rows, c),
               state=0.1 * f(slots, heads, ref.HEAD, ref.HEAD))
    return inp


def _run_wkv(hip, inp, heads, first, starts, source, to, fmt, max_rows=None):
    rows, slots = len(inp["r"]), len(inp["state"])
    dev = {k: hip.to_device(v) for k, v in inp.items() if v is not None}
    p = lambda k: dev[k].ptr if k in dev else 0
    batch, held = _batch(hip, starts, source, to, slots, rows, max_rows)
    nbytes = rows * heads * ref.HEAD * ref.SIZE[fmt]
    out = _guarded(hip, nbytes)
    ws_bytes = native.rwkv7_wkv_rows_workspace_bytes(heads)
    ws = _guarded(hip, ws_bytes)
    hip.rwkv7_wkv_rows(native.Rwkv7WkvRowsArgs(batch, heads, int(first), *[p(k) for k in native.RWKV7_WKV_VECTORS],
                                               p("v_first"), p("state"), out.ptr, ws.ptr, fmt))
    raw = out.readback(np.uint8, nbytes)
    _spare_untouched(out, nbytes)
    _spare_untouched(ws, ws_bytes)
    state = dev["state"].readback(np.float32).reshape(inp["state"].shape)
    v_first = dev["v_first"].readback(np.float32).reshape(rows, -1)
    for b in [out, ws, *held, *dev.values()]:
        b.free()
    return raw.reshape(rows, -1), state, v_first


def _check_wkv(hip, inp, heads, first, starts, source, to, fmt, max_rows=None):
    rows = len(inp["r"])
    raw, state, v_first = _run_wkv(hip, inp, heads, first, starts, source, to, fmt, max_rows)
    want, bound, want_state, off = ref.wkv_rows(inp, heads, first, starts, source, to)
    live = np.zeros(rows, bool)
    for _, a, b in ref.spans(starts, rows):
        live[a:b] = True
    got = ref.values(np.ascontiguousarray(raw).reshape(-1), fmt).reshape(rows, -1)
    _near(got[live], want[live], bound[live] + ref.STEP[fmt] * np.abs(want[live]) + ref.TINY[fmt])
    assert np.all(raw[~live] == FILL)
    finite = np.isfinite(want_state).all((2, 3))
    assert np.array_equal(np.isfinite(state).all((2, 3)), finite)
    diff = np.linalg.norm(state.astype(np.float64) - want_state, axis=(2, 3))
    assert np.all(diff[finite] <= off[finite]), np.max(diff[finite] / np.maximum(off[finite], 1e-300))
    assert np.array_equal(v_first[live], inp["v" if first else "v_first"][live])
    assert np.array_equal(v_first[~live], inp["v_first"][~live])


@pytest.mark.parametrize("counts", [[1], [1, 1, 1, 1, 1], [2, 0, 7, 4, 1], [8, 9], [15, 16, 17], [33], [64, 1, 0, 31], [130, 3]])
@pytest.mark.parametrize("heads,first,fmt", [(1, False, native.F32), (3, True, native.BF16), (2, False, native.F16)])
def test_wkv_rows(hip, counts, heads, first, fmt):
    rng = np.random.default_rng(sum(counts) * 7 + heads)
    starts, source, to, slots, rows = _lay(rng, counts, tail=2)
    _check_wkv(hip, _wkv_inputs(rng, rows, heads, first, slots), heads, first, starts, source, to, fmt)


@pytest.mark.parametrize("heads,counts", [(1, [1500]), (2, [700, 90, 1, 260]), (64, [700, 1500, 13, 0, 40, 900, 1]),
                                          (4, [20] * 150 + [640, 0, 1] + [13] * 149 + [900])])
def test_wkv_rows_long(hip, heads, counts):
    """Long sequences, which may be shared out over their length."""
    rng = np.random.default_rng(len(counts))
    starts, source, to, slots, rows = _lay(rng, counts)
    _check_wkv(hip, _wkv_inputs(rng, rows, heads, False, slots), heads, False, starts, source, to, native.F32)


@pytest.mark.parametrize("most", [3, 20, 45])
def test_wkv_rows_of_many_heads(hip, most):
    """More heads than the card takes at once, of sequences of few rows and of some more."""
    rng = np.random.default_rng(most)
    starts, source, to, slots, rows = _lay(rng, list(rng.integers(0, most, 50)) + [most], tail=1)
    _check_wkv(hip, _wkv_inputs(rng, rows, 24, most == 20, slots), 24, most == 20, starts, source, to, native.BF16)


@pytest.mark.parametrize("starts", [[0, 0], [3, 8], [5, 120], [100, 300], [0, 640], [0, 0, 5, 25], [2, 4, 400, 400], [0, 100, 600]])
def test_wkv_rows_fewer_than_stated(hip, starts):
    """Sequences, one among them, that bring fewer rows than the launch goes by."""
    rng = np.random.default_rng(sum(starts))
    n = len(starts) - 1
    _check_wkv(hip, _wkv_inputs(rng, 640, 3, False, 2 * n), 3, False, starts, range(n), range(n, 2 * n), native.F32, max_rows=640)


@pytest.mark.parametrize("starts", [[0, 600, 300, 640], [0, 200, 150, 500], [0, 700, 500], [-4, 300, 500], [500, 20]])
def test_wkv_rows_starts_that_fall(hip, starts):
    """Starts that fall or leave the rows: anything in those rows and slots, nothing outside of them."""
    rng = np.random.default_rng(12)
    n = len(starts) - 1
    inp = _wkv_inputs(rng, 640, 2, False, 2 * n)
    raw, state, _ = _run_wkv(hip, inp, 2, False, starts, range(n), range(n, 2 * n), native.F32, 640)
    assert np.array_equal(state[:n], inp["state"][:n])
    assert np.all(raw[max(min(max(starts), 640), 0):] == FILL)


@pytest.mark.parametrize("count", [3, 20, 200])
def test_wkv_rows_slots(hip, count):
    """From and to the same slot, one slot for several, none, no slots; a bound on the rows that is too low."""
    rng = np.random.default_rng(count)
    starts, rows = [2, 2 + count, 2 + 2 * count, 2 + 3 * count, 2 + 3 * count], 4 + 3 * count
    for source, to in (([1, 3, 3, 0], [1, 0, 2, 3]), ([-1, 4, 2, 2], [-1, 0, 4, 1]), ([-2, 0, 1, 1], [3, 2, -5, 3])):
        inp = _wkv_inputs(rng, rows, 2, False, 4)
        _check_wkv(hip, inp, 2, False, starts, source, to, native.F32, max_rows=None if source[0] else 1)
    _check_wkv(hip, inp, 2, False, starts, [0, 1, 2, 3], [0, 1, 2, 3], native.F32, max_rows=1)


@pytest.mark.parametrize("count", [5, 37])
def test_wkv_rows_like_keys(hip, count):
    """The same key row after row, at full adaptation and hardly any decay: the rows' products are as far from
    independent as they can be."""
    rng = np.random.default_rng(count)
    inp = _wkv_inputs(rng, count, 2, False, 3)
    inp["k"][:] = inp["k"][0] + 1e-3 * inp["k"]
    inp["a_lora"][:] = 20.0
    inp["w_lora"][:] = -20.0
    _check_wkv(hip, inp, 2, False, [0, count], [1], [2], native.F32)


@pytest.mark.parametrize("count", [6, 45])
def test_wkv_rows_extreme_gates(hip, count):
    """The fastest decay in every row, gates far off on both sides, keys of zeros, large values."""
    rng = np.random.default_rng(count)
    inp = _wkv_inputs(rng, count, 2, False, 3)
    inp["w_lora"][:] = 30.0
    inp["a_lora"][::2] = -100.0
    inp["k"][3::7] = 0.0
    inp["v"][1::5] *= np.float32(1e10)
    _check_wkv(hip, inp, 2, False, [0, count], [1], [2], native.F32)


@pytest.mark.parametrize("count,at", [(6, 3), (50, 21), (300, 170)])
@pytest.mark.parametrize("name,value", [("v", np.nan), ("k", np.inf), ("r", np.nan), ("w_lora", np.nan), ("gate", np.inf),
                                        ("a_lora", np.nan)])
def test_wkv_rows_not_finite(hip, count, at, name, value):
    """What is not finite changes no row before its own, no other head and no other sequence."""
    rng = np.random.default_rng(at)
    starts, source, to, slots, rows = _lay(rng, [count, 9])
    inp = _wkv_inputs(rng, rows, 2, False, slots)
    clean = ref.values(_run_wkv(hip, inp, 2, False, starts, source, to, native.F32)[0].reshape(-1), native.F32).reshape(rows, 2, -1)
    inp[name][at, 64 + 5] = value
    raw, state, _ = _run_wkv(hip, inp, 2, False, starts, source, to, native.F32)
    got = ref.values(raw.reshape(-1), native.F32).reshape(rows, 2, -1)
    assert np.array_equal(got[:, 0], clean[:, 0]) and np.array_equal(got[count:], clean[count:])
    with np.errstate(all="ignore"):
        want, bound, want_state, _ = ref.wkv_rows(inp, 2, False, starts, source, to)
    want, bound = want.reshape(rows, 2, -1), bound.reshape(rows, 2, -1)
    _near(got[:at], want[:at], bound[:at])
    assert not np.isfinite(got[at, 1]).all()
    if name in ("r", "gate"):   # these leave the state as it is
        _near(got[at + 1:], want[at + 1:], bound[at + 1:])
        assert np.isfinite(state[to[0]]).all()
    else:
        assert np.isnan(got[at + 1:count, 1]).all()


def test_wkv_rows_is_the_single_row_operator(hip):
    """Row after row through si_hip_rwkv7_wkv gives the same to the bounds of both."""
    rng = np.random.default_rng(77)
    heads, rows = 2, 40
    inp = _wkv_inputs(rng, rows, heads, False, 2)
    raw, state, _ = _run_wkv(hip, inp, heads, False, [0, rows], [0], [1], native.F32)
    _, bound, _, off = ref.wkv_rows(inp, heads, False, [0, rows], [0], [1])
    dev = {k: hip.to_device(v) for k, v in inp.items()}
    c = heads * ref.HEAD * 4
    out = hip.alloc(rows * c)
    for t in range(rows):
        at = lambda k: dev[k].ptr + (t * c if inp[k].ndim == 2 else 0)
        hip.rwkv7_wkv(native.Rwkv7WkvArgs(heads, 0, *[at(k) for k in native.RWKV7_WKV_VECTORS], at("v_first"),
                                          dev["state"].ptr, out.ptr + t * c))
    one = out.readback(np.float32).reshape(rows, -1)
    assert np.all(np.abs(one - raw.view(np.float32)) <= 2 * bound)
    last = dev["state"].readback(np.float32).reshape(inp["state"].shape)[0]
    assert np.all(np.linalg.norm(last.astype(np.float64) - state[1], axis=(1, 2)) <= 2 * off[1])


# ---- beam selection ----------------------------------------------------------------------------------

def _run_beams(hip, logits, scores, done, slots, beams, candidates, fmt, end_token=-1, pad=0, in_place=False):
    """logits: FP32 values; rows lie len + pad values apart."""
    rows, vocab = logits.shape
    wide = np.full((rows, vocab + pad), 1e30, np.float32)
    wide[:, :vocab] = logits
    raw = ref.encode(wide, fmt)
    shown = ref.values(raw.reshape(-1), fmt).reshape(rows, -1)[:, :vocab]
    sequences = rows // beams
    dl, ds = hip.to_device(raw), hip.to_device(np.asarray(scores, np.float32))
    dd = None if done is None else _i32(hip, done)
    dt = None if slots is None else _i32(hip, slots)
    nbytes = sequences * candidates * 4
    outs = {k: _guarded(hip, nbytes) for k in ("parents", "tokens", "scores", "done", "from", "to")}
    if in_place:
        outs["scores"], outs["done"], outs["to"] = ds, dd, dt
    size = native.beam_select_workspace_bytes(sequences, beams, candidates, vocab)
    ws = _guarded(hip, size)
    ptr = lambda b: 0 if b is None else b.ptr
    hip.beam_select(native.BeamSelectArgs(
        dl.ptr, ds.ptr, ptr(dd), ptr(dt), outs["parents"].ptr, outs["tokens"].ptr, outs["scores"].ptr,
        outs["done"].ptr if end_token >= 0 else 0, outs["from"].ptr if dt else 0, outs["to"].ptr if dt else 0, ws.ptr,
        vocab, vocab + pad, sequences, beams, candidates, fmt, end_token))
    got = {k: b.readback(np.float32 if k == "scores" else np.int32, sequences * candidates) for k, b in outs.items()}
    _spare_untouched(ws, size)
    for k, b in outs.items():
        if not (in_place and k in ("scores", "done", "to")):
            _spare_untouched(b, nbytes)
    for b in {id(b): b for b in [dl, ds, dd, dt, ws, *outs.values()] if b is not None}.values():
        b.free()
    return got, shown


def _check_beams(hip, logits, scores, done, slots, beams, candidates, fmt, end_token=-1, **more):
    got, shown = _run_beams(hip, logits, scores, done, slots, beams, candidates, fmt, end_token, **more)
    with np.errstate(all="ignore"):
        want = ref.beam_select(shown, np.asarray(scores, np.float32), done, slots, beams, candidates, end_token)
    keys = ["parents", "tokens"] + (["done"] if end_token >= 0 else []) + (["from", "to"] if slots is not None else [])
    for k in keys:
        assert np.array_equal(got[k], want[k]), k
    # one rounding to FP32; the sum's exponentials are off by at most 2^-21 (3 roundings, and |x - m| up to 64 of them that count)
    w = want["scores"]
    finite = np.isfinite(w)
    assert np.array_equal(np.isfinite(got["scores"]), finite)
    assert np.all(np.abs(got["scores"][finite] - w[finite]) <= ref.U * np.abs(w[finite]) + 2.0 ** -21)
    assert np.all(got["scores"][~finite] == -np.inf)


@pytest.mark.parametrize("vocab", [1, 2, 63, 64, 1000, 2048, 2049, 5001, 65536])
@pytest.mark.parametrize("sequences,beams,twice", [(1, 1, False), (2, 4, False), (3, 5, True), (1, 16, True), (2, 16, False)])
def test_beam_select(hip, vocab, sequences, beams, twice):
    rng = np.random.default_rng(vocab + beams)
    rows = sequences * beams
    logits = (2.5 * rng.standard_normal((rows, vocab))).astype(np.float32)
    scores = -4 * rng.random(rows)
    slots = None if twice else rng.permutation(rows + 3)[:rows]
    for fmt in FORMATS:
        _check_beams(hip, logits, scores, None, slots, beams, beams * (2 if twice else 1), fmt, pad=0 if vocab % 2 else 3)


def test_beam_select_many_rows(hip):
    """So many rows that a wave takes several tiles of one."""
    rng = np.random.default_rng(4)
    logits = (3 * rng.standard_normal((320, 40000))).astype(np.float32)
    for k in (8, 16):
        _check_beams(hip, logits, -2 * rng.random(320), None, rng.permutation(320) if k == 8 else None, 8, k, native.F32)


def test_beam_select_parts_of_many_tiles(hip):
    """A wave's part in more tiles than it looks at together; rows among them that rise, and rows of few different values."""
    rng = np.random.default_rng(5)
    logits = rng.standard_normal((3104, 9000), dtype=np.float32)
    logits[::7].sort(axis=1)
    logits[3::7] = np.round(logits[3::7])
    _check_beams(hip, logits, -2 * rng.random(3104), None, rng.permutation(3104), 16, 16, native.F32)


@pytest.mark.parametrize("fmt", FORMATS)
def test_beam_select_ties(hip, fmt):
    """Equal logits, equal beams, zeros of both signs: the lowest first; more equal values than are ranked together."""
    rng = np.random.default_rng(6)
    for vocab in (700, 4500):
        logits = rng.integers(-2, 3, (8, vocab)).astype(np.float32)
        logits[4:] = logits[4]
        logits[4:, 5::3] *= -1.0
        logits[4:] = np.where(logits[4:] == 0, np.where(np.arange(vocab) % 2, 0.0, -0.0), logits[4:])
        scores = np.array([-1, -1, -2, -1, -3, -3, -3, -3], np.float32)
        _check_beams(hip, logits, scores, None, np.arange(8), 4, 4, fmt)
        _check_beams(hip, np.zeros_like(logits), scores, None, None, 4, 32, fmt)
        _check_beams(hip, np.sort(logits, 1), scores, None, None, 4, 7, fmt)


def test_beam_select_equal_over_many_parts(hip):
    """More equal logits over a row's parts than are ranked together; parts of them masked; one beam's tokens before the next's."""
    logits = np.zeros((4, 70000), np.float32)
    logits[1, :65000] = -np.inf
    logits[2, ::3] = 1.0
    logits[3] = np.arange(70000) // 7000
    _check_beams(hip, logits, np.array([-1, -1, -2, -2]), None, None, 2, 32, native.F32)
    _check_beams(hip, logits, np.array([-1, -1, -1, -1]), None, np.arange(4), 4, 4, native.F16)
    _check_beams(hip, logits[:, ::-1], np.zeros(4), None, None, 4, 29, native.BF16)


@pytest.mark.parametrize("fmt", FORMATS)
def test_beam_select_masks(hip, fmt):
    """Masked logits (-infinity, and the type's lowest), rows with nothing left, beams that are none, NaN and infinity."""
    rng = np.random.default_rng(7)
    low = {native.F32: -3.0e38, native.F16: -65504.0, native.BF16: -3.0e38}[fmt]
    logits = (2 * rng.standard_normal((16, 3000))).astype(np.float32)
    logits[0, 100:] = -np.inf
    logits[1] = -np.inf
    logits[2, :2990] = low
    logits[3] = low
    logits[4, 77] = np.nan
    logits[5, 2500] = np.inf
    logits[6, 3:] = -np.inf
    logits[8:12] = -np.inf
    logits[9, 5] = 1.0
    logits[12:] = -np.inf
    scores = -rng.random(16)
    scores[7] = -np.inf
    scores[14] = np.nan
    for k in (4, 8, 32):
        _check_beams(hip, logits, scores, None, np.arange(16)[::-1].copy() if k == 4 else None, 4, k, fmt)


def test_beam_select_ended_beams(hip):
    rng = np.random.default_rng(8)
    logits = (2 * rng.standard_normal((24, 900))).astype(np.float32)
    logits[:, 17] += 6   # the end token is likely
    scores = -3 * rng.random(24)
    done = (rng.random(24) < 0.4).astype(np.int32)
    done[8:16] = 1
    logits[9] = np.nan   # an ended beam's logits are not looked at
    scores[10] = -np.inf
    for in_place in (False, True):
        _check_beams(hip, logits, scores, done, np.arange(24), 8, 8, native.F32, end_token=17, in_place=in_place)
    _check_beams(hip, logits, scores, done, None, 8, 3, native.BF16, end_token=899)


# ---- slot moves ----------------------------------------------------------------------------------------

@pytest.mark.parametrize("sizes", [[1], [1000, 24, 1024], [2500, 16, 4096], [3, 17, 16384], [16, 16400, 40000, 16384 * 3 + 5], [4097] * 70])
@pytest.mark.parametrize("shift", [0, 1, 4])
def test_copy_slots(hip, sizes, shift):
    rng = np.random.default_rng(len(sizes))
    slots = 9
    host = [rng.integers(0, 256, (slots, n), dtype=np.uint8) for n in sizes]
    dev = []
    for a in host:
        b = _guarded(hip, a.nbytes + shift)
        b.upload(a, shift)
        dev.append(b)
    source, to = [4, 4, 7, -1, 2, 9, 8, 5], [0, 1, 7, 3, -1, 6, 12, 2]
    ds, dt = _i32(hip, source), _i32(hip, to)
    hip.copy_slots(native.slot_arrays([(b.ptr + shift, n) for b, n in zip(dev, sizes)]), slots, ds.ptr, dt.ptr, len(to))
    for a, b in zip(host, dev):
        want = a.copy()
        want[0], want[1], want[2] = a[4], a[4], a[5]
        assert np.array_equal(b.readback(np.uint8, a.nbytes, shift).reshape(a.shape), want)
        _spare_untouched(b, a.nbytes + shift)
        if shift:
            assert np.all(b.readback(np.uint8, shift) == FILL)
        b.free()


# ---- recorded, far and beside one another ---------------------------------------------------------------

def test_recorded_calls_read_their_arrays_at_each_replay(hip):
    """A plan of all four operators, replayed with other row starts, slots and values, beside eager work."""
    rng = np.random.default_rng(12)
    heads, rows, slots, n = 2, 300, 6, 128
    plans, held = [], []

    def new(x):
        held.append(hip.to_device(x))
        return held[-1]
    inp = _wkv_inputs(rng, rows, heads, False, slots)
    dev = {k: new(v) for k, v in inp.items()}
    starts, source, to = new(np.zeros(4, np.int32)), new(np.zeros(3, np.int32)), new(np.zeros(3, np.int32))
    batch = native.RowBatch(starts.ptr, source.ptr, to.ptr, 3, slots, rows, rows)
    x = _mix_inputs(rng, rows, n, 2, False, slots)
    mix = {k: new(v) for k, v in x.items() if v is not None}
    mixed, out = hip.alloc(2 * rows * n * 4), hip.alloc(rows * n * 4)
    ws = hip.alloc(native.rwkv7_wkv_rows_workspace_bytes(heads))
    beam_ws = hip.alloc(native.beam_select_workspace_bytes(1, 4, 4, n))
    scores, slot = new(np.zeros(4, np.float32)), new(np.arange(4, dtype=np.int32))
    picked = {k: new(np.zeros(4, np.int32)) for k in ("parents", "tokens", "from")}

    def body():
        hip.layernorm_mix_rows(native.LayernormMixRowsArgs(batch, mix["x"].ptr, 0, mix["weight"].ptr, mix["bias"].ptr, mix["mix"].ptr,
                                                           mix["state"].ptr, 0, mixed.ptr, n, 2, native.F32, 1e-5))
        hip.rwkv7_wkv_rows(native.Rwkv7WkvRowsArgs(batch, heads, 0, *[dev[k].ptr for k in native.RWKV7_WKV_VECTORS],
                                                   dev["v_first"].ptr, dev["state"].ptr, out.ptr, ws.ptr, native.F32))
        # the first rows of the mixed ones as logits; the slots of beams move in place
        hip.beam_select(native.BeamSelectArgs(mixed.ptr, scores.ptr, 0, slot.ptr, picked["parents"].ptr, picked["tokens"].ptr,
                                              scores.ptr, 0, picked["from"].ptr, slot.ptr, beam_ws.ptr, n, n, 1, 4, 4, native.F32, -1))
        hip.copy_slots(native.slot_arrays([(mix["state"].ptr, 4 * n)]), slots, picked["from"].ptr, slot.ptr, 4)
    plan = hip.record(body)
    state, shift = inp["state"].copy(), x["state"].copy()
    given, beam_slots = np.zeros(4, np.float32), np.arange(4)
    for turn, (at, a, b) in enumerate((([0, 40, 40, 300], [0, 1, 2], [0, 1, 2]), ([0, 250, 255, 270], [3, -1, 4], [5, 0, 4]),
                                       ([0, 0, 290, 300], [1, 2, 5], [1, 2, 3]), ([0, 1, 2, 6], [4, 4, 4], [0, 1, 2]))):
        starts.upload(np.asarray(at, np.int32))
        source.upload(np.asarray(a, np.int32))
        to.upload(np.asarray(b, np.int32))
        scale = np.float32(1 + turn)
        dev["r"].upload(inp["r"] * scale)
        plan.launch()
        now = {**inp, "r": inp["r"] * scale, "state": state}
        want, bound, after, off = ref.wkv_rows(now, heads, False, at, a, b)
        live = np.isfinite(want)
        got = out.readback(np.float32).reshape(rows, n)
        assert np.all(np.abs(got - want)[live] <= bound[live] + 1e-30)
        new_state = dev["state"].readback(np.float32).reshape(inp["state"].shape)
        assert np.all(np.linalg.norm(new_state.astype(np.float64) - after, axis=(2, 3)) <= off + 1e-30)
        state = new_state
        _, mixes, mix_off, rows_kept, kept_off, _ = ref.mix_rows(x["x"], None, x["weight"], x["bias"], x["mix"], shift, at, a, b, 1e-5)
        got = mixed.readback(np.float32).reshape(2, rows, n)
        live = np.isfinite(mixes)
        assert np.all(np.abs(got - mixes)[live] <= mix_off[live] + 1e-30)
        if at[-1] >= 4 and at[0] == 0:
            best = ref.beam_select(got[0, :4].astype(np.float64), given, None, beam_slots, 4, 4, -1)
            assert np.array_equal(picked["parents"].readback(np.int32), best["parents"])
            assert np.array_equal(picked["tokens"].readback(np.int32), best["tokens"])
            beam_slots = slot.readback(np.int32)
            assert np.array_equal(beam_slots, best["to"])
            given = scores.readback(np.float32)
            for f, t in zip(best["from"], best["to"]):
                rows_kept[t], kept_off[t] = rows_kept[f].copy(), kept_off[f].copy()
        shift = mix["state"].readback(np.float32).reshape(slots, n)
        assert np.all(np.abs(shift - rows_kept) <= kept_off + 1e-30)
    plan.destroy()
    for b in [*held, mixed, out, ws, beam_ws]:
        b.free()


def test_rows_and_slots_far_into_their_arrays(hip):
    """Rows and slots more than 4 GiB into their buffers, logits more than 2."""
    rng = np.random.default_rng(13)
    # 540000 rows of 32 heads: 4.4 GB an array; only the last 43 are sequences' rows, and slot 8600 is 4.5 GB into the states
    heads, rows, slots, tail = 32, 540000, 8601, 43
    width = heads * 64
    inp = _wkv_inputs(rng, tail, heads, False, 1)
    dev, held = {}, []
    for k, v in inp.items():
        in_rows = v.ndim == 2
        b = hip.alloc(rows * width * 4 if in_rows else slots * v.nbytes if k == "state" else v.nbytes)
        b.upload(v, (rows - tail) * width * 4 if in_rows else (slots - 1) * v.nbytes if k == "state" else 0)
        dev[k] = b
    starts = np.array([rows - tail, rows - 40, rows], np.int32)
    batch, held = _batch(hip, starts, [slots - 1, slots - 1], [slots - 2, slots - 3], slots, rows, 40)
    out, ws = hip.alloc(rows * width * 4), hip.alloc(native.rwkv7_wkv_rows_workspace_bytes(heads))
    hip.rwkv7_wkv_rows(native.Rwkv7WkvRowsArgs(batch, heads, 0, *[dev[k].ptr for k in native.RWKV7_WKV_VECTORS],
                                               dev["v_first"].ptr, dev["state"].ptr, out.ptr, ws.ptr, native.F32))
    want, bound, state, off = ref.wkv_rows({**inp, "state": np.repeat(inp["state"], 3, 0)}, heads, False, [0, 3, tail], [0, 0], [1, 2])
    got = out.readback(np.float32, tail * width, (rows - tail) * width * 4).reshape(tail, width)
    _near(got, want, bound)
    size = width * 64
    for i, slot in ((1, slots - 2), (2, slots - 3)):
        s = dev["state"].readback(np.float32, size, slot * size * 4).reshape(heads, 64, 64)
        assert np.all(np.linalg.norm(s - state[i], axis=(1, 2)) <= off[i])
    # the same rows, mixed (their state 8600 slots in, too)
    x = _mix_inputs(rng, tail, width, 1, False, 1)
    small = [hip.to_device(x[k]) for k in ("weight", "bias", "mix")]
    dev["r"].upload(x["x"], (rows - tail) * width * 4)
    shift = hip.alloc(slots * width * 4)
    shift.upload(x["state"], (slots - 1) * width * 4)
    hip.layernorm_mix_rows(native.LayernormMixRowsArgs(batch, dev["r"].ptr, 0, *[b.ptr for b in small], shift.ptr, 0, out.ptr, width,
                                                       1, native.F32, 1e-5))
    want, bound = ref.mix_rows(x["x"], None, x["weight"], x["bias"], x["mix"], np.repeat(x["state"], 3, 0), [0, 3, tail], [0, 0],
                               [1, 2], 1e-5)[1:3]
    _near(out.readback(np.float32, tail * width, (rows - tail) * width * 4).reshape(1, tail, width), want, bound)
    # logits: four rows 1.2 GB apart
    logits = (2 * rng.standard_normal((4, 3000))).astype(np.float32)
    stride = 300_000_000
    for i in range(4):
        out.upload(logits[i], 4 * stride * i) if 4 * (stride * i + 3000) <= out.nbytes else None
    assert 4 * (3 * stride + 3000) <= out.nbytes and 4 * 3 * stride > 1 << 31
    scores, ids = hip.to_device(np.zeros(4, np.float32)), [hip.alloc(16) for _ in range(3)]
    hip.beam_select(native.BeamSelectArgs(out.ptr, scores.ptr, 0, 0, ids[0].ptr, ids[1].ptr, ids[2].ptr, 0, 0, 0, ws.ptr, 3000, stride,
                                          1, 4, 4, native.F32, -1))
    best = ref.beam_select(logits.astype(np.float64), np.zeros(4), None, None, 4, 4, -1)
    assert np.array_equal(ids[0].readback(np.int32), best["parents"]) and np.array_equal(ids[1].readback(np.int32), best["tokens"])
    # a slot 4.5 GB into the states onto the first one
    pair = [_i32(hip, [slots - 2]), _i32(hip, [0])]
    hip.copy_slots(native.slot_arrays([(dev["state"].ptr, size * 4)]), slots, pair[0].ptr, pair[1].ptr, 1)
    assert np.array_equal(dev["state"].readback(np.uint8, size * 4), dev["state"].readback(np.uint8, size * 4, (slots - 2) * size * 4))
    for b in [*dev.values(), *held, out, ws, shift, scores, *ids, *pair, *small]:
        b.free()


def test_refusals(hip):
    """Everything that a call refuses, before anything is launched."""
    b = hip.alloc(1 << 20)
    far = [hip.alloc(1 << 16) for _ in range(24)]
    f = [x.ptr for x in far]
    A, U = native.ERR_ARGUMENT, native.ERR_UNSUPPORTED

    def refused(call, args, status):
        with pytest.raises(native.HipError) as e:
            call(args)
        assert e.value.status == status, e.value

    def changed(make, base, changes):
        for change, status in changes:
            yield make({**base, **change}), status, change
    rows = dict(row_starts=f[0], from_=f[1], to=f[2], sequences=2, slots=3, rows=4, max_rows=4)
    batches = [(dict(row_starts=0), A), (dict(row_starts=f[0] + 2), A), (dict(from_=0), A), (dict(to=0), A), (dict(sequences=0), A),
               (dict(sequences=4097), A), (dict(slots=0), A), (dict(rows=0), A), (dict(rows=(1 << 20) + 1), A), (dict(max_rows=0), A),
               (dict(max_rows=5), A)]
    mix = dict(batch=native.RowBatch(**rows), x=f[3], residual=0, weight=f[4], bias=f[5], mix=f[6], state=f[7], updated=0, output=f[8],
               n=64, mixes=2, output_format=native.BF16, eps=1e-5)
    make_mix = lambda a: native.LayernormMixRowsArgs(**a)
    for change, status in batches:
        refused(hip.layernorm_mix_rows, make_mix({**mix, "batch": native.RowBatch(**{**rows, **change})}), status)
    for args, status, _ in changed(make_mix, mix, [
            (dict(x=0), A), (dict(x=f[3] + 1), A), (dict(weight=0), A), (dict(bias=0), A), (dict(mix=0), A), (dict(state=0), A),
            (dict(output=0), A), (dict(output=f[8] + 1), A), (dict(n=0), A), (dict(n=8193), A), (dict(mixes=-1), A), (dict(mixes=9), A),
            (dict(eps=-1.0), A), (dict(eps=float("nan")), A), (dict(eps=float("inf")), A), (dict(output_format=native.Q8_0), U),
            (dict(residual=f[9]), A), (dict(updated=f[9]), A), (dict(output=f[3]), A), (dict(state=f[3]), A), (dict(state=f[8]), A),
            (dict(residual=f[9], updated=f[3]), A), (dict(residual=f[9], updated=f[9]), A), (dict(output=f[0]), A)]):
        refused(hip.layernorm_mix_rows, args, status)
    names = native.RWKV7_WKV_VECTORS
    big = hip.alloc(native.rwkv7_wkv_rows_workspace_bytes(1))
    wkv = dict(batch=native.RowBatch(**rows), heads=1, first_layer=0, **{n: f[3 + i] for i, n in enumerate(names)}, v_first=f[18],
               state=f[19], output=f[20], workspace=big.ptr, output_format=native.F32)
    make_wkv = lambda a: native.Rwkv7WkvRowsArgs(**a)
    for change, status in batches:
        refused(hip.rwkv7_wkv_rows, make_wkv({**wkv, "batch": native.RowBatch(**{**rows, **change})}), status)
    for args, status, _ in changed(make_wkv, wkv, [(dict(heads=0), A), (dict(heads=1025), A), (dict(output_format=native.Q4_0), U),
                                                   (dict(output=f[20] + 4), A), (dict(state=f[19] + 8), A), (dict(workspace=0), A),
                                                   (dict(workspace=big.ptr + 8), A), (dict(v_first=0), A), (dict(output=f[3]), A),
                                                   (dict(state=f[18]), A), (dict(workspace=f[3]), A), (dict(output=f[18]), A),
                                                   (dict(first_layer=1, v_first=f[5]), A)] +
                                   [(dict([(n, 0)]), A) for n in names] + [(dict([(n, f[3 + i] + 2)]), A) for i, n in enumerate(names)]):
        refused(hip.rwkv7_wkv_rows, args, status)
    beam = dict(logits=f[0], scores=f[1], done=f[2], slots=f[3], parents=f[4], tokens=f[5], new_scores=f[6], new_done=f[7], from_=f[8],
                to=f[9], workspace=b.ptr, vocab=100, stride=100, sequences=2, beams=4, candidates=4, logits_format=native.F16, end_token=3)
    for args, status, _ in changed(lambda a: native.BeamSelectArgs(**a), beam, [
            (dict(vocab=0), A), (dict(vocab=(1 << 21) + 1, stride=1 << 22), A), (dict(stride=99), A), (dict(stride=(1 << 32) + 1), A),
            (dict(sequences=0), A), (dict(sequences=16385), A), (dict(beams=0), A), (dict(beams=17), A), (dict(candidates=0), A),
            (dict(candidates=33), A), (dict(candidates=5), A), (dict(logits_format=native.Q8_0), U), (dict(end_token=-2), A),
            (dict(end_token=100), A), (dict(end_token=-1), A), (dict(slots=0), A), (dict(logits=0), A), (dict(logits=f[0] + 1), A),
            (dict(scores=0), A), (dict(done=f[2] + 1), A), (dict(parents=0), A), (dict(tokens=0), A), (dict(new_scores=0), A),
            (dict(from_=0), A), (dict(to=0), A), (dict(workspace=0), A), (dict(workspace=b.ptr + 4), A), (dict(parents=f[4], tokens=f[4]), A),
            (dict(tokens=f[0]), A), (dict(from_=f[3]), A), (dict(new_scores=f[1] + 4), A), (dict(new_done=f[1]), A),
            (dict(workspace=f[0]), A)]):
        refused(hip.beam_select, args, status)
    for arrays, slots, source, to, moves in (([], 3, f[1], f[2], 1), ([(0, 4)], 3, f[1], f[2], 1), ([(f[0], 0)], 3, f[1], f[2], 1),
                                             ([(f[0], (1 << 36) + 1)], 3, f[1], f[2], 1), ([(f[0], 4)], 0, f[1], f[2], 1),
                                             ([(f[0], 4)], 1 << 31, f[1], f[2], 1), ([(f[0], 4)], 3, 0, f[2], 1),
                                             ([(f[0], 4)], 3, f[1], f[2] + 1, 1), ([(f[0], 4)], 3, f[1], f[2], 0),
                                             ([(f[0], 4)], 3, f[1], f[2], (1 << 20) + 1), ([(f[0], 4), (f[0] + 8, 4)], 3, f[1], f[2], 1),
                                             ([(f[0], 4)], 3, f[0] + 8, f[2], 1), ([(f[0], 4)], 3, f[1], f[0], 1),
                                             ([(f[0], 1)] * 4097, 3, f[1], f[2], 1)):
        with pytest.raises(native.HipError) as e:
            hip.copy_slots(native.slot_arrays(arrays), slots, source, to, moves)
        assert e.value.status == A
    for x in [b, big, *far]:
        x.free()
