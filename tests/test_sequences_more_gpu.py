"""More of the operators over many sequences, beside tests/test_sequences_gpu.py: sizes that wrap, what falling starts leave
alone, cut sequences of a first layer and with 16-bit outputs, 16-bit logits in several groups of tiles."""
import numpy as np
import pytest

from sharpinference_amd import native
from tests import sequences_reference as ref
from tests.test_sequences_gpu import (FILL, FORMATS, _check_beams, _check_wkv, _lay, _mix_inputs, _run_mix, _run_wkv,
                                      _wkv_inputs)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("size,slots", [(1 << 36, 1 << 28), ((1 << 36) - 4096, (1 << 31) - 1), (1 << 35, (1 << 29) + 1),
                                        (1 << 33, (1 << 31) - 1)])
def test_copy_slots_beyond_the_address_space(hip, size, slots):
    """slots * slot_bytes at 2^64 and beyond (modulo that, these arrays would be small or lie anywhere): refused."""
    b = hip.alloc(1 << 16)
    pair = [hip.to_device(np.full(1, -1, np.int32)) for _ in range(2)]
    with pytest.raises(native.HipError) as e:
        hip.copy_slots(native.slot_arrays([(b.ptr, size)]), slots, pair[0].ptr, pair[1].ptr, 1)
    assert e.value.status == native.ERR_ARGUMENT
    for x in [b, *pair]:
        x.free()


@pytest.mark.parametrize("heads,counts", [(1, [1500]), (2, [700, 90, 1, 260]), (5, [333, 13, 901])])
@pytest.mark.parametrize("first,fmt", [(True, native.BF16), (True, native.F16), (True, native.F32), (False, native.BF16),
                                       (False, native.F16)])
def test_wkv_rows_cut(hip, heads, counts, first, fmt):
    """Sequences cut into stretches: the first layer's values, which two passes write, and 16-bit outputs."""
    rng = np.random.default_rng(heads * 11 + len(counts))
    starts, source, to, slots, rows = _lay(rng, counts, tail=2)
    _check_wkv(hip, _wkv_inputs(rng, rows, heads, first, slots), heads, first, starts, source, to, fmt)


@pytest.mark.parametrize("starts", [[0, 600, 300, 640], [0, 200, 150, 500], [0, 700, 500], [-4, 300, 500], [500, 20], [0, 30, 20, 600],
                                    [9, 3, 12, 5]])
@pytest.mark.parametrize("most", [8, 640])
def test_wkv_rows_outside_of_falling_starts(hip, starts, most):
    """Rows and slots of no sequence whose starts rise within the rows stay as they are."""
    rng = np.random.default_rng(len(starts))
    n = len(starts) - 1
    inp = _wkv_inputs(rng, 640, 2, True, 2 * n)
    raw, state, v_first = _run_wkv(hip, inp, 2, True, starts, range(n), range(n, 2 * n), native.F32, most)
    outside, untouched = np.ones(640, bool), np.ones(2 * n, bool)
    for s, a, b in ref.spans(starts, 640):
        outside[a:b] = False
        untouched[n + s] = False
    assert np.all(raw[outside] == FILL)
    assert np.array_equal(v_first[outside], inp["v_first"][outside])
    assert np.array_equal(state[untouched], inp["state"][untouched])


def _specials(x):
    return np.where(np.isnan(x), 2, np.where(np.isinf(x), np.sign(x), 0))


@pytest.mark.parametrize("fmt", FORMATS)
def test_mix_rows_what_is_not_finite(hip, fmt):
    """NaN is NaN and an infinity one of the same sign, value by value: rows that go on from no slot, infinite mixes, biases."""
    rng = np.random.default_rng(21)
    starts, slots, n, rows = [0, 4, 9, 10], 4, 130, 10
    inp = _mix_inputs(rng, rows, n, 3, True, slots)
    inp["mix"][1, 7] = np.inf
    inp["bias"][9] = -np.inf
    inp["x"][6, 2] = np.nan
    inp["state"][1, 3] = np.inf
    with np.errstate(all="ignore"):
        _, want, _, held, _, _ = ref.mix_rows(inp["x"], inp["residual"], inp["weight"], inp["bias"], inp["mix"], inp["state"], starts,
                                              [5, 1, -1], [0, 2, 3], 1e-5)
        _, raw, state = _run_mix(hip, inp, starts, [5, 1, -1], [0, 2, 3], slots, fmt)
        got = ref.values(raw, fmt).reshape(want.shape)
    assert np.array_equal(_specials(got), _specials(want))
    assert np.array_equal(_specials(state), _specials(held))


@pytest.mark.parametrize("count,at", [(6, 3), (50, 21), (300, 170)])
def test_wkv_rows_infinite_gates_and_biases(hip, count, at):
    """An infinity behind the normalisation stays in its value, with its sign."""
    rng = np.random.default_rng(at)
    inp = _wkv_inputs(rng, count, 2, False, 2)
    inp["gate"][at, 70], inp["gate"][at - 1, 5] = np.inf, -np.inf
    inp["lnx_bias"][9], inp["lnx_bias"][80] = np.inf, -np.inf
    raw, state, _ = _run_wkv(hip, inp, 2, False, [0, count], [0], [1], native.F32)
    with np.errstate(all="ignore"):
        want = ref.wkv_rows(inp, 2, False, [0, count], [0], [1])[0]
    assert np.array_equal(_specials(raw.view(np.float32)), _specials(want))
    assert np.isfinite(state).all()


@pytest.mark.parametrize("fmt", [native.F16, native.BF16])
def test_beam_select_16_bit_parts_of_many_tiles(hip, fmt):
    """More tiles a part than a wave looks at together; rows that rise, so that every group replaces the list, rows that fall,
    rows of few different values."""
    rng = np.random.default_rng(fmt)
    logits = rng.standard_normal((4096, 14000), dtype=np.float32)
    logits[::64].sort(axis=1)
    logits[1::64] = -np.sort(-logits[1::64], axis=1)
    logits[2::5] = np.round(logits[2::5])
    _check_beams(hip, logits, -2 * rng.random(4096), None, rng.permutation(4096), 16, 16, fmt)
