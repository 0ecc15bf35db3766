"""The time-mix core at the ends of its inputs' range, against 64-bit numpy with the bounds of tests/sequences_reference.py."""
import numpy as np
import pytest

from sharpinference_amd import native
from tests import sequences_reference as ref
from tests.test_sequences_gpu import _near, _run_wkv, _wkv_inputs

pytestmark = pytest.mark.gpu

# The references' bounds are relative.  A FP32 result under 2^-126 is off by up to 2^-150 whatever its size: at the fastest decay
# (0.545 a row) a value of the state, whose up to 8 operations a row may each be off by that, by at most 8 / (1 - 0.545) * 2^-150,
# under 2^-145, and a head's 64 * 64 values, by their root of the sum of squares, by 64 times as much.
UNDERFLOW = 64 * 2.0 ** -145


def _check(hip, inp, heads, count, underflow=0.0):
    """One sequence of every row, from slot 1 into slot 2."""
    raw, state, _ = _run_wkv(hip, inp, heads, False, [0, count], [1], [2], native.F32)
    want, bound, want_state, off = ref.wkv_rows(inp, heads, False, [0, count], [1], [2])
    _near(ref.values(raw.reshape(-1), native.F32).reshape(count, -1), want, bound + ref.STEP[native.F32] * np.abs(want))
    assert np.isfinite(state).all()
    assert np.all(np.linalg.norm(state.astype(np.float64) - want_state, axis=(2, 3)) <= off + underflow)


@pytest.mark.parametrize("count,at", [(6, 4), (16, 14), (40, 30), (400, 30), (400, 254)])
def test_large_key_before_a_large_readout(hip, count, at):
    """A row whose k * k_k is near 2^60.5 (its square's sum fits FP32) and the next one's r near 2^63.7, at the fastest
    decay: the sum of their products passes FP32, which no value of the formulas does.  key = k (1 + (a - 1) k_a) is 0
    throughout, so nothing of that size enters the state."""
    rng = np.random.default_rng(count)
    inp = _wkv_inputs(rng, count, 2, False, 3)
    inp["w_lora"][:] = 30.0
    inp["a0"][:] = 0.0
    inp["a_lora"][:] = 0.0     # a is 1/2, exactly
    inp["k_a"][:] = 2.0
    inp["k_k"][:] = 1.0
    inp["k"][at] = np.float32(2.0 ** 60) * np.sign(inp["k"][at]) * (1.4 + 0.2 * rng.random(128).astype(np.float32))
    inp["r"][at] = 0.0
    inp["r"][at + 1] = np.sign(inp["k"][at]) * np.float32(2.0 ** 63.4) * (1 + 0.4 * rng.random(128).astype(np.float32))
    inp["state"] *= np.float32(1e-6)
    _check(hip, inp, 2, count, UNDERFLOW)


@pytest.mark.parametrize("count", [1, 5, 13, 20, 33, 400])
def test_decays_at_both_ends(hip, count):
    """w0 of plus and minus infinity: the fastest decay and none, in every row (and in no row that a block does not have)."""
    rng = np.random.default_rng(count)
    inp = _wkv_inputs(rng, count, 2, False, 3)
    inp["w0"][3::7] = np.inf
    inp["w0"][5::7] = -np.inf
    _check(hip, inp, 2, count)
