"""CPU checks of the operators over many sequences: what is refused without a device, and the 64-bit references that the
GPU tests compare with (against the oracle and against plain enumeration; mistakes planted in them pass their bounds)."""
import ctypes

import numpy as np
import pytest

import oracle as orc
from sharpinference_amd import native
from tests import sequences_reference as ref


@pytest.mark.parametrize("args", [(0, 4, 4, 100), (1, 0, 4, 100), (1, 17, 4, 100), (1, 4, 0, 100), (1, 4, 33, 100), (1, 4, 4, 0),
                                  (1, 4, 4, (1 << 21) + 1), (16385, 4, 4, 100)])
def test_beam_workspace_refusals(args):
    with pytest.raises(native.HipError) as e:
        native.beam_select_workspace_bytes(*args)
    assert e.value.status == native.ERR_ARGUMENT


@pytest.mark.parametrize("heads", [0, -1, 1025])
def test_wkv_workspace_refusals(heads):
    with pytest.raises(native.HipError) as e:
        native.rwkv7_wkv_rows_workspace_bytes(heads)
    assert e.value.status == native.ERR_ARGUMENT


def test_calls_without_a_context_or_an_output():
    lib = native.lib()
    for call in (lib.si_hip_layernorm_mix_rows, lib.si_hip_rwkv7_wkv_rows, lib.si_hip_beam_select):
        assert call(None, None) == native.ERR_ARGUMENT
        assert b"null context" in lib.si_hip_last_error(None)
    assert lib.si_hip_copy_slots(None, None, 0, 1, None, None, 1) == native.ERR_ARGUMENT
    assert lib.si_hip_rwkv7_wkv_rows_workspace_bytes(1, None) == native.ERR_ARGUMENT
    assert lib.si_hip_beam_select_workspace_bytes(1, 1, 1, 1, None) == native.ERR_ARGUMENT


def test_workspaces_follow_the_shapes():
    assert native.beam_select_workspace_bytes(1, 4, 4, 65536) < 1 << 20
    assert native.beam_select_workspace_bytes(2, 16, 32, 200064) < 1 << 25
    assert {native.rwkv7_wkv_rows_workspace_bytes(h) for h in (1, 32, 1024)} == {native.rwkv7_wkv_rows_workspace_bytes(12)}


def test_argument_structures_are_the_headers():
    """Sizes of the C structures (x86-64): pointers 8, int32 and float 4."""
    assert ctypes.sizeof(native.RowBatch) == 40
    assert ctypes.sizeof(native.LayernormMixRowsArgs) == 40 + 8 * 8 + 16
    assert ctypes.sizeof(native.Rwkv7WkvRowsArgs) == 40 + 8 + 15 * 8 + 4 * 8 + 8
    assert ctypes.sizeof(native.BeamSelectArgs) == 11 * 8 + 16 + 20 + 4
    assert ctypes.sizeof(native.SlotArray) == 16


def _inputs(rng, rows, heads, first):
    c = heads * ref.HEAD
    f = lambda *s: rng.standard_normal(s).astype(np.float32)
    return dict(r=f(rows, c), k=f(rows, c), v=f(rows, c), w_lora=f(rows, c), a_lora=f(rows, c), gate=f(rows, c),
                v_lora=None if first else f(rows, c), w0=f(c), a0=f(c), v0=None if first else f(c), k_k=1 + 0.1 * f(c), k_a=f(c),
                r_k=0.1 * f(c), lnx_weight=f(c), lnx_bias=f(c), v_first=f(rows, c), state=0.3 * f(2, heads, 64, 64))


def test_scan_reference_is_the_oracles_update():
    rng = np.random.default_rng(1)
    heads, rows = 2, 5
    inp = _inputs(rng, rows, heads, True)
    _, _, state, _ = ref.wkv_rows(inp, heads, True, [0, rows], [0], [1])
    S = inp["state"][0].copy()
    sig = lambda x: (1 / (1 + np.exp(-x.astype(np.float64)))).astype(np.float32)
    for t in range(rows):
        decay = np.exp(-0.606531 * sig(inp["w_lora"][t] + inp["w0"])).astype(np.float32)
        a = sig(inp["a_lora"][t] + inp["a0"])
        sk = (inp["k"][t] * inp["k_k"]).reshape(heads, 64)
        kn = (sk / np.linalg.norm(sk, axis=1, keepdims=True)).astype(np.float32).reshape(-1)
        key = (inp["k"][t] * (1 + (a - 1) * inp["k_a"])).astype(np.float32)
        orc.rwkv7_wkv_update(S, inp["r"][t], decay, key, inp["v"][t], kn, a)
    assert np.allclose(S, state[1], rtol=1e-4, atol=1e-4)


@pytest.mark.parametrize("name,change", [("k_a", lambda x: 0 * x), ("w0", lambda x: x + 0.01), ("a0", lambda x: x - 0.01),
                                         ("r_k", lambda x: 1.01 * x), ("gate", lambda x: 1.0001 * x), ("k_k", lambda x: x[::-1])])
def test_scan_bounds_catch_mistakes(name, change):
    """A mistake in one factor moves outputs or state past the bounds."""
    rng = np.random.default_rng(2)
    inp = _inputs(rng, 40, 1, False)
    out, bound, state, off = ref.wkv_rows(inp, 1, False, [0, 40], [0], [1])
    wrong, _, wrong_state, _ = ref.wkv_rows({**inp, name: np.ascontiguousarray(change(inp[name]), np.float32)}, 1, False, [0, 40], [0], [1])
    moved = np.linalg.norm(wrong_state[1] - state[1]) > off[1, 0]
    assert moved or np.any(np.abs(wrong - out) > bound)


def test_mix_reference_is_the_oracles_layernorm():
    rng = np.random.default_rng(3)
    x = rng.standard_normal((4, 200)).astype(np.float32)
    w, b, m = (rng.standard_normal(200).astype(np.float32) for _ in range(3))
    state = rng.standard_normal((2, 200)).astype(np.float32)
    _, out, bound, held, _, _ = ref.mix_rows(x, None, w, b, m[None], state, [0, 1, 4], [1, -1], [0, 1], 1e-5)
    n = np.stack([orc.layernorm(r, w, b, 1e-5) for r in x]).astype(np.float64)
    before = np.stack([state[1], np.zeros(200), n[1], n[2]])
    assert np.allclose(out[0], n + (before - n) * m, rtol=1e-4, atol=1e-5)
    assert np.allclose(held, [n[0], n[3]], rtol=1e-5, atol=1e-5)
    assert np.all(bound < 1e-4)
    shifted = ref.mix_rows(x, None, w, b, m[None], state, [0, 4], [1], [0], 1e-5)[1]   # one sequence in place of two
    assert np.any(np.abs(shifted - out) > bound)


def test_beam_reference_against_enumeration():
    rng = np.random.default_rng(4)
    for _ in range(20):
        beams, vocab, k = int(rng.integers(1, 5)), int(rng.integers(1, 7)), int(rng.integers(1, 9))
        x = rng.integers(-2, 3, (beams, vocab)).astype(np.float64)
        x[rng.random((beams, vocab)) < 0.2] = -np.inf
        scores = -rng.integers(0, 3, beams).astype(np.float64)
        got = ref.beam_select(x, scores, None, None, beams, k, -1)
        every = []
        for b in range(beams):
            for t in range(vocab):
                if np.isfinite(x[b, t]):
                    m = x[b].max()
                    every.append((scores[b] + (x[b, t] - m) - np.log(np.exp(x[b] - m).sum()), b, t))
        every.sort(key=lambda e: (-e[0], e[1], e[2]))
        every = every[:k]
        assert got["parents"].tolist() == [e[1] for e in every] + [-1] * (k - len(every))
        assert got["tokens"].tolist() == [e[2] for e in every] + [-1] * (k - len(every))
        assert np.allclose(got["scores"][:len(every)], [e[0] for e in every])


def test_beam_reference_hands_slots_on():
    # beam 0 has no candidates left, beam 2 three: its first keeps slot 7, the others take 5 and 6 in order
    x = np.full((3, 4), -np.inf)
    x[2] = [0, 3, 2, 1]
    got = ref.beam_select(x, np.zeros(3), None, [5, 6, 7], 3, 3, -1)
    assert got["parents"].tolist() == [2, 2, 2] and got["tokens"].tolist() == [1, 2, 3]
    assert got["from"].tolist() == [7, 7, 7] and got["to"].tolist() == [7, 5, 6]
    # nothing at all: every slot stays somebody's
    got = ref.beam_select(np.full((3, 4), -np.inf), np.zeros(3), None, [5, 6, 7], 3, 3, -1)
    assert got["parents"].tolist() == [-1] * 3 and got["from"].tolist() == [-1] * 3 and got["to"].tolist() == [5, 6, 7]
