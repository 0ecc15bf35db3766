"""Rwkv7RowsSession where LoRA ranks exceed the model's width, against the oracle's token steps.

The token-by-token session, whose steps take wide models only, is held within 3e-4 * (1 + |t|) of the oracle's logits and
1e-4 * (1 + |t|) of its states (tests/test_rwkv_gpu.py).  The oracle and the session are two FP32 computations of that
exactness, and differ by at most twice as much, as two sessions do (tests/test_rwkv_rows_gpu.py).
"""
import numpy as np
import pytest

import oracle as orc
from sharpinference_amd import rwkv7
from sharpinference_amd.rwkv7_rows import Rwkv7RowsSession
from tests.test_rwkv_gpu import oracle_cfg
from tests.test_rwkv_rows_gpu import _near, _states_near

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hidden,ranks", [(128, (288, 160, 32, 416)), (64, (96, 96, 64, 256))])
def test_prompt_of_a_narrow_model(hip, hidden, ranks):
    w, a, v, g = ranks
    cfg = rwkv7.Rwkv7Config(layers=3, hidden=hidden, heads=hidden // 64, ffn=2 * hidden, vocab=300, rank_w=w, rank_a=a, rank_v=v,
                            rank_g=g)
    weights = rwkv7.synth_weights(cfg, seed=5)
    zeros = [tuple(np.zeros_like(x) for x in layer) for layer in rwkv7.synth_state(cfg)]
    model = orc.Rwkv7Oracle(oracle_cfg(cfg), weights, zeros)
    tokens = np.random.default_rng(hidden).integers(0, cfg.vocab, 21).tolist()
    want = np.stack([model.step(t)[1].copy() for t in tokens])
    session = Rwkv7RowsSession(hip, cfg, weights, slots=2)
    try:
        got = session.step([tokens[:16]], [-1], [1])
        _near(got, want[:16], "first logits")
        _near(session.step([tokens[16:]], [1], [1]), want[16:], "logits")
        _states_near(session, 1, model.state, "prompt")
    finally:
        session.close()
