"""RWKV-7 over many rows a step (sharpinference_amd/rwkv7_rows.py) against the token-by-token session,
which has its own tests against the oracle: prompts in pieces of 16, sequences beside one another, beam
search with its moves of states.

The token-by-token session's tests hold its logits within 3e-4 * (1 + |t|) of the oracle's and its states within
1e-4 * (1 + |t|) (tests/test_rwkv_gpu.py); two sessions of that exactness differ by at most twice as much.  A
log-probability is a logit less the logarithm of a mean of exponentials of logits, and so off by at most twice what
the logits are.
"""
import numpy as np
import pytest

from sharpinference_amd import rwkv7
from sharpinference_amd.rwkv7_rows import Hypothesis, Rwkv7RowsSession
from tests.test_rwkv_gpu import small_cfg

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def model():
    cfg = small_cfg(layers=3)
    return cfg, rwkv7.synth_weights(cfg, seed=31)


LOGITS, STATES = 6e-4, 2e-4


def _near(a, b, what, gate=LOGITS):
    assert np.all(np.abs(a - b) <= gate * (1 + np.abs(b))), f"{what}: {np.max(np.abs(a - b) / (1 + np.abs(b)))}"


def _by_tokens(hip, model, tokens):
    """(logits of every token, states) of the token-by-token session."""
    cfg, weights = model
    one = rwkv7.Rwkv7DecodeSession(hip, cfg, weights)
    logits = []
    for t in tokens:
        one.forward_token(t)
        logits.append(one.read_logits())
    states = [one.read_state(l) for l in range(cfg.layers)]
    one.close()
    return np.stack(logits), states


def _states_near(session, slot, states, what):
    for l, want in enumerate(states):
        for name, got, ref in zip(("att", "ffn", "wkv"), session.read_state(l, slot), want):
            _near(got, ref, f"{what}: layer {l} {name}", STATES)


def test_prompt_in_pieces(hip, model):
    cfg, weights = model
    tokens = np.random.default_rng(1).integers(0, cfg.vocab, 45).tolist()
    logits, states = _by_tokens(hip, model, tokens)
    session = Rwkv7RowsSession(hip, cfg, weights, slots=3)
    try:
        _near(session.prefill(tokens, 2), logits[-1], "logits")
        _states_near(session, 2, states, "prompt")
        # the same from the beginning again, in one row a step, into another slot
        for i, t in enumerate(tokens[:5]):
            got = session.step([[t]], [-1 if i == 0 else 0], [0])
            _near(got[0], logits[i], f"token {i}")
        _states_near(session, 2, states, "the other slot")
    finally:
        session.close()


def test_sequences_beside_one_another(hip, model):
    """Prompts and single tokens in one step, a shared beginning, a step whose state is not kept."""
    cfg, weights = model
    rng = np.random.default_rng(2)
    a, b = rng.integers(0, cfg.vocab, 9).tolist(), rng.integers(0, cfg.vocab, 6).tolist()
    la, sa = _by_tokens(hip, model, a)
    lb, sb = _by_tokens(hip, model, b)
    session = Rwkv7RowsSession(hip, cfg, weights, slots=4)
    try:
        got = session.step([a[:8], b[:5]], [-1, -1], [1, 3])
        _near(got, np.concatenate([la[:8], lb[:5]]), "prompts")
        # both go on, and a third from a's state with b's token
        forked, _ = _by_tokens(hip, model, a[:8] + b[5:6])
        got = session.step([a[8:], b[5:], b[5:6]], [1, 3, 1], [0, 3, -1])
        _near(got, np.stack([la[8], lb[5], forked[-1]]), "next tokens")
        _states_near(session, 0, sa, "a")
        _states_near(session, 3, sb, "b")
    finally:
        session.close()


def _search(hip, model, prompt, beams, steps, end):
    """(hypotheses, largest logit) of beam search on the host over the token-by-token session."""
    cfg, weights = model
    peak = 0.0
    one = rwkv7.Rwkv7DecodeSession(hip, cfg, weights)

    def log_softmax(x):
        nonlocal peak
        peak = max(peak, float(np.abs(x).max()))
        x = x.astype(np.float64) - x.max()
        return x - np.log(np.exp(x).sum())
    for t in prompt:
        one.forward_token(t)
    keep = lambda: [one.read_state(l) for l in range(cfg.layers)]
    live = [([], 0.0, keep(), log_softmax(one.read_logits()))]
    for _ in range(steps):
        every = []
        for i, (tokens, score, _, log) in enumerate(live):
            if tokens and tokens[-1] == end:
                every.append((-score, i, end))
            else:
                every += [(-(score + log[t]), i, int(t)) for t in np.argsort(-log, kind="stable")[:beams]]
        chosen, after = sorted(every)[:beams], []
        for minus, i, t in chosen:
            tokens, _, state, log = live[i]
            if tokens and tokens[-1] == end:
                after.append((tokens, -minus, state, log))
                continue
            one.load_state(state)
            one.forward_token(t)
            after.append((tokens + [t], -minus, keep(), log_softmax(one.read_logits())))
        live = after
    one.close()
    return [Hypothesis(tokens, score) for tokens, score, _, _ in live], peak


@pytest.mark.parametrize("prompts,beams,ended", [(1, 4, False), (2, 5, True), (1, 1, False), (1, 16, False)])
def test_beam_search(hip, model, prompts, beams, ended):
    cfg, weights = model
    rng = np.random.default_rng(beams)
    given = [rng.integers(0, cfg.vocab, n).tolist() for n in (18, 3)[:prompts]]
    steps = 4
    end = None
    if ended:   # a token that the first prompt's best beams use
        end = _search(hip, model, given[0], beams, 2, -1)[0][0].tokens[-1]
    want = [_search(hip, model, p, beams, steps, -1 if end is None else end) for p in given]
    session = Rwkv7RowsSession(hip, cfg, weights)
    try:
        for _ in range(2):   # the plans are recorded once and replayed
            found = session.beam_search(given, beams, steps, end)
            for got, (ref, peak) in zip(found, want):
                assert [h.tokens for h in got] == [h.tokens for h in ref]
                assert np.allclose([h.score for h in got], [h.score for h in ref], rtol=0,
                                   atol=steps * 2 * LOGITS * (1 + peak))
        if ended:
            assert any(end in h.tokens for h in found[0])
    finally:
        session.close()


def test_refusals(hip, model):
    cfg, weights = model
    session = Rwkv7RowsSession(hip, cfg, weights, slots=4)
    try:
        for sequences, source, to in (([], [], []), ([[1] * 17], [-1], [0]), ([[1], []], [-1], [0]), ([[1]], [4], [0]),
                                      ([[1]], [-1], [-2]), ([[1], [2]], [-1, -1], [1, 1]), ([[1], [2]], [0, 1], [1, 2]),
                                      ([[cfg.vocab]], [-1], [0]), ([[-1]], [-1], [0])):
            with pytest.raises(ValueError):
                session.step(sequences, source, to)
        for args in (([[1]], 5, 2), ([[1]], 0, 2), ([], 1, 2), ([[1]], 2, 0), ([[1]], 2, 2, cfg.vocab), ([[]], 2, 2)):
            with pytest.raises(ValueError):
                session.beam_search(*args)
    finally:
        session.close()
