"""64-bit references of the operators over many sequences, with the bounds that go with them.

Bounds count roundings: a FP32 rounding is off by at most U = 2^-24 of its result, an output
rounded to a type by at most half its step (STEP).
"""
import numpy as np

from sharpinference_amd import native

U = 2.0 ** -24
HEAD = 64
RHO = 1 - 1 / 512
GROUP_EPS = float(np.float32(64e-5))
STEP = {native.F32: 2.0 ** -24, native.F16: 2.0 ** -11, native.BF16: 2.0 ** -8}
TINY = {native.F32: 2.0 ** -149, native.F16: 2.0 ** -24, native.BF16: 2.0 ** -133}
SIZE = {native.F32: 4, native.F16: 2, native.BF16: 2}


def values(raw, fmt):
    """64-bit values of the bytes of an output."""
    if fmt == native.F32:
        return raw.view(np.float32).astype(np.float64)
    if fmt == native.F16:
        return raw.view(np.float16).astype(np.float64)
    return (raw.view(np.uint16).astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def encode(x, fmt):
    """FP32 values as the bytes of a type (BF16: truncated, so exact in what it decodes to)."""
    x = np.ascontiguousarray(x, np.float32)
    with np.errstate(over="ignore"):
        return x if fmt == native.F32 else x.astype(np.float16) if fmt == native.F16 else (x.view(np.uint32) >> 16).astype(np.uint16)


def taken(state, slot):
    """What a sequence goes on from."""
    if slot == -1:
        return np.zeros_like(state[0])
    return state[slot] if 0 <= slot < len(state) else np.full_like(state[0], np.nan)


def spans(starts, rows):
    """(sequence, first, last) of the sequences that have rows."""
    return [(s, a, b) for s, (a, b) in enumerate(zip(starts[:-1], starts[1:])) if 0 <= a < b <= rows]


def layernorm(x, residual, weight, bias, eps):
    """(updated, norm, bound of norm): the mean of n values is off by log2(n) / 2 + 10 roundings of their mean
    magnitude (sums in trees of at most 32 in a row), the rest by a few roundings of each factor."""
    u = x if residual is None else x + residual   # FP32, as the operator rounds it
    v = u.astype(np.float64)
    n = v.shape[-1]
    c = v - v.mean(-1, keepdims=True)
    inv = 1 / np.sqrt((c * c).mean(-1, keepdims=True) + float(np.float32(eps)))
    norm = c * inv * weight + bias
    sums = 32 + np.log2(n)
    mean_off = sums * U * np.abs(v).mean(-1, keepdims=True)
    # c: the mean's error and one rounding; inv: half the relative error of the variance, which a shift of
    # the mean changes only in the second order
    shift = (mean_off * inv) ** 2
    bound = (mean_off + U * np.abs(c)) * inv * np.abs(weight) + (sums + 8) * U * (np.abs(c) * inv * np.abs(weight)) + \
        shift * np.abs(c) * inv * np.abs(weight) + 2 * U * (np.abs(norm) + np.abs(bias))
    return u, norm, bound


def mix_rows(x, residual, weight, bias, mix, state, starts, source, to, eps):
    """(updated, outputs [mixes or 1][rows][n], bounds, state, its bounds); rows in no sequence are NaN in the first two."""
    rows, n = x.shape
    u, norm, off = layernorm(x, residual, weight.astype(np.float64), bias.astype(np.float64), eps)
    before, before_off = np.full((rows, n), np.nan), np.zeros((rows, n))
    held, held_off = state.astype(np.float64).copy(), np.zeros(state.shape)
    live = np.zeros(rows, bool)
    for s, a, b in spans(starts, rows):
        live[a:b] = True
        before[a], before[a + 1:b] = taken(state, source[s]), norm[a:b - 1]
        before_off[a + 1:b] = off[a:b - 1]
        if 0 <= to[s] < len(state):
            held[to[s]], held_off[to[s]] = norm[b - 1], off[b - 1]
    if mix is None or len(mix) == 0:
        out, bound, held, held_off = norm[None].copy(), off[None], state.astype(np.float64), np.zeros(state.shape)
    else:
        m = mix.astype(np.float64)[:, None]
        out = norm + (before - norm) * m
        bound = off * np.abs(1 - m) + before_off * np.abs(m) + 4 * U * (np.abs(norm) + np.abs(before)) * (1 + np.abs(m))
    out[:, ~live] = np.nan
    return u, out, bound, held, held_off, live


def _sigmoid(x):
    return 1 / (1 + np.exp(-x))


def wkv_rows(inp, heads, first, starts, source, to):
    """(out, bound, state, bound per head, v_first): the recurrence in 64 bits, and how far FP32 may be off.

    A step's state S' = S G + v k^T, G = diag(w) - kn (kn a)^T, comes from its factors with at most C
    roundings a term (sums of 64 products, then of up to 16 rows; exponentials and quotients a few
    each): an error D_t with |D_t| <= d_t in Frobenius norm, a head at a time.  After T steps the state is off by
    sum_t D_t P_t, P_t = G_(t+1) .. G_T; by Cauchy and Schwarz, with weights rho^(T - t), a readout of it by r is off by at
    most sqrt(sum rho^(T - t)) sqrt(r^T M r), M = sum_t d_t^2 rho^(t - T) P_t^T P_t, and the state by the root of
    M's largest eigenvalue in place of r^T M r.  A readout adds C roundings of |S| |r|; the GroupNorm divides by the
    root of its variance; the output is rounded once.
    """
    rows = len(inp["r"])
    d = {k: v.astype(np.float64) for k, v in inp.items() if v is not None and v.dtype == np.float32}
    per = lambda x: x.reshape(-1, heads, HEAD)
    decay = per(np.exp(float(np.float32(-0.606531)) * _sigmoid(d["w_lora"] + d["w0"])))
    a = per(_sigmoid(d["a_lora"] + d["a0"]))
    sk = per(d["k"] * d["k_k"])
    kn = sk / np.sqrt(np.maximum((sk * sk).sum(-1, keepdims=True), 1e-24))
    key = per(d["k"]) * (1 + (a - 1) * per(d["k_a"][None]))
    value = d["v"] if first else d["v"] + (d["v_first"] - d["v"]) * _sigmoid(d["v_lora"] + d["v0"])
    value, r = per(value), per(d["r"])
    ak = kn * a
    out, bound = np.full((rows, heads, HEAD), np.nan), np.zeros((rows, heads, HEAD))
    state = d["state"].copy()
    off = np.zeros((len(state), heads))
    C = (64 + 16 + 20) * U
    lw, lb, rk, gate = per(d["lnx_weight"][None])[0], per(d["lnx_bias"][None])[0], per(d["r_k"][None])[0], per(d["gate"])
    norm = lambda x: np.linalg.norm(x, axis=-1)
    for s, first_row, last_row in spans(starts, rows):
        S, M, weights = taken(d["state"], source[s]).copy(), np.zeros((heads, HEAD, HEAD)), 0.0
        for t in range(first_row, last_row):
            G = np.zeros((heads, HEAD, HEAD))
            G[:, np.arange(HEAD), np.arange(HEAD)] = decay[t]
            G -= kn[t][:, :, None] * ak[t][:, None, :]
            size = np.linalg.norm(S, axis=(1, 2))
            step = C * (size * (1 + norm(ak[t])) + norm(value[t]) * norm(key[t]))
            weights = weights * RHO + 1
            M = G.transpose(0, 2, 1) @ M @ G / RHO + step[:, None, None] ** 2 * np.eye(HEAD)
            S = S @ G + value[t][:, :, None] * key[t][:, None, :]
            y = (S @ r[t][:, :, None])[..., 0]
            y_off = np.sqrt(weights * np.einsum("hi,hij,hj->h", r[t], M, r[t])) + C * np.linalg.norm(S, axis=(1, 2)) * norm(r[t])
            mean = y.mean(-1, keepdims=True)
            inv = 1 / np.sqrt(((y - mean) ** 2).mean(-1, keepdims=True) + GROUP_EPS)
            ln = (y - mean) * inv
            bonus = (key[t] * r[t] * rk).sum(-1, keepdims=True)
            out[t] = (ln * lw + lb + value[t] * bonus) * gate[t]
            size_b = (np.abs(key[t] * r[t] * rk)).sum(-1, keepdims=True) * np.abs(value[t])
            # the norm of a vector error y_off bounds each of its values; through the normalisation it at most triples
            ln_off = 3 * y_off[:, None] * inv + 80 * U * (np.abs(ln) + np.abs(mean) * inv)
            bound[t] = (ln_off * np.abs(lw) + 100 * U * (np.abs(lb) + size_b) + 4 * U * np.abs(ln * lw)) * np.abs(gate[t]) + \
                4 * U * np.abs(out[t])
        if 0 <= to[s] < len(state):
            state[to[s]] = S
            off[to[s]] = np.sqrt(weights * np.linalg.eigvalsh(np.where(np.isfinite(M), M, 0))[:, -1])
    return out.reshape(rows, -1), bound.reshape(rows, -1), state, off


def beam_select(logits, scores, done, slots, beams, candidates, end_token):
    """Per sequence, in 64 bits; logits [sequences * beams][vocab] values."""
    out = {k: [] for k in ("parents", "tokens", "scores", "done", "from", "to")}
    for s in range(len(logits) // beams):
        pairs = []
        for b in range(beams):
            row, given = logits[s * beams + b], float(scores[s * beams + b])
            if done is not None and done[s * beams + b]:
                if np.isfinite(given):
                    pairs.append((-given, b, end_token))
                continue
            if np.isnan(row).any() or (row == np.inf).any() or not np.isfinite(given) or not (row > -np.inf).any():
                continue
            m = row.max()
            score = given + ((row - m) - np.log(np.exp(row - m).sum()))
            best = np.lexsort((np.arange(len(row)), -row))[:candidates]
            pairs += [(-score[t], b, int(t)) for t in best if np.isfinite(row[t])]
        pairs = sorted(pairs)[:candidates]
        pairs += [(np.inf, -1, -1)] * (candidates - len(pairs))
        mine = None if slots is None else list(slots[s * beams:(s + 1) * beams])
        spare = [] if mine is None else [mine[b] for b in range(beams) if all(p[1] != b for p in pairs)]
        seen = set()
        for minus, parent, token in pairs:
            out["parents"].append(parent)
            out["tokens"].append(token)
            out["scores"].append(-minus)
            out["done"].append(int(token >= 0 and token == end_token))
            if mine is not None:
                out["from"].append(mine[parent] if parent >= 0 else -1)
                out["to"].append(spare.pop(0) if parent < 0 or parent in seen else mine[parent])
            seen.add(parent)
    return {k: np.array(v, np.float64 if k == "scores" else np.int64) for k, v in out.items()}
