"""The operators of a recurrent model's step over many sequences at once, and of a beam search over them, as they are timed.

  mix   LayerNorm of `rows` token rows (behind the residual's addition), mixed with the row before: the inputs of the
        products that follow
  scan  the time-mix core of a layer over packed sequences: the gated recurrence S = S diag(w) - (S kn)(kn a)^T + v k^T of
        every head, its readout, GroupNorm, bonus and gate
  beam  the best candidates over beams and vocabulary, and the state slots that they take over
  move  those slots' contents, array after array

A batch holds `sequences` sequences; sequence s brings count(s) rows, spread between the case's bounds by a fixed
low-discrepancy sequence, so a case is one workload and a seed its data.  States lie in slots, in any order; a call reads
slot from[s] and writes slot to[s], so that a step can be taken again.
"""
import math

import numpy as np
import torch

own = False

F32, F64, EPS = torch.float32, torch.float64, 1e-5
HEAD, GROUP_EPS, DECAY = 64, 64e-5, -0.606531
FORMATS = {"f32": 0, "f16": 1, "bf16": 30}
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _mix(name, sequences, rows, n, mixes, out, residual):
    return {"name": name, "kind": "mix", "sequences": sequences, "lo": rows[0], "hi": rows[1], "n": n, "mixes": mixes,
            "out": out, "residual": residual}


def _scan(name, sequences, rows, heads, out, first=False, fresh=False):
    return {"name": name, "kind": "scan", "sequences": sequences, "lo": rows[0], "hi": rows[1], "heads": heads, "out": out,
            "first": first, "fresh": fresh}


def _beam(name, sequences, beams, vocab, fmt, keep, ended=0.0):
    return {"name": name, "kind": "beam", "sequences": sequences, "beams": beams, "vocab": vocab, "fmt": fmt, "keep": keep,
            "ended": ended}


def _move(name, arrays, slots, units, moves, kind="f32"):
    return {"name": name, "kind": "move", "arrays": arrays, "slots": slots, "units": units, "moves": moves, "unit": kind}


def listed():
    return [
        # decode: one row for each of 16 sequences, the six inputs of a 2048-wide layer's time-mix products
        _mix("mix_tokens", 16, (1, 1), 2048, 6, "bf16", True),
        # prompts of five sequences packed behind one another: ragged counts
        _mix("mix_prompts", 5, (300, 1500), 2048, 6, "bf16", True),
        # the channel-mix input of a wide model: one mix, FP32 out
        _mix("mix_channel", 3, (1, 2777), 4096, 1, "f32", False),
        # decode: one row for each of 64 sequences, bound by the states
        _scan("scan_tokens", 64, (1, 1), 32, "bf16"),
        # a few positions checked at once (drafted tokens), the first layer
        _scan("scan_drafts", 7, (3, 6), 32, "f32", first=True),
        # one prompt of a 2048-wide model: 32 heads on 256 compute units
        _scan("scan_prompt", 1, (4001, 4001), 32, "bf16"),
        # prompts of eight sequences beside one another, ragged, with new sequences among them
        _scan("scan_prompts", 8, (500, 3000), 32, "bf16", fresh=True),
        # a long text through a narrow model
        _scan("scan_long", 1, (8191, 8191), 12, "f16"),
        # one sequence of four beams over a vocabulary of 65536: latency counts
        _beam("beam_few", 1, 4, 65536, "f32", "slots"),
        # 24 sequences of eight beams over a vocabulary of 200064, 16-bit logits; ended beams among them
        _beam("beam_batch", 24, 8, 200064, "bf16", "slots", 0.15),
        # the states of a 24-layer model after a selection: both shift rows and 32 heads of 64 x 64 of each layer
        _move("move_states", 24, 24, 2 * 2048 + 32 * 64 * 64, 16),
        # pages of a cache (16 KiB keys, as many values) that two sequences share and one is about to write
        _move("move_pages", 2, 3001, 16384, 300, "u8"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["mix", "mix", "scan", "scan", "scan", "beam", "beam", "move"])
    if kind == "mix":
        n = _log(rng, 32, 8192)
        n = n if rng.random() < 0.3 else max(32, n // 32 * 32)
        mixes = rng.choice([1, 1, 6, 6, rng.randint(2, 5)])
        rows = _log(rng, 1, max(1, min(4096, 8000000 // n)))
        sequences = _log(rng, 1, min(rows, 256))
        most = max(1, rows // sequences)
        return {"kind": kind, "sequences": sequences, "lo": rng.randint(1, most), "hi": most, "n": n, "mixes": mixes,
                "out": rng.choice(["bf16", "bf16", "f16", "f32"]), "residual": rng.random() < 0.6}
    if kind == "scan":
        heads = _log(rng, 1, 64)
        most = _log(rng, 1, 4000) if rng.random() < 0.7 else 1
        sequences = _log(rng, 1, max(1, min(128, 40000 // most, 200000 // (heads * most))))
        return {"kind": kind, "sequences": sequences, "lo": rng.randint(1, most), "hi": most, "heads": heads,
                "out": rng.choice(["bf16", "bf16", "f16", "f32"]), "first": rng.random() < 0.2, "fresh": rng.random() < 0.4}
    if kind == "beam":
        beams, sequences = rng.randint(1, 16), _log(rng, 1, 32)
        vocab = _log(rng, 32, max(64, min(200064, 30000000 // (beams * sequences))))
        return {"kind": kind, "sequences": sequences, "beams": beams, "vocab": vocab, "keep": rng.choice(["slots", "double"]),
                "fmt": rng.choice(["f32", "f32", "f16", "bf16"]), "ended": rng.choice([0.0, 0.2])}
    slots = _log(rng, 2, 1000)
    units = _log(rng, 16, max(32, min(200000, 40000000 // slots)))
    arrays = _log(rng, 1, max(1, min(64, 80000000 // (slots * units))))
    return {"kind": kind, "arrays": arrays, "slots": slots, "units": units, "unit": rng.choice(["f32", "u8"]),
            "moves": _log(rng, 1, max(1, slots // 2))}


# ---- the batch ------------------------------------------------------------------------------

def _spread(lo, hi, count, turn):
    """`count` whole numbers between lo and hi (by their logarithm), the largest among them."""
    share = (np.arange(count) * turn) % 1.0
    return np.rint((lo + 1) * ((hi + 1) / (lo + 1)) ** (1 - share) - 1).astype(np.int64)


def _counts(case):
    """Rows of each of the case's sequences."""
    return _spread(case["lo"], case["hi"], case["sequences"], 0.6180339887)


# ---- inputs ---------------------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _randn(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def _rand(g, *shape):
    return torch.rand(*shape, device="cuda", generator=g)


def _ints(values):
    return torch.tensor(np.asarray(values), dtype=torch.int32, device="cuda")


def _batch(g, case):
    """Where each sequence's rows and states lie: twice as many slots as sequences and one more, in any order."""
    counts = _counts(case)
    starts = np.concatenate([[0], np.cumsum(counts)])
    n = case["sequences"]
    order = torch.randperm(2 * n + 1, device="cuda", generator=g).to(torch.int32)
    source = order[:n].clone()
    if case.get("fresh"):
        source[::3] = -1   # new sequences: from a state of zeros
    return {"starts": _ints(starts), "from": source, "to": order[n:2 * n].clone(), "slots": 2 * n + 1,
            "rows": int(starts[-1]), "most": int(counts.max())}


def _inputs(case, seed):
    g, kind = _gen(seed), case["kind"]
    if kind == "mix":
        inp, n = _batch(g, case), case["n"]
        shape = (inp["rows"], n)
        inp.update(x=_randn(g, *shape) * 2 + 0.1, residual=_randn(g, *shape) if case["residual"] else None,
                   weight=1 + 0.1 * _randn(g, n), bias=0.1 * _randn(g, n), mix=_rand(g, case["mixes"], n),
                   state=_randn(g, inp["slots"], n))
        return inp
    if kind == "scan":
        inp, c = _batch(g, case), case["heads"] * HEAD
        rows = inp["rows"]
        for name in ("r", "k", "v"):
            inp[name] = _randn(g, rows, c)
        inp.update(w_lora=_randn(g, rows, c) * 0.5, a_lora=_randn(g, rows, c) * 0.5, gate=_rand(g, rows, c) * 2)
        # channels from slow decay (thousands of positions) to fast
        inp["w0"] = torch.linspace(-7, 1, HEAD, device="cuda").repeat(case["heads"]) + 0.3 * _randn(g, c)
        inp.update(a0=_randn(g, c), k_k=1 + 0.1 * _randn(g, c), k_a=_rand(g, c), r_k=0.1 * _randn(g, c),
                   lnx_weight=1 + 0.1 * _randn(g, c), lnx_bias=0.1 * _randn(g, c),
                   state=0.1 * _randn(g, inp["slots"], case["heads"], HEAD, HEAD))
        inp["v_lora"], inp["v0"] = (None, None) if case["first"] else (_randn(g, rows, c) * 0.5, _randn(g, c))
        inp["v_first"] = torch.zeros(rows, c, device="cuda") if case["first"] else _randn(g, rows, c)
        return inp
    if kind == "beam":
        s, b, v = case["sequences"], case["beams"], case["vocab"]
        logits = _randn(g, s * b, v)
        logits *= 2.5
        return {"logits": logits.to(TYPES[case["fmt"]]), "scores": -4 * _rand(g, s * b),
                "done": (_rand(g, s * b) < case["ended"]).to(torch.int32),
                "slots": torch.randperm(s * b, device="cuda", generator=g).to(torch.int32)}
    shape = (case["slots"], case["units"])
    if case["unit"] == "u8":
        arrays = [torch.randint(0, 256, shape, device="cuda", generator=g, dtype=torch.uint8) for _ in range(case["arrays"])]
    else:
        arrays = [_randn(g, *shape) for _ in range(case["arrays"])]
    order = torch.randperm(case["slots"], device="cuda", generator=g).to(torch.int32)
    n = case["moves"]
    # sources may repeat and are no destinations; every fourth child stays where its parent was
    source = order[n:][torch.randint(0, case["slots"] - n, (n,), device="cuda", generator=g)]
    to = torch.where(torch.arange(n, device="cuda") % 4 == 3, source, order[:n])
    return {"arrays": arrays, "from": source.contiguous(), "to": to.contiguous()}


def prepare(case, seed):
    inp = _inputs(case, seed)
    state = {"case": case, "inp": inp}
    empty = lambda *s, dtype=F32: torch.empty(*s, device="cuda", dtype=dtype)
    if case["kind"] == "mix":
        shape = (inp["rows"], case["n"])
        state["bufs"] = {"updated": empty(*shape) if case["residual"] else None,
                         "out": empty(case["mixes"], *shape, dtype=TYPES[case["out"]])}
    elif case["kind"] == "scan":
        state["bufs"] = {"out": empty(inp["rows"], case["heads"] * HEAD, dtype=TYPES[case["out"]])}
    elif case["kind"] == "beam":
        keep = case["beams"] * (1 if case["keep"] == "slots" else 2)
        count = case["sequences"] * keep
        state["bufs"] = {"scores": empty(count)}
        state["bufs"].update({k: empty(count, dtype=torch.int32) for k in ("parents", "tokens", "done", "from", "to")})
    else:
        state["bufs"] = {}
    return state


# ---- the calls of a user's program -------------------------------------------------------------

_hip = None


def _context():
    """The program's one context."""
    global _hip
    if _hip is None:
        from sharpinference_amd import native
        _hip = native.HipContext(0)
    return _hip


class _Owner:
    """Keeps a state's device memory until the context's stream is done with it."""

    def __init__(self, *held):
        self.held = held

    def __del__(self):
        if _hip is not None:   # (None as the interpreter ends)
            _hip.sync()


def _program(state):
    """What a program sets up once for its buffers: the calls with their arguments.

    The context has a stream of its own, which torch's does not wait for, nor it for torch's.  So
    what torch fills is waited for here, once; whoever reads outputs waits for the context
    (or the device) first; and the memory goes back to torch only behind the context's work.
    """
    from sharpinference_amd import native
    hip, case, inp, bufs = _context(), state["case"], state["inp"], state["bufs"]
    p = lambda t: 0 if t is None else t.data_ptr()
    workspace, size = None, 0
    if case["kind"] == "scan":
        size = native.rwkv7_wkv_rows_workspace_bytes(case["heads"])
    elif case["kind"] == "beam":
        keep = case["beams"] * (1 if case["keep"] == "slots" else 2)
        size = native.beam_select_workspace_bytes(case["sequences"], case["beams"], keep, case["vocab"])
    if size:
        workspace = torch.empty(size, dtype=torch.uint8, device="cuda")
    state["owner"] = _Owner(inp, bufs, workspace)
    torch.cuda.synchronize()
    if case["kind"] in ("mix", "scan"):
        batch = native.RowBatch(p(inp["starts"]), p(inp["from"]), p(inp["to"]), case["sequences"], inp["slots"],
                                inp["rows"], inp["most"])
    if case["kind"] == "mix":
        args = native.LayernormMixRowsArgs(batch, p(inp["x"]), p(inp["residual"]), p(inp["weight"]), p(inp["bias"]),
                                           p(inp["mix"]), p(inp["state"]), p(bufs["updated"]), p(bufs["out"]), case["n"],
                                           case["mixes"], FORMATS[case["out"]], EPS)
        outs = ([] if bufs["updated"] is None else [bufs["updated"]]) + [bufs["out"], inp["state"]]

        def call():
            hip.layernorm_mix_rows(args)
            return outs
        return call
    if case["kind"] == "scan":
        vectors = [p(inp[name]) for name in native.RWKV7_WKV_VECTORS]
        args = native.Rwkv7WkvRowsArgs(batch, case["heads"], int(case["first"]), *vectors, p(inp["v_first"]),
                                       p(inp["state"]), p(bufs["out"]), p(workspace), FORMATS[case["out"]])
        outs = [bufs["out"], inp["state"]] + ([inp["v_first"]] if case["first"] else [])

        def call():
            hip.rwkv7_wkv_rows(args)
            return outs
        return call
    if case["kind"] == "beam":
        slots = case["keep"] == "slots"
        args = native.BeamSelectArgs(p(inp["logits"]), p(inp["scores"]), p(inp["done"]), p(inp["slots"]) if slots else 0,
                                     p(bufs["parents"]), p(bufs["tokens"]), p(bufs["scores"]), p(bufs["done"]),
                                     p(bufs["from"]) if slots else 0, p(bufs["to"]) if slots else 0, p(workspace),
                                     case["vocab"], case["vocab"], case["sequences"], case["beams"], keep,
                                     FORMATS[case["fmt"]], 0)
        outs = [bufs[k] for k in ("parents", "tokens", "scores", "done") + (("from", "to") if slots else ())]

        def call():
            hip.beam_select(args)
            return outs
        return call
    width = case["units"] * inp["arrays"][0].element_size()
    arrays = native.slot_arrays([(p(a), width) for a in inp["arrays"]])
    args = (arrays, case["slots"], p(inp["from"]), p(inp["to"]), case["moves"])

    def call():
        hip.copy_slots(*args)
        return inp["arrays"]
    return call


# ---- the plain forms ----------------------------------------------------------------------------

def _taken(state, slots, at):
    """What the slots of sequences hold; zeros for -1."""
    held = state[at.clamp(min=0).long()]
    return held * (at >= 0).to(held.dtype).reshape(-1, *[1] * (held.dim() - 1))


def _plain_mix(state):
    case, inp = state["case"], state["inp"]
    u = inp["x"] if inp["residual"] is None else inp["x"] + inp["residual"]
    c = u - u.mean(-1, keepdim=True)
    n = c / torch.sqrt((c * c).mean(-1, keepdim=True) + EPS) * inp["weight"] + inp["bias"]
    starts = inp["starts"].long()
    shifted = torch.cat([n[:1], n[:-1]])
    shifted[starts[:-1]] = _taken(inp["state"], inp["slots"], inp["from"])
    out = n[None] + (shifted - n)[None] * inp["mix"][:, None]
    inp["state"][inp["to"].long()] = n[starts[1:] - 1]
    return ([] if inp["residual"] is None else [u]) + [out.to(TYPES[case["out"]]), inp["state"]]


def _gates(inp, case, t):
    """(decay, unit keys, their share in the update, keys, values) of every row, [rows, heads, 64] of type t."""
    rows = inp["rows"]
    x = lambda name: inp[name].to(t)
    h = lambda y: y.reshape(rows, case["heads"], HEAD)
    decay = torch.exp(DECAY * torch.sigmoid(x("w_lora") + x("w0")))
    a = torch.sigmoid(x("a_lora") + x("a0"))
    sk = h(x("k") * x("k_k"))
    kn = sk / torch.sqrt((sk * sk).sum(-1, keepdim=True).clamp(min=1e-24))
    key = x("k") + (a - 1) * (x("k") * x("k_a"))
    value = x("v")
    if not case["first"]:
        value = value + (x("v_first") - value) * torch.sigmoid(x("v_lora") + x("v0"))
    return h(decay), kn, kn * h(a), h(key), h(value)


def _plain_scan(state):
    case, inp = state["case"], state["inp"]
    rows, c = inp["rows"], case["heads"] * HEAD
    decay, kn, ak, key, value = _gates(inp, case, F32)
    r = inp["r"].reshape(rows, -1, HEAD)
    counts = _counts(case)
    order = np.argsort(-counts, kind="stable")
    first = inp["starts"][:-1][_ints(order).long()].long()
    S = _taken(inp["state"], inp["slots"], inp["from"])[_ints(order).long()]
    y = torch.empty(rows, case["heads"], HEAD, device="cuda")
    # a recurrence: one step a position, of all sequences that have it
    for t in range(inp["most"]):
        n = int((counts > t).sum())
        at, s = first[:n] + t, S[:n]
        seen = (s * kn[at].unsqueeze(2)).sum(-1, keepdim=True)
        s.mul_(decay[at].unsqueeze(2))
        s.add_(value[at].unsqueeze(3) * key[at].unsqueeze(2) - seen * ak[at].unsqueeze(2))
        y[at] = (s * r[at].unsqueeze(2)).sum(-1)
    inp["state"][inp["to"][_ints(order).long()].long()] = S
    d = y - y.mean(-1, keepdim=True)
    ln = (d / torch.sqrt((d * d).mean(-1, keepdim=True) + GROUP_EPS)).reshape(rows, c) * inp["lnx_weight"] + inp["lnx_bias"]
    bonus = (key * r * inp["r_k"].reshape(-1, HEAD)).sum(-1, keepdim=True)
    out = (ln + (value * bonus).reshape(rows, c)) * inp["gate"]
    outs = [out.to(TYPES[case["out"]]), inp["state"]]
    if case["first"]:
        inp["v_first"].copy_(inp["v"])
        outs.append(inp["v_first"])
    return outs


def _plain_beam(state):
    case, inp = state["case"], state["inp"]
    s, b, v = case["sequences"], case["beams"], case["vocab"]
    keep = b * (1 if case["keep"] == "slots" else 2)
    # 64 bits: candidates next to one another keep their order
    x = inp["logits"].to(F64)
    x = x - x.amax(-1, keepdim=True)
    x = x - torch.log(torch.exp(x).sum(-1, keepdim=True)) + inp["scores"].to(F64)[:, None]
    ended = inp["done"] != 0
    token = torch.arange(v, device="cuda")
    # an ended beam's one candidate is itself, under the end token (0)
    x = torch.where(ended[:, None], torch.where(token == 0, inp["scores"].to(F64)[:, None], -math.inf), x).reshape(s, b * v)
    flat = torch.arange(b * v, device="cuda")
    scores, places = [], []
    for _ in range(keep):   # the best, the lowest of equals, and then without it
        best = x.amax(1)
        place = torch.where(x == best[:, None], flat, b * v).amin(1)
        x[torch.arange(s, device="cuda"), place] = -math.inf
        scores.append(best)
        places.append(place)
    scores, places = torch.stack(scores, 1), torch.stack(places, 1)
    none = torch.isinf(scores)
    parents, tokens = torch.where(none, -1, places // v), torch.where(none, -1, places % v)
    done = ((tokens == 0) & ~none).to(torch.int32)
    outs = [t.reshape(-1).to(torch.int32) for t in (parents, tokens)] + [scores.to(F32).reshape(-1), done.reshape(-1)]
    if case["keep"] != "slots":
        return outs
    # the first child keeps its parent's slot, the others take those of childless beams in turn
    mine = parents[:, :, None] == torch.arange(b, device="cuda")
    kept = (mine & (torch.cumsum(mine.int(), 1) == 1)).any(2)
    free = ~mine.any(1)
    slots = inp["slots"].reshape(s, b)
    spare = torch.sort(torch.where(free, torch.arange(b, device="cuda"), b), dim=1).values.clamp(max=b - 1)
    turn = (torch.cumsum((~kept).int(), 1) - 1).clamp(min=0)
    source = torch.where(none, -1, torch.gather(slots, 1, parents.clamp(min=0)))
    to = torch.where(kept, source, torch.gather(slots, 1, torch.gather(spare, 1, turn)))
    return outs + [source.reshape(-1).to(torch.int32), to.reshape(-1).to(torch.int32)]


def _plain_move(state):
    inp = state["inp"]
    source, to = inp["from"].long(), inp["to"].long()
    for a in inp["arrays"]:
        a[to] = a[source]
    return inp["arrays"]


PLAIN = {"mix": _plain_mix, "scan": _plain_scan, "beam": _plain_beam, "move": _plain_move}


def run(state):
    if own:
        if "call" not in state:
            state["call"] = _program(state)
        return state["call"]()
    return PLAIN[state["case"]["kind"]](state)


# ---- what a pass cannot do without --------------------------------------------------------------

def work(case):
    kind = case["kind"]
    if kind == "mix":
        counts = _counts(case)
        count = int(counts.sum()) * case["n"]
        size = 4 if case["out"] == "f32" else 2
        moved = 4 + (8 if case["residual"] else 0) + size * case["mixes"]
        return {"bytes": count * moved + 4 * case["n"] * (2 + case["mixes"] + 2 * case["sequences"]),
                "flops": count * (8 + 2 * case["mixes"])}
    if kind == "scan":
        pairs = int(_counts(case).sum()) * case["heads"]   # rows times heads
        size = 4 if case["out"] == "f32" else 2
        read = 4 * HEAD * (6 if case["first"] else 8) + (4 * HEAD if case["first"] else 0)
        return {"bytes": pairs * (read + size * HEAD) + case["sequences"] * case["heads"] * 8 * HEAD * HEAD,
                "flops": pairs * (9 * HEAD * HEAD + 40 * HEAD)}
    if kind == "beam":
        count = case["sequences"] * case["beams"] * case["vocab"]
        return {"bytes": count * (4 if case["fmt"] == "f32" else 2) + 40 * case["sequences"] * case["beams"],
                "flops": 3 * count}
    moved = case["moves"] - case["moves"] // 4   # the rest stays in its place
    return {"bytes": 2 * moved * case["arrays"] * case["units"] * (1 if case["unit"] == "u8" else 4), "flops": 0}


# ---- the same results in 64 bits ----------------------------------------------------------------

def _exact_scan(case, inp):
    rows, heads = inp["rows"], case["heads"]
    wide = {k: t.double() if torch.is_tensor(t) and t.is_floating_point() else t for k, t in inp.items()}
    per = lambda name: wide[name].view(rows, heads, HEAD)
    own_ = lambda name: wide[name].view(heads, HEAD)
    sig = lambda z: 1 / (1 + torch.exp(-z))
    decay = torch.exp(DECAY * sig(per("w_lora") + own_("w0")))
    adapt = sig(per("a_lora") + own_("a0"))
    unit = per("k") * own_("k_k")
    unit = unit / unit.norm(dim=2, keepdim=True)
    key = per("k") * (1 + (adapt - 1) * own_("k_a"))
    value = per("v")
    if not case["first"]:
        mixed = sig(per("v_lora") + own_("v0"))
        value = value * (1 - mixed) + per("v_first") * mixed
    states = wide["state"].clone()
    y = torch.empty(rows, heads, HEAD, 1, dtype=F64, device="cuda")
    at = inp["starts"].tolist()
    for s, (source, to) in enumerate(zip(inp["from"].tolist(), inp["to"].tolist())):
        S = torch.zeros(heads, HEAD, HEAD, dtype=F64, device="cuda") if source < 0 else wide["state"][source].clone()
        for t in range(at[s], at[s + 1]):
            # S (diag(w) - kn (kn a)^T) + v k^T
            turn = torch.diag_embed(decay[t]) - unit[t].unsqueeze(2) * (unit[t] * adapt[t]).unsqueeze(1)
            S = torch.baddbmm(value[t].unsqueeze(2) * key[t].unsqueeze(1), S, turn)
            y[t] = torch.bmm(S, per("r")[t].unsqueeze(2))
        states[to] = S
    y = y[..., 0]
    var, mean = torch.var_mean(y, dim=2, keepdim=True, correction=0)
    norm = (y - mean) * torch.rsqrt(var + GROUP_EPS) * own_("lnx_weight") + own_("lnx_bias")
    bonus = torch.einsum("rhj,rhj,hj->rh", key, per("r"), own_("r_k")).unsqueeze(2)
    out = ((norm + value * bonus) * per("gate")).reshape(rows, -1)
    return [out, states] + ([wide["v"]] if case["first"] else [])


def _exact_beam(case, inp):
    b, v = case["beams"], case["vocab"]
    keep = b * (1 if case["keep"] == "slots" else 2)
    found = {k: [] for k in ("parents", "tokens", "scores", "done", "from", "to")}
    for s in range(case["sequences"]):
        rows = inp["logits"][s * b:(s + 1) * b].double()
        given = inp["scores"][s * b:(s + 1) * b].tolist()
        ended = inp["done"][s * b:(s + 1) * b].tolist()
        log = rows - torch.logsumexp(rows, 1, keepdim=True)
        every = []
        for i in range(b):
            if ended[i]:
                every.append((-given[i], i, 0))
                continue
            top = torch.sort(log[i], descending=True, stable=True)
            every += [(-(given[i] + x), i, t) for x, t in zip(top.values[:keep].tolist(), top.indices[:keep].tolist())]
        every = sorted(every)[:keep]
        every += [(math.inf, -1, -1)] * (keep - len(every))
        slots = inp["slots"][s * b:(s + 1) * b].tolist()
        spare = [slots[i] for i in range(b) if all(c[1] != i for c in every)]
        taken = set()
        for minus, parent, token in every:
            found["parents"].append(parent)
            found["tokens"].append(token)
            found["scores"].append(-minus)
            found["done"].append(int(token == 0))
            found["from"].append(slots[parent] if parent >= 0 else -1)
            if case["keep"] == "slots":
                found["to"].append(spare.pop(0) if parent < 0 or parent in taken else slots[parent])
            taken.add(parent)
    names = ("parents", "tokens", "scores", "done") + (("from", "to") if case["keep"] == "slots" else ())
    return [torch.tensor(found[k], dtype=F64, device="cuda") if k == "scores" else _ints(found[k]) for k in names]


def exact(case, seed):
    inp, kind = _inputs(case, seed), case["kind"]
    if kind == "beam":
        return _exact_beam(case, inp)
    if kind == "move":
        pairs = dict(zip(inp["to"].tolist(), inp["from"].tolist()))
        at = torch.tensor([pairs.get(i, i) for i in range(case["slots"])], device="cuda")
        held = [a.index_select(0, at) for a in inp["arrays"]]
        return [a.double() if a.is_floating_point() else a for a in held]
    if kind == "scan":
        return _exact_scan(case, inp)
    u = inp["x"].double() if inp["residual"] is None else inp["x"].double() + inp["residual"].double()
    var, mean = torch.var_mean(u, dim=1, keepdim=True, correction=0)
    n = (u - mean) * torch.rsqrt(var + EPS) * inp["weight"].double() + inp["bias"].double()
    states, at = inp["state"].double(), inp["starts"].tolist()
    before = torch.empty_like(n)
    held = states.clone()
    for s, (source, to) in enumerate(zip(inp["from"].tolist(), inp["to"].tolist())):
        a, b = at[s], at[s + 1]
        before[a] = 0 if source < 0 else states[source]
        before[a + 1:b] = n[a:b - 1]
        held[to] = n[b - 1]
    out = torch.stack([n * (1 - m) + before * m for m in inp["mix"].double()])
    return ([] if inp["residual"] is None else [u]) + [out, held]
