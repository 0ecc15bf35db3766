"""The operators of a serving step over many sequences at once, as they are timed.

  norm    RMSNorm of `rows` token rows (with the residual's addition) into 8-bit rows, one scale a row
  gemm    Y = X . W^T of 8-bit rows with a scale for each token and each output channel
  append  the batch's new rows: rotary embedding of q and k, k and v into the pages of a paged cache
  attend  the batch's new rows against the pages: causal attention with shared KV heads

A batch holds `sequences` sequences; sequence s brings its newest new(s) positions and has length(s) positions in the
cache, those included.  Both are spread between the case's bounds by a fixed low-discrepancy sequence, so a case is
one workload and a seed its data.  Pages lie shuffled in the pool.

Cache pages: F16 [page][kv_head][position][head] values; Q4_0 [page][kv_head] blocks of bytes, first
[position][head / 2] (byte j of a position: value 2j in the low nibble, 2j + 1 in the high one), then FP16 scales
[head / 32][position]: value = scale * (nibble - 8).
"""
import math

import numpy as np
import torch

own = False

F32, F64, EPS = torch.float32, torch.float64, 1e-5
FORMATS = {"f16": 1, "q4_0": 2, "bf16": 30}
OUT_TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
ROPE_SCALE, ROPE_BASE = 1.19, 10000.0


def _attend(name, fmt, out, sequences, new, context, **more):
    return {"name": name, "kind": "attend", "fmt": fmt, "out": out, "sequences": sequences, "new_lo": new[0],
            "new_hi": new[1], "ctx_lo": context[0], "ctx_hi": context[1],
            **{"heads": 24, "kv_heads": 8, "head": 128, "page": 64, **more}}


def _append(name, fmt, sequences, new, context, **more):
    return {"name": name, "kind": "append", "fmt": fmt, "sequences": sequences, "new_lo": new[0], "new_hi": new[1],
            "ctx_lo": context[0], "ctx_hi": context[1],
            **{"heads": 24, "kv_heads": 8, "head": 128, "rotary": 96, "page": 64, **more}}


def listed():
    return [
        # decode: the norm before a projection of one token (the smallest call, bound by its launch)
        {"name": "norm_token", "kind": "norm", "rows": 1, "n": 2048, "residual": True},
        # prompts packed behind one another: a ragged token count
        {"name": "norm_prompt", "kind": "norm", "rows": 4093, "n": 4096, "residual": True},
        # decode of one token: the 8192-wide projection of a 2048-wide model, bound by reading the weights
        {"name": "gemm_token", "kind": "gemm", "m": 1, "rows": 8192, "cols": 2048, "residual": False},
        # decode of a batch of 40 sequences back into the residual stream, a ragged number of channels
        {"name": "gemm_batch", "kind": "gemm", "m": 40, "rows": 5000, "cols": 8192, "residual": True},
        # prompts: the largest product of a layer
        {"name": "gemm_prompt", "kind": "gemm", "m": 4093, "rows": 8192, "cols": 4096, "residual": False},
        # decode: one new position for each of 64 sequences, 4-bit pages
        _append("append_tokens", "q4_0", 64, (1, 1), (100, 4000)),
        # prompts of five sequences, 4-bit pages
        _append("append_prompts_q4", "q4_0", 5, (300, 1500), (0, 0)),
        # prompts continued behind far positions, FP16 pages of 16, narrow heads, one KV head for eight
        _append("append_prompts_f16", "f16", 3, (700, 2000), (30000, 60000), heads=32, kv_heads=4, head=64, rotary=64,
                page=16),
        # decode of four short conversations: latency counts
        _attend("attend_few", "q4_0", "bf16", 4, (1, 1), (40, 500)),
        # decode of a full batch, lengths over more than a decade
        _attend("attend_batch", "q4_0", "bf16", 64, (1, 1), (500, 16000)),
        # a few positions checked at once (drafted tokens) on long FP16 caches, pages of 16
        _attend("attend_drafts_f16", "f16", "f16", 7, (3, 5), (3000, 9000), heads=32, kv_heads=4, head=64, page=16),
        # prompts: chunks of up to 2000 new positions, earlier ones in the cache
        _attend("attend_prompts", "q4_0", "bf16", 3, (500, 2000), (0, 4000)),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "gemm", "gemm", "append", "append", "attend", "attend", "attend"])
    if kind == "norm":
        n = _log(rng, 64, 16384)
        n = n if rng.random() < 0.3 else max(16, n // 16 * 16)
        return {"kind": kind, "rows": _log(rng, 1, max(1, 16000000 // n)), "n": n, "residual": rng.random() < 0.7}
    if kind == "gemm":
        rows, cols = _log(rng, 64, 16384), 16 * _log(rng, 4, 512)
        return {"kind": kind, "m": _log(rng, 1, max(1, min(4096, int(1.3e11 / (rows * cols))))), "rows": rows,
                "cols": cols, "residual": rng.random() < 0.5}
    kv = rng.choice([1, 2, 4, 8])
    case = {"kind": kind, "fmt": rng.choice(["q4_0", "q4_0", "f16"]), "heads": kv * rng.randint(1, 8), "kv_heads": kv,
            "head": rng.choice([64, 128, 128]), "page": rng.choice([16, 32, 64, 128])}
    if kind == "append":
        case["rotary"] = rng.choice([case["head"], case["head"], 3 * case["head"] // 4, 2 * rng.randint(1, case["head"] // 2)])
        width = (case["heads"] + 2 * kv) * case["head"]
        rows = _log(rng, 1, max(1, min(4096, 20000000 // width)))
        case["sequences"] = _log(rng, 1, min(rows, 256))
        most = max(1, rows // case["sequences"])
        case.update(new_lo=rng.randint(1, most), new_hi=most, ctx_lo=0)
        case["ctx_hi"] = _log(rng, 1, max(1, min(60000, 400000000 // (case["sequences"] * kv * case["head"]))))
        return case
    case["out"] = rng.choice(["f16", "bf16"])
    case["sequences"] = _log(rng, 1, 64)
    most = 1000000000 // (case["sequences"] * kv * case["head"])   # positions of a sequence
    new = 1 if rng.random() < 0.5 else _log(rng, 1, 2000)
    case.update(new_lo=rng.randint(1, new), new_hi=new)
    scores = 250000000 // (case["sequences"] * case["heads"] * new)   # positions against which all new rows go
    case["ctx_hi"] = _log(rng, 1, max(2, min(60000, most - new, scores - new)))
    case["ctx_lo"] = rng.randint(0, case["ctx_hi"])
    if (case["ctx_hi"] + new) * case["sequences"] * case["heads"] * new > 400000000:   # few positions, many rows
        case["sequences"] = max(1, 400000000 // ((case["ctx_hi"] + new) * case["heads"] * new))
    return case


# ---- the batch ------------------------------------------------------------------------------

def _spread(lo, hi, count, turn):
    """`count` whole numbers between lo and hi (by their logarithm), the largest among them."""
    share = (np.arange(count) * turn) % 1.0
    return np.rint((lo + 1) * ((hi + 1) / (lo + 1)) ** (1 - share) - 1).astype(np.int64)


def _batch(case):
    """(new positions, lengths) of the case's sequences."""
    new = _spread(case["new_lo"], case["new_hi"], case["sequences"], 0.6180339887)
    return new, new + _spread(case["ctx_lo"], case["ctx_hi"], case["sequences"], 0.7548776662)


def _head_bytes(case):
    """Bytes of one position's key (or value) of one KV head."""
    return 2 * case["head"] if case["fmt"] == "f16" else case["head"] // 2 + case["head"] // 16


# ---- inputs ---------------------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _randn(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def _codes(g, rows, cols):
    """Rows of 8-bit codes as quantized normal values give them, and their scales."""
    q = _randn(g, rows, cols).mul_(32).round_().clamp_(-127, 127).to(torch.int8)
    return q, torch.rand(rows, device="cuda", generator=g) * 0.03 + 0.01


def _ints(values):
    return torch.tensor(np.asarray(values), dtype=torch.int32, device="cuda")


def _pool(g, case, pages):
    """A pool's pages, keys or values: stale rows included."""
    kv, ps, d = case["kv_heads"], case["page"], case["head"]
    if case["fmt"] == "f16":
        return _randn(g, pages, kv, ps, d).half()
    pool = torch.randint(0, 256, (pages, kv, ps * _head_bytes(case)), device="cuda", generator=g, dtype=torch.uint8)
    scales = pool[:, :, ps * d // 2:].view(torch.float16)
    scales.copy_((torch.rand(scales.shape, device="cuda", generator=g) * 0.15 + 0.15).half())
    return pool


def _inputs(case, seed):
    g, kind = _gen(seed), case["kind"]
    if kind == "norm":
        shape = (case["rows"], case["n"])
        return {"hidden": _randn(g, *shape) * 3, "residual": _randn(g, *shape) if case["residual"] else None,
                "weight": 1 + 0.1 * _randn(g, case["n"])}
    if kind == "gemm":
        x, xs = _codes(g, case["m"], case["cols"])
        w, ws = _codes(g, case["rows"], case["cols"])
        return {"x": x, "xs": xs, "w": w, "ws": ws * 0.02,
                "residual": _randn(g, case["m"], case["rows"]) if case["residual"] else None}
    new, lengths = _batch(case)
    ps = case["page"]
    held = -(-lengths // ps)
    pages = int(held.sum()) + 3
    order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
    table = torch.full((len(held), int(held.max())), -1, dtype=torch.int32, device="cuda")
    table[torch.arange(table.shape[1], device="cuda") < _ints(held)[:, None]] = order[:int(held.sum())]
    starts = np.concatenate([[0], np.cumsum(new)])
    rows, h, d = int(starts[-1]), case["heads"], case["head"]
    inp = {"table": table, "starts": _ints(starts), "lengths": _ints(lengths), "rows": rows, "pages": pages,
           "most": int(new.max()), "longest": int(lengths.max()), "k": _pool(g, case, pages), "v": _pool(g, case, pages)}
    if kind == "append":
        i = torch.arange(case["rotary"] // 2, device="cuda", dtype=F32)
        inp["freq"] = 1.0 / torch.pow(torch.tensor(ROPE_BASE, device="cuda"), 2.0 * i / case["rotary"])
        inp["qkv"] = _randn(g, rows, (h + 2 * case["kv_heads"]) * d)
    else:
        inp["q"] = _randn(g, rows, h * d)
    return inp


def prepare(case, seed):
    inp = _inputs(case, seed)
    state = {"case": case, "inp": inp}
    empty = lambda *s, dtype=F32: torch.empty(*s, device="cuda", dtype=dtype)
    if case["kind"] == "norm":
        shape = (case["rows"], case["n"])
        state["bufs"] = {"updated": empty(*shape), "q": empty(*shape, dtype=torch.int8), "scale": empty(shape[0]),
                         "values": empty(*shape)}
    elif case["kind"] == "gemm":
        state["bufs"] = {"y": empty(case["m"], case["rows"])}
    elif case["kind"] == "append":
        kv = (inp["rows"], case["kv_heads"] * case["head"])
        state["bufs"] = {"query": empty(inp["rows"], case["heads"] * case["head"]), "keys": empty(*kv),
                         "values": empty(*kv)}
    else:
        state["bufs"] = {"out": empty(inp["rows"], case["heads"] * case["head"], dtype=OUT_TYPES[case["out"]])}
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
    workspace = None
    if case["kind"] == "attend":
        workspace = torch.empty(native.paged_attention_workspace_bytes(case["heads"], case["kv_heads"], case["head"]),
                                dtype=torch.uint8, device="cuda")
    state["owner"] = _Owner(inp, bufs, workspace)
    torch.cuda.synchronize()
    if case["kind"] == "norm":
        updated = bufs["updated"] if case["residual"] else None
        args = (p(inp["hidden"]), p(inp["residual"]), p(inp["weight"]), p(updated), p(bufs["q"]), p(bufs["scale"]),
                case["rows"], case["n"], EPS)
        back = (p(bufs["q"]), p(bufs["scale"]), p(bufs["values"]), case["rows"], case["n"])
        outs = [inp["hidden"] if updated is None else updated, bufs["scale"], bufs["values"]]

        def call():
            hip.residual_rms_norm_i8(*args)
            hip.dequant_i8(*back)
            return outs
        return call
    if case["kind"] == "gemm":
        args = (p(inp["x"]), p(inp["xs"]), p(inp["w"]), p(inp["ws"]), p(bufs["y"]), case["m"], case["rows"],
                case["cols"], p(inp["residual"]))

        def call():
            hip.gemm_i8(*args)
            return bufs["y"]
        return call
    batch = native.PagedBatch(p(inp["table"]), p(inp["starts"]), p(inp["lengths"]), case["sequences"],
                              inp["table"].shape[1], inp["rows"], inp["most"])
    cache = native.PagedCache(p(inp["k"]), p(inp["v"]), inp["pages"], case["page"], case["kv_heads"], case["head"],
                              FORMATS[case["fmt"]])
    if case["kind"] == "append":
        args = native.PagedAppendArgs(batch, cache, p(inp["qkv"]), p(inp["freq"]), p(bufs["query"]), case["heads"],
                                      case["rotary"], ROPE_SCALE)
        if case["fmt"] == "f16":
            def call():
                hip.paged_kv_append(args)
                return [bufs["query"], inp["k"], inp["v"]]
            return call

        def call():
            hip.paged_kv_append(args)
            hip.paged_kv_read(batch, cache, p(bufs["keys"]), p(bufs["values"]))
            return [bufs["query"], bufs["keys"], bufs["values"]]
        return call
    args = native.PagedAttentionArgs(batch, cache, p(inp["q"]), p(bufs["out"]), p(workspace), case["heads"],
                                     FORMATS[case["out"]])

    def call():
        hip.paged_attention(args)
        return bufs["out"]
    return call


# ---- the plain forms ----------------------------------------------------------------------------

def _plain_norm(state):
    inp = state["inp"]
    u = inp["hidden"] if inp["residual"] is None else inp["hidden"] + inp["residual"]
    # 64 bits from here: a value next to the border of two codes takes the same one in every form
    x = u.to(F64)
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * inp["weight"].to(F64)
    scale = (y.abs().amax(-1, keepdim=True) / 127).to(F32)
    codes = torch.round(y / scale.to(F64)).to(torch.int8)
    return [u, scale[:, 0], codes.to(F32) * scale]


def _plain_gemm(state):
    inp = state["inp"]
    y = torch.matmul(inp["x"].to(F32), inp["w"].to(F32).t()) * inp["xs"][:, None] * inp["ws"][None, :]
    return y if inp["residual"] is None else y + inp["residual"]


def _places(inp, page):
    """(sequence, position) of every row of the batch, and the page and slot that hold it."""
    row = torch.arange(inp["rows"], device="cuda")
    s = torch.searchsorted(inp["starts"][1:].to(torch.int64), row, right=True)
    pos = inp["lengths"][s] - inp["starts"][s + 1] + row
    return s, pos, inp["table"][s, pos // page].long(), pos % page


def _quantize(x):
    """[..., head] FP32 -> (codes 0..15, FP16 scales) of blocks of 32."""
    b = x.reshape(*x.shape[:-1], -1, 32)
    at = b.abs().argmax(-1, keepdim=True)
    scale = (torch.gather(b, -1, at) / -8).to(torch.float16)
    d = scale.to(F32)
    codes = torch.where(d == 0, 8.0, (torch.round(b / torch.where(d == 0, 1.0, d)) + 8).clamp(0, 15))
    return codes.reshape(x.shape).to(torch.uint8), scale[..., 0]


def _unpack(pool, case):
    """FP32 values [..., position, head] of 4-bit pages [..., bytes]."""
    ps, d = case["page"], case["head"]
    nib = pool[..., :ps * d // 2].reshape(*pool.shape[:-1], ps, d // 2)
    v = torch.stack([nib & 15, nib >> 4], -1).reshape(*pool.shape[:-1], ps, d // 32, 32).to(F32) - 8
    scale = pool[..., ps * d // 2:].contiguous().view(torch.float16).reshape(*pool.shape[:-1], d // 32, ps)
    return (v * scale.transpose(-1, -2).to(F32).unsqueeze(-1)).reshape(*pool.shape[:-1], ps, d)


def _store(pool, case, page, slot, x):
    """Rows x [rows, kv, head] into the pages; returns the values that they hold from then on."""
    kv, ps, d = case["kv_heads"], case["page"], case["head"]
    if case["fmt"] == "f16":
        pool[page, :, slot] = x.to(torch.float16)
        return pool
    codes, scale = _quantize(x)
    pool[:, :, :ps * d // 2].view(-1, kv, ps, d // 2)[page, :, slot] = codes[..., 0::2] | (codes[..., 1::2] << 4)
    pool[:, :, ps * d // 2:].view(torch.float16).view(-1, kv, d // 32, ps)[page, :, :, slot] = scale
    v = (codes.to(F32) - 8).reshape(*x.shape[:-1], -1, 32) * scale.to(F32).unsqueeze(-1)
    return v.reshape(x.shape[0], -1)


def _plain_append(state):
    case, inp = state["case"], state["inp"]
    h, kv, d, half = case["heads"], case["kv_heads"], case["head"], case["rotary"] // 2
    _, pos, page, slot = _places(inp, case["page"])
    x = inp["qkv"].reshape(inp["rows"], -1, d)
    # angles of far positions, and values next to a code's border: 64 bits
    angle = pos.to(F64)[:, None] * inp["freq"].to(F64)[None]
    scale = float(np.float32(ROPE_SCALE))
    cos, sin = (torch.cos(angle) * scale)[:, None], (torch.sin(angle) * scale)[:, None]
    a, b = x[:, :h + kv, :half].to(F64), x[:, :h + kv, half:2 * half].to(F64)
    turned = torch.cat([(a * cos - b * sin).to(F32), (b * cos + a * sin).to(F32), x[:, :h + kv, 2 * half:]], -1)
    return [turned[:, :h].reshape(inp["rows"], -1), _store(inp["k"], case, page, slot, turned[:, h:]),
            _store(inp["v"], case, page, slot, x[:, h + kv:])]


def _plain_attend(state):
    case, inp = state["case"], state["inp"]
    h, kv, d, ps, n = case["heads"], case["kv_heads"], case["head"], case["page"], case["sequences"]
    s, pos, _, _ = _places(inp, ps)
    pages = inp["table"].clamp(min=0).long()   # [sequences, pages]; what lies behind a sequence's end is masked
    k, v = (t[pages] for t in (inp["k"], inp["v"]))
    k, v = (t.to(F32) if case["fmt"] == "f16" else _unpack(t, case) for t in (k, v))
    k, v = (t.transpose(1, 2).reshape(n, kv, -1, d) for t in (k, v))
    at = torch.arange(inp["rows"], device="cuda") - inp["starts"][s]
    q = torch.zeros(n, inp["most"], h, d, device="cuda")
    last = torch.full((n, inp["most"]), -1, device="cuda", dtype=torch.int64)
    q[s, at], last[s, at] = inp["q"].reshape(-1, h, d), pos.long()
    q = q.reshape(n, inp["most"], kv, h // kv, d).permute(0, 2, 3, 1, 4).reshape(n, kv, -1, d)
    scores = torch.matmul(q, k.transpose(2, 3)).reshape(n, kv, h // kv, inp["most"], -1) / math.sqrt(d)
    seen = torch.arange(k.shape[2], device="cuda") <= last[..., None]   # [sequences, new, positions]
    scores = scores.masked_fill(~seen[:, None, None], -math.inf)
    e = torch.exp(scores - scores.amax(-1, keepdim=True).clamp(min=torch.finfo(F32).min))
    e = e / e.sum(-1, keepdim=True).clamp(min=torch.finfo(F32).tiny)
    out = torch.matmul(e.reshape(n, kv, -1, k.shape[2]), v).reshape(n, h, inp["most"], d)
    return out[s, :, at].reshape(inp["rows"], h * d).to(OUT_TYPES[case["out"]])


PLAIN = {"norm": _plain_norm, "gemm": _plain_gemm, "append": _plain_append, "attend": _plain_attend}


def run(state):
    if own:
        if "call" not in state:
            state["call"] = _program(state)
        return state["call"]()
    return PLAIN[state["case"]["kind"]](state)


# ---- what a pass cannot do without --------------------------------------------------------------

def work(case):
    kind = case["kind"]
    if kind == "norm":
        # the codes are written, and so are the values that they stand for
        count = case["rows"] * case["n"]
        moved = 4 + (8 if case["residual"] else 0) + 1 + 4
        return {"bytes": count * moved + 4 * case["n"] + 4 * case["rows"], "flops": 8 * count}
    if kind == "gemm":
        m, r, c = case["m"], case["rows"], case["cols"]
        return {"bytes": (m + r) * (c + 4) + 4 * m * r * (2 if case["residual"] else 1), "flops": 2 * m * r * c}
    new, lengths = _batch(case)
    rows, d, kv = int(new.sum()), case["head"], case["kv_heads"]
    if kind == "append":
        width = (case["heads"] + 2 * kv) * d
        kept = 2 * kv * _head_bytes(case)
        back = 0 if case["fmt"] == "f16" else 8 * kv * d   # the values that the codes stand for
        return {"bytes": rows * (4 * width + 4 * case["heads"] * d + kept + back), "flops": 6 * rows * width}
    seen = sum(int(n) * (int(l) - int(n)) + int(n) * (int(n) + 1) // 2 for n, l in zip(new, lengths))
    return {"bytes": int(lengths.sum()) * 2 * kv * _head_bytes(case) + rows * case["heads"] * d * 6,
            "flops": 4 * seen * case["heads"] * d}


# ---- the same results in 64 bits ----------------------------------------------------------------

def _exact_cache_values(pool, case, page_of, count):
    """[kv, count, head] values of one sequence's first `count` positions, in 64 bits."""
    ps, d = case["page"], case["head"]
    p = pool[page_of[:-(-count // ps)].long()]
    if case["fmt"] == "f16":
        v = p.to(F64)
    else:
        low, high = (p[:, :, :ps * d // 2].to(torch.int64) % 16, p[:, :, :ps * d // 2].to(torch.int64) // 16)
        codes = torch.empty(p.shape[0], p.shape[1], ps * d, device="cuda", dtype=F64)
        codes[..., 0::2], codes[..., 1::2] = low.to(F64), high.to(F64)
        scales = p[:, :, ps * d // 2:].contiguous().view(torch.float16).to(F64).reshape(p.shape[0], -1, d // 32, ps)
        v = (codes.reshape(p.shape[0], -1, ps, d) - 8) * scales.permute(0, 1, 3, 2).repeat_interleave(32, 3)
    return v.permute(1, 0, 2, 3).reshape(p.shape[1], -1, d)[:, :count]


def _exact_held(x, fmt):
    """The values that a cache of this format holds for FP32 rows x [rows, n]."""
    if fmt == "f16":
        return x.half().to(F64)
    blocks = x.reshape(-1, 32).to(F64)
    low, high = blocks.amin(1), blocks.amax(1)
    first = blocks.gather(1, blocks.abs().max(1).indices[:, None])[:, 0]
    top = torch.where(-low > high, low, torch.where(high > -low, high, first))
    d = (top / -8).half().to(F64)[:, None]
    ratio = (blocks / torch.where(d == 0, 1.0, d)).float().to(F64)
    return (torch.where(d == 0, 0.0, ratio.round().clamp(-8, 7)) * d).reshape(x.shape)


def exact(case, seed):
    inp, kind = _inputs(case, seed), case["kind"]
    if kind == "norm":
        u = inp["hidden"] if inp["residual"] is None else (inp["hidden"].to(F64) + inp["residual"].to(F64)).float()
        scales, values = [], []
        for part, w in ((p, inp["weight"].to(F64)) for p in u.split(1024)):
            part = part.to(F64)
            y = part * torch.rsqrt(part.pow(2).sum(1) / case["n"] + EPS)[:, None] * w
            scales.append(y.abs().max(1).values / 127)
            step = scales[-1].float().to(F64)[:, None]
            values.append((y / step).round() * step)
        return [u.to(F64), torch.cat(scales), torch.cat(values)]
    if kind == "gemm":
        w = inp["w"].to(F64).t().contiguous()
        y = torch.cat([x.to(F64) @ w for x in inp["x"].split(1024)])
        y = y * inp["xs"].to(F64)[:, None] * inp["ws"].to(F64)
        return y if inp["residual"] is None else y + inp["residual"].to(F64)
    new, lengths = _batch(case)
    h, kv, d, ps = case["heads"], case["kv_heads"], case["head"], case["page"]
    starts = np.concatenate([[0], np.cumsum(new)])
    if kind == "append":
        pos = torch.cat([torch.arange(l - n, l, device="cuda") for n, l in zip(new.tolist(), lengths.tolist())])
        x = inp["qkv"].to(F64).reshape(inp["rows"], -1, d)
        half, turned = case["rotary"] // 2, x.clone()
        wave = torch.polar(torch.full((), float(np.float32(ROPE_SCALE)), dtype=F64, device="cuda"),
                           pos.to(F64)[:, None] * inp["freq"].to(F64))[:, None]
        pair = torch.complex(x[:, :h + kv, :half], x[:, :h + kv, half:2 * half]) * wave
        turned[:, :h + kv, :half], turned[:, :h + kv, half:2 * half] = pair.real, pair.imag
        k, v = turned[:, h:h + kv].float(), x[:, h + kv:].float()
        held = [_exact_held(t.reshape(inp["rows"], -1), case["fmt"]) for t in (k, v)]
        query = turned[:, :h].reshape(inp["rows"], -1)
        if case["fmt"] != "f16":
            return [query] + held
        pools = [inp["k"].to(F64), inp["v"].to(F64)]
        for s, (a, b) in enumerate(zip(starts[:-1], starts[1:])):
            for page in set((pos[a:b] // ps).tolist()):
                rows = torch.nonzero(pos[a:b] // ps == page)[:, 0] + int(a)
                for pool, t in zip(pools, held):
                    pool[int(inp["table"][s, page])][:, pos[rows] % ps] = t[rows].reshape(-1, kv, d).transpose(0, 1)
        return [query] + pools
    out = torch.empty(inp["rows"], h, d, device="cuda", dtype=F64)
    for s, (n, length) in enumerate(zip(new.tolist(), lengths.tolist())):
        k, v = (_exact_cache_values(inp[t], case, inp["table"][s], length) for t in ("k", "v"))
        q = inp["q"][starts[s]:starts[s] + n].to(F64).reshape(n, h, d)
        hidden = torch.arange(length, device="cuda")[None] > torch.arange(length - n, length, device="cuda")[:, None]
        for head in range(h):
            scores = (q[:, head] @ k[head * kv // h].t().contiguous()) * d ** -0.5
            out[starts[s]:starts[s] + n, head] = torch.softmax(scores.masked_fill(hidden, -math.inf), 1) @ v[head * kv // h]
    return out.reshape(inp["rows"], -1)
