"""RWKV-7 over up to 16 rows a step: prompts in pieces of 16 rows, several sequences at once, beam search.

The rows of a step belong to sequences whose states lie in slots
(si_hip_row_batch); a layer is the norm and token mix of all rows, the
projections as batched products (weights read once for the rows), the
time-mix core of every sequence's rows, and the channel mix.  Weights,
layers and formulas are Rwkv7DecodeSession's, products and states FP32.  The
reference runs the graph token after token
(PortableRwkv7GraphProvider.cs:190-292) and has no search.
"""
from __future__ import annotations

from typing import Dict, List, NamedTuple, Optional, Sequence

import numpy as np

from . import native
from .rwkv7 import LAYER_VECTORS, Rwkv7Config, Rwkv7Weights

ROWS = 16          # of a step: the batched products' most
LN_EPS = 1e-5


class Hypothesis(NamedTuple):
    """A beam's tokens behind its prompt, and the sum of their log-probabilities."""
    tokens: List[int]
    score: float


class Rwkv7RowsSession:
    """Device-resident model, the states of `slots` sequences, and recorded steps."""

    def __init__(self, hip: native.HipContext, cfg: Rwkv7Config, weights: Rwkv7Weights, slots: int = ROWS):
        if cfg.head_size != 64:
            raise ValueError("the RWKV-7 step takes heads of 64")
        if slots < 1:
            raise ValueError("a session needs a slot")
        self.hip, self.cfg, self.slots = hip, cfg, int(slots)
        self._bufs: List[native.DeviceBuffer] = []
        self._plans: Dict[tuple, native.Plan] = {}
        D, F, V = cfg.hidden, cfg.ffn, cfg.vocab
        up, new = self._upload, self._alloc
        self.embed, self.head = up(weights.embed), up(weights.head)
        self.norms = {n: up(getattr(weights, n)) for n in ("ln0_weight", "ln0_bias", "ln_out_weight", "ln_out_bias")}
        self.layers = []
        for l in range(cfg.layers):
            W = weights.layers[l]
            L = {n: up(W[n]) for n in (*cfg.matrix_shapes(l), *LAYER_VECTORS, "mix")}
            L["att_prev"], L["ffn_prev"] = new(4 * D * slots), new(4 * D * slots)
            L["wkv"] = new(4 * D * 64 * slots)
            self.layers.append(L)
        # a step's inputs: row starts, slots, the rows that count, tokens
        self.starts, self.from_, self.to, self.control, self.tokens = new(4 * (ROWS + 1)), new(4 * ROWS), new(4 * ROWS), new(8), \
            new(4 * ROWS)
        rows = lambda width: new(4 * ROWS * width)
        self.embedded, self.hidden, self.norm, self.mixed = rows(D), [rows(D), rows(D)], rows(D), rows(6 * D)
        self.r, self.k, self.v, self.att, self.add, self.v_first = (rows(D) for _ in range(6))
        self.lora = {n: rows(rank) for n, rank in (("w", cfg.rank_w), ("a", cfg.rank_a), ("g", cfg.rank_g), ("v", cfg.rank_v))}
        self.activated = rows(max(cfg.rank_w, cfg.rank_g))   # of one LoRA vector at a time
        self.lora_out = {n: rows(D) for n in "wagv"}
        self.ffn, self.ffn_relu = rows(F), rows(F)
        self.logits = rows(V)
        self.workspace = new(native.rwkv7_wkv_rows_workspace_bytes(cfg.heads))
        # beam search
        self.parents, self.scores, self.done = new(4 * ROWS), new(4 * ROWS), new(4 * ROWS)
        self.beam_from, self.beam_slots = new(4 * ROWS), new(4 * ROWS)
        self.select_workspace: Dict[tuple, native.DeviceBuffer] = {}
        self.state_arrays = native.slot_arrays([(L[n].ptr, size) for L in self.layers
                                                for n, size in (("att_prev", 4 * D), ("ffn_prev", 4 * D), ("wkv", 4 * D * 64))])

    # -- buffers -------------------------------------------------------------------
    def _alloc(self, nbytes: int) -> native.DeviceBuffer:
        b = self.hip.alloc(max(int(nbytes), 16))
        self._bufs.append(b)
        return b

    def _upload(self, arr: np.ndarray) -> native.DeviceBuffer:
        b = self._alloc(arr.nbytes)
        b.upload(np.ascontiguousarray(arr))
        return b

    # -- one step, as launches ---------------------------------------------------------
    def _batch(self, slots_in: native.DeviceBuffer, slots_out: native.DeviceBuffer, most: int) -> native.RowBatch:
        return native.RowBatch(self.starts.ptr, slots_in.ptr, slots_out.ptr, ROWS, self.slots, ROWS, most)

    def _step(self, batch: native.RowBatch) -> None:
        hip, cfg = self.hip, self.cfg
        D, F, fmt = cfg.hidden, cfg.ffn, cfg.weight_format
        product = lambda w, x, y, rows, cols, f=fmt: hip.batch_matvec(f, w, x, self.control.ptr, y, ROWS, rows, cols)

        def norm(x, residual, weight, bias, mix, mixes, state, updated, out):
            hip.layernorm_mix_rows(native.LayernormMixRowsArgs(batch, x, residual, weight, bias, mix, state, updated, out, D, mixes,
                                                               native.F32, LN_EPS))
        for row in range(ROWS):
            hip.gather_row(cfg.embed_format, self.embed.ptr, cfg.vocab, D, self.tokens.ptr + 4 * row,
                           self.embedded.ptr + 4 * D * row)
        x, other = self.hidden[0].ptr, self.hidden[1].ptr
        norm(self.embedded.ptr, 0, self.norms["ln0_weight"].ptr, self.norms["ln0_bias"].ptr, 0, 0, 0, 0, x)
        residual = 0
        for l, L in enumerate(self.layers):
            p = {n: b.ptr for n, b in L.items()}
            norm(x, residual, p["ln1_weight"], p["ln1_bias"], p["mix"], 6, p["att_prev"], other if residual else 0, self.mixed.ptr)
            if residual:
                x, other = other, x
            mixed = [self.mixed.ptr + 4 * ROWS * D * m for m in range(6)]   # r, w, k, v, a, g
            for name, m, y in (("receptance", 0, self.r), ("key", 2, self.k), ("value", 3, self.v)):
                product(p[name], mixed[m], y.ptr, D, D)
            ranks = {"w": (1, cfg.rank_w, "tanh"), "a": (4, cfg.rank_a, None), "g": (5, cfg.rank_g, "sigmoid")}
            if l > 0:
                ranks["v"] = (3, cfg.rank_v, None)
            for name, (m, rank, function) in ranks.items():
                hidden = self.lora[name].ptr
                product(p[name + "1"], mixed[m], hidden, rank, D)
                if function:
                    hip.t0_elementwise(function, hidden, 0, self.activated.ptr, ROWS * rank)
                    hidden = self.activated.ptr
                product(p[name + "2"], hidden, self.lora_out[name].ptr, D, rank)
            out = {n: b.ptr for n, b in self.lora_out.items()}
            hip.rwkv7_wkv_rows(native.Rwkv7WkvRowsArgs(
                batch, cfg.heads, int(l == 0), self.r.ptr, self.k.ptr, self.v.ptr, out["w"], out["a"], out["g"], out["v"], p["w0"],
                p["a0"], p["v0"], p["k_k"], p["k_a"], p["r_k"], p["lnx_weight"], p["lnx_bias"], self.v_first.ptr, p["wkv"],
                self.att.ptr, self.workspace.ptr, native.F32))
            product(p["output"], self.att.ptr, self.add.ptr, D, D)
            norm(x, self.add.ptr, p["ln2_weight"], p["ln2_bias"], p["ffn_mix"], 1, p["ffn_prev"], other, self.norm.ptr)
            x, other = other, x
            product(p["ffn_key"], self.norm.ptr, self.ffn.ptr, F, D)
            hip.t0_elementwise("relu", self.ffn.ptr, 0, self.ffn_relu.ptr, ROWS * F)
            hip.t0_elementwise("square", self.ffn_relu.ptr, 0, self.ffn.ptr, ROWS * F)
            product(p["ffn_value"], self.ffn.ptr, self.add.ptr, D, F)
            residual = self.add.ptr
        norm(x, residual, self.norms["ln_out_weight"].ptr, self.norms["ln_out_bias"].ptr, 0, 0, 0, other, self.norm.ptr)
        product(self.head.ptr, self.norm.ptr, self.logits.ptr, cfg.vocab, D, cfg.head_format)

    def _plan(self, key: tuple, body) -> native.Plan:
        if key not in self._plans:
            self._plans[key] = self.hip.record(body)
        return self._plans[key]

    # -- steps -----------------------------------------------------------------------------
    def step(self, sequences: Sequence[Sequence[int]], from_: Sequence[int], to: Sequence[int]) -> np.ndarray:
        """The next tokens of some sequences (16 in all, at most): sequence s goes on from slot from_[s] (-1: from the
        beginning) and leaves its state in slot to[s] (-1: nowhere; a sequence without tokens leaves none).  Returns the logits of
        every row [rows, vocab]."""
        counts = [len(t) for t in sequences]
        rows = sum(counts)
        if not sequences or len(sequences) > ROWS or rows < 1 or rows > ROWS:
            raise ValueError(f"a step takes 1 to {ROWS} rows of as many sequences at most, not {rows} of {len(sequences)}")
        if len(from_) != len(counts) or len(to) != len(counts):
            raise ValueError("a slot to go on from and one to leave the state in for each sequence")
        if any(not -1 <= s < self.slots for s in (*from_, *to)):
            raise ValueError(f"slots are -1 or 0..{self.slots - 1}")
        kept = [s for s in to if s >= 0]
        if len(set(kept)) != len(kept) or any(s in kept and (to[i] != s) for i, s in enumerate(from_)):
            raise ValueError("a slot that one sequence writes may not be another's")
        tokens = np.concatenate([np.asarray(t, np.int32).reshape(-1) for t in sequences]).astype(np.int32)
        if np.any((tokens < 0) | (tokens >= self.cfg.vocab)):
            raise ValueError(f"tokens lie in 0..{self.cfg.vocab - 1}")
        starts = np.full(ROWS + 1, rows, np.int32)
        starts[:len(counts) + 1] = np.concatenate([[0], np.cumsum(counts)])
        pad = lambda x: np.concatenate([np.asarray(x, np.int32), np.full(ROWS - len(x), -1, np.int32)])
        for buf, value in ((self.starts, starts), (self.from_, pad(from_)), (self.to, pad(to)),
                           (self.control, np.array([0, rows], np.int32)), (self.tokens, np.pad(tokens, (0, ROWS - rows)))):
            buf.upload(value.astype(np.int32))
        most = 1 if max(counts) == 1 else ROWS
        self._plan(("step", most), lambda: self._step(self._batch(self.from_, self.to, most))).launch()
        return self.logits.readback(np.float32, rows * self.cfg.vocab).reshape(rows, -1)

    def prefill(self, tokens: Sequence[int], slot: int) -> np.ndarray:
        """A whole prompt into a slot, 16 rows a step; returns the last row's logits."""
        if len(tokens) < 1:
            raise ValueError("a prompt has a token at least")
        source, logits = -1, None
        for i in range(0, len(tokens), ROWS):
            logits = self.step([tokens[i:i + ROWS]], [source], [slot])
            source = slot
        return logits[-1]

    def beam_search(self, prompts: Sequence[Sequence[int]], beams: int, steps: int,
                    end_token: Optional[int] = None) -> List[List[Hypothesis]]:
        """The `beams` best continuations of each prompt by `steps` tokens (fewer behind an end token), best first.
        The states take slots 0 to len(prompts) * beams - 1.

        A token is one replayed plan: the candidates of all beams, the moves of their states, and the step of the tokens they
        chose; only the choices come back."""
        n = len(prompts)
        if n < 1 or beams < 1 or n * beams > min(ROWS, self.slots):
            raise ValueError(f"{n} prompts of {beams} beams: 1 to {min(ROWS, self.slots)} rows")
        if steps < 1:
            raise ValueError("a search takes a step at least")
        end = -1 if end_token is None else int(end_token)
        if not -1 <= end < self.cfg.vocab:
            raise ValueError(f"the end token lies in 0..{self.cfg.vocab - 1}")
        rows, vocab = n * beams, self.cfg.vocab
        first = np.stack([self.prefill(p, s * beams) for s, p in enumerate(prompts)])
        # every prompt begins with one beam, in its first slot
        logits = np.zeros((rows, vocab), np.float32)
        logits[::beams] = first
        scores = np.full(ROWS, -np.inf, np.float32)
        scores[:rows:beams] = 0.0
        self.logits.upload(logits)
        self.scores.upload(scores)
        self.done.upload(np.zeros(ROWS, np.int32))
        self.beam_slots.upload(np.arange(ROWS, dtype=np.int32))
        self.starts.upload(np.minimum(np.arange(ROWS + 1), rows).astype(np.int32))
        self.control.upload(np.array([0, rows], np.int32))
        self.tokens.upload(np.zeros(ROWS, np.int32))
        size = (n, beams)
        if size not in self.select_workspace:
            self.select_workspace[size] = self._alloc(native.beam_select_workspace_bytes(n, beams, beams, vocab))
        done = self.done.ptr if end >= 0 else 0
        select = native.BeamSelectArgs(self.logits.ptr, self.scores.ptr, done, self.beam_slots.ptr, self.parents.ptr, self.tokens.ptr,
                                       self.scores.ptr, done, self.beam_from.ptr, self.beam_slots.ptr, self.select_workspace[size].ptr,
                                       vocab, vocab, n, beams, beams, native.F32, end)

        def choose():
            self.hip.beam_select(select)
            self.hip.copy_slots(self.state_arrays, self.slots, self.beam_from.ptr, self.beam_slots.ptr, rows)

        def choose_and_step():
            choose()
            self._step(self._batch(self.beam_slots, self.beam_slots, 1))
        history = []
        for i in range(steps):
            # (the last choice needs no step behind it; a beam that has ended is stepped with the rest, and its logits do not count)
            last = i == steps - 1
            self._plan((last, n, beams, end), choose if last else choose_and_step).launch()
            history.append((self.parents.readback(np.int32, rows), self.tokens.readback(np.int32, rows)))
        final = self.scores.readback(np.float32, rows)
        found = []
        for s in range(n):
            found.append([])
            for b in range(beams):
                if not np.isfinite(final[s * beams + b]):
                    continue
                at, tokens = b, []
                for parents, chosen in reversed(history):
                    tokens.append(int(chosen[s * beams + at]))
                    at = int(parents[s * beams + at])
                tokens.reverse()
                if end >= 0 and end in tokens:
                    tokens = tokens[:tokens.index(end) + 1]
                found[-1].append(Hypothesis(tokens, float(final[s * beams + b])))
        return found

    # -- states -------------------------------------------------------------------------------
    def read_state(self, layer: int, slot: int):
        """(att_prev, ffn_prev, wkv) of a slot, as Rwkv7DecodeSession has them."""
        D, L = self.cfg.hidden, self.layers[layer]
        return (L["att_prev"].readback(np.float32, D, 4 * D * slot), L["ffn_prev"].readback(np.float32, D, 4 * D * slot),
                L["wkv"].readback(np.float32, D * 64, 4 * D * 64 * slot).reshape(self.cfg.heads, 64, 64))

    def close(self) -> None:
        for plan in self._plans.values():
            plan.destroy()
        self._plans = {}
        for b in self._bufs:
            b.free()
        self._bufs = []
