"""CPU checks of Rwkv7RowsSession: what a step's launches read and write lies in the session's buffers, and no launch writes
over what a later one still reads, also where LoRA ranks exceed the model's width."""
import numpy as np
import pytest

from sharpinference_amd import native, rwkv7
from sharpinference_amd.rwkv7_rows import ROWS, Rwkv7RowsSession


class _Buffer:
    def __init__(self, ptr, nbytes):
        self.ptr, self.nbytes = ptr, nbytes

    def upload(self, host, offset=0):
        assert offset + host.nbytes <= self.nbytes


class _Ranges:
    """Stands in for a HipContext: launches nothing, follows which launch wrote what last."""

    def __init__(self):
        self.buffers, self.next, self.writes, self.read_from = [], 1 << 20, [], []

    def alloc(self, nbytes):
        self.buffers.append(_Buffer(self.next, nbytes))
        self.next += (nbytes + 4095) // 4096 * 4096 + 4096
        return self.buffers[-1]

    def _inside(self, ptr, nbytes):
        assert any(b.ptr <= ptr and ptr + nbytes <= b.ptr + b.nbytes for b in self.buffers), (ptr, nbytes)

    def _writes(self, who, ptr, nbytes):
        self._inside(ptr, nbytes)
        self.writes.append((who, ptr, ptr + nbytes))

    def _reads(self, ptr, nbytes):
        """Who wrote [ptr, ptr + nbytes), which has one writer."""
        self._inside(ptr, nbytes)
        for who, first, last in reversed(self.writes):
            if first < ptr + nbytes and ptr < last:
                assert first <= ptr and ptr + nbytes <= last, f"{who} wrote a part of it"
                return who
        return None

    def gather_row(self, fmt, table, rows, cols, index, out):
        self._inside(index, 4)
        self._writes("gather", out, 4 * cols)

    def batch_matvec(self, fmt, w, x, control, y, batch, rows, cols):
        self.read_from.append((w, self._reads(x, 4 * batch * cols)))
        self._writes("product", y, 4 * batch * rows)

    def t0_elementwise(self, op, left, right, out, count):
        assert self._reads(left, 4 * count) in ("product", "relu")
        self._writes(op, out, 4 * count)

    def layernorm_mix_rows(self, args):
        rows = 4 * args.batch.rows * args.n
        if args.mixes or args.residual:   # (the first norm's input is written row by row)
            self._reads(args.x, rows)
        else:
            self._inside(args.x, rows)
        if args.residual:
            assert self._reads(args.residual, rows) == "product"
            self._writes("sum", args.updated, rows)
        self._writes("norm", args.output, rows * max(args.mixes, 1))

    def rwkv7_wkv_rows(self, args):
        rows = 4 * args.batch.rows * args.heads * 64
        for name in ("r", "k", "v", "w_lora", "a_lora", "gate") + (() if args.first_layer else ("v_lora",)):
            assert self._reads(getattr(args, name), rows) == "product", name
        self._writes("core", args.output, rows)


@pytest.mark.parametrize("hidden,ranks", [(128, (32, 32, 32, 256)), (128, (288, 160, 32, 416)), (64, (96, 96, 64, 256)),
                                          (256, (32, 64, 32, 64))])
def test_step_stays_in_its_buffers(hidden, ranks):
    w, a, v, g = ranks
    cfg = rwkv7.Rwkv7Config(layers=2, hidden=hidden, heads=hidden // 64, ffn=2 * hidden, vocab=64, rank_w=w, rank_a=a, rank_v=v,
                            rank_g=g)
    hip = _Ranges()
    session = Rwkv7RowsSession(hip, cfg, rwkv7.synth_weights(cfg, seed=1), slots=2)
    session._step(session._batch(session.from_, session.to, ROWS))
    read_from = dict(hip.read_from)
    for l, L in enumerate(session.layers):
        loras = "wag" + ("v" if l else "")
        for name in ["receptance", "key", "value", "ffn_key"] + [n + "1" for n in loras]:
            assert read_from[L[name].ptr] == "norm", (l, name)
        second = {"w": "tanh", "g": "sigmoid", "a": "product", "v": "product"}
        for n in loras:
            assert read_from[L[n + "2"].ptr] == second[n], (l, n)
    assert read_from[session.head.ptr] == "norm"
