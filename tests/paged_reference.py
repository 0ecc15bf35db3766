"""Plain 64-bit numpy forms of the paged cache: page layout, quantization,
rotary append and attention, written from their definitions."""
import numpy as np

Q4_0, F16 = 2, 1


class Pool:
    """Key (or value) pages of a pool as host bytes."""

    def __init__(self, fmt, pages, kv_heads, page_size, head, rng=None):
        self.fmt, self.pages, self.kv, self.ps, self.d = fmt, pages, kv_heads, page_size, head
        per = 2 * head * page_size if fmt == F16 else page_size * (head // 2 + head // 16)
        # stale bytes: any nibbles, scales (and FP16 values) that are infinities and NaN among them
        rng = rng or np.random.default_rng(0)
        self.raw = rng.integers(0, 256, (pages, kv_heads, per), dtype=np.uint8)

    def values_view(self):
        assert self.fmt == F16
        return self.raw.view(np.float16).reshape(self.pages, self.kv, self.ps, self.d)

    def nibble_view(self):
        return self.raw[:, :, :self.ps * self.d // 2].reshape(self.pages, self.kv, self.ps, self.d // 2)

    def get_scales(self):
        return self.raw[:, :, self.ps * self.d // 2:].copy().view(np.float16).reshape(
            self.pages, self.kv, self.d // 32, self.ps)

    def put_scale(self, page, h, block, slot, value):
        at = self.ps * self.d // 2 + 2 * (block * self.ps + slot)
        self.raw[page, h, at:at + 2] = np.frombuffer(np.float16(value).tobytes(), np.uint8)

    def store(self, page, slot, x):
        """x [kv, d] FP32 at one place."""
        if self.fmt == F16:
            v = self.raw.view(np.float16).reshape(self.pages, self.kv, self.ps, self.d)
            with np.errstate(over="ignore"):
                v[page, :, slot] = x.astype(np.float16)
            return
        codes, scales = quantize(x)
        self.nibble_view()[page, :, slot] = codes[:, 0::2] | codes[:, 1::2] << 4
        for h in range(self.kv):
            for b in range(self.d // 32):
                self.put_scale(page, h, b, slot, scales[h, b])

    def load(self, page, slot):
        """[kv, d] in 64 bits."""
        if self.fmt == F16:
            return self.raw.view(np.float16).reshape(self.pages, self.kv, self.ps, self.d)[page, :, slot].astype(np.float64)
        nib = self.nibble_view()[page, :, slot]
        codes = np.stack([nib & 15, nib >> 4], -1).reshape(self.kv, self.d).astype(np.float64)
        at = self.ps * self.d // 2
        sc = np.stack([self.raw[page, :, at + 2 * (b * self.ps + slot):][:, :2].copy().view(np.float16)[:, 0]
                       for b in range(self.d // 32)], -1).astype(np.float64)
        return (codes - 8) * np.repeat(sc, 32, -1)


def quantize(x):
    """FP32 [..., d] -> (nibbles uint8 [..., d], FP16 scales [..., d / 32])."""
    b = x.reshape(*x.shape[:-1], -1, 32).astype(np.float32)
    with np.errstate(all="ignore"):
        at = np.argmax(np.where(np.isnan(b), -1, np.abs(b)), -1)[..., None]
        d = (np.take_along_axis(b, at, -1) / np.float32(-8)).astype(np.float16)
        bad = np.any(~(np.abs(b) <= 65504), -1, keepdims=True)
        df = d.astype(np.float32)
        q = np.clip(np.rint(b / np.where(df == 0, np.float32(1), df)) + 8, 0, 15)
        q = np.where(bad | (df == 0), 8, q)
    d = np.where(bad, np.float16(np.nan), np.where(df == 0, np.float16(0), d))   # zeros have the scale +0
    return q.reshape(x.shape).astype(np.uint8), d[..., 0]


def place(table, starts, lengths, page_size, pages, t):
    """(sequence, position, page) of batch row t; page None: nowhere."""
    for s in range(len(lengths)):
        if starts[s] <= t < starts[s + 1]:
            p = int(lengths[s]) - int(starts[s + 1]) + t
            if not 0 <= p < table.shape[1] * page_size:
                return s, p, None
            page = int(table[s, p // page_size])
            return s, p, page if 0 <= page < pages else None
    return None, None, None


def rotate(x, position, freq, rotary, scale):
    """x [heads, d] FP32 rotated in 64 bits, as FP32."""
    half = rotary // 2
    a = float(position) * freq.astype(np.float64)
    c, s = np.cos(a) * float(np.float32(scale)), np.sin(a) * float(np.float32(scale))
    v = x.astype(np.float64).copy()
    lo, hi = x[:, :half].astype(np.float64), x[:, half:rotary].astype(np.float64)
    v[:, :half], v[:, half:rotary] = lo * c - hi * s, hi * c + lo * s
    return v.astype(np.float32)


def attention(q, keys, values, visible):
    """One row: q [heads, d], keys / values [positions, kv, d] in 64 bits, the
    first `visible` positions seen.  Returns (out [heads, d], mean |v| [heads,
    d], score slack [heads]): the weights' mean of |v| and the largest
    sum |q| |k| / sqrt(d) that a score's rounding grows with."""
    heads, d = q.shape
    kv = keys.shape[1]
    out, mag, slack = np.zeros((heads, d)), np.zeros((heads, d)), np.zeros(heads)
    if visible <= 0:
        return out, mag, slack
    for h in range(heads):
        k, v = keys[:visible, h * kv // heads], values[:visible, h * kv // heads]
        s = k @ q[h].astype(np.float64) / np.sqrt(d)
        slack[h] = np.max(np.abs(k) @ np.abs(q[h]).astype(np.float64)) / np.sqrt(d)
        p = np.exp(s - np.max(s))
        p /= p.sum()
        out[h], mag[h] = p @ v, p @ np.abs(v)
    return out, mag, slack
