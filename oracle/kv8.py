"""The decode step over a cache in 8 bits, restated in numpy from the formulas of include/zwgpu.h:
rotary positions, the cache's append and values, the attention over it (64 bits) with a bound
on the kernels' error, and the rules on the logits (the f32 operations, one by one)."""
import numpy as np

BLOCK = 32


def rope(x, cos, sin, pos, interleaved):
    """x f32 [n][heads][d] rotated to positions pos [n], the f32 operations of the definition."""
    rot = 2 * cos.shape[1]
    y = x.copy()
    a = x[..., 0:rot:2] if interleaved else x[..., : rot // 2]
    b = x[..., 1:rot:2] if interleaved else x[..., rot // 2: rot]
    c, s = cos[pos][:, None], sin[pos][:, None]
    ra, rb = a * c - b * s, a * s + b * c
    if interleaved:
        y[..., 0:rot:2], y[..., 1:rot:2] = ra, rb
    else:
        y[..., : rot // 2], y[..., rot // 2: rot] = ra, rb
    return y


def quantise(rows):
    """int8 values and the f32 scale of a block's rows [32][d]."""
    top = np.abs(rows).max()
    if not np.isfinite(rows).all():
        return np.zeros(rows.shape, np.int8), np.float32(np.nan)
    if top == 0:
        return np.zeros(rows.shape, np.int8), np.float32(0)
    return np.rint(127.0 * rows.astype(np.float64) / np.float64(top)).astype(np.int8), np.float32(top) / np.float32(127)


class Cache:
    """The cache's contents in the order of tokens: ints [side][n_batch][n_head_kv][n_ctx][d]."""

    def __init__(self, n_batch, n_head_kv, d, n_ctx):
        self.n_batch, self.n_head_kv, self.d, self.n_ctx = n_batch, n_head_kv, d, n_ctx
        self.ints = np.zeros((2, n_batch, n_head_kv, n_ctx, d), np.int8)
        self.scale = np.zeros((2, n_batch, n_head_kv, n_ctx // BLOCK), np.float32)
        self.open = np.zeros((2, n_batch, n_head_kv, BLOCK, d), np.float32)
        self.tag = np.full((n_batch, n_head_kv), -1, np.int32)

    def values(self, dtype=np.float32):
        return self.ints.astype(dtype) * np.repeat(self.scale, BLOCK, axis=-1)[..., None].astype(dtype)

    def append(self, k, v, past, count=None):
        """k, v f32 [n_batch][n][n_head_kv][d] at past [n_batch]."""
        n = k.shape[1]
        for b in range(self.n_batch):
            p, m = int(past[b]), n if count is None else int(count[b])
            if m == 0:
                continue
            b0, b1 = p // BLOCK, (p + m - 1) // BLOCK
            for h in range(self.n_head_kv):
                for side, x in ((0, k), (1, v)):
                    rows = np.zeros(((b1 - b0 + 1) * BLOCK, self.d), np.float32)
                    held = p - b0 * BLOCK
                    if held and self.tag[b, h] == b0:
                        rows[:held] = self.open[side, b, h, :held]
                    elif held:
                        old = self.ints[side, b, h, b0 * BLOCK: b0 * BLOCK + held].astype(np.float32)
                        rows[:held] = old * self.scale[side, b, h, b0]
                    rows[held: held + m] = x[b, :m, h]
                    for j in range(b0, b1 + 1):
                        part = rows[(j - b0) * BLOCK: (j - b0 + 1) * BLOCK]
                        q, t = quantise(part)
                        self.ints[side, b, h, j * BLOCK: (j + 1) * BLOCK] = q
                        self.scale[side, b, h, j] = t
                    self.open[side, b, h] = rows[-BLOCK:]
                self.tag[b, h] = b1


def attention(q, k, v, past, count, first, pieces, out_half_step=0.0):
    """q [n_batch][n][n_head][d] over the cache's values k, v [n_batch][n_head_kv][n_ctx][d], all in
    64 bits. Returns the output (rows behind count: NaN) and a bound on a kernel's error.

    The bound, per output, with S = sum over d of |q k| / sqrt(d) the largest over the row's keys:
      - a query in one f16 piece is off by 2^-12 of an element, in two by 2^-23 of its largest
        (whichever is larger counts for both: at most 2^-11 and 2^-22 with the subnormal pieces of
        elements far below the largest one); a bf16 query (pieces 0) is exact;
      - its product with exact integers is summed in f32, truncated: at most d + 16 steps of 2^-23;
        the scale, unit and log2(e) factors round three times more;
      - exp2 is off by 2^-22, and by the score's rounding; numerator and denominator both: twice;
      - a probability is off by 2^-12 or 2^-22 in its pieces, its value scale's ratio by 2^-23;
      - sums over the keys: one step of 2^-23 per key at the most, and 32 more for the merges;
      - all relative to sum p |v| / sum p, and the half step of the output's type;
      - a probability's last piece ends at f16's smallest step: 2^15 p vs / ref (ref the largest
        value scale the call's rows see, sum p >= 1) is off by half of 2^-24 at the least, which is
        2^-40 of ref, so 2^-40 of the largest value, for each key and int8 unit of 127. Calls of more
        than 48 query rows to a kv head hold 2^11 p vs / ref with p up to 2^4 (a maximum that is at
        most 4 too low, so sum p >= 1 as before): half of 2^-24 there is 2^-36 of ref."""
    B, n, H, d = q.shape
    group = H // k.shape[1]
    out, tol = np.full(q.shape, np.nan), np.zeros(q.shape)
    for b in range(B):
        p, m = int(past[b]), n if count is None else int(count[b])
        lo = 0 if first is None else int(first[b])
        for i in range(m):
            hi = p + i + 1
            for h in range(H):
                if lo >= hi:
                    out[b, i, h] = 0
                    continue
                kk, vv = k[b, h // group, lo:hi].astype(np.float64), v[b, h // group, lo:hi].astype(np.float64)
                qq = q[b, i, h].astype(np.float64)
                s = kk @ qq / np.sqrt(d)
                e = np.exp(s - s.max())
                w = e / e.sum()
                out[b, i, h] = w @ vv
                # largest |q| in every place where a piece may be subnormal
                size = (np.abs(kk) @ np.maximum(np.abs(qq), np.abs(qq).max() * 2.0 ** -11)).max() / np.sqrt(d)
                piece = {0: 0.0, 1: 2.0 ** -11, 2: 2.0 ** -22}[pieces]
                ds = size * (piece + (d + 20) * 2.0 ** -23) + 2.0 ** -22 * (1 + np.abs(s).max())
                rel = 2 * ds + (2.0 ** -11 if pieces < 2 else 2.0 ** -21) + (hi - lo + 32) * 2.0 ** -23
                least = (hi - lo) * (2.0 ** -40 if n * group <= 48 else 2.0 ** -36) * np.abs(v[b, h // group, :p + m]).max()
                tol[b, i, h] = rel * (w @ np.abs(vv)) + out_half_step * np.abs(out[b, i, h]) + least
    return out, tol * 1.01 + 1e-30


def logits(x, recent, window, repeat, presence, frequency, bias_ids, bias, allow):
    """One row: the rules' f32 operations, and the first index of the largest (-1: none)."""
    f, x = np.float32, x.copy()
    ids, times = np.unique(np.asarray(recent[max(0, len(recent) - window):], np.int64), return_counts=True)
    for t, c in zip(ids, times):
        if 0 <= t < len(x):
            y = x[t] * (f(1) / f(repeat)) if x[t] > 0 else x[t] * f(repeat)
            x[t] = y - (f(c) * f(frequency) + f(presence))
    add = np.zeros_like(x)
    for t, a in zip(bias_ids, bias):
        if 0 <= t < len(x):
            add[t] += f(a)
    x = np.where(add != 0, x + add, x)
    if allow is not None:
        t = np.arange(len(x))
        x = np.where((allow.view(np.uint32)[t // 32] >> (t % 32).astype(np.uint32)) & 1, x, f(-np.inf))
    seen = np.where(np.isnan(x), f(-np.inf), x)
    return x, int(seen.argmax()) if seen.max() > -np.inf else -1
