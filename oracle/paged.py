"""The cache in pages and trees of drafted tokens, restated in numpy from the formulas of include/zwgpu.h: the
append (the f32 operations one by one, one rounding), the attention in 64 bits with a bound on the kernels'
error, the acceptance and the rows it keeps."""
import numpy as np

from oracle.kv8 import rope


def ancestors(parent):
    """For each token of a tree, its index and those above it."""
    above = []
    for i, a in enumerate(parent):
        above.append([i] + (above[a] if a >= 0 else []))
    return above


def seen_slots(past, count, first, n_slots, parent=None):
    """seen [count][n_slots]: which slots each query of a sequence sees."""
    seen = np.zeros((count, n_slots), bool)
    above = None if parent is None else ancestors(parent[:count])
    for i in range(count):
        if parent is None:
            seen[i, : past + i + 1] = True
        else:
            seen[i, :past] = True
            seen[i, [past + j for j in above[i]]] = True
    seen[:, :first] = False
    return seen


def positions(past, count, parent=None):
    if parent is None:
        return past + np.arange(count)
    return past + np.array([len(a) - 1 for a in ancestors(parent[:count])], int)


def rotated(x, cos, sin, pos, interleaved):
    return rope(x, cos, sin, pos, interleaved)


def accept(tokens, ids, parent):
    """The agreed tokens' indices, and the model's token after the last one."""
    path = [0]
    while True:
        at = path[-1]
        below = [i for i in range(len(tokens)) if parent[i] == at and tokens[i] == ids[at]]
        if not below:
            return path, int(ids[at])
        path.append(below[0])


def attention(q, k, v, seen, pieces, half_step, big):
    """q [n][n_head][d] over a sequence's k, v [n_head_kv][n_slots][d] (values in f64, finite where seen), seen
    [n][n_slots]. Returns the output and a bound on a kernel's error.

    The bound, per output, with S the largest sum over d of |q k| / sqrt(d) of the row's keys:
      - a query in one f16 piece is off by 2^-12 of an element, in two by 2^-23 of its largest (whichever is larger
        counts for both: at most 2^-11 and 2^-22 with the subnormal pieces of elements far below the largest one);
        a bf16 query (pieces 0) is exact;
      - its product with exact keys is summed in f32, truncated: at most d + 16 steps of 2^-23; the scale, unit and
        log2(e) factors round three times more;
      - exp2 is off by 2^-22, and by the score's rounding; numerator and denominator both: twice;
      - a probability in f16 pieces is off by 2^-12 or 2^-22, both in what weighs the value and, where the sum takes
        the rounded one, in that; one rounded to bf16 by 2^-8: it weighs and is summed alike, so the output is off by
        2^-8 of the sum of w |v - o|, no more than 2^-8 (sum of w |v| + |o|);
      - sums over the keys: one step of 2^-23 per key at the most, and 32 more for the merges;
      - all relative to sum p |v| / sum p, and the half step of the output's type;
      - a probability's last f16 piece ends at f16's smallest step: 2^15 p is off by half of 2^-24 at the least,
        2^-40 of the largest probability for each key (calls that hold 2^11 p, with p up to 2^4, `big`: 2^-36)."""
    n, H, d = q.shape
    group = H // k.shape[0]
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    rows = np.flatnonzero(seen.any(1))
    used = np.flatnonzero(seen.any(0))
    if len(rows) == 0:
        return out, tol + 1e-30
    mask, number = seen[np.ix_(rows, used)], seen[rows].sum(1)[:, None]
    for h in range(H):
        kk, vv, qq = k[h // group, used], v[h // group, used], q[rows, h].astype(np.float64)
        s = np.where(mask, qq @ kk.T / np.sqrt(d), -np.inf)
        e = np.exp(s - s.max(1, keepdims=True))
        w = e / e.sum(1, keepdims=True)
        o = w @ vv
        held = np.maximum(np.abs(qq), np.abs(qq).max(1, keepdims=True) * 2.0 ** -11)
        size = np.where(mask, held @ np.abs(kk).T, 0).max(1, keepdims=True) / np.sqrt(d)
        piece = {0: 0.0, 1: 2.0 ** -11, 2: 2.0 ** -22}[pieces]
        ds = size * (piece + (d + 20) * 2.0 ** -23) + 2.0 ** -22 * (1 + np.abs(np.where(mask, s, 0)).max(1, keepdims=True))
        rel = 2 * ds + {0: 0.0, 1: 2.0 ** -11, 2: 2.0 ** -21}[pieces] + (number + 32) * 2.0 ** -23
        if pieces == 0:  # the sum of w |v - o|, a column at a time
            off = 2.0 ** -8 * np.stack([(w * np.abs(vv[:, c][None] - o[:, c][:, None])).sum(1) for c in range(d)], 1)
        else:
            most = np.array([np.abs(vv[m]).max() for m in mask])[:, None]
            off = number * (2.0 ** -36 if big else 2.0 ** -40) * most
        out[rows, h], tol[rows, h] = o, rel * (w @ np.abs(vv)) + off + half_step * np.abs(o)
    return out, tol * 1.01 + 1e-30
