"""Inputs for which attention's roundings of fp32 rows can be told apart, and a bound that is near them.

The bound of kv_forms.attention_near is dominated by what D additions in fp32 may do.  Here a row has two values that are not 0, so its scores are
sums of two products, and a window leaves it 9 keys at most: what is left is what the operands hold.  All relative to sum p |v|:
  scores   A = the largest sum |q k| scale of a row; the queries' two parts hold 2^-22, a product of parts is exact, the additions of two products of two parts
           each (adding 0 is exact) and the two factors (scale times log2(e), two fp32 roundings of it, and the row's own power of two) are at most 8 roundings:
           A (2^-22 + 8 2^-24).  A weight is exp of that and its sum of weights moves as well: twice it.
  argument of exp2: score - m + 8 in one rounding, of a number of at most 16 + 2 A log2(e): that times 2^-24 ln 2, twice (weight, sum).
  weights  two parts 2^-22, exp2 itself 2^-22, and the same in their sum.
  sums     9 keys in at most 32 + 8 additions of a product and 16 of a join (4 waves, 2 levels), each at most 2^-23, for values and weights.
           Shifts by the maximum in a join: exp2 of a difference that is a rounding off, 2^-24 (16 + 2 A log2(e)) ln 2 and 2^-22 once more.
  output   half a step of fp32.
`emulate` is the operator with operands of that many parts, all else in 64 bits."""
import numpy as np

WINDOW = 9
# sequences (rows, keys), nq, nk, D: few rows (16 and 32 columns of a head's group) and prompts, of each head size
CASES = [(seqs, 4, 2, D) for D in (64, 96, 128, 192, 256) for seqs in ([(3, 40), (2, 9), (8, 300)], [(14, 70), (5, 5)], [(45, 70), (66, 90)])]
SCALE = 1.5


def inputs(rng, n, keys, nq, nk, D):
    """q [n][nq][D] with two values a row, k and v [keys][nk][D] fp32, v of one sign."""
    q = np.zeros((n, nq, D), np.float32)
    for i in range(n):
        for h in range(nq):
            at = rng.choice(D, 2, replace=False)
            q[i, h, at] = rng.uniform(1, 2, 2) * rng.choice([-1, 1], 2)
    k = (rng.uniform(0.5, 1.5, (keys, nk, D)) * rng.choice([-1, 1], (keys, nk, D))).astype(np.float32)
    v = rng.uniform(1, 2, (keys, nk, D)) ** 3
    return q, k, v.astype(np.float32)


def seen(rows, keys):
    """[rows][keys] of a causal window of 9."""
    pos, key = np.arange(keys - rows, keys)[:, None], np.arange(keys)[None]
    return (key <= pos) & (key > pos - WINDOW)


def parts(x, count):
    """What `count` fp16 parts hold of x, relative to a power of two that puts the row's largest in [2^14, 2^15)."""
    up = 2.0 ** (14 - np.floor(np.log2(np.abs(x).max(-1, keepdims=True))))
    x, held = x * up, 0.0
    for _ in range(count):
        held = held + (x - held).astype(np.float16).astype(np.float64)
    return held / up


def emulate(q, k, v, scale, see, q_parts, w_parts):
    """One head in 64 bits: rows q [n][D] over k, v [L][D]."""
    s = np.where(see, (parts(q.astype(np.float64), q_parts) @ k.astype(np.float64).T) * scale, -np.inf)
    w = 256 * np.exp(s - s.max(-1, keepdims=True))
    p = sum_ = 0.0
    for _ in range(w_parts):
        p = p + (w - p).astype(np.float16).astype(np.float64)
    sum_ = p.sum(-1, keepdims=True)
    return p @ v.astype(np.float64) / sum_


def excess(out, q, k, v, scale, see):
    """How far out [n][D] fp32 is outside the bound, at most (below 0: nowhere)."""
    q, k, v = q.astype(np.float64), k.astype(np.float64), v.astype(np.float64)
    s = np.where(see, (q @ k.T) * scale, -np.inf)
    p = np.exp(s - s.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    want, weight = p @ v, p @ np.abs(v)
    A = np.where(see, np.abs(q) @ np.abs(k).T, 0).max(-1) * scale
    arg = (16 + 2 * A * 1.4427) * 2.0 ** -24 * 0.6932
    rel = 2 * A * (2.0 ** -22 + 8 * 2.0 ** -24) + 4 * arg + 6 * 2.0 ** -22 + 2 * (32 + 8 + 16) * 2.0 ** -23
    tol = rel[:, None] * weight + 2.0 ** -24 * np.abs(want)
    return (np.abs(out.astype(np.float64) - want) - tol).max()
