"""The operators around the paged 4-bit cache in 64 bits, from their definitions (include/beglin_qgemv.h), and how far the
kernels may be off.

Roundings, relative to the value: half a step, 2^-24 (fp32), 2^-11 (fp16), 2^-8 (bf16); fp16 below its normal range 2^-25
absolute."""
import numpy as np

HALF = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
LEAST = {"float32": 2.0 ** -149, "float16": 2.0 ** -25, "bfloat16": 2.0 ** -133}


# ------------------------------------------------------------------ heads
def heads(x, norm, w, eps, w_add, rope, pos, rot, style):
    """[T][n][D] in 64 bits; style 0 none, 1 half, 2 pairs."""
    x = x.astype(np.float64)
    if norm == 2:
        x = x - x.mean(-1, keepdims=True)
    if norm:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + np.float64(np.float32(eps)))
        if w is not None:
            x = x * (w.astype(np.float64) + np.float64(np.float32(w_add)))
    if not style:
        return x
    h = rot // 2
    ok = (pos >= 0) & (pos < len(rope))
    row = rope[np.where(ok, pos, 0)].astype(np.float64)[:, None]
    c, s = row[..., :h], row[..., h:]
    i, j = (slice(0, h), slice(h, rot)) if style == 1 else (slice(0, rot, 2), slice(1, rot, 2))
    y = x.copy()
    y[..., i] = x[..., i] * c - x[..., j] * s
    y[..., j] = x[..., j] * c + x[..., i] * s
    return y


# ------------------------------------------------------------------ the cache's values
def kept(x):
    """What fp32 rows [..., D] become in the cache, as fp16 (numpy rounds 64 bits to fp16 at once)."""
    g = x.reshape(*x.shape[:-1], -1, 32)
    bad = ~np.isfinite(g).all(-1, keepdims=True)
    g = np.clip(np.where(bad, 0, g), np.float32(-32768), np.float32(32768)).astype(np.float32)
    m = g.min(-1, keepdims=True).astype(np.float16)
    fm = m.astype(np.float32)
    s = np.maximum(np.float32(0), (g.max(-1, keepdims=True) - fm) * (np.float32(1) / np.float32(15))).astype(np.float16)
    fs = s.astype(np.float32)
    r = np.float32(1) / np.where(fs > 0, fs, np.float32(1))
    c = np.where(fs > 0, np.clip(np.rint((g - fm) * r), 0, 15), 0)
    v = (c.astype(np.float64) * s.astype(np.float64) + m.astype(np.float64)).astype(np.float16)
    return np.where(bad, np.float16(np.nan), v).reshape(x.shape)


def record_values(rec, D):
    """(K, V) values [16][D] fp16 of one record of 20 D bytes, from the addresses of each code, step and floor."""
    G = D // 32
    out = []
    for half in (0, 1):
        part = rec[10 * D * half:10 * D * (half + 1)]
        steps = part[8 * D:].copy().view(np.float16).astype(np.float64)
        v = np.zeros((16, D), np.float16)
        for t in range(16):
            for e in range(D):
                if half == 0:
                    b, j, i = e // (8 * G), e // 8 % G, e % 8
                    byte, high = ((b * 16 + t) * G + j) * 4 + (i & 1) * 2 + i // 4, i // 2 % 2
                    at = (e // 32 * 16 + t) * 2
                    s, m = steps[at], steps[at + 1]
                else:
                    b, r = t // 4, t % 4
                    byte, high = (b * (D // 2) + e // 2) * 4 + r, e % 2
                    at = (e // 32 * 4 + b) * 8 + r % 2 * 2 + r // 2
                    s, m = steps[at], steps[at + 4]
                v[t, e] = np.float16((part[byte] >> (4 * high) & 15) * s + m)
        out.append(v)
    return out


def pack(k, v):
    """Records [n][20 D] of values' codes, from rows k and v [n][16][D] fp32."""
    n, _, D = k.shape
    G = D // 32
    rec = np.zeros((n, 20 * D), np.uint8)
    for half, x in enumerate((k, v)):
        g = x.reshape(n, 16, G, 32).astype(np.float32)
        m = g.min(-1).astype(np.float16)
        s = np.maximum(np.float32(0), (g.max(-1) - m.astype(np.float32)) * (np.float32(1) / np.float32(15))).astype(np.float16)
        fs = s.astype(np.float32)[..., None]
        r = np.float32(1) / np.where(fs > 0, fs, np.float32(1))
        c = np.where(fs > 0, np.clip(np.rint((g - m.astype(np.float32)[..., None]) * r), 0, 15), 0).astype(np.uint8)
        c = c.reshape(n, 16, D)
        part = rec[:, 10 * D * half:10 * D * (half + 1)]
        sm = part[:, 8 * D:]
        for t in range(16):
            for e in range(0, D, 2):
                if half == 0:
                    for i in (e, e + 1):
                        b, j, q = i // (8 * G), i // 8 % G, i % 8
                        part[:, ((b * 16 + t) * G + j) * 4 + (q & 1) * 2 + q // 4] |= c[:, t, i] << (4 * (q // 2 % 2))
                else:
                    part[:, (t // 4 * (D // 2) + e // 2) * 4 + t % 4] = c[:, t, e] | c[:, t, e + 1] << 4
            for gi in range(G):
                at = ((gi * 16 + t) * 2, (gi * 16 + t) * 2 + 1) if half == 0 else \
                     ((gi * 4 + t // 4) * 8 + t % 2 * 2 + t % 4 // 2, (gi * 4 + t // 4) * 8 + t % 2 * 2 + t % 4 // 2 + 4)
                for a, z in zip(at, (s, m)):
                    sm[:, 2 * a:2 * a + 2] = z[:, t, gi].copy().view(np.uint8).reshape(n, 2)
    return rec


# ------------------------------------------------------------------ attention
def attention(q, k, v, scale, seen, sink):
    """One head: rows q [n][D] over keys k, values v [L][D] in 64 bits; seen [n][L].  Returns out, and sum_j p_j |v_j| of the
    normalised weights (what a relative error of the weights is multiplied by), and the largest |score| a row sees."""
    s = (q.astype(np.float64) @ k.astype(np.float64).T) * np.float64(np.float32(scale))
    s = np.where(seen, s, -np.inf)
    top = s.max(-1, initial=-np.inf, keepdims=True)
    if sink is not None:
        top = np.maximum(top, np.float64(sink))
    ref = np.where(np.isfinite(top), top, 0)
    p = np.where(seen, np.exp(s - ref), 0.0)
    total = p.sum(-1, keepdims=True)
    if sink is not None:
        total = total + np.exp(np.float64(sink) - ref)
    p = np.where(total > 0, p / np.where(total > 0, total, 1), 0)
    v = v.astype(np.float64)
    return p @ v, p @ np.abs(v), np.where(seen, np.abs(s), 0).max(-1, initial=0)


def attention_near(out, q, k, v, scale, seen, sink, kind, name):
    """out [n][D] of one head, from rows q of type `kind` over the cache's values k, v [L][D], is attention within the kernel's
    roundings (all relative):
      scores   q is exact as an operand (two parts of it hold 2^-22 for fp32 rows), D products are summed in fp32, and the sum is scaled
               and shifted: A (2 D + 32) 2^-24 + A 2^-22 (fp32 rows), A the largest sum |q_i k_i| scale that the row sees; both the weight and the
               sum of weights follow it: twice that.  A merge of partial sums shifts by the maximum once more, which the 32 holds.
      weights  fp16: 2^-11, two parts: 2^-22; exp2 itself 2^-22.  A weight below 2^-22 of the largest is off by at
               most 2^-33 of it (weights are 2^8 exp2(s - m) with m at most 7 below the largest score, and fp16 errs by 2^-25 below 2^-14).
      sums     32 products in a matrix instruction and L / 32 instructions and joins, each at most 2^-23.
      output   half a step of its type.
    All but the last multiply sum p |v|.  NaN is where the formula has it: a row that sees a NaN among its keys or in itself, and the
    values that see one among V's."""
    D, n = q.shape[-1], len(k)
    out, q = out.astype(np.float64), q.astype(np.float64)
    k, v = k.astype(np.float64), v.astype(np.float64)
    parts = kind == "float32"
    lost = (seen & ~np.isfinite(k).all(-1)[None]).any(-1) | (~np.isfinite(q).all(-1) & seen.any(-1))
    nan = lost[:, None] | ((seen[:, :, None] & ~np.isfinite(v)[None]).any(1) if not np.isfinite(v).all() else False)
    assert np.array_equal(np.isnan(out), np.broadcast_to(nan, out.shape)), (name, "NaN")
    kk, vv, x = np.where(np.isfinite(k), k, 0), np.where(np.isfinite(v), v, 0), np.where(np.isfinite(q), q, 0)
    want, weight, _ = attention(x, kk, vv, scale, seen, sink)
    A = np.where(seen, np.abs(x) @ np.abs(kk).T, 0).max(-1, initial=0) * abs(scale)
    if sink is not None:
        A = np.maximum(A, abs(float(sink)))
    ds = A * ((2 * D + 32) * 2.0 ** -24 + (2.0 ** -22 if parts else 0))
    rel = (2.0 ** -22 if parts else 2.0 ** -11) + 2.0 ** -21 + 2 * ds + (32 + n / 32 + 800) * 2.0 ** -23
    tol = rel[:, None] * weight + n * 2.0 ** -33 * np.abs(vv).max(initial=0)
    tol = tol * (1 + HALF[kind]) + HALF[kind] * np.abs(want) + LEAST[kind] + 1e-30
    off = np.where(nan, 0, np.abs(out - want) - tol)[~lost]
    worst = off.max(initial=-1.0)
    assert worst <= 0, (name, worst, np.argwhere(off > 0)[:3])
