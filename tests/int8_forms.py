"""Plain forms of the int8 operators in numpy: every fp32 step of the definitions is one numpy fp32 operation, so the
products, the codes and the SwiGLU rows compare bit for bit; the norms are computed in 64 bits."""
import numpy as np

F = np.float32


def quantize(x):
    """fp32 rows -> (int8 codes, fp32 scales), one scale per row (q4_quant_act_i8's steps with the row as the group)."""
    x = np.asarray(x, F)
    bits = np.maximum((x.view(np.uint32) & 0x7FFFFFFF).max(-1), F(1e-8).view(np.uint32)).astype(np.uint32)
    top = bits.view(F)
    fine = bits < 0x7F800000
    with np.errstate(invalid="ignore", over="ignore"):
        scale = (top / F(127)).astype(F)
        inv = np.where(fine, F(1) / scale, F(0)).astype(F)
        p = np.where(fine[..., None], x, F(0)) * inv[..., None]
    q = np.trunc(p + np.where(p >= 0, F(0.5), F(-0.5)).astype(F))
    return np.clip(q, -128, 127).astype(np.int8), scale


def product(q, qs, codes, scales, bias=None):
    """fp32(exact sum) * (qs * scales) + bias, each step rounded."""
    acc = q.astype(np.float64) @ codes.astype(np.float64).T              # below 2^53: exact
    with np.errstate(invalid="ignore", over="ignore"):
        y = acc.astype(F) * (qs[:, None] * scales[None, :])
        return y if bias is None else y + bias


def swiglu(g, u):
    with np.errstate(over="ignore", invalid="ignore"):
        e = np.exp(-g.astype(np.float64)).astype(F)
        return g / (F(1) + e) * u


def mlp(x, gate, up, down):
    q, s = quantize(x)
    h = swiglu(product(q, s, *gate), product(q, s, *up))
    return h, product(*quantize(h), *down)


def normed(kind, v, w=None, b=None, eps=1e-6, w_add=0.0):
    """The norms in 64 bits: kind 0 none, 1 rms, 2 layer."""
    v = v.astype(np.float64)
    if kind == 0:
        return v
    if kind == 2:
        v = v - v.mean(-1, keepdims=True)
    with np.errstate(over="ignore", invalid="ignore"):
        n = v / np.sqrt((v * v).mean(-1, keepdims=True) + np.float64(F(eps)))
        if w is not None:
            n = n * (w.astype(np.float64) + np.float64(F(w_add)))
        return n if b is None else n + b.astype(np.float64)


def weights(rng, out, inn):
    """Codes over their whole range and scales of their own for each channel."""
    return rng.integers(-127, 128, (out, inn)).astype(np.int8), rng.uniform(2e-4, 9e-4, out).astype(F)


def routed(x, idx, w, gate, up, down, shared=None):
    """The routed FFN of int8 experts: gate / up / down are lists of (codes, scales), idx / w [T][K]; ids outside the stack
    are skipped.  Experts are added in ascending order, then k, each step one fp32 operation."""
    T, K = idx.shape
    q, s = quantize(x)
    out = np.zeros((T, x.shape[1]), F)
    pair = {}
    for e in range(len(gate)):
        ts, ks = np.nonzero(idx == e)
        if len(ts):
            h = swiglu(product(q[ts], s[ts], *gate[e]), product(q[ts], s[ts], *up[e]))
            y = product(*quantize(h), *down[e])
            pair.update({(t, k): y[i] for i, (t, k) in enumerate(zip(ts, ks))})
    for t in range(T):
        for e, k in sorted((int(idx[t, k]), k) for k in range(K) if (t, k) in pair):
            out[t] = out[t] + w[t, k] * pair[t, k]
    if shared:
        out = out + mlp(x, *shared)[1]
    return out
