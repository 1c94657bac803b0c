"""The int8 operators around a transformer block's feed-forward half, as cases that can be timed and compared.

Weights hold one int8 code per value and one fp32 scale per output channel (kind Q8C); activations
are int8 with one fp32 scale per token:

  linear   fp32 columns, quantized by the call, times one tensor or a fused group
  linear8  columns that the caller quantized, outputs in fp32, fp16 or bf16
  mlp      gate+up, SwiGLU, down, both products in int8
  norm     the end of a block and the norm before the next one in a call: the block's output is
           normed (or not), scaled, gated and added to the residual stream, and the new residual row
           is normed, to floats or to int8 codes with a scale per token
  block    norm to int8 codes, then the fused products that read them
  moe      a routed layer of int8 experts for a few tokens: router, top-K, experts, shared experts

With `own` false, `run` is elementary torch arithmetic; with `own` true, the library's calls.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # one token through a small model's gate projection (Qwen2.5-1.5B: 8960 x 1536): latency counts
        dict(name="linear_token", call="linear", rows="8960", cols=1536, m=1, bias=False),
        # eight sequences decoding: the fused q/k/v products of an 8B model, with biases
        dict(name="linear_qkv_batch8", call="linear", rows="4096,1024,1024", cols=4096, m=8, bias=True),
        # a prompt chunk of 64 tokens, quantized by the norm before it
        dict(name="linear8_chunk64", call="linear8", rows="14336", cols=4096, m=64, bias=False, y="bf16"),
        # a long prompt: the largest product of an 8B model
        dict(name="linear8_prompt4096", call="linear8", rows="14336", cols=4096, m=4096, bias=True, y="bf16"),
        # odd everything: an odd number of tokens, of channels and of inputs
        dict(name="linear8_ragged", call="linear8", rows="1001", cols=1411, m=333, bias=True, y="f16"),
        # 32 sequences decoding: an 8B model's whole MLP block
        dict(name="mlp_batch32", call="mlp", hidden=4096, inner=14336, m=32),
        # one token: residual add, RMS norm and its int8 codes
        dict(name="norm_token", call="norm", t=1, h=4096, x="f32", f="f32", post="none", pre="rms", gate="none", out="i8"),
        # a long prompt's rows in bf16: residual add and RMS norm
        dict(name="norm_prompt4096", call="norm", t=4096, h=4096, x="bf16", f="bf16", post="none", pre="rms", gate="none", out="bf16"),
        # a norm after the block as well, a gate per token and channel, layer norms, rows of an odd width
        dict(name="norm_sandwich_ragged", call="norm", t=777, h=2883, x="f32", f="f16", post="layer", pre="layer", gate="full", out="f16"),
        # a prompt of 512 tokens: the norm to int8 codes and the fused gate+up products that read them
        dict(name="block_prompt512", call="block", t=512, h=1536, rows="8960,8960", x="bf16", f="bf16", post="rms", pre="rms",
             gate="channel", y="bf16"),
        # a routed layer (DeepSeek-V2-Lite: 64 experts, top 6, two shared): one token, and 32 sequences
        dict(name="moe_token", call="moe", experts=64, top=6, hidden=2048, inner=1408, shared=2816, m=1),
        dict(name="moe_batch32", call="moe", experts=64, top=6, hidden=2048, inner=1408, shared=2816, m=32),
    ]


def _log_int(rng, lo, hi):
    return int(round(2 ** rng.uniform(math.log2(lo), math.log2(hi))))


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        call = rng.choice(["linear", "linear8", "linear8", "mlp", "norm", "norm", "block", "moe", "moe"])
        bias = rng.random() < 0.5
        rows = lambda hi: ",".join(str(_log_int(rng, 64, hi)) for _ in range(rng.choice([1, 1, 2, 3])))  # noqa: E731
        norm = lambda: dict(x=rng.choice(["f32", "f16", "bf16"]), f=rng.choice(["f32", "f16", "bf16"]),  # noqa: E731
                            post=rng.choice(["none", "rms", "layer"]), pre=rng.choice(["rms", "layer"]),
                            gate=rng.choice(["none", "channel", "token", "full"]))
        if call == "linear":
            c = dict(call=call, rows=rows(14336), cols=_log_int(rng, 128, 14336), m=_log_int(rng, 1, 512), bias=bias)
        elif call == "linear8":
            c = dict(call=call, rows=rows(14336), cols=_log_int(rng, 128, 14336), m=_log_int(rng, 1, 4096), bias=bias,
                     y=rng.choice(["f32", "f16", "bf16"]))
        elif call == "mlp":
            c = dict(call=call, hidden=_log_int(rng, 512, 4096), inner=_log_int(rng, 1024, 14336), m=_log_int(rng, 1, 512))
        elif call == "norm":
            c = dict(call=call, t=_log_int(rng, 1, 8192), h=_log_int(rng, 64, 8192), out=rng.choice(["f32", "f16", "bf16", "i8"]), **norm())
        elif call == "block":
            c = dict(call=call, t=_log_int(rng, 1, 2048), h=_log_int(rng, 512, 4096), rows=rows(8960), y=rng.choice(["f32", "f16", "bf16"]),
                     **norm())
        else:
            e = rng.choice([8, 16, 32, 64])
            c = dict(call=call, experts=e, top=rng.randint(1, min(e, 8)), hidden=64 * _log_int(rng, 8, 45), inner=64 * _log_int(rng, 4, 45),
                     shared=rng.choice([0, 64 * _log_int(rng, 4, 44)]), m=_log_int(rng, 1, 64))
        if _cost(c) <= most:
            return c


# --------------------------------------------------------------------------------------- the inputs
class _State:
    ctx, tensors = None, ()

    def __del__(self):
        try:
            if self.ctx is not None:
                torch.cuda.synchronize()
                for t in self.tensors:
                    t.free()
                self.ctx.close()
        except Exception:
            pass


_STREAM = None


def _stream():
    """The stream that the program queues the library's work on."""
    global _STREAM
    if _STREAM is None:
        _STREAM = torch.cuda.Stream()
    return _STREAM


def _rows(case):
    return [int(r) for r in case["rows"].split(",")]


def _codes(gen, *shape):
    """int8 codes of normal weights, as rounding each row by its largest value leaves them."""
    out = torch.empty(shape, dtype=torch.int8, device="cuda")
    for part in out.reshape(-1, shape[-1]).split(1 << 14):
        part.copy_(torch.randn(part.shape, generator=gen, device="cuda").mul_(33.0).round_().clamp_(-127, 127))
    return out


def _scales(gen, *shape):
    return torch.rand(shape, generator=gen, device="cuda").mul_(4e-4).add_(4e-4)


def _build(case, seed):
    """The inputs of a case, from its seed alone."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = _State()
    s.case = case
    call, m = case["call"], case.get("m", case.get("t"))
    rand = lambda *shape: torch.randn(shape, generator=gen, device="cuda")  # noqa: E731
    if call in ("norm", "block"):
        t, h = case["t"], case["h"]
        x = TYPES[case["x"]]
        f = TYPES[case["f"]]
        hot = 1.0 + 30.0 * (torch.rand(h, generator=gen, device="cuda") < 0.004)     # a residual stream's few large channels
        s.x = (rand(t, h) * 3 * hot).to(x)
        s.f = (rand(t, h) * 0.5 + 0.1).to(f)
        shape = {"none": None, "channel": (1, h), "token": (t, 1), "full": (t, h)}[case["gate"]]
        s.gate = None if shape is None else (rand(*shape) * 0.3 + 0.5).to(f)
        s.alpha = 0.25 if case["gate"] == "full" else 1.0
        s.post_w, s.post_b, s.pre_w, s.pre_b = (1 + 0.1 * rand(h), 0.1 * rand(h), 1 + 0.1 * rand(h), 0.1 * rand(h))
        s.eps = 1e-6
    if call in ("linear", "mlp", "moe"):
        k = case["cols"] if call == "linear" else case["hidden"]
        s.x = rand(m, k) * (1.0 + 15.0 * (torch.rand(k, generator=gen, device="cuda") < 0.004))
    if call == "linear8":
        # what a norm writes: codes whose rows are a multiple of 16 bytes apart, and a scale per row
        k = case["cols"]
        s.xq = torch.zeros((m, (k + 15) // 16 * 16), dtype=torch.int8, device="cuda")
        s.xq[:, :k] = rand(m, k).mul_(30.0).round_().clamp_(-127, 127)
        s.xs = torch.rand(m, generator=gen, device="cuda") * 0.02 + 0.01
    if call in ("linear", "linear8", "block"):
        k = case["h"] if call == "block" else case["cols"]
        s.w = [(_codes(gen, r, k), _scales(gen, r)) for r in _rows(case)]
        s.b = [rand(r) if case.get("bias") else None for r in _rows(case)]
    if call == "mlp":
        h, i = case["hidden"], case["inner"]
        s.w = [(_codes(gen, o, k), _scales(gen, o)) for o, k in ((i, h), (i, h), (h, i))]
    if call == "moe":
        e, h, i, sh = (case[n] for n in ("experts", "hidden", "inner", "shared"))
        s.router = rand(e, h) / h ** 0.5
        s.w = [(_codes(gen, e, o, k), _scales(gen, e, o)) for o, k in ((i, h), (i, h), (h, i))]
        s.sh = [(_codes(gen, o, k), _scales(gen, o)) for o, k in ((sh, h), (sh, h), (h, sh))] if sh else None
    return s


def _bind(s):
    """The library's handles, and the buffers that its calls write."""
    import beglin_amd as B

    case, call = s.case, s.case["call"]
    stream = _stream()
    s.ctx = B.Context(0, stream.cuda_stream)
    bound = []

    def one(codes, scales):
        t = s.ctx.bind(B.K_Q8C, codes, scales, *codes.shape)         # from where they lie, on the device
        bound.append(t)
        return t

    def stack(codes, scales):
        each = [one(c, v) for c, v in zip(codes, scales)]
        del bound[-len(each):]                            # the stack owns its experts
        t = s.ctx.experts_from_tensors(each)
        bound.append(t)
        return t

    new = lambda *shape, dtype=torch.float32: torch.empty(shape, dtype=dtype, device="cuda")  # noqa: E731
    if call == "moe":
        s.t = [stack(*w) for w in s.w]
        s.ts = [one(*w) for w in s.sh] if s.sh else None
        s.y = new(*s.x.shape)
    elif call != "norm":
        s.t = [one(*w) for w in s.w]
    if call in ("linear", "linear8", "block"):
        m = case["t"] if call == "block" else case["m"]
        s.ys = [new(m, r, dtype=TYPES[case.get("y", "f32")]) for r in _rows(case)]
    if call == "mlp":
        s.hid, s.y = new(case["m"], case["inner"]), new(*s.x.shape)
    if call in ("norm", "block"):
        t, h = s.x.shape
        s.x_out = new(t, h, dtype=s.x.dtype)
        i8 = call == "block" or case["out"] == "i8"
        s.y = None if i8 else new(t, h, dtype=TYPES[case["out"]])
        s.yq, s.yscale = (new(t, (h + 15) // 16 * 16, dtype=torch.int8), new(t)) if i8 else (None, None)
        kinds = {"none": B.NORM_NONE, "rms": B.NORM_RMS, "layer": B.NORM_LAYER}
        s.post, s.pre = kinds[case["post"]], kinds[case["pre"]]
        s.act = None
    if call in ("linear", "mlp"):
        s.act = B.ACT_W4A8
    s.tensors = bound


def prepare(case, seed):
    s = _build(case, seed)
    if own:
        torch.cuda.synchronize()
        _bind(s)
    return s


# ------------------------------------------------------------------------------ the library's calls
def _own_norm(s):
    layer = s.case["pre"] == "layer"
    s.ctx.norm(s.x, y=s.y, yq=s.yq, yscale=s.yscale, kind=s.pre, w=s.pre_w, b=s.pre_b if layer else None, eps=s.eps,
               x_out=s.x_out, branch=s.f, branch_kind=s.post, branch_w=s.post_w if s.post else None,
               branch_b=s.post_b if s.case["post"] == "layer" else None, branch_eps=s.eps, gate=s.gate, alpha=s.alpha)


def _run_own(s):
    call, ctx = s.case["call"], s.ctx
    if call == "linear":
        if len(s.t) == 1:
            ctx.matmul(s.t[0], s.x, s.ys[0], act=s.act, bias_dev=s.b[0])
        else:
            ctx.matmul_group(s.t, s.x, s.ys, act=s.act, biases=s.b)
        return s.ys
    if call == "linear8":
        ctx.matmul_i8(s.t, s.xq, s.xs, s.ys, biases=s.b)
        return s.ys
    if call == "mlp":
        ctx.mlp(*s.t, s.x, s.y, act=s.act, h_dev=s.hid)
        return {"h": s.hid, "y": s.y}
    if call == "moe":
        ctx.moe_layer(s.router, *s.t, s.ts, s.x, s.case["top"], s.y)
        return s.y
    _own_norm(s)
    if call == "block":
        ctx.matmul_i8(s.t, s.yq, s.yscale, s.ys)
        return {"x": s.x_out, "y": s.ys}
    if s.yq is None:
        return {"x": s.x_out, "y": s.y}
    with torch.cuda.stream(_stream()):                     # the values that the codes stand for
        return {"x": s.x_out, "y": s.yq[:, :s.x.shape[1]].float() * s.yscale[:, None]}


# ----------------------------------------------------------------------------------- the plain forms
def _quant(x):
    """fp32 rows as int8 codes (held as floats) and a scale per row: the largest value becomes 127; halves go
    away from zero.  Every step is one fp32 operation, since a code next to a border follows the last bit."""
    s = x.abs().amax(-1, keepdim=True).clamp_min(1e-8)
    s = s / torch.full_like(s, 127.0)
    p = x * (1.0 / s)
    return torch.trunc(p + torch.where(p >= 0, 0.5, -0.5)).clamp_(-128, 127), s


def _product(q, qs, codes, scales, bias=None):
    """Codes times codes, exact in 64 bits, then the two scales; q [M][K] with scales qs [M][1]."""
    acc = (q.double() @ codes.double().t()).float()
    y = acc * (qs * scales)
    return y if bias is None else y + bias


def _swiglu(g, u):
    """fp32 operations, with the exponential rounded once from 64 bits."""
    return g / (1.0 + torch.exp(-g.double()).float()) * u


def _normed(kind, v, w, b, eps):
    if kind == "none":
        return v
    if kind == "layer":
        d = v - v.mean(-1, keepdim=True)
        return d / torch.sqrt((d * d).mean(-1, keepdim=True) + eps) * w + b
    return v / torch.sqrt((v * v).mean(-1, keepdim=True) + eps) * w


def _plain_norm(s, wide):
    """The new residual rows, and what the next norm makes of them; in 64 bits where codes follow the values."""
    case = s.case
    up = (lambda t: t.double()) if wide else (lambda t: t.float())
    n = _normed(case["post"], up(s.f), up(s.post_w), up(s.post_b), s.eps)
    if s.gate is not None:
        n = n * up(s.gate)
    x = (up(s.x) + s.alpha * n).to(s.x.dtype)
    return x, _normed(case["pre"], up(x), up(s.pre_w), up(s.pre_b), s.eps)


def _experts(w, xq, pick, k):
    """Products of a stack's experts with their tokens' codes: w [E][O][K] int8, xq [T][K]; one row for each of the T*k
    pairs, `pick` their experts.  Few pairs read their own experts, many read every expert once for all tokens."""
    if pick.numel() < w.shape[0]:
        return torch.bmm(w[pick].double(), xq.repeat_interleave(k, 0).double().unsqueeze(-1)).squeeze(-1)
    every = xq.double() @ w.reshape(-1, w.shape[-1]).double().t()
    every = every.reshape(xq.shape[0], w.shape[0], -1)
    return every[torch.arange(pick.numel(), device=pick.device) // k, pick]


def _expert_rows(w, hq, pick, k):
    """The same for the down products: row p of hq belongs to pair p alone."""
    if pick.numel() < w.shape[0]:
        return torch.bmm(w[pick].double(), hq.double().unsqueeze(-1)).squeeze(-1)
    token = torch.arange(pick.numel(), device=pick.device) // k
    spread = torch.zeros((w.shape[0], pick.numel() // k, hq.shape[1]), dtype=torch.float64, device=hq.device)
    spread[pick, token] = hq.double()
    return torch.bmm(spread, w.double().transpose(1, 2).contiguous())[pick, token]


def _plain_moe(s):
    k = s.case["top"]
    x, t = s.x, s.x.shape[0]
    p = torch.softmax((x.double() @ s.router.double().t()).float().double(), -1).float()
    order = torch.argsort(p, dim=-1, descending=True, stable=True)[:, :k]      # ties: the lowest expert first
    pick = order.sort(-1).values                                               # experts' rows are added in ascending order
    weight = p.gather(1, pick)
    pick = pick.reshape(-1)
    xq, xs = _quant(x)
    gate, up, down = s.w
    pair = xs.repeat_interleave(k, 0)
    g = _experts(gate[0], xq, pick, k).float() * (pair * gate[1][pick])
    u = _experts(up[0], xq, pick, k).float() * (pair * up[1][pick])
    hq, hs = _quant(_swiglu(g, u))
    y = _expert_rows(down[0], hq, pick, k).float() * (hs * down[1][pick])
    y = (y.reshape(t, k, -1) * weight.unsqueeze(-1)).sum(1)
    if s.sh is None:
        return y
    (gw, gs), (uw, us), (dw, ds) = s.sh
    hq, hs = _quant(_swiglu(_product(xq, xs, gw, gs), _product(xq, xs, uw, us)))
    return y + _product(hq, hs, dw, ds)


def _run_plain(s):
    case = s.case
    call = case["call"]
    if call in ("linear", "linear8"):
        q, qs = _quant(s.x) if call == "linear" else (s.xq[:, :case["cols"]], s.xs[:, None])
        return [_product(q, qs, *w, b).to(TYPES[case.get("y", "f32")]) for w, b in zip(s.w, s.b)]
    if call == "mlp":
        q, qs = _quant(s.x)
        h = _swiglu(_product(q, qs, *s.w[0]), _product(q, qs, *s.w[1]))
        return {"h": h, "y": _product(*_quant(h), *s.w[2])}
    if call == "moe":
        return _plain_moe(s)
    x, y = _plain_norm(s, call == "block" or case["out"] == "i8")
    if call == "block":
        q, qs = _quant(y.float())
        return {"x": x, "y": [_product(q, qs, *w).to(TYPES[case["y"]]) for w in s.w]}
    if case["out"] == "i8":
        q, qs = _quant(y.float())
        return {"x": x, "y": q * qs}
    return {"x": x, "y": y.to(TYPES[case["out"]])}


def run(s):
    return _run_own(s) if own else _run_plain(s)


# ------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    call, m = case["call"], case.get("m", case.get("t"))
    size = {"f32": 4, "f16": 2, "bf16": 2, "i8": 1}
    if call in ("linear", "linear8", "block"):
        k, n = case["h" if call == "block" else "cols"], sum(_rows(case))
        data = n * (k + 4.0) + (4.0 * n if case.get("bias") else 0.0) + m * n * size[case.get("y", "f32")]
        flops = 2.0 * m * n * k
        if call == "linear":
            return {"bytes": data + 4.0 * m * k, "flops": flops}
        if call == "linear8":
            return {"bytes": data + m * (k + 4.0), "flops": flops}
        norm = work(dict(case, call="norm", out="i8"))
        return {"bytes": data + norm["bytes"] - m * (k + 4.0), "flops": flops + norm["flops"]}     # the codes stay inside
    if call == "mlp":
        h, i = case["hidden"], case["inner"]
        return {"bytes": 3.0 * h * i + 4.0 * (2 * i + h) + 4.0 * m * (2 * h + i), "flops": 6.0 * m * h * i}
    if call == "norm":
        h = case["h"]
        gate = {"none": 0, "channel": h, "token": m, "full": m * h}[case["gate"]]
        weights = sum({"none": 0, "rms": 1, "layer": 2}[case[n]] for n in ("post", "pre")) * 4.0 * h
        data = m * h * (2.0 * size[case["x"]] + size[case["f"]] + size[case["out"]]) + gate * size[case["f"]] + weights
        return {"bytes": data + (4.0 * m if case["out"] == "i8" else 0.0), "flops": 12.0 * m * h}
    e, h, i, sh, k = (case[n] for n in ("experts", "hidden", "inner", "shared", "top"))
    touched = e * (1.0 - (1.0 - k / e) ** m)                                      # expected, for independent tokens
    return {"bytes": touched * (3.0 * h * i + 4.0 * (2 * i + h)) + 3.0 * h * sh + 4.0 * e * h + 8.0 * m * h,
            "flops": 6.0 * m * (k * h * i + h * sh) + 2.0 * m * e * h}


def _cost(case):
    """Bytes and operations of a case in one figure, for the limit on drawn cases."""
    w = work(case)
    return w["bytes"] / 2e12 + w["flops"] / 3e13


# --------------------------------------------------------------------------------------- in 64 bits
def _exact_quant(x):
    """int8 values of fp32 rows as the definition has them (the code of a value is that of the fp32 quotient's rounding)."""
    x = x.float()
    top = torch.clamp_min(torch.amax(torch.abs(x), dim=1), 1e-8)
    scale = torch.div(top, torch.full_like(top, 127.0))
    steps = torch.mul(x, torch.reciprocal(scale)[:, None])
    code = torch.sign(steps) * torch.floor(steps.abs() + 0.5)
    return code.clamp_(-128, 127).to(torch.int8), scale


def _exact_dot(q, scale, codes, scales, bias=None):
    y = torch.matmul(q.double() * scale.double()[:, None], (codes.double() * scales.double()[:, None]).t())
    return y if bias is None else y + bias.double()


def _exact_hidden(q, scale, gate, up):
    """h = silu(g) u, where g and u are fp32 values (an exact sum, times the rounded product of its scales) and so is each step."""
    each = []
    for codes, scales in (gate, up):
        total = torch.matmul(q.double(), codes.double().t())
        each.append(total.float() * torch.mul(scale[:, None], scales[None, :]))
    g, u = each
    return torch.mul(torch.div(g, torch.add(torch.exp(g.double().neg()).float(), 1.0)), u)


def _exact_norm(kind, v, w, b, eps):
    if kind == "none":
        return v
    if kind == "layer":
        var, mean = torch.var_mean(v, dim=1, unbiased=False, keepdim=True)
        return (v - mean) * torch.rsqrt(var + eps) * w.double() + b.double()
    return v * torch.rsqrt(v.pow(2).mean(dim=1, keepdim=True) + eps) * w.double()


def exact(case, seed):
    s = _build(case, seed)
    call = case["call"]
    if call in ("linear", "linear8"):
        q, scale = _exact_quant(s.x) if call == "linear" else (s.xq[:, :case["cols"]], s.xs)
        return [_exact_dot(q, scale, *w, b) for w, b in zip(s.w, s.b)]
    if call == "mlp":
        h = _exact_hidden(*_exact_quant(s.x), s.w[0], s.w[1])
        return {"h": h.double(), "y": _exact_dot(*_exact_quant(h), *s.w[2])}
    if call == "moe":
        score = torch.matmul(s.x.double(), s.router.double().t())
        prob = torch.exp(score - torch.logsumexp(score, 1, keepdim=True))
        chosen = torch.topk(prob, case["top"], dim=1).indices
        q, scale = _exact_quant(s.x)
        y = torch.zeros_like(score[:, :1]).expand(-1, s.x.shape[1]).clone()
        for e in range(case["experts"]):
            t = (chosen == e).any(1).nonzero()[:, 0]
            if len(t):
                gate, up, down = ((c[e], v[e]) for c, v in s.w)
                y[t] += prob[t, e][:, None] * _exact_dot(*_exact_quant(_exact_hidden(q[t], scale[t], gate, up)), *down)
        if s.sh:
            y += _exact_dot(*_exact_quant(_exact_hidden(q, scale, s.sh[0], s.sh[1])), *s.sh[2])
        return y
    n = _exact_norm(case["post"], s.f.double(), s.post_w, s.post_b, s.eps)
    if s.gate is not None:
        n = s.gate.double() * n
    x = torch.add(s.x.double(), n, alpha=s.alpha)
    y = _exact_norm(case["pre"], x.to(s.x.dtype).double(), s.pre_w, s.pre_b, s.eps)
    if call == "block" or case["out"] == "i8":
        q, scale = _exact_quant(y)
        y = [_exact_dot(q, scale, *w) for w in s.w] if call == "block" else q.double() * scale.double()[:, None]
    return {"x": x, "y": y}
