"""The operators between a layer's q/k/v products and its output product, as cases that can be timed and compared.

  heads    queries and keys normed head by head (or not) and rotated by their positions, in one pass
  append   the same, with the keys and the values written to a paged cache that holds them in 4 bits;
           the values that the cache then stands for are read back
  attn     attention of a ragged batch over such a cache: single tokens, a few tokens a sequence, prompts

The cache holds groups of 32 values of a head as codes c of 4 bits, a step s and a floor m in fp16: the value is
fp16(c * s + m).  16 tokens of a head are one record of 20 * D bytes (D values a head, G = D / 32), K before V:

  K codes  [4 b][16 tokens][G j][4 bytes]   dword j of (b, token): the token's values 8 * (G * b + j) + 0 .. 7
  K steps  [G][16 tokens]                   s and m, two fp16
  V codes  [4 b][16 n][G j][4 bytes]        byte r: token 4 * b + r, values 2 * G * n + 2 * j (low) and + 1 (high)
  V steps  [G][4 b][8 fp16]                 s of tokens 4 * b + 0, 2, 1, 3, then m of the same

With `own` false, `run` is elementary torch arithmetic; with `own` true, the library's calls.
"""
import math
import random

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


# ---------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # one token of a small model (12 query heads, 2 of keys): rotation alone, latency counts
        dict(name="heads_token", call="heads", t=1, nq=12, nk=2, d=128, rot=128, style="half", norm="none", x="f32", y="f32", span=4096),
        # a long prompt of an 8B model's heads: RMS norms and rotation, bf16
        dict(name="heads_prompt4096", call="heads", t=4096, nq=32, nk=8, d=128, rot=128, style="half", norm="rms", x="bf16", y="bf16", span=8192),
        # odd numbers of tokens and heads, part of each head rotated in neighbouring pairs, layer norms, far positions
        dict(name="heads_ragged", call="heads", t=777, nq=15, nk=5, d=96, rot=64, style="pairs", norm="layer", x="f16", y="f16", span=131072),
        # eight sequences decoding: the step's keys and values into the cache
        dict(name="append_batch8", call="append", t=8, nq=32, nk=8, d=128, rot=128, style="half", norm="rms", x="bf16", y="bf16", span=8192,
             page=64, skip=0.0),
        # a long prompt's keys and values into the cache
        dict(name="append_prompt4096", call="append", t=4096, nq=32, nk=8, d=128, rot=128, style="half", norm="none", x="bf16", y="bf16", span=8192,
             page=64, skip=0.0),
        # an odd number of tokens, small pages, padding tokens without a place, fp32 rows whose queries leave as fp16
        dict(name="append_ragged", call="append", t=1001, nq=10, nk=5, d=64, rot=32, style="pairs", norm="rms", x="f32", y="f16", span=20000,
             page=16, skip=0.1),
        # one token of a small model after a short prompt, fp32: latency counts
        dict(name="attn_token", call="attn", seqs=1, rows=1, lo=300, hi=300, nq=12, nk=2, d=128, x="f32", page=16, window=0, sink=False, mix=1),
        # 32 sequences of an 8B model decoding, of very different lengths
        dict(name="attn_batch32", call="attn", seqs=32, rows=1, lo=100, hi=8192, nq=32, nk=8, d=128, x="bf16", page=64, window=0, sink=False, mix=2),
        # one sequence with a very long context
        dict(name="attn_long131072", call="attn", seqs=1, rows=1, lo=131072, hi=131072, nq=32, nk=8, d=128, x="bf16", page=128, window=0,
             sink=False, mix=3),
        # three tokens a sequence at once (drafted ones that are checked together), wide heads, one of keys for all, fp32
        dict(name="attn_drafts_wide", call="attn", seqs=5, rows=3, lo=1000, hi=20000, nq=8, nk=1, d=256, x="f32", page=32, window=0, sink=False, mix=4),
        # a batch in which prompts run in chunks beside single tokens: small heads, a window, and a sink in each row's sum
        dict(name="attn_chunks", call="attn", seqs=9, rows=600, lo=1, hi=5000, nq=64, nk=8, d=64, x="f16", page=16, window=512, sink=True, mix=5),
        # a whole long prompt
        dict(name="attn_prompt4096", call="attn", seqs=1, rows=4096, lo=4096, hi=4096, nq=32, nk=8, d=128, x="bf16", page=64, window=0, sink=False,
             mix=6),
    ]


def _log_int(rng, lo, hi):
    return int(round(2 ** rng.uniform(math.log2(lo), math.log2(hi))))


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        call = rng.choice(["heads", "append", "append", "attn", "attn", "attn", "attn"])
        d = rng.choice([64, 64, 96, 128, 128, 128, 192, 256])
        nk = rng.choice([1, 2, 3, 4, 5, 8, 8, 16])
        c = dict(call=call, nq=nk * rng.choice([1, 2, 3, 4, 4, 5, 7, 8, 16]), nk=nk, d=d, x=rng.choice(["f32", "f16", "bf16", "bf16"]))
        if call != "attn":
            c.update(t=_log_int(rng, 1, 8192), rot=rng.choice([d, d, 32 * rng.randint(1, d // 32)]), style=rng.choice(["half", "pairs"]),
                     norm=rng.choice(["none", "rms", "rms", "layer"]), y=rng.choice([c["x"], "f32", "f16", "bf16"]),
                     span=_log_int(rng, 8192, 131072))
            if call == "append":
                c.update(page=rng.choice([16, 32, 48, 64, 128, 256]), skip=rng.choice([0.0, 0.0, 0.05, 0.5]))
        else:
            rows = rng.choice([1, 1, rng.randint(2, 8), _log_int(rng, 9, 4096)])
            seqs = _log_int(rng, 1, 64 if rows < 9 else 8)
            hi = max(rows, _log_int(rng, 1, 131072 if rows < 9 else 16384))
            c.update(seqs=seqs, rows=rows, lo=max(1, _log_int(rng, 1, hi)), hi=hi, page=rng.choice([16, 32, 48, 64, 128, 256]),
                     window=rng.choice([0, 0, _log_int(rng, 16, 8192)]), sink=rng.random() < 0.3, mix=rng.randint(0, 10 ** 6))
            padded = seqs * hi * nk * d, seqs * rows * c["nq"] * hi          # the plain form's rectangles
            if max(padded) > 1 << 30:
                continue
        if _cost(c) <= most:
            return c


def _lengths(case):
    """Rows of q and keys of each sequence: the last has the most of both, the others spread over the logarithm."""
    rng = random.Random(case["mix"])
    rows, lens = [], []
    for i in range(case["seqs"]):
        last = i == case["seqs"] - 1
        n = case["hi"] if last else _log_int(rng, case["lo"], case["hi"])
        r = case["rows"] if last or case["rows"] < 9 else _log_int(rng, 1, case["rows"])
        lens.append(n)
        rows.append(min(n, r))
    return rows, lens


# --------------------------------------------------------------------------------------- the inputs
class _State:
    ctx = None

    def __del__(self):
        try:
            if self.ctx is not None:
                torch.cuda.synchronize()
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


def _codes(x):
    """Codes, steps and floors of groups of 32: x [..., 32] fp32; every step is one operation in fp32 or fp16."""
    x = x.clamp(-32768.0, 32768.0)
    m = x.amin(-1, keepdim=True).half()
    s = ((x.amax(-1, keepdim=True) - m.float()) / 15.0).half().clamp_min(0.0)
    c = torch.round((x - m.float()) * (1.0 / s.float()))
    return torch.where(s > 0, c, 0.0).clamp(0, 15), s, m


def _fill(record, x, half, d):
    """Packs rows x [n][16][d] as the K (half 0) or V (half 1) part of records [n][20 * d]."""
    n, g = x.shape[0], d // 32
    c, s, m = _codes(x.reshape(n, 16, g, 32))
    c = c.to(torch.uint8).reshape(n, 16, d)
    part = record[:, 10 * d * half:10 * d * (half + 1)]
    if half == 0:
        v = c.reshape(n, 16, 4, g, 8).permute(0, 2, 1, 3, 4)                     # n, b, token, j, value
        pairs = torch.stack([v[..., i] | v[..., i + 2] << 4 for i in (0, 4, 1, 5)], -1)
        steps = torch.cat([s, m], -1).permute(0, 2, 1, 3)                        # n, group, token, (s, m)
    else:
        v = c.reshape(n, 4, 4, 16, g, 2).permute(0, 1, 3, 4, 2, 5)               # n, b, unit, j, r, (low, high)
        pairs = v[..., 0] | v[..., 1] << 4
        steps = torch.stack([s, m], 0).reshape(2, n, 4, 2, 2, g)                 # (s, m), n, b, r / 2, r % 2, group
        steps = steps.permute(1, 5, 2, 0, 4, 3)
    part[:, :8 * d] = pairs.reshape(n, 8 * d)
    part[:, 8 * d:] = steps.contiguous().reshape(n, -1).view(torch.uint8)


def _rope(span, rot):
    """Cosines and sines of each position: [span][rot / 2] and [span][rot / 2], from angles in 64 bits."""
    at = torch.arange(span, device="cuda", dtype=torch.float64)
    f = 10000.0 ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
    a = at[:, None] * f
    return torch.cat([a.cos(), a.sin()], 1).float()


def _build(case, seed):
    """The inputs of a case, from its seed alone."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = _State()
    s.case = case
    nq, nk, d = case["nq"], case["nk"], case["d"]
    rand = lambda *shape: torch.randn(shape, generator=gen, device="cuda")  # noqa: E731
    hot = lambda *shape: 1.0 + 7.0 * (torch.rand(shape, generator=gen, device="cuda") < 0.02)  # noqa: E731  keys have a few large channels
    x = TYPES[case["x"]]
    if case["call"] != "attn":
        t = case["t"]
        both = rand(t, nq + 2 * nk, d)                                            # the q/k/v products' rows
        both[:, nq:nq + nk] *= hot(nk, d)
        both = both.to(x)
        s.q, s.k, s.v = both[:, :nq], both[:, nq:nq + nk], both[:, nq + nk:]
        s.q_w, s.k_w = 1 + 0.1 * rand(d), 1 + 0.1 * rand(d)
        s.eps = 1e-6
        first = torch.randint(0, case["span"] - t + 1, (1,), generator=gen, device="cuda") if case["span"] > t else 0
        s.pos = (torch.arange(t, device="cuda") + first).clamp_max(case["span"] - 1).int()
        s.rope = _rope(case["span"], case["rot"])
        if case["call"] == "append":
            page = case["page"]
            s.pages = (t + page - 1) // page + 3
            order = torch.randperm(s.pages, generator=gen, device="cuda")
            at = torch.arange(t, device="cuda") + 5                               # the sequence's pages, from inside the first one
            s.slots = (order[at // page] * page + at % page).int()
            s.slots[torch.rand(t, generator=gen, device="cuda") < case["skip"]] = -1
        return s
    rows, lens = _lengths(case)
    page = case["page"]
    each = [(n + page - 1) // page for n in lens]
    s.pages = sum(each) + 2
    order = torch.randperm(s.pages, generator=gen, device="cuda").int()
    s.table = torch.zeros((len(lens), max(each)), dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(each):
        s.table[i, :n] = order[at:at + n]
        at += n
    s.lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    s.start = torch.tensor([sum(rows[:i]) for i in range(len(rows) + 1)], dtype=torch.int32, device="cuda")
    s.total, s.most, s.longest = sum(rows), max(rows), max(lens)
    s.cache = torch.zeros((s.pages, nk, page // 16, 20 * d), dtype=torch.uint8, device="cuda")
    channels = hot(d)
    records = s.cache.reshape(-1, 20 * d)
    for part in records.split(1 << 14):
        _fill(part, rand(len(part), 16, d) * channels, 0, d)
        _fill(part, rand(len(part), 16, d), 1, d)
    s.q = rand(s.total, nq, d).to(x)
    s.sink = rand(nq) if case["sink"] else None
    s.scale = d ** -0.5
    # which sequence each row belongs to, and its place there
    s.of = torch.tensor([i for i, r in enumerate(rows) for _ in range(r)], device="cuda")
    s.nth = torch.tensor([j for r in rows for j in range(r)], device="cuda")
    return s


def _bind(s):
    """The library's handles, and the buffers that its calls write."""
    import beglin_amd as B

    case = s.case
    s.ctx = B.Context(0, _stream().cuda_stream)
    zeros = lambda like, kind: torch.zeros(like.shape, dtype=kind, device="cuda")  # noqa: E731
    if case["call"] == "attn":
        s.kv = B.KVCache(s.pages, case["page"], case["nk"], case["d"], data=s.cache)
        s.out = zeros(s.q, s.q.dtype)
        return
    s.norm = {"none": B.NORM_NONE, "rms": B.NORM_RMS, "layer": B.NORM_LAYER}[case["norm"]]
    s.style = {"half": B.ROT_HALF, "pairs": B.ROT_PAIRS}[case["style"]]
    s.q_out = zeros(s.q, TYPES[case["y"]])
    if case["call"] == "heads":
        s.k_out = zeros(s.k, TYPES[case["y"]])
    else:
        s.kv = B.KVCache(s.pages, case["page"], case["nk"], case["d"])
        s.k_read, s.v_read = zeros(s.k, torch.float16), zeros(s.v, torch.float16)


def prepare(case, seed):
    s = _build(case, seed)
    if own:
        torch.cuda.synchronize()
        _bind(s)
        torch.cuda.synchronize()
    return s


# ------------------------------------------------------------------------------ the library's calls
def _run_own(s):
    call, ctx = s.case["call"], s.ctx
    if call == "attn":
        ctx.attention(s.kv, s.q, s.out, s.start, s.lens, s.table, scale=s.scale, window=s.case["window"], sink=s.sink, max_rows=s.most,
                      max_len=s.longest)
        return s.out
    how = dict(norm=s.norm, q_w=s.q_w, k_w=s.k_w, eps=s.eps, rope=s.rope, pos=s.pos, rot=s.style)
    if call == "heads":
        ctx.heads(s.q, s.k, s.q_out, s.k_out, **how)
        return {"q": s.q_out, "k": s.k_out}
    ctx.kv_append(s.kv, s.slots, s.k, s.v, q=s.q, q_out=s.q_out, **how)
    ctx.kv_read(s.kv, s.slots, s.k_read, s.v_read)
    return {"q": s.q_out, "k": s.k_read, "v": s.v_read}


# ----------------------------------------------------------------------------------- the plain forms
def _turned(s, x, w, wide):
    """Heads x [T][n][D] normed and rotated; in 64 bits where codes follow the values."""
    case = s.case
    up = (lambda t: t.double()) if wide else (lambda t: t.float())
    x = up(x)
    if case["norm"] == "layer":
        x = x - x.mean(-1, keepdim=True)
    if case["norm"] != "none":
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + s.eps) * up(w)
    rot = case["rot"]
    c, n = up(s.rope[s.pos.long()]).unsqueeze(1).chunk(2, -1)
    a, b = (x[..., :rot // 2], x[..., rot // 2:rot]) if case["style"] == "half" else (x[..., 0:rot:2], x[..., 1:rot:2])
    a, b = a * c - b * n, b * c + a * n
    turned = torch.cat([a, b], -1) if case["style"] == "half" else torch.stack([a, b], -1).flatten(-2)
    return torch.cat([turned, x[..., rot:]], -1)


def _kept(s, x):
    """The values that the cache stands for after rows x [T][n][D], 0 where a token has no place."""
    c, step, floor = _codes(x.float().unflatten(-1, (-1, 32)))
    v = (c * step.float() + floor.float()).half().flatten(-2)
    return torch.where(s.slots[:, None, None] >= 0, v, 0)


def _values(record, half, d):
    """fp32 values [n][16][d] of the K (half 0) or V (half 1) part of records [n][20 * d]."""
    n, g = record.shape[0], d // 32
    part = record[:, 10 * d * half:10 * d * (half + 1)]
    code, steps = part[:, :8 * d], part[:, 8 * d:].contiguous().view(torch.float16).float()
    code = torch.stack([code & 15, code >> 4], -1)
    if half == 0:
        code = code.reshape(n, 4, 16, g, 8)[..., [0, 4, 1, 5, 2, 6, 3, 7]].permute(0, 2, 1, 3, 4)
        step, floor = steps.reshape(n, g, 16, 2).permute(3, 0, 2, 1)
    else:
        code = code.reshape(n, 4, 16, g, 4, 2).permute(0, 1, 4, 2, 3, 5)
        step, floor = steps.reshape(n, g, 4, 2, 2, 2).permute(3, 0, 2, 5, 4, 1).reshape(2, n, 16, g)
    code = code.reshape(n, 16, g, 32).float()
    return (code * step.unsqueeze(-1) + floor.unsqueeze(-1)).half().float().reshape(n, 16, d)


def _plain_attn(s):
    case = s.case
    nq, nk, d = case["nq"], case["nk"], case["d"]
    seqs, most = case["seqs"], s.most
    record = s.cache[s.table.long()].transpose(1, 2).reshape(-1, 20 * d)          # seqs, heads, pages, tiles
    k, v = (_values(record, half, d).reshape(seqs, nk, -1, d) for half in (0, 1))
    n = k.shape[2]
    at = torch.arange(most, device="cuda")
    row = (s.start[:-1, None] + at).clamp_max(s.total - 1).long()                 # rows of a rectangle, some of the next sequence
    q = s.q[row].float().reshape(seqs, most, nk, nq // nk, d).permute(0, 2, 3, 1, 4)
    score = torch.matmul(q.reshape(seqs, nk, -1, d), k.transpose(2, 3).contiguous()).reshape(seqs, nq, most, n) * s.scale
    pos = (s.lens - (s.start[1:] - s.start[:-1]))[:, None] + at
    key = torch.arange(n, device="cuda")
    seen = (key <= pos[..., None]) & (key < s.lens[:, None, None])
    if case["window"]:
        seen &= key > pos[..., None] - case["window"]
    score = score.masked_fill(~seen[:, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    if s.sink is not None:
        top = torch.maximum(top, s.sink[:, None, None])
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    if s.sink is not None:
        total = total + torch.exp(s.sink[:, None, None] - top)
    out = torch.matmul((p / total).reshape(seqs, nk, -1, n), v).reshape(seqs, nq, most, d)
    return out[s.of, :, s.nth].to(s.q.dtype)


def _run_plain(s):
    if s.case["call"] == "attn":
        return _plain_attn(s)
    y = TYPES[s.case["y"]]
    if s.case["call"] == "heads":
        return {"q": _turned(s, s.q, s.q_w, False).to(y), "k": _turned(s, s.k, s.k_w, False).to(y)}
    return {"q": _turned(s, s.q, s.q_w, False).to(y), "k": _kept(s, _turned(s, s.k, s.k_w, True)), "v": _kept(s, s.v)}


def run(s):
    return _run_own(s) if own else _run_plain(s)


# ------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    nq, nk, d, size = case["nq"], case["nk"], case["d"], SIZE[case["x"]]
    if case["call"] != "attn":
        t, out = case["t"], SIZE[case["y"]]
        data = t * (4.0 * case["rot"] + 4.0) + (8.0 * d if case["norm"] != "none" else 0.0)
        if case["call"] == "heads":
            return {"bytes": data + t * (nq + nk) * d * (size + out), "flops": 12.0 * t * (nq + nk) * d}
        # the cache is written and read once, the values read are written
        data += t * (nq * d * (size + out) + 2.0 * nk * d * size) + (1 - case["skip"]) * t * 2.0 * nk * d * (2 * 0.625 + 2)
        return {"bytes": data, "flops": 12.0 * t * (nq + 2 * nk) * d}
    keys, pairs = 0, 0
    for r, n in zip(*_lengths(case)):
        window = case["window"] or n
        keys += n - max(0, n - r + 1 - window)
        full = max(0, min(r, n - window))                                         # rows that see a whole window
        pairs += full * min(window, n) + sum(min(window, n - r + i + 1) for i in range(r - full))
    rows = sum(_lengths(case)[0])
    return {"bytes": keys * nk * d * 1.25 + 2.0 * rows * nq * d * size, "flops": 4.0 * pairs * nq * d}


def _cost(case):
    """Bytes and operations of a case in one figure, for the limit on drawn cases."""
    w = work(case)
    return w["bytes"] / 2e12 + w["flops"] / 3e13


# --------------------------------------------------------------------------------------- in 64 bits
def _exact_kept(x, slots):
    """What the cache stands for, group by group, from fp32 rows [T][n][D]."""
    x = torch.clamp(x.reshape(-1, 32), min=-32768.0, max=32768.0)
    floor = torch.min(x, dim=1).values.to(torch.float16).to(torch.float32)
    step = torch.relu(torch.div(torch.max(x, dim=1).values - floor, 15.0).to(torch.float16).to(torch.float32))
    inverse = torch.reciprocal(step)
    code = torch.mul(torch.sub(x, floor[:, None]), inverse[:, None]).round().clamp_(min=0.0, max=15.0)
    code[step == 0] = 0.0
    value = torch.addcmul(floor.double()[:, None], code.double(), step.double()[:, None]).to(torch.float16).double()
    value = value.reshape(len(slots), -1)
    value[slots < 0] = 0.0
    return value


def _exact_values(record, half, d):
    """The values of records' K or V part, each from the addresses of its code, step and floor."""
    g = d // 32
    t = torch.arange(16, device="cuda")[:, None]
    e = torch.arange(d, device="cuda")
    if half == 0:
        i = e % 8
        byte = ((e // (8 * g) * 16 + t) * g + e // 8 % g) * 4 + (i & 1) * 2 + i // 4
        high = (i // 2 % 2).expand(16, d)
        step = (e // 32 * 16 + t) * 2
        floor = step + 1
    else:
        byte = ((t // 4 * 16 + e // (2 * g)) * g + e % (2 * g) // 2) * 4 + t % 4
        high = (e % 2).expand(16, d)
        step = (e // 32 * 4 + t // 4) * 8 + t % 2 * 2 + t % 4 // 2
        floor = step + 4
    at = 10 * d * half
    steps = record[:, at + 8 * d:at + 10 * d].contiguous().view(torch.float16).double()
    code = torch.bitwise_and(torch.bitwise_right_shift(record[:, at + byte].int(), 4 * high.int()), 15)
    return torch.addcmul(steps[:, floor], code.double(), steps[:, step]).to(torch.float16).double()


def exact(case, seed):
    s = _build(case, seed)
    nq, nk, d = case["nq"], case["nk"], case["d"]
    if case["call"] != "attn":
        def heads(x, w):
            x = x.to(torch.float64)
            if case["norm"] == "layer":
                var, mean = torch.var_mean(x, dim=2, unbiased=False, keepdim=True)
                x = torch.mul((x - mean) * torch.rsqrt(var + s.eps), w)
            elif case["norm"] == "rms":
                x = torch.mul(x * torch.rsqrt(x.pow(2).sum(2, keepdim=True) / d + s.eps), w)
            half = case["rot"] // 2
            table = s.rope.double().index_select(0, s.pos.long())
            turn = torch.complex(table[:, :half], table[:, half:])[:, None]
            if case["style"] == "half":
                z = torch.complex(x[..., :half].contiguous(), x[..., half:2 * half].contiguous()) * turn
                parts = [z.real, z.imag, x[..., 2 * half:]]
            else:
                z = torch.view_as_complex(x[..., :2 * half].reshape(*x.shape[:2], half, 2)) * turn
                parts = [torch.view_as_real(z).reshape(*x.shape[:2], 2 * half), x[..., 2 * half:]]
            return torch.cat(parts, dim=2)

        q, k = heads(s.q, s.q_w), heads(s.k, s.k_w)
        if case["call"] == "heads":
            return {"q": q, "k": k}
        return {"q": q, "k": _exact_kept(k.float().contiguous(), s.slots).reshape(k.shape),
                "v": _exact_kept(s.v.float().contiguous(), s.slots).reshape(k.shape)}
    rows, lens = _lengths(case)
    page, g = case["page"], nq // nk
    out = torch.zeros((s.total, nq, d), dtype=torch.float64, device="cuda")
    begin = 0
    for i, (r, n) in enumerate(zip(rows, lens)):
        pages = s.table[i, :(n + page - 1) // page].long()
        pos = torch.arange(n - r, n, device="cuda")[:, None]
        key = torch.arange(n, device="cuda")[None]
        hidden = key > pos
        if case["window"]:
            hidden = hidden | (key + case["window"] <= pos)
        for h in range(nk):
            record = s.cache[pages, h].reshape(-1, 20 * d)
            k, v = (_exact_values(record, half, d).reshape(-1, d)[:n] for half in (0, 1))
            for j in range(h * g, (h + 1) * g):
                score = torch.mm(s.q[begin:begin + r, j].double(), k.t()).mul_(s.scale).masked_fill_(hidden, -math.inf)
                if s.sink is not None:
                    score = torch.cat([score, s.sink[j].double().expand(r, 1)], 1)
                p = torch.softmax(score, 1)[:, :n]
                out[begin:begin + r, j] = torch.mm(p, v)
        begin += r
    return out
