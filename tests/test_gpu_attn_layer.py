"""A layer's attention as a decoder runs it, step after step: q/k/v products, heads and append, attention, output product.  A prompt
batch first, then single tokens as a captured graph beside eager calls.  Every step is checked from the inputs that it found on
the device: rows that are normed and rotated within their roundings, the cache's values exactly (but for one code in 10^4, where a value lies on
a border), attention within kv_forms.attention_near's bounds, and the output product of the codes exactly."""
import numpy as np
import pytest

import int8_forms as I
import kv_forms as F

pytestmark = pytest.mark.gpu
H, NQ, NK, D, PAGE, WIDE = 320, 8, 2, 64, 16, 12


@pytest.fixture(scope="module")
def torch_dev():
    import torch
    assert torch.cuda.is_available(), "gpu tests need a GPU"
    return torch


@pytest.mark.parametrize("kind", ["bfloat16", "float16", "float32"])
def test_prompt_and_decode(torch_dev, kind):
    import beglin_amd as B
    torch = torch_dev
    rng = np.random.default_rng(3)
    stream = torch.cuda.Stream()
    c = B.Context(0, stream.cuda_stream)
    dt = getattr(torch, kind)
    dev = lambda v: torch.from_numpy(v).cuda()  # noqa: E731
    S, prompt = 3, [40, 1, 9]
    rope = np.concatenate([np.cos(a := np.arange(256)[:, None] * 10000.0 ** (-np.arange(0, D, 2) / D)), np.sin(a)], 1).astype(np.float32)
    norms = [(1 + 0.1 * rng.standard_normal(n)).astype(np.float32) for n in (H, D, D)]
    weights = [I.weights(rng, n * D, H) for n in (NQ, NK, NK)] + [I.weights(rng, H, NQ * D)]
    with torch.cuda.stream(stream):
        if kind == "float32":                                # fp32 rows: the products of other formats give no other type
            w = [c.quantize(B.K_Q8G64, dev((rng.standard_normal((n, k)) / k ** 0.5).astype(np.float32)))
                 for n, k in ((NQ * D, H), (NK * D, H), (NK * D, H), (H, NQ * D))]
        else:
            w = [c.bind(B.K_Q8C, x[0], x[1], *x[0].shape) for x in weights]
        rd, nd = dev(rope), [dev(x) for x in norms]
        table = dev(rng.permutation(S * WIDE).astype(np.int32).reshape(S, WIDE))
        tab = table.cpu().numpy()
        caches = [B.KVCache(S * WIDE, PAGE, NK, D) for _ in range(2)]
        for x in caches:
            x.data.fill_(0xFF)

        class Rows:
            """The buffers of a step of T rows."""

            def __init__(self, T):
                new = lambda *s, t=torch.float32: torch.zeros(s, dtype=t, device="cuda")  # noqa: E731
                self.T = T
                self.x, self.n, self.xq, self.xs = new(T, H), new(T, H), new(T, H, t=torch.int8), new(T)
                qkv = new(T, (NQ + 2 * NK) * D, t=dt)
                cut = (0, NQ * D, (NQ + NK) * D, (NQ + 2 * NK) * D)
                self.parts = [qkv[:, a:b] for a, b in zip(cut, cut[1:])]
                if kind == "float32":
                    self.parts = [p.contiguous() for p in self.parts]
                self.q, self.k, self.v = (p.unflatten(1, (-1, D)) for p in self.parts)
                self.qr, self.att = new(T, NQ, D, t=dt), new(T, NQ, D, t=dt)
                self.aq, self.as_, self.y = new(T, NQ * D, t=torch.int8), new(T), new(T, H)
                self.slots, self.pos, self.start, self.lens = (new(n, t=torch.int32) for n in (T, T, S + 1, S))

        def step(r, cache, rows, most):
            if kind == "float32":
                c.norm(r.x, y=r.n, w=nd[0])
                c.matmul_group(w[:3], r.n, r.parts)
            else:
                c.norm(r.x, yq=r.xq, yscale=r.xs, w=nd[0])
                c.matmul_i8(w[:3], r.xq, r.xs, r.parts)
            c.kv_append(cache, r.slots, r.k, r.v, q=r.q, q_out=r.qr, norm=B.NORM_RMS, q_w=nd[1], k_w=nd[2], rope=rd, pos=r.pos)
            c.attention(cache, r.qr, r.att, r.start, r.lens, table, max_rows=rows, max_len=most)
            if kind == "float32":
                c.matmul(w[3], r.att.flatten(1), r.y)
            else:
                c.norm(r.att.flatten(1), yq=r.aq, yscale=r.as_, kind=B.NORM_NONE)
                c.matmul_i8(w[3], r.aq, r.as_, r.y)

        held_k, held_v = [np.zeros((0, NK, D), np.float16)] * S, [np.zeros((0, NK, D), np.float16)] * S

        def inputs(r, rows):
            """rows[s] more tokens of each sequence."""
            before = [len(k) for k in held_k]
            pos = np.concatenate([np.arange(b, b + n) for b, n in zip(before, rows)]).astype(np.int32)
            of = np.repeat(np.arange(S), rows)
            r.x.copy_(dev(rng.standard_normal((r.T, H)).astype(np.float32)))
            r.pos.copy_(dev(pos))
            r.slots.copy_(dev((tab[of, pos // PAGE] * PAGE + pos % PAGE).astype(np.int32)))
            r.start.copy_(dev(np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)))
            r.lens.copy_(dev((np.array(before) + rows).astype(np.int32)))
            return pos, of

        def check(r, rows, pos, of, cache):
            stream.synchronize()
            host = lambda t: t.float().cpu().numpy()  # noqa: E731
            q, k, v = host(r.q), host(r.k), host(r.v)
            want = F.heads(q, 1, norms[1], 1e-6, 0.0, rope, pos, D, 1)
            off = np.abs(host(r.qr) - want) - ((2.0 ** -24 + F.HALF[kind]) * (1 + 1e-6) * np.abs(want) + 2.0 ** -19 * np.abs(want).max(-1, keepdims=True))
            assert off.max() <= 0
            gk, gv = (torch.zeros((r.T, NK, D), dtype=torch.float16, device="cuda") for _ in range(2))
            c.kv_read(cache, r.slots, gk, gv)
            stream.synchronize()
            gk, gv = gk.cpu().numpy(), gv.cpu().numpy()
            assert np.array_equal(gv, F.kept(v))
            assert (gk != F.kept(F.heads(k, 1, norms[2], 1e-6, 0.0, rope, pos, D, 1).astype(np.float32))).mean() <= 1e-4
            for s in range(S):
                held_k[s], held_v[s] = np.concatenate([held_k[s], gk[of == s]]), np.concatenate([held_v[s], gv[of == s]])
                n, have = rows[s], len(held_k[s])
                seen = np.arange(have)[None] <= np.arange(have - n, have)[:, None]
                for h in range(NQ):
                    F.attention_near(host(r.att)[of == s, h], host(r.qr)[of == s, h], held_k[s][:, h // 4], held_v[s][:, h // 4], D ** -0.5, seen, None, kind,
                                     (s, h))
            if kind != "float32":
                codes, scale = I.quantize(host(r.att).reshape(r.T, -1))
                assert np.array_equal(r.aq.cpu().numpy(), codes)
                assert np.array_equal(host(r.y), I.product(codes, scale, *weights[3]))
            assert torch.isfinite(r.y).all()

        first = Rows(sum(prompt))
        pos, of = inputs(first, prompt)
        for cache in caches:
            step(first, cache, max(prompt), max(prompt))
        check(first, prompt, pos, of, caches[0])
        one, eager = Rows(S), Rows(S)
        one.start.copy_(torch.arange(S + 1))
        step(eager, B.KVCache(S * WIDE, PAGE, NK, D), 1, PAGE * WIDE)          # scratch for the capture (no keys: lens are 0)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step(one, caches[0], 1, PAGE * WIDE)
        for _ in range(6):
            pos, of = inputs(one, [1] * S)
            for a in ("x", "pos", "slots", "start", "lens"):
                getattr(eager, a).copy_(getattr(one, a))
            graph.replay()
            step(eager, caches[1], 1, PAGE * WIDE)
            check(one, [1] * S, pos, of, caches[0])
            assert torch.equal(one.att, eager.att) and torch.equal(one.y, eager.y)
        assert torch.equal(caches[0].data, caches[1].data)
    for x in w:
        x.free()
    c.close()
