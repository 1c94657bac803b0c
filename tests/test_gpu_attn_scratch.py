"""bgl_attn_dev's scratch and captures: what a context's first call reserves, and what a call that is refused leaves behind."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch_dev():
    import torch
    assert torch.cuda.is_available(), "gpu tests need a GPU"
    return torch


def ints(torch, *v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


class Seqs:
    """Sequences of (rows, keys) over a cache that a context of its own has filled."""

    def __init__(self, torch, seqs, nq, nk, D, dtype, page=16, seed=0):
        import beglin_amd as B
        gen = torch.Generator(device="cuda").manual_seed(seed)
        rand = lambda *s: torch.randn(s, generator=gen, device="cuda")  # noqa: E731
        wide = max((n + page - 1) // page for _, n in seqs)
        self.cache = B.KVCache(len(seqs) * wide, page, nk, D)
        self.table = torch.arange(len(seqs) * wide, dtype=torch.int32, device="cuda").reshape(-1, wide)
        places = len(seqs) * wide * page
        c = B.Context(0, torch.cuda.current_stream().cuda_stream)
        c.kv_append(self.cache, torch.arange(places, dtype=torch.int32, device="cuda"), rand(places, nk, D), rand(places, nk, D))
        torch.cuda.synchronize()
        c.close()
        self.start = ints(torch, *np.concatenate([[0], np.cumsum([r for r, _ in seqs])]).tolist())
        self.lens = ints(torch, *[n for _, n in seqs])
        self.q = rand(sum(r for r, _ in seqs), nq, D).to(dtype)
        self.out = torch.full_like(self.q, 7.0)
        self.how = dict(max_rows=max(r for r, _ in seqs), max_len=max(n for _, n in seqs))

    def call(self, c, out=None, **how):
        c.attention(self.cache, self.q, self.out if out is None else out, self.start, self.lens, self.table, **{**self.how, **how})


PROMPTS = {"one prompt": ([(40, 40)], 4, 2), "one long prompt": ([(300, 900)], 8, 8), "a prompt and tokens": ([(50, 60), (1, 200), (1, 7)], 8, 2),
           "a token": ([(1, 30)], 4, 2), "prompts and tokens, two kernels": ([(70, 2500), (1, 2500), (60, 60)], 16, 2)}


@pytest.mark.parametrize("first", PROMPTS, ids=list(PROMPTS))
@pytest.mark.parametrize("kind", ["float32", "bfloat16"])
def test_decode_is_captured_after_any_first_call(torch_dev, first, kind):
    """A prompt, then the step of single rows as a graph, with no other call between them."""
    import beglin_amd as B
    torch, (seqs, nq, nk) = torch_dev, PROMPTS[first]
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        prompt = Seqs(torch, seqs, nq, nk, 64, getattr(torch, kind))
        step = Seqs(torch, [(1, 700), (1, 1), (1, 90)], 8, 2, 128, getattr(torch, kind), seed=1)
        c, other = B.Context(0, st.cuda_stream), B.Context(0, st.cuda_stream)
        prompt.call(c)
        st.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            step.call(c)
        assert (step.out == 7).all()
        want = torch.empty_like(step.out)
        for i in range(4):
            step.q.mul_(0.9)
            step.lens[0] -= 100
            step.out.fill_(7.0)
            g.replay()
            step.call(other, want)
            prompt.call(c)
            st.synchronize()
            assert torch.equal(step.out, want) and torch.isfinite(want.float()).all(), i
        c.close()
        other.close()


def captured(torch, c, st, call, mark):
    """A graph of a call that may be refused, which is all that it then lacks, and the refusal's code."""
    import beglin_amd as B
    g, code = torch.cuda.CUDAGraph(), 0
    with torch.cuda.graph(g, stream=st):
        try:
            call(c)
        except B.BglError as e:
            code = e.code
        mark.add_(1)
    return g, code


@pytest.mark.parametrize("seqs,nk,longest", [([(90, 90), (1, 90), (40, 90)], 64, 4000), ([(90, 90), (1, 90), (40, 90)], 1, 4000), ([(90, 90), (1, 90)], 200, 90),
                                             ([(40, 3000)], 1, 3000)], ids=str)
def test_a_refused_call_has_launched_nothing(torch_dev, seqs, nk, longest):
    """A context's first call inside a capture: refused as a whole where it needs scratch (two kernels, or keys in parts), or captured as a whole."""
    import beglin_amd as B
    torch = torch_dev
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        b = Seqs(torch, seqs, nk, nk, 64, torch.float16)
        c, other = B.Context(0, st.cuda_stream), B.Context(0, st.cuda_stream)
        mark, want = torch.zeros(4, device="cuda"), torch.empty_like(b.out)
        b.call(other, want, max_len=longest)
        st.synchronize()
        g, code = captured(torch, c, st, lambda c: b.call(c, max_len=longest), mark)
        assert code in (0, B.E_CAPTURE) and (code or longest == 90)
        for i in range(3):
            b.out.fill_(7.0)
            g.replay()
            st.synchronize()
            assert (mark == i + 1).all() and ((b.out == 7).all() if code else torch.equal(b.out, want))
        b.call(c, max_len=longest)
        st.synchronize()
        assert torch.equal(b.out, want)
        c.close()
        other.close()


def test_a_prompt_without_scratch_is_captured_first(torch_dev):
    """One sequence whose keys are in one part needs none: a context's first call may be inside a capture."""
    import beglin_amd as B
    torch = torch_dev
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        b = Seqs(torch, [(60, 60)], 4, 2, 64, torch.float16)
        c, other = B.Context(0, st.cuda_stream), B.Context(0, st.cuda_stream)
        mark, want = torch.zeros(4, device="cuda"), torch.empty_like(b.out)
        st.synchronize()
        g, code = captured(torch, c, st, b.call, mark)
        assert code == 0
        for _ in range(3):
            b.q.mul_(0.5)
            g.replay()
            b.call(other, want)
            st.synchronize()
            assert torch.equal(b.out, want)
        c.close()
        other.close()
