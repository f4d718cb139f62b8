"""GPU: the operators over a paged cache together, as a server runs them: prompts of different lengths packed into one
step, one of them continued later, then single tokens for the whole batch from a captured graph, each request with its own
sampling settings, pages handed out as sequences grow.  A two-layer model with random weights; the other side computes every
sequence from its tokens alone, in float64 from the same bf16 weights."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

HIDDEN, QH, KH, D, VOCAB, LAYERS, PAGE, EPS = 512, 8, 2, 64, 5000, 2, 16, 1e-6


class Model:
    def __init__(self, dev, seed):
        g = torch.Generator().manual_seed(seed)

        def make(*shape, scale):
            return (torch.randn(shape, generator=g) * scale).bfloat16().to(dev)

        self.embedding = make(VOCAB, HIDDEN, scale=1.0)
        self.layers = [dict(qkv=make((QH + 2 * KH) * D, HIDDEN, scale=HIDDEN ** -0.5), o=make(HIDDEN, QH * D, scale=(QH * D) ** -0.5),
                            qn=make(D, scale=0.1) + 1, kn=make(D, scale=0.1) + 1) for _ in range(LAYERS)]
        self.head = make(VOCAB, HIDDEN, scale=3 * HIDDEN ** -0.5)
        angle = torch.arange(256, dtype=torch.float64)[:, None] * 1e4 ** (-(torch.arange(D, dtype=torch.float64) % (D // 2)) / (D // 2))
        self.cos, self.sin = angle.cos().float().to(dev), angle.sin().float().to(dev)


def _alone(m, tokens):
    """Logits of the last of one sequence's tokens, from all of them, in float64."""
    x = m.embedding[tokens].double()
    n = len(tokens)
    cos, sin = m.cos[:n, None].double(), m.sin[:n, None].double()

    def turned(v, w):
        v = v / (v.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * w.double()
        return v * cos + torch.cat((-v[..., D // 2:], v[..., :D // 2]), -1) * sin

    for p in m.layers:
        qkv = (x @ p["qkv"].double().T).view(n, QH + 2 * KH, D)
        q, k, v = turned(qkv[:, :QH], p["qn"]), turned(qkv[:, QH:QH + KH], p["kn"]), qkv[:, QH + KH:]
        k, v = (t.repeat_interleave(QH // KH, 1) for t in (k, v))
        s = (q.transpose(0, 1) @ k.permute(1, 2, 0)) * D ** -0.5
        s = s.masked_fill(torch.ones((n, n), dtype=torch.bool, device=s.device).triu(1), float("-inf"))
        x = x + (torch.softmax(s, -1) @ v.transpose(0, 1)).transpose(0, 1).reshape(n, QH * D) @ p["o"].double().T
    return x[-1] @ m.head.double().T


class Server:
    """The batch's pages and what each sequence has of them."""

    def __init__(self, dev, model, requests, room):
        self.m, self.dev = model, dev
        self.keys, self.values = ([torch.full((requests * room, KH, PAGE, D), float("nan"), dtype=torch.bfloat16, device=dev)
                                   for _ in range(LAYERS)] for _ in range(2))
        self.free = list(range(requests * room))[::-1]
        self.table = torch.full((requests, room), -1, dtype=torch.int32, device=dev)
        self.lengths = torch.zeros(requests, dtype=torch.int32, device=dev)
        self.held = [0] * requests

    def grow(self, b, n):
        old = -(-self.held[b] // PAGE)
        self.held[b] += n
        for j in range(old, -(-self.held[b] // PAGE)):
            self.table[b, j] = self.free.pop()
        self.lengths[b] = self.held[b]

    def step(self, tokens, starts):
        """Hidden rows of packed tokens; ``starts`` None: one a sequence."""
        from moss_tts._runtime import paged

        m = self.m
        x = m.embedding[tokens]
        for i, p in enumerate(m.layers):
            q = paged.qk_rope(x @ p["qkv"].T, p["qn"], p["kn"], m.cos, m.sin, self.keys[i], self.values[i], self.table,
                              self.lengths, EPS, starts=starts)
            if starts is None:
                o = paged.decode_attention(q, self.keys[i], self.values[i], self.table, self.lengths)
            else:
                o = paged.prompt_attention(q, self.keys[i], self.values[i], self.table, self.lengths, starts)
            x = x + o @ p["o"].T
        return x


def _near(got, want, what):
    # two layers whose every product, sum and attention is rounded to bf16 (2^-8 of a value each, about ten in a row)
    got, want = got.double(), want.double()
    err = float((got - want).norm() / want.norm())
    print(f"{what}: {err:.2e}", flush=True)
    assert err < 10 * 2.0 ** -8, what


def test_prompts_then_tokens(dev):
    from moss_tts._runtime import sampling

    g = torch.Generator().manual_seed(1)
    m = Model(dev, 2)
    prompts = [37, 5, 100]
    server = Server(dev, m, len(prompts), 12)
    told = [torch.randint(0, VOCAB, (n,), generator=g).tolist() for n in prompts]
    settings = dict(temperature=torch.tensor([0.0, 0.8, 1.2], device=dev), top_k=torch.tensor([0, 50, 0], dtype=torch.int32, device=dev),
                    top_p=torch.tensor([1.0, 0.9, 0.7], device=dev), min_p=torch.tensor([0.0, 0.0, 0.02], device=dev))

    # step 1: two whole prompts and the first 60 tokens of the third; step 2: the rest of it, and padding
    first = [prompts[0], prompts[1], 60]
    for b, n in enumerate(first):
        server.grow(b, n)
    packed = torch.tensor(told[0] + told[1] + told[2][:60], device=dev)
    x = server.step(packed, torch.tensor([0, *np.cumsum(first)], dtype=torch.int32, device=dev))
    last = [x[36], x[41], None]
    server.grow(2, 40)
    packed = torch.tensor(told[2][60:] + [0] * 8, device=dev)
    x = server.step(packed, torch.tensor([0, 0, 0, 40], dtype=torch.int32, device=dev))
    last[2] = x[39]
    logits = torch.stack(last) @ m.head.T
    for b in range(3):
        _near(logits[b], _alone(m, told[b]), f"prompt {b}")

    # single tokens: one captured step, replayed as the sequences grow
    tokens = torch.zeros(3, dtype=torch.int64, device=dev)
    uniform = torch.zeros(3, device=dev)
    for b in range(3):
        server.grow(b, 1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        sampling.sample(server.step(tokens, None) @ m.head.T, uniform, **settings)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out_logits = server.step(tokens, None) @ m.head.T
        drawn = sampling.sample(out_logits, uniform, **settings)
    nxt = sampling.sample(logits, torch.rand(3, generator=g).to(dev), **settings)
    for i in range(20):
        if i:
            for b in range(3):
                server.grow(b, 1)
        for b in range(3):
            told[b].append(int(nxt[b]))
        tokens.copy_(nxt)
        uniform.copy_(torch.rand(3, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        nxt = drawn.clone()
        assert torch.equal(nxt, sampling.sample(out_logits, uniform, **settings))
        if i % 5 == 4:
            for b in range(3):
                _near(out_logits[b], _alone(m, told[b]), f"token {i} of request {b}")
    assert ((nxt >= 0) & (nxt < VOCAB)).all()
    assert int(nxt[0]) == int((out_logits[0] == out_logits[0].max()).nonzero()[0])  # temperature 0: the first of the largest
