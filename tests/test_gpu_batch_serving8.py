"""GPU: a server's steps over a cache in 8 bits, as they are used together: one voice's long instruction is taken in once and its
pages named by every request's table, the requests' own prompts follow in one packed step, then single tokens from a captured
graph whose attention takes the shared rows once, whose logits are adjusted by what was said and drawn from.  A two-layer model
with random weights; the other side computes each last token in float64 from the rows that the cache holds, read back by
``gather``."""
import numpy as np
import pytest
import torch

from oracle import paged as o
from paged_helpers import values
from test_gpu_batch_serving import D, EPS, KH, LAYERS, PAGE, QH, VOCAB, Model, _near

pytestmark = pytest.mark.gpu

PREFIX, REQUESTS, ROOM = 2048, 20, 3  # 19 x 2048 rows of two KV heads saved: enough to be shared


class Server:
    def __init__(self, dev, model):
        self.m, self.dev = model, dev
        pages = PREFIX // PAGE + REQUESTS * ROOM
        angle = torch.arange(PREFIX + 64, dtype=torch.float64)[:, None] * 1e4 ** (-(torch.arange(D, dtype=torch.float64) % (D // 2)) / (D // 2))
        self.cos, self.sin = angle.cos().float().to(dev), angle.sin().float().to(dev)
        # memory as another program left it: e4m3's NaN, bytes that are no scale
        self.caches = []
        for _ in range(LAYERS):
            codes = torch.full((pages, 2, KH, PAGE, D), 0x7f, dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn)
            scales = torch.full((pages, 2, KH, PAGE), 255, dtype=torch.uint8, device=dev)
            self.caches.append((codes[:, 0], codes[:, 1], (scales[:, 0], scales[:, 1])))
        self.free = list(range(pages))[::-1]
        self.table = torch.full((REQUESTS, PREFIX // PAGE + ROOM), -1, dtype=torch.int32, device=dev)
        self.lengths = torch.zeros(REQUESTS, dtype=torch.int32, device=dev)
        self.held = [0] * REQUESTS
        self.groups = torch.zeros(REQUESTS, dtype=torch.int32, device=dev)
        self.shared = torch.full((REQUESTS,), PREFIX, dtype=torch.int32, device=dev)

    def grow(self, b, n):
        old = -(-self.held[b] // PAGE)
        self.held[b] += n
        for j in range(old, -(-self.held[b] // PAGE)):
            self.table[b, j] = self.free.pop()
        self.lengths[b] = self.held[b]

    def share(self, b):
        self.table[b, :PREFIX // PAGE] = self.table[0, :PREFIX // PAGE]
        self.held[b] = PREFIX
        self.lengths[b] = PREFIX

    def step(self, tokens, starts):
        from moss_tts._runtime import paged

        x = self.m.embedding[tokens]
        for p, (keys, vals, scales) in zip(self.m.layers, self.caches):
            q = paged.qk_rope(x @ p["qkv"].T, p["qn"], p["kn"], self.cos, self.sin, keys, vals, self.table, self.lengths, EPS,
                              starts=starts, scales=scales)
            if starts is None:
                y = paged.shared_decode_attention(q, keys, vals, self.table, self.lengths, self.groups, self.shared, scales=scales)
            else:
                y = paged.prompt_attention(q, keys, vals, self.table, self.lengths, starts, scales=scales)
            x = x + y @ p["o"].T
        return x

    def last_logits(self, b, token):
        """The last token's logits in float64 from the rows that the cache holds."""
        from moss_tts._runtime import paged

        m, n = self.m, self.held[b]
        starts = torch.tensor([0] + [0] * b + [n] * (REQUESTS - b), dtype=torch.int32, device=self.dev)
        x = m.embedding[token].double()
        cos, sin = self.cos[n - 1].double(), self.sin[n - 1].double()
        for p, (keys, vals, scales) in zip(m.layers, self.caches):
            k, v = (t.double().repeat_interleave(QH // KH, 1) for t in paged.gather(keys, vals, self.table, self.lengths, starts, n, scales=scales))
            q = (p["qkv"].double() @ x)[:QH * D].view(QH, D)
            q = q / (q.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * p["qn"].double()
            q = q * cos + torch.cat((-q[:, D // 2:], q[:, :D // 2]), -1) * sin
            w = torch.softmax((k * q).sum(-1) * D ** -0.5, 0)
            x = x + p["o"].double() @ (w[..., None] * v).sum(0).reshape(-1)
        return m.head.double() @ x


def test_a_voice_and_its_requests(dev):
    from moss_tts._runtime import sampling

    g = torch.Generator().manual_seed(5)
    m = Model(dev, 6)
    server = Server(dev, m)
    voice = torch.randint(0, VOCAB, (PREFIX,), generator=g).to(dev)
    own = [torch.randint(0, VOCAB, (1 + i % 9,), generator=g).tolist() for i in range(REQUESTS)]

    # the instruction, once; then every request's own prompt behind it, and padding
    server.grow(0, PREFIX)
    server.step(voice, torch.tensor([0] + [PREFIX] * REQUESTS, dtype=torch.int32, device=dev))
    for b in range(1, REQUESTS):
        server.share(b)
    for b in range(REQUESTS):
        server.grow(b, len(own[b]))
    counts = [len(t) for t in own]
    starts = torch.tensor([0, *np.cumsum(counts)], dtype=torch.int32, device=dev)
    x = server.step(torch.tensor(sum(own, []) + [0] * 5, device=dev), starts)
    logits = x[(starts[1:] - 1).long()] @ m.head.T
    for b in (0, 1, 8, 19):
        _near(logits[b], server.last_logits(b, own[b][-1]), f"prompt of request {b}")

    # single tokens: one captured step with its draw, replayed as the sequences grow
    history = torch.zeros((REQUESTS, 40), dtype=torch.int64, device=dev)
    said = torch.tensor(counts, dtype=torch.int32, device=dev)
    prompt = said.clone()
    for b in range(REQUESTS):
        history[b, :counts[b]] = torch.tensor(own[b], device=dev)
    mask = torch.full((1, (VOCAB + 31) // 32), -1, dtype=torch.int32, device=dev)
    mask[0, :100] = 0  # no token below 3200
    penalties = dict(tokens=history, lengths=said, prompt=prompt, repetition=1.2, presence=torch.rand(REQUESTS, generator=g).to(dev),
                     frequency=0.3, mask=mask)
    settings = dict(temperature=0.8, top_k=50, top_p=0.9)
    tokens = torch.zeros(REQUESTS, dtype=torch.int64, device=dev)
    uniform = torch.zeros(REQUESTS, device=dev)

    def draw(raw):
        adjusted = sampling.adjust(raw, **penalties)
        return adjusted, sampling.sample(adjusted, uniform, **settings)

    uniform.copy_(torch.rand(REQUESTS, generator=g))
    _, nxt = draw(logits)
    for b in range(REQUESTS):
        server.grow(b, 1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        draw(server.step(tokens, None) @ m.head.T)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        raw = server.step(tokens, None) @ m.head.T
        adjusted, drawn = draw(raw)
    for i in range(12):
        if i:
            for b in range(REQUESTS):
                server.grow(b, 1)
        tokens.copy_(nxt)
        history[torch.arange(REQUESTS, device=dev), said.long()] = nxt
        said += 1
        uniform.copy_(torch.rand(REQUESTS, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        nxt = drawn.clone()
        assert ((nxt >= 3200) & (nxt < VOCAB)).all()
        again = draw(raw)
        assert torch.equal(again[0], adjusted) and torch.equal(again[1], drawn)
        if i % 4 == 3:
            for b in (0, 7, 19):
                _near(raw[b], server.last_logits(b, int(tokens[b])), f"token {i} of request {b}")
                n = int(said[b])
                want = o.adjust(values(raw[b]), history[b, :n].cpu().numpy(), int(prompt[b]), 1.2, float(penalties["presence"][b]), 0.3, [],
                                mask[0].cpu().numpy())
                got = values(adjusted[b])
                assert np.array_equal(np.isneginf(got), np.isneginf(want))
                fine = np.isfinite(want)
                # a rounding to bf16 of what a few fp32 steps leave of terms up to |logit| + 12 x 0.3 + 1
                assert (np.abs(got[fine] - want[fine]) <= 2.0 ** -8 * np.abs(want[fine]) + 2.0 ** -20 * (np.abs(values(raw[b])[fine]) * 1.2 + 5)).all()
