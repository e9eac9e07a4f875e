"""A whole decode step, products and all: projections, norms and rotation, the cache,
attention, the output projection, penalties, the next tokens -- eager and as a
captured graph whose lengths, positions and random numbers change on the device."""
import numpy as np
import pytest
import torch

import _step

pytestmark = pytest.mark.gpu


class Server:
    def __init__(self, Q, gpu, kind, B=5, K=512, H=8, HK=2, V=4096, page=32, block=8, most=96):
        self.Q, self.B, self.K, self.H, self.HK, self.D, self.V, self.most = Q, B, K, H, HK, K // H, V, most
        rng = np.random.default_rng(3)
        g = torch.Generator(device=gpu).manual_seed(3)
        w = lambda m: torch.from_numpy(Q.quantize_rows_q4_K(rng.standard_normal((m, K), dtype=np.float32) * np.float32(K ** -0.5))).to(gpu)  # noqa: E731
        self.w = {"q": w(K), "k": w(HK * self.D), "v": w(HK * self.D), "o": w(K), "out": w(V)}
        self.embed = torch.randn(V, K, device=gpu, generator=g)
        norm = 1 + 0.1 * torch.randn(self.D, device=gpu, generator=g)
        self.rope = Q.Rope(self.D, mode="neox", q_norm=norm, k_norm=norm)
        per = -(-most // page)
        table = torch.randperm(B * per, device=gpu, generator=g).view(B, per).int()
        self.cache = [torch.zeros(B * per, page, HK, self.D, dtype=torch.uint8, device=gpu).view(kind) for _ in range(2)]
        self.cache += [torch.zeros(B * per, page // block, HK, device=gpu) for _ in range(2)]
        self.pages = Q.KV8Pages(*self.cache, table=table)
        self.lens = torch.zeros(B, dtype=torch.int32, device=gpu)
        self.tokens = (torch.arange(B, device=gpu) * 11 + 1).int()
        self.uniform, self.logits = torch.zeros(B, device=gpu), torch.zeros(B, V, device=gpu)
        self.history = torch.full((B, most), -1, dtype=torch.int32, device=gpu)
        self.start = torch.arange(B + 1, dtype=torch.int64, device=gpu) * most
        self.repeat = torch.full((B,), 1.3, device=gpu)
        self.rules = dict(temperature=torch.tensor([0.0, 0.7, 1.0, 1.0, 1.3], device=gpu), top_k=torch.tensor([0, 40, 0, 0, 5], dtype=torch.int32, device=gpu),
                          top_p=torch.tensor([1.0, 0.95, 0.9, 1.0, 0.8], device=gpu), min_p=torch.tensor([0.0, 0.05, 0.0, 0.0, 0.1], device=gpu))
        self.attn, self.lp = torch.zeros(B, H, self.D, device=gpu), torch.zeros(B, device=gpu)
        self.ws = Q.kv8_attention_workspace(self.attn, self.pages, self.lens, most)
        self.ws_sample = Q.sample_workspace(self.logits)
        self.row = torch.arange(B, device=gpu)

    def step(self):
        Q, B, K = self.Q, self.B, self.K
        mul = lambda n, x: Q.mul_mat_vec_q(self.w[n], K, x, out=torch.empty(B, self.w[n].shape[0], device=x.device))  # noqa: E731
        x = self.embed[self.tokens.long()]
        q, k, v = (mul(n, x).view(B, -1, self.D) for n in "qkv")
        Q.rope(self.rope, q, k, self.lens, q_out=q, k_out=k)
        at = self.lens.long()
        self.lens += 1
        Q.kv8_store(self.pages, k, v, self.lens, self.most)
        Q.kv8_attention(q, self.pages, self.lens, self.most, out=self.attn, workspace=self.ws)
        h = x + mul("o", self.attn.view(B, K))
        h = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + 1e-6)
        Q.mul_mat_vec_q(self.w["out"], K, h, out=self.logits)
        Q.logits_adjust(self.logits, repeat=self.repeat, history=self.history.view(-1), history_start=self.start, out=self.logits)
        Q.sample(self.logits, self.uniform, out=self.tokens, logprob=self.lp, workspace=self.ws_sample, **self.rules)
        self.history[self.row, at] = self.tokens


@pytest.mark.parametrize("kind", [torch.int8, torch.float8_e4m3fn])
def test_decode_steps_eager_and_in_a_graph(Q, gpu, kind):
    steps = 12
    g = torch.Generator(device=gpu).manual_seed(1)
    u = torch.rand(steps, 5, device=gpu, generator=g)
    a, b = Server(Q, gpu, kind), Server(Q, gpu, kind)
    want = []
    for i in range(steps):
        a.uniform.copy_(u[i])
        a.step()
        want.append((a.tokens.clone(), a.lp.clone()))
        for r in range(a.B):
            t, k, p, m = (float(a.rules[n][r]) for n in ("temperature", "top_k", "top_p", "min_p"))
            token, lp, margin = _step.sample(a.logits[r], float(u[i, r]), t, int(k), p, m)
            assert margin < 2.0 ** -36 or (int(a.tokens[r]) == token and abs(float(a.lp[r]) - lp) <= 2.0 ** -24 * abs(lp) + 1e-10)
    # the same in a graph: one step to warm up, taken back
    b.step()
    torch.cuda.synchronize()
    first = (torch.arange(b.B, device=gpu) * 11 + 1).int()
    for t in (b.lens, *b.cache[2:]):
        t.zero_()
    for t in b.cache[:2]:
        t.view(torch.uint8).zero_()
    b.history.fill_(-1)
    b.tokens.copy_(first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.step()
    for i in range(steps):
        b.uniform.copy_(u[i])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(b.tokens, want[i][0]) and torch.equal(b.lp, want[i][1]), i
    for x, y in zip(a.cache, b.cache):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
