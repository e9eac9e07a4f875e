"""One decode step of a layer and the output projection for a batch of up to
eight requests that share a long prefix, each with an adapter, a history and a
grammar of its own, on random weights:

    x -> Q4_K products q, k, v + the requests' adapters -> k, v into the requests'
    own pages -> attention over the shared prefix and the own tokens -> Q4_K
    product o + adapters -> Q6_K output projection -> penalties, biases and
    masks -> the next tokens

What the requests share is read once for all of them: the quantised weights by
mul_mat_vec_q, the prefix's keys and values by prefix_attention.  (A layer's
norms, rotary positions and feed-forward part are left out.)

    python examples/shared_prefix_decode.py [--requests 8] [--prefix 4096] [--steps 4]
"""
import argparse
import importlib.util
import os
import sys

import numpy as np
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def package():
    if "q4k_amd" not in sys.modules:
        spec = importlib.util.spec_from_file_location("q4k_amd", os.path.join(ROOT, "gemv-q4_k-optimization_amd", "__init__.py"))
        sys.modules["q4k_amd"] = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(sys.modules["q4k_amd"])
    return sys.modules["q4k_amd"]


class Decoder:
    """The weights, caches and workspaces that a server keeps between steps."""

    def __init__(self, requests=8, prefix=4096, embd=4096, heads=32, heads_kv=8, vocab=32768, adapters=4, rank=16, page=64,
                 most_new=256, seed=0):
        Q = self.Q = package()
        dev = self.dev = torch.device("cuda:0")
        rng = np.random.default_rng(seed)
        g = torch.Generator(device=dev).manual_seed(seed)
        self.B, self.K, self.H, self.HK, self.D, self.V = requests, embd, heads, heads_kv, embd // heads, vocab
        self.prefix, self.page, self.most = prefix, page, most_new

        def q4(rows, k):
            w = rng.standard_normal((rows, k), dtype=np.float32) * np.float32(k ** -0.5)
            return torch.from_numpy(Q.quantize_rows_q4_K(w, nthreads=16)).to(dev)

        kv = heads_kv * self.D
        self.w = {"q": q4(embd, embd), "k": q4(kv, embd), "v": q4(kv, embd), "o": q4(embd, embd)}
        out = rng.standard_normal((vocab, embd), dtype=np.float32) * np.float32(embd ** -0.5)
        self.w_out = torch.from_numpy(Q.quantize_rows_q6_K(out, nthreads=16)).to(dev)
        self.embed = torch.randn(vocab, embd, device=dev, generator=g)

        def lora(rows):
            a = (torch.randn(adapters, rank, embd, device=dev, generator=g) * embd ** -0.5).half()
            b = (torch.randn(adapters, rows, rank, device=dev, generator=g) * 0.1).half()
            return Q.LoraAdapters(a, b, scale=torch.full((adapters,), 2.0, device=dev))

        self.lora = {n: lora(w.shape[0]) for n, w in self.w.items()}
        self.adapter = torch.arange(requests, dtype=torch.int32, device=dev) % (adapters + 1) - 1  # -1: none
        # the prefix's keys and values, written once; pages of the requests' own
        half = lambda *s: torch.randn(*s, device=dev, generator=g).half()  # noqa: E731
        self.pre = Q.KVPages(half(1, prefix, heads_kv, self.D), half(1, prefix, heads_kv, self.D))
        per = -(-most_new // page)
        self.own_k, self.own_v = (torch.zeros(requests * per, page, heads_kv, self.D, dtype=torch.float16, device=dev) for _ in range(2))
        self.table = torch.randperm(requests * per, device=dev, generator=g).view(requests, per).int()
        self.own = Q.KVPages(self.own_k, self.own_v, table=self.table)
        self.lens = torch.zeros(requests, dtype=torch.int32, device=dev)
        self.steps = 0  # taken: what every request has generated, known without asking the device
        self.row = torch.arange(requests, device=dev)
        # histories: what each request has generated, one list of `most_new` places each
        self.history = torch.full((requests, most_new), -1, dtype=torch.int32, device=dev)
        self.history_start = torch.arange(requests + 1, dtype=torch.int64, device=dev) * most_new
        self.penalty = [torch.full((requests,), x, device=dev) for x in (1.1, 0.05, 0.1)]
        self.bias_ids = torch.full((requests,), 2, dtype=torch.int32, device=dev)   # token 2 never
        self.bias = torch.full((requests,), -float("inf"), device=dev)
        self.bias_start = torch.arange(requests + 1, dtype=torch.int64, device=dev)
        # a grammar for the first request: the first half of the vocabulary only
        self.mask = torch.zeros(1, -(-vocab // 32), dtype=torch.int32, device=dev)
        self.mask[:, :vocab // 64] = -1
        self.mask_rows = torch.where(self.row == 0, 0, -1).int()
        f32 = lambda *s: torch.empty(*s, device=dev)  # noqa: E731
        self.buf = {n: f32(requests, w.shape[0]) for n, w in self.w.items()}
        self.attn, self.logits = f32(requests, heads, self.D), f32(requests, vocab)
        self.ws_lora = Q.lora_workspace(self.lora["q"], requests)
        self.ws_attn = Q.prefix_attention_workspace(self.attn, self.pre, prefix, self.own, self.lens, most_new)

    def project(self, name, x):
        """The shared Q4_K product and, in place, each request's adapter."""
        y = self.Q.mul_mat_vec_q(self.w[name], self.K, x, out=self.buf[name])
        return self.Q.lora_add(self.lora[name], x, self.adapter, base=y, out=y, workspace=self.ws_lora)

    def step(self, tokens):
        """tokens int64 [requests] -> the next tokens."""
        if self.steps == self.most:
            raise ValueError(f"the requests' own pages hold {self.most} tokens each")
        self.steps += 1
        Q, B = self.Q, self.B
        x = self.embed[tokens]
        q, k, v = (self.project(n, x) for n in "qkv")
        # the new token's key and value go to the end of its request's own pages
        at = self.lens.long()
        pages = self.table[self.row, at // self.page].long()
        self.own_k[pages, at % self.page] = k.view(B, self.HK, self.D).half()
        self.own_v[pages, at % self.page] = v.view(B, self.HK, self.D).half()
        self.lens += 1
        Q.prefix_attention(q.view(B, self.H, self.D), self.pre, self.prefix, self.own, self.lens, self.most, out=self.attn,
                           workspace=self.ws_attn)
        h = x + self.project("o", self.attn.view(B, self.K))
        h = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + 1e-6)
        Q.mul_mat_vec_q(self.w_out, self.K, h, out=self.logits, wtype=Q.GGML_TYPE_Q6_K)
        rep, freq, pres = self.penalty
        Q.logits_adjust(self.logits, repeat=rep, frequency=freq, presence=pres, history=self.history.view(-1),
                        history_start=self.history_start, bias_ids=self.bias_ids, bias=self.bias, bias_start=self.bias_start,
                        mask=self.mask, mask_rows=self.mask_rows, out=self.logits)
        nxt = self.logits.argmax(-1)
        self.history[self.row, at] = nxt.int()
        return nxt


def main():
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--requests", type=int, default=8)
    ap.add_argument("--prefix", type=int, default=4096)
    ap.add_argument("--steps", type=int, default=4)
    a = ap.parse_args()
    d = Decoder(requests=a.requests, prefix=a.prefix, most_new=max(256, a.steps))
    tokens = torch.arange(a.requests, device=d.dev) + 5
    for i in range(a.steps):
        tokens = d.step(tokens)
        print(f"step {i}: {tokens.tolist()}", flush=True)


if __name__ == "__main__":
    main()
