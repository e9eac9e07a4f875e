"""The example of a decode step runs all batch operators together with the
quantised products; each operator's part of it against 64 bits."""
import importlib.util
import os

import pytest
import torch

import _batch
import _common

pytestmark = pytest.mark.gpu


def test_shared_prefix_decode_example(Q, gpu):
    spec = importlib.util.spec_from_file_location("shared_prefix_decode", os.path.join(_common.ROOT, "examples", "shared_prefix_decode.py"))
    ex = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ex)
    d = ex.Decoder(requests=5, prefix=300, embd=512, heads=8, heads_kv=2, vocab=1000, page=16, most_new=32, rank=8, seed=3)
    tokens = torch.arange(5, device=gpu) + 5
    seen = []
    for step in range(20):
        hist = d.history.clone()
        nxt = d.step(tokens)
        if step in (0, 19):
            # the o projection of this step: product, then the adapters' part added in place
            x = d.attn.view(5, 512)
            y = Q.mul_mat_vec_q(d.w["o"], 512, x)
            ad = d.lora["o"]
            want, tol = _batch.lora(*ad.tensors[:2], x, d.adapter, y, ad.tensors[2])
            _batch.assert_close(d.buf["o"], want, tol, "o projection")
            pre = (*d.pre.tensors[:2], torch.zeros(1, dtype=torch.int32))
            lens = [step + 1] * 5
            want, _, tol, _ = _batch.attention(d.buf["q"].view(5, 8, 64), [(r, r + 1) for r in range(5)], pre, (d.own_k, d.own_v, d.table),
                                               (300, lens), 64 ** -0.5)
            _batch.assert_close(d.attn, want, tol, "attention")
        assert d.lens.tolist() == [step + 1] * 5
        assert (d.logits[:, 2] == -float("inf")).all() and (nxt != 2).all()
        assert (d.logits[0, 480:] == -float("inf")).all() and int(nxt[0]) < 480   # the grammar's first 15 words
        assert torch.equal(d.history[:, step], nxt.int()) and torch.equal(d.history[:, :step], hist[:, :step])
        seen.append(nxt.tolist())
        tokens = nxt
    # the same from the start: equal bits, so equal tokens
    d2 = ex.Decoder(requests=5, prefix=300, embd=512, heads=8, heads_kv=2, vocab=1000, page=16, most_new=32, rank=8, seed=3)
    tokens = torch.arange(5, device=gpu) + 5
    for step in range(20):
        tokens = d2.step(tokens)
        assert tokens.tolist() == seen[step]


def test_shared_prefix_decode_example_ends_with_its_pages(Q, gpu):
    spec = importlib.util.spec_from_file_location("shared_prefix_decode", os.path.join(_common.ROOT, "examples", "shared_prefix_decode.py"))
    ex = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ex)
    d = ex.Decoder(requests=2, prefix=20, embd=512, heads=8, heads_kv=2, vocab=256, page=16, most_new=3, rank=8, seed=3)
    tokens = torch.arange(2, device=gpu)
    for _ in range(3):
        tokens = d.step(tokens)
    with pytest.raises(ValueError):
        d.step(tokens)
    assert d.lens.tolist() == [3, 3]
