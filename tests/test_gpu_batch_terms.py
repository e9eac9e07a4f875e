"""F32 activations, queries and probabilities keep the bits that q4k_batch.h
states: results of single products against 64 bits, at bounds that no kernel
without the smallest of a value's terms meets."""
import pytest
import torch

import _batch
import _batch_terms as T

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("N,K,M,r,A", [(1, 256, 64, 8, 1), (7, 264, 70, 16, 3), (17, 333, 65, 5, 4), (64, 512, 130, 24, 2), (40, 320, 96, 96, 2),
                                       (33, 256, 300, 200, 1), (700, 512, 200, 64, 3), (700, 2048, 100, 40, 40), (520, 4096, 64, 16, 2),
                                       (600, 256, 14336, 16, 2)])
def test_adapters_keep_24_bits(Q, gpu, dtype, N, K, M, r, A):
    a, b, x, ids, base, scale, want, tol = T.lora_inputs(gpu, N, K, M, r, A, dtype, N + M)
    got = Q.lora_add(Q.LoraAdapters(a, b, scale=scale), x, ids, base=base)
    _batch.assert_close(got, want.cpu(), tol.cpu(), "lora")


# rows of a KV head: streamed by 16 and 32, and shared (F16: from 193; 256 dimensions: from 33)
@pytest.mark.parametrize("kv", [F16, BF16])
@pytest.mark.parametrize("B,H,hk,D", [(1, 1, 1, 64), (3, 8, 2, 128), (11, 4, 2, 80), (150, 4, 2, 64), (90, 6, 2, 128), (5, 4, 4, 256), (30, 4, 2, 256)])
def test_attention_keeps_f32(Q, gpu, kv, B, H, hk, D):
    q, k, v, want, tol = T.score_inputs(gpu, B, H, hk, D, kv, B + D)
    lse = torch.empty(B, H, device=gpu)
    Q.prefix_attention(q, Q.KVPages(k[None], v[None]), 1, scale=1.0, lse=lse)
    _batch.assert_close(lse, want.cpu(), tol.cpu(), "score")
    for n in (3, 33, 64):
        q, k, v, want, tol = T.probability_inputs(gpu, B, H, hk, D, n, kv, B + n)
        got = Q.prefix_attention(q, Q.KVPages(k[None], v[None]), n, scale=1.0)
        _batch.assert_close(got, want.cpu(), tol.cpu(), f"probability of {n}")
