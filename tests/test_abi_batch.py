"""Argument checks of the batch operators (include/q4k_batch.h) that need no GPU."""
import ctypes

import pytest

FAKE = 0x10000  # never dereferenced by the host checks
OK, EUNSUPPORTED, EINVAL = 0, 1, 2


def lora(Q, **kw):
    d = dict(type=1, rank=8, n_adapters=2, a=FAKE, nb_a=512, nb_a_adapter=4096, b=FAKE, nb_b=16, nb_b_adapter=1024, scale=None, ranks=None)
    d.update(kw)
    return Q.q4k_lora(*d.values())


def lora_call(Q, l, ne00=256, ne01=64, x=FAKE, N=2, nb11=1024, ids=FAKE, base=FAKE, nb21=256, dst=FAKE + 4096, nb1=256, ws=None, wb=0):
    return Q.lib().q4k_lora_add(ctypes.byref(l), ne00, ne01, x, N, nb11, ids, base, nb21, dst, nb1, ws, wb, None)


@pytest.mark.parametrize("desc", [dict(type=0), dict(type=12), dict(rank=0), dict(rank=257), dict(n_adapters=-1), dict(a=None), dict(b=None),
                                  dict(nb_a=510), dict(nb_a=513), dict(nb_b=14), dict(a=FAKE + 1), dict(scale=FAKE + 2), dict(ranks=FAKE + 1),
                                  dict(nb_b_adapter=-2)])
def test_lora_descriptor_checks(Q, desc):
    assert lora_call(Q, lora(Q, **desc)) == EINVAL


@pytest.mark.parametrize("kw", [dict(ne00=-1), dict(ne01=-1), dict(N=-1), dict(x=None), dict(ids=None), dict(dst=None), dict(x=FAKE + 2),
                                dict(ids=FAKE + 1), dict(dst=FAKE + 2), dict(nb11=1020), dict(nb11=1026), dict(nb1=252), dict(nb21=252),
                                dict(base=FAKE + 4096, nb21=512), dict(ne00=1 << 33)])
def test_lora_call_checks(Q, kw):
    assert lora_call(Q, lora(Q), **kw) == EINVAL


def test_lora_empty_and_workspace(Q):
    L, l = Q.lib(), lora(Q)
    assert lora_call(Q, l, N=0, x=None, ids=None, dst=None) == OK
    assert lora_call(Q, l, ne01=0) == OK
    assert L.q4k_lora_add(None, 256, 64, FAKE, 1, 1024, FAKE, None, 0, FAKE, 256, None, 0, None) == EINVAL
    size = lambda n, **kw: L.q4k_lora_workspace_bytes(ctypes.byref(lora(Q, **kw)), 256, 64, n)  # noqa: E731
    assert size(8) >= 8 * 8 * 4 and size(16) >= size(8)
    assert size(-1) == 0 and size(8, rank=0) == 0 and size(1 << 40) == 0
    assert L.q4k_lora_workspace_bytes(None, 256, 64, 8) == 0


def pages(Q, **kw):
    d = dict(k=FAKE, v=FAKE, n_pages=8, page_size=16, nb_k_page=32768, nb_k_token=2048, nb_k_head=256, nb_v_page=32768, nb_v_token=2048,
             nb_v_head=256, table=FAKE, table_stride=4, table_len=4)
    d.update(kw)
    return Q.q4k_kv_pages(*d.values())


def attn(Q, prefix=None, suffix=None, **kw):
    pre, suf = pages(Q, **(prefix or {})), pages(Q, **(suffix or {}))
    d = dict(q_type=0, kv_type=1, n_head=32, n_head_kv=8, head_dim=128, scale=1.0, n_tokens=2, n_requests=2, n_q=1, q_start=None, q=FAKE,
             nb_q_token=16384, nb_q_head=512, prefix=ctypes.pointer(pre), n_prefix=64, suffix=ctypes.pointer(suf), suffix_len=FAKE,
             max_suffix=64, dst=FAKE, nb_dst_token=16384, nb_dst_head=512, lse=None)
    d.update(kw)
    a = Q.q4k_prefix_attn_args(*d.values())
    return Q.lib().q4k_prefix_attn(ctypes.byref(a), None, 0, None), Q.lib().q4k_prefix_attn_workspace_bytes(ctypes.byref(a))


@pytest.mark.parametrize("kw", [
    dict(q_type=30), dict(q_type=12), dict(kv_type=0), dict(n_head=0), dict(n_head_kv=0), dict(n_head=33), dict(head_dim=0), dict(n_tokens=-1),
    dict(n_tokens=3), dict(n_q=-1), dict(n_prefix=-1), dict(max_suffix=-1), dict(q=None), dict(dst=None), dict(q=FAKE + 2), dict(dst=FAKE + 2),
    dict(lse=FAKE + 2), dict(q_start=FAKE + 2), dict(nb_q_token=16386), dict(nb_q_head=508), dict(nb_dst_head=508), dict(prefix=None),
    dict(suffix=None), dict(suffix_len=None), dict(suffix_len=FAKE + 2), dict(n_prefix=65), dict(max_suffix=65), dict(prefix=dict(k=None)),
    dict(suffix=dict(v=None)), dict(suffix=dict(n_pages=0)), dict(prefix=dict(page_size=0)), dict(suffix=dict(table=FAKE + 2)),
    dict(suffix=dict(table_len=-1)), dict(suffix=dict(table=None, table_len=5)), dict(suffix=dict(table_stride=-1)), dict(n_prefix=1 << 40)])
def test_prefix_attn_checks(Q, kw):
    parts = {k: v for k, v in kw.items() if isinstance(v, dict)}
    rest = {k: v for k, v in kw.items() if not isinstance(v, dict)}
    if rest.get("prefix", 1) is None or rest.get("suffix", 1) is None:
        pre, suf = pages(Q), pages(Q)
        d = dict(prefix=ctypes.pointer(pre), suffix=ctypes.pointer(suf))
        d.update(rest)
        a = Q.q4k_prefix_attn_args(0, 1, 32, 8, 128, 1.0, 2, 2, 1, None, FAKE, 16384, 512, d["prefix"], 64, d["suffix"], FAKE, 64, FAKE, 16384, 512, None)
        assert Q.lib().q4k_prefix_attn(ctypes.byref(a), None, 0, None) == EINVAL
        return
    assert attn(Q, **parts, **rest) == (EINVAL, 0)


@pytest.mark.parametrize("kw", [dict(head_dim=12), dict(head_dim=264), dict(prefix=dict(k=FAKE + 8)), dict(suffix=dict(nb_v_token=2056))])
def test_prefix_attn_unsupported(Q, kw):
    if kw.get("head_dim") == 264:
        kw = dict(kw, nb_q_head=2048, nb_dst_head=2048)
    assert attn(Q, **kw) == (EUNSUPPORTED, 0)


def test_prefix_attn_empty(Q):
    assert attn(Q, n_tokens=0, n_requests=0)[0] == OK
    assert attn(Q, n_tokens=0, n_q=0)[0] == OK
    assert Q.lib().q4k_prefix_attn(None, None, 0, None) == EINVAL
    assert Q.lib().q4k_prefix_attn_workspace_bytes(None) == 0


def logits(Q, src=FAKE, V=100, N=2, nb=400, dst=FAKE + 4096, nbd=400, **kw):
    r = Q.q4k_logits_rules()
    for k, v in kw.items():
        setattr(r, k, v)
    return Q.lib().q4k_logits_adjust(src, V, N, nb, ctypes.byref(r), dst, nbd, None)


@pytest.mark.parametrize("kw", [
    dict(V=-1), dict(N=-1), dict(src=None), dict(dst=None), dict(src=FAKE + 2), dict(dst=FAKE + 1), dict(nb=396), dict(nb=402), dict(nbd=396),
    dict(dst=FAKE, nbd=800), dict(V=1 << 33), dict(history=FAKE), dict(history_start=FAKE), dict(history=FAKE, history_start=FAKE + 4),
    dict(n_history=-1), dict(bias_ids=FAKE, bias=FAKE), dict(bias=FAKE), dict(n_bias=-1), dict(repeat=FAKE + 2), dict(mask_rows=FAKE),
    dict(mask=FAKE, n_masks=2, nb_mask=12), dict(mask=FAKE, n_masks=2, nb_mask=18), dict(mask=FAKE, n_masks=1, nb_mask=16), dict(n_masks=-1)])
def test_logits_checks(Q, kw):
    assert logits(Q, **kw) == EINVAL


def test_logits_empty(Q):
    assert logits(Q, N=0, src=None, dst=None) == OK
    assert logits(Q, V=0) == OK
    assert Q.lib().q4k_logits_adjust(FAKE, 100, 2, 400, None, FAKE, 400, None) == EINVAL


def test_binding_refuses_tensors_in_host_memory(Q):
    import torch
    f16, f32 = torch.float16, torch.float32
    with pytest.raises(ValueError):
        Q.logits_adjust(torch.zeros(2, 100, dtype=f32))
    with pytest.raises(ValueError):
        Q.LoraAdapters(torch.zeros(2, 8, 256, dtype=f16), torch.zeros(2, 64, 8, dtype=f16))
    with pytest.raises(ValueError):
        Q.KVPages(torch.zeros(2, 16, 2, 64, dtype=f16), torch.zeros(2, 16, 2, 64, dtype=f16))


def test_lora_rows_past_the_kernels_offsets(Q):
    """Values of a row are counted in 31 bits of bytes of a 16-bit row: up to 2^30 of them."""
    l = lora(Q, nb_a=1 << 33, nb_a_adapter=1 << 34)
    for K in ((1 << 30) + 1, (1 << 31) - 8192):
        assert lora_call(Q, l, ne00=K, N=1) == EUNSUPPORTED
        assert Q.lib().q4k_lora_workspace_bytes(ctypes.byref(l), K, 64, 1) == 0
    assert Q.lib().q4k_lora_workspace_bytes(ctypes.byref(l), 1 << 30, 64, 1) > 0


@pytest.mark.parametrize("K,rank,adapters,type", [(4096, 16, 256, 1), (4096, 16, 16, 1), (14336, 16, 4, 30), (4096, 8, 4, 1), (14336, 64, 16, 30),
                                                  (256, 200, 2, 1), (0, 16, 2, 1), (2304, 24, 40000, 30)])
def test_lora_workspace_serves_every_smaller_batch(Q, K, rank, adapters, type):
    """The size for n tokens is enough for fewer, so it never falls as n rises."""
    L, l = Q.lib(), lora(Q, rank=rank, n_adapters=adapters, type=type)
    sizes = [L.q4k_lora_workspace_bytes(ctypes.byref(l), K, 64, n) for n in [*range(1, 2200), 4095, 4096, 4097, 65536, 1 << 20]]
    assert sizes == sorted(sizes)
