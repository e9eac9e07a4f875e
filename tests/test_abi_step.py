"""Argument checks of the operators of a decode step (include/q4k_step.h) that need no GPU."""
import ctypes

import pytest
import torch

FAKE = 0x10000  # never dereferenced by the host checks
OK, EUNSUPPORTED, EINVAL = 0, 1, 2


def rows(Q, **kw):
    d = dict(src=FAKE, dst=FAKE + 65536, src_type=0, dst_type=0, n_head=8, nb_src_token=4096, nb_src_head=512, nb_dst_token=4096,
             nb_dst_head=512, norm=None)
    d.update(kw)
    return Q.q4k_rope_rows(*d.values())


def rope(Q, q={}, k={}, **kw):
    d = dict(head_dim=128, n_rot=128, mode=0, eps=1e-6, freq_base=1e4, freq_scale=1.0, ext_factor=0.0, attn_factor=1.0, beta_fast=32.0,
             beta_slow=1.0, n_ctx_orig=0, freq_factors=None, n_tokens=2, pos=FAKE)
    d.update(kw)
    a = Q.q4k_rope_args(*d.values())
    for name, r in (("q", q), ("k", k)):
        if r is not None:
            setattr(a, name, ctypes.pointer(rows(Q, **r)))
    return Q.lib().q4k_rope(ctypes.byref(a), None)


@pytest.mark.parametrize("kw", [
    dict(head_dim=0), dict(n_rot=130), dict(n_rot=3), dict(n_rot=-2), dict(mode=1), dict(mode=8), dict(eps=-1.0), dict(eps=float("nan")), dict(freq_base=0.0),
    dict(freq_base=float("nan")), dict(freq_scale=float("inf")), dict(ext_factor=1.0), dict(ext_factor=1.0, n_ctx_orig=4096, freq_scale=0.0),
    dict(ext_factor=1.0, n_ctx_orig=4096, freq_base=1.0), dict(ext_factor=1.0, n_ctx_orig=4096, beta_slow=0.0), dict(freq_factors=FAKE + 2),
    dict(n_tokens=-1), dict(n_tokens=1 << 31), dict(pos=None), dict(pos=FAKE + 2), dict(q=dict(src=None)), dict(k=dict(dst=None)),
    dict(q=dict(src=FAKE + 2)), dict(q=dict(src_type=12)), dict(q=dict(src_type=1)), dict(k=dict(src_type=1, dst_type=30)), dict(q=dict(n_head=-1)),
    dict(q=dict(nb_src_head=508)), dict(q=dict(nb_dst_head=256)), dict(q=dict(nb_src_token=4098)), dict(k=dict(norm=FAKE + 1)), dict(q=dict(nb_dst_token=256)),
    dict(q=dict(dst=FAKE, nb_dst_token=8192)), dict(q=dict(dst=FAKE, dst_type=1))])
def test_rope_checks(Q, kw):
    assert rope(Q, **kw) == EINVAL


def test_rope_unsupported_and_empty(Q):
    assert rope(Q, head_dim=258, n_rot=2, q=dict(nb_src_head=2048, nb_dst_head=2048), k=dict(nb_src_head=2048, nb_dst_head=2048)) == EUNSUPPORTED
    assert rope(Q, head_dim=127, n_rot=64) == EUNSUPPORTED
    assert rope(Q, q=dict(n_head=1 << 30)) == EUNSUPPORTED
    assert rope(Q, n_tokens=0, pos=None) == OK
    assert rope(Q, q=None, k=None) == OK
    assert rope(Q, q=dict(n_head=0, src=None), k=None) == OK
    assert Q.lib().q4k_rope(None, None) == EINVAL


def test_rope_binding(Q):
    x, pos = torch.zeros(3, 4, 64), torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError):
        Q.rope(Q.Rope(64), x, None, pos)
    with pytest.raises(ValueError):
        Q.rope(Q.Rope(64), None, None, pos)
    with pytest.raises(ValueError):
        Q.Rope(64, mode="half")
    with pytest.raises(ValueError):
        Q.Rope(64, q_norm=torch.ones(64))
    for kw in (dict(n_rot=66), dict(n_rot=5), dict(ext_factor=1.0), dict(freq_base=-1.0)):
        with pytest.raises(Q.Q4KError):
            Q.Rope(64, **kw)


def kv8(Q, **kw):
    d = dict(type=24, n_head_kv=8, head_dim=128, block=16, k=FAKE, v=FAKE, n_pages=8, page_size=16, nb_k_page=16384, nb_k_token=1024,
             nb_k_head=128, nb_v_page=16384, nb_v_token=1024, nb_v_head=128, k_scale=FAKE, v_scale=FAKE, nb_s_page=32, nb_s_block=32,
             nb_s_head=4, table=FAKE, table_stride=4, table_len=4)
    d.update(kw)
    return Q.q4k_kv8_pages(*d.values())


def kv8_rows(Q, name, pages={}, **kw):
    d = dict(pages=ctypes.pointer(kv8(Q, **pages)) if pages is not None else None, type=0, n_tokens=2, n_requests=2, n_q=1, q_start=None, len=FAKE,
             max_len=64, k=FAKE, v=FAKE, nb_k_token=4096, nb_k_head=512, nb_v_token=4096, nb_v_head=512)
    d.update(kw)
    a = Q.q4k_kv8_rows(*d.values())
    return getattr(Q.lib(), name)(ctypes.byref(a), None)


PAGES_INVALID = [dict(type=0), dict(type=1), dict(n_head_kv=0), dict(head_dim=0), dict(block=0), dict(block=32), dict(k=None), dict(v_scale=None),
                 dict(n_pages=0), dict(page_size=0), dict(k_scale=FAKE + 2), dict(nb_s_head=2), dict(table=FAKE + 2), dict(table_len=-1),
                 dict(table_len=3), dict(table_stride=-1), dict(table=None, table_len=5)]
PAGES_UNSUPPORTED = [dict(head_dim=120), dict(head_dim=272), dict(k=FAKE + 8), dict(nb_v_token=1032), dict(nb_k_page=16392)]


@pytest.mark.parametrize("name", ["q4k_kv8_store", "q4k_kv8_load"])
def test_kv8_rows_checks(Q, name):
    for pages in PAGES_INVALID:
        assert kv8_rows(Q, name, pages) == EINVAL, pages
    for pages in PAGES_UNSUPPORTED:
        assert kv8_rows(Q, name, pages, nb_k_head=2048, nb_v_head=2048) == EUNSUPPORTED, pages
    for kw in (dict(pages=None), dict(type=12), dict(n_tokens=-1), dict(n_tokens=3), dict(n_requests=-1), dict(n_q=-1), dict(n_q=2), dict(q_start=FAKE + 2),
               dict(len=None), dict(len=FAKE + 1), dict(max_len=-1), dict(max_len=65), dict(k=FAKE + 2), dict(nb_v_head=508), dict(nb_k_token=4098)):
        assert kv8_rows(Q, name, **kw) == EINVAL, kw
    big = dict(page_size=1 << 30, table_len=4)
    assert kv8_rows(Q, name, big, max_len=(1 << 30) + 1) == EUNSUPPORTED
    assert kv8_rows(Q, name, n_tokens=5, n_requests=1 << 16, n_q=1 << 16, q_start=FAKE) == EUNSUPPORTED
    assert kv8_rows(Q, name, n_tokens=0, n_requests=0, len=None, k=None, v=None) == OK
    assert kv8_rows(Q, name, n_tokens=0, n_q=0) == OK
    assert getattr(Q.lib(), name)(None, None) == EINVAL


def test_kv8_store_needs_both(Q):
    assert kv8_rows(Q, "q4k_kv8_store", k=None) == EINVAL and kv8_rows(Q, "q4k_kv8_store", v=None) == EINVAL
    assert kv8_rows(Q, "q4k_kv8_load", k=None, v=None) == OK


def test_kv8_binding_refuses_host_memory(Q):
    k = torch.zeros(2, 16, 2, 64, dtype=torch.int8)
    with pytest.raises(ValueError):
        Q.KV8Pages(k, k, torch.zeros(2, 1, 2), torch.zeros(2, 1, 2))


def kv8_attn(Q, pages={}, **kw):
    d = dict(pages=ctypes.pointer(kv8(Q, **pages)) if pages is not None else None, q_type=0, n_head=32, scale=1.0, n_tokens=2, n_requests=2, n_q=1,
             q_start=None, len=FAKE, max_len=64, q=FAKE, nb_q_token=16384, nb_q_head=512, dst=FAKE, nb_dst_token=16384, nb_dst_head=512, lse=None)
    d.update(kw)
    a = Q.q4k_kv8_attn_args(*d.values())
    return Q.lib().q4k_kv8_attn(ctypes.byref(a), None, 0, None), Q.lib().q4k_kv8_attn_workspace_bytes(ctypes.byref(a))


def test_kv8_attn_checks(Q):
    for pages in PAGES_INVALID:
        assert kv8_attn(Q, pages) == (EINVAL, 0), pages
    for pages in PAGES_UNSUPPORTED:
        assert kv8_attn(Q, pages, nb_q_head=2048, nb_dst_head=2048) == (EUNSUPPORTED, 0), pages
    for kw in (dict(pages=None), dict(q_type=24), dict(q_type=12), dict(n_head=0), dict(n_head=33), dict(n_tokens=-1), dict(n_tokens=3), dict(n_requests=-1),
               dict(n_q=-1), dict(q_start=FAKE + 2), dict(len=None), dict(len=FAKE + 2), dict(max_len=-1), dict(max_len=65), dict(q=None), dict(dst=None),
               dict(q=FAKE + 2), dict(dst=FAKE + 1), dict(lse=FAKE + 2), dict(nb_q_token=16386), dict(nb_q_head=508), dict(nb_dst_head=508)):
        assert kv8_attn(Q, **kw) == (EINVAL, 0), kw
    assert kv8_attn(Q, dict(page_size=1 << 30), max_len=(1 << 30) + 1) == (EUNSUPPORTED, 0)
    assert kv8_attn(Q, n_tokens=0, n_requests=0, q=None, dst=None, len=None)[0] == OK
    assert kv8_attn(Q, n_tokens=0, n_q=0)[0] == OK
    assert Q.lib().q4k_kv8_attn(None, None, 0, None) == EINVAL and Q.lib().q4k_kv8_attn_workspace_bytes(None) == 0


def sample(Q, src=FAKE, V=100, N=2, nb=400, tokens=FAKE, logprob=None, **kw):
    r = Q.q4k_sample_rules()
    for k, v in kw.items():
        setattr(r, k, v)
    return Q.lib().q4k_sample(src, V, N, nb, ctypes.byref(r), tokens, logprob, None, 0, None)


@pytest.mark.parametrize("kw", [
    dict(V=-1), dict(N=-1), dict(src=None), dict(tokens=None), dict(src=FAKE + 2), dict(tokens=FAKE + 2), dict(logprob=FAKE + 1), dict(nb=396), dict(nb=402),
    dict(V=1 << 33), dict(N=1 << 33), dict(temperature=FAKE + 2), dict(top_k=FAKE + 1), dict(top_p=FAKE + 3), dict(min_p=FAKE + 2), dict(uniform=FAKE + 2)])
def test_sample_checks(Q, kw):
    assert sample(Q, **kw) == EINVAL


def test_sample_empty_unsupported_and_binding(Q):
    assert sample(Q, N=0, src=None, tokens=None) == OK
    assert sample(Q, V=(1 << 30) + 4, N=1) == EUNSUPPORTED
    assert Q.lib().q4k_sample(FAKE, 100, 2, 400, None, FAKE, None, None, 0, None) == EINVAL
    size = Q.lib().q4k_sample_workspace_bytes
    assert size(-1, 4) == 0 and size(4, -1) == 0 and size(1 << 40, 4) == 0
    for V in (1000, 32768, 151936, 1 << 30):
        sizes = [size(V, n) for n in [*range(1, 600), 4096]]
        assert sizes == sorted(sizes)
    with pytest.raises(ValueError):
        Q.sample(torch.zeros(2, 100), torch.zeros(2))
