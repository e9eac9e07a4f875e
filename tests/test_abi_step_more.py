"""More argument checks of the operators of a decode step that need no GPU."""
import pytest

from test_abi_step import EINVAL, EUNSUPPORTED, kv8_rows

#: strides by which rows or scales of the cache would lie on each other
OVERLAPPING = [dict(nb_k_head=0), dict(nb_k_head=112), dict(nb_v_token=0), dict(nb_v_token=-112), dict(nb_k_page=64), dict(nb_s_head=0), dict(nb_s_page=0),
               dict(nb_s_block=0, block=8), dict(nb_v_page=0), dict(nb_k_token=16)]


@pytest.mark.parametrize("pages", OVERLAPPING)
def test_kv8_store_refuses_overlapping_pages(Q, pages):
    assert kv8_rows(Q, "q4k_kv8_store", pages) == EINVAL


@pytest.mark.parametrize("pages", OVERLAPPING + [dict(nb_k_head=-128), dict(nb_k_page=-16384, nb_s_page=-32)])
def test_kv8_load_takes_them(Q, pages):
    assert kv8_rows(Q, "q4k_kv8_load", dict(pages, head_dim=pages.get("head_dim", 120))) == EUNSUPPORTED  # (as far as the checks go without a device)


@pytest.mark.parametrize("pages", [dict(nb_s_block=0), dict(n_pages=1, table_len=1, page_size=64, nb_k_page=0, nb_v_page=0, nb_s_page=0, nb_s_block=32),
                                   dict(n_head_kv=1, nb_k_head=0, nb_v_head=0, nb_s_head=0), dict(nb_k_token=-1024, nb_k_head=-128)])
def test_kv8_store_takes_strides_of_one_and_below_zero(Q, pages):
    # (what the check lets through ends at the missing device)
    import torch
    if torch.cuda.is_available():
        pytest.skip("addresses that are none")
    assert kv8_rows(Q, "q4k_kv8_store", pages) not in (EINVAL,)
