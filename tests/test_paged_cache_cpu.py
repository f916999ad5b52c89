"""What ``PagedCache`` refuses, and the state it begins with."""

import pytest
import torch

SIZES = dict(layers=2, requests=3, pages=10, page_size=16, kv_heads=2, head_dim=128, device="cpu")


@pytest.mark.parametrize("over,says", [
    (dict(layers=0), "layers"), (dict(requests=0), "requests"), (dict(pages=0), "pages"), (dict(kv_heads=-1), "kv_heads"), (dict(width=0), "width"),
    (dict(page_size=8), "power of two"), (dict(page_size=24), "power of two"), (dict(head_dim=64), "head_dim"), (dict(requests=2049), "2048"),
])
def test_sizes_that_no_kernel_takes(over, says):
    from tybok_b200.paged import PagedCache

    with pytest.raises(ValueError, match=says):
        PagedCache(**{**SIZES, **over})


def test_a_new_cache_holds_nothing():
    from tybok_b200.paged import PagedCache

    cache = PagedCache(**SIZES, width=4)
    assert cache.k_pages.shape == cache.v_pages.shape == (2, 10, 2, 16, 128)
    assert cache.key_lens.tolist() == [0, 0, 0] and cache.block_table.shape == (3, 4)
    assert cache.free_count.tolist() == [10] and sorted(cache.free_pages.tolist()) == list(range(10))


def test_attend_needs_a_step_and_a_layer():
    from tybok_b200.paged import PagedCache

    cache = PagedCache(**SIZES)
    qkv, table = torch.zeros(4, 8 * 128, dtype=torch.bfloat16), torch.zeros(64, 64)
    with pytest.raises(RuntimeError, match="before the first step"):
        cache.attend(0, qkv, table, table, heads=4)
    with pytest.raises(NotImplementedError):  # the sizes agree; there is no such operator on a CPU
        cache.step(torch.ones(3, dtype=torch.int32), tokens=4)
    cache.plan = ()
    for layer in (-1, 2):
        with pytest.raises(IndexError, match="of 2"):
            cache.attend(layer, qkv, table, table, heads=4)
