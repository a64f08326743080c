"""The handles of serving: a cache's memory stays the memory that its calls go by."""
import gc

import pytest
import torch

FIELDS = ("k_codes", "k_scales", "v", "pages", "kv_heads", "page_size", "head_dim", "device", "struct")


@pytest.mark.parametrize("name", FIELDS)
def test_a_cache_is_read_only(fa, name):
    cache = fa.PagedCache.__new__(fa.PagedCache)
    with pytest.raises(AttributeError):
        setattr(cache, name, None)
    with pytest.raises(AttributeError):
        delattr(cache, name)


@pytest.mark.gpu
def test_a_cache_keeps_its_memory(fa, cuda):
    """Neither the caller's tensors nor their replacement take the memory away from the calls."""
    codes = torch.zeros(4, 1, 16, 32, dtype=torch.uint8, device="cuda")
    scales = torch.full((4, 1, 16, 2), 127, dtype=torch.uint8, device="cuda")
    v = torch.zeros(4, 1, 16, 64, dtype=torch.float16, device="cuda")
    cache = fa.PagedCache(codes, scales, v)
    at = [t.data_ptr() for t in (cache.k_codes, cache.k_scales, cache.v)]
    v.data = torch.ones_like(v)
    del codes, scales
    gc.collect()
    new = [torch.full((4, 1, 16, 64), 3.0, dtype=torch.float16, device="cuda") for _ in range(8)]
    assert not {t.data_ptr() for t in new} & set(at)
    x = torch.full((1, 1, 64), 2.0, dtype=torch.float16, device="cuda")
    page, first = torch.tensor([[2]], dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    fa.cache_append(cache, x, x, page, first)
    assert at == [t.data_ptr() for t in (cache.k_codes, cache.k_scales, cache.v)]
    assert bool((cache.v[2, 0, 0] == 2).all()) and bool((v == 1).all()) and all(bool((t == 3).all()) for t in new)
    assert bool((fa.paged_attention(x, cache, page, first + 1) == 2).all())
    assert fa.status_query() == fa.OK


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(0, 32, 2), (8, 0, 2)])
def test_an_empty_rotary_table_is_not_none(fa, cuda, shape):
    """Keys are not stored unrotated where a table was asked for."""
    cache = fa.PagedCache.empty(2, 16, 1, 64)
    cache.v.zero_()
    x = torch.ones(1, 1, 64, dtype=torch.float16, device="cuda")
    page, first = torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="empty"):
        fa.cache_append(cache, x, x, page, first, Q=x, table=torch.empty(shape, device="cuda"))
    with pytest.raises((ValueError, fa.Fp4AttnError)):
        fa.rotary(x[None], torch.empty(shape, device="cuda"))
    assert not cache.v.any() and fa.status_query() == fa.OK


def test_page_numbers_are_integers(fa):
    """Of any integer type and as lists; fractions and truth values are not cut to page 0."""
    from fp4attn_b200 import paged
    for t in (torch.int8, torch.uint8, torch.int16, torch.int32, torch.int64):
        got = paged._page_numbers(torch.tensor([3, 0, 7], dtype=t), "src")
        assert got.dtype == torch.int32 and got.tolist() == [3, 0, 7]
    assert paged._page_numbers([5, 1], "src").tolist() == [5, 1]
    assert paged._page_numbers(range(3), "src").tolist() == [0, 1, 2]
    assert paged._page_numbers([], "src").shape == (0,)
    for bad in ([0.7], [1.0, 2.0], [True], torch.tensor([0.0])):
        with pytest.raises(TypeError, match="src"):
            paged._page_numbers(bad, "src")
    for bad in ([2 ** 31], [2 ** 32], torch.tensor([-2 ** 31 - 1])):
        with pytest.raises(ValueError, match="src"):
            paged._page_numbers(bad, "src")


@pytest.mark.gpu
def test_block_tables_on_a_device_by_its_number(fa, cuda):
    pool = fa.PagePool(8, 16)
    seq = pool.new()
    pool.extend(seq, 20)
    for device in (0, "cuda", "cuda:0", torch.device("cuda", 0)):
        t = pool.block_table([seq], device=device)
        assert t.device == torch.device("cuda", 0) and t.tolist() == [pool.table(seq)]
    assert pool.block_table([seq]).device.type == "cpu"
