"""What a call of the paged attention takes, by its sizes: host code, no GPU."""
import ctypes
import gc

import pytest

from fastforward_amd import _lib
from fastforward_amd import cache as C


def _cache(page_size=64, kv_heads=8, head_dim=128):
    """A cache object without pages, for its plans."""
    import torch
    c = C.PagedCache.__new__(C.PagedCache)
    c.pages, c.page_size, c.kv_heads, c.head_dim, c.dtype = 1, page_size, kv_heads, head_dim, torch.bfloat16
    c._hold(torch.empty(0), torch.empty(0), None, None)
    return c


def _asked(page_size, kv_heads, head_dim, fp8, t, heads, width, batch, starts):
    need = ctypes.c_int64(-1)
    sizes = _lib.PagedCacheStruct(0, 0, 0, 0, 1, page_size, kv_heads, head_dim, fp8)
    _lib.call("ff_attention_paged_workspace", ctypes.byref(sizes), heads, width, batch, starts, t, ctypes.byref(need))
    return need.value


def test_sizes_are_not_kept_without_bound():
    """A serving process sees ever new sizes: nothing of the cache grows with them."""
    c = _cache()
    for t in range(1, 3000):
        assert c.attend_workspace(t, 32, 64, 1, True) >= 0

    def entries(x):
        return sum(len(v) for v in vars(x).values() if isinstance(v, (dict, list, set)))
    gc.collect()
    assert entries(c) == 0 and C.attend_workspace.cache_info().currsize <= 1024


def test_tile_choice_is_followed():
    """A tile choice that is set after a size was asked for holds for the next call of that size."""
    args = (64, 8, 128, False, 200, 32, 64, 1, True)
    first = C.attend_workspace(*args)
    try:
        seen = set()
        for tile in (1, 2, 3):
            _lib.call("ff_set_tuning", 14, tile)
            assert C.attend_workspace(*args) == _asked(*args)
            seen.add(C.attend_workspace(*args))
        assert len(seen) == 3
    finally:
        _lib.call("ff_set_tuning", 14, 0)
    assert C.attend_workspace(*args) == first == _asked(*args)


def test_launches_past_their_limit_are_refused():
    """131073 tiles for each of 128 key heads are 2^32 threads, which no launch has."""
    sizes = (16, 128, 64, False)
    assert C.attend_workspace(*sizes, 1 << 20, 128, 1, 65000, True) >= 0
    with pytest.raises(RuntimeError, match="too large"):
        C.attend_workspace(*sizes, 1 << 20, 128, 1, 65536, True)
    rows = C.attend_workspace(*sizes, 65536, 128, 1, 65536, False)      # a decode step of as many sequences
    assert rows >= 0


def test_workspace_of_many_sequences():
    """Only split tiles leave partial sums, and they are about as many as workgroups, however many
    sequences there are: what grows with them is a note of 8 bytes a row and head, and the list."""
    for t in (64, 1024, 4096, 65536):
        for fp8 in (False, True):
            need = C.attend_workspace(64, 8, 128, fp8, t, 32, 128, t, False)
            assert 0 < need <= (40 << 20) + t * (32 * 8 + 8), (t, need)


def test_one_long_sequence_among_many():
    """A decode step's rows are split over keys where the table reaches far, whether starts say which rows
    are whose or not."""
    for t in (100, 1024, 4096):
        for width in (65, 1024):
            plain = C.attend_workspace(64, 8, 128, False, t, 32, width, t, False)
            assert C.attend_workspace(64, 8, 128, False, t, 32, width, t, True) >= plain > 4 << 20
