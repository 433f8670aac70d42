"""Paged key/value cache and the attention that reads it, on gfx950 kernels.

No reference counterpart (its step runs a prompt once and keeps nothing): a prompt that
is kept and continued, by a question after a cached image or token by token.
``PagedCache`` holds one layer's keys and values in pages that a table hands to
sequences; ``write`` puts new tokens there, ``attend`` is the causal attention of those
tokens over their sequences (beside ``ops.attention_direct``, which has no cache), ``read``
gives contiguous rows back.

The calls share their arguments: ``table`` (B, W) int32, position p of sequence b lying in
page ``table[b, p // page_size]``; ``lengths`` (B,) int32, the sequences' positions with
the call's tokens; ``starts`` (B + 1,) int32, rising from 0 to at most T: sequence b has
rows ``starts[b] .. starts[b + 1] - 1`` of the T rows, its LAST positions. Without
``starts`` every sequence has one row (T = B), as in a decode step. The three live on the
GPU, are read by the kernels alone and may change between replays of a captured graph.

Like the other ops: shape, dtype and device violations raise AssertionError before any
launch, outputs are fresh tensors, launches go to the current stream and can be captured
(no host sync, no device-dependent grid).
"""
import ctypes

import torch

from ._lib import PagedCacheStruct, call, entry, planned, stream

BF16, E4M3, I32 = torch.bfloat16, torch.float8_e4m3fn, torch.int32
_ROWS, _POSITIONS = 1 << 24, (1 << 31) - (1 << 16)


@planned
def attend_workspace(page_size, kv_heads, head_dim, fp8, t, heads, width, batch, starts):
    """Bytes of workspace ff_attention_paged needs (0: none) for a table (batch, width) and, where
    ``starts`` is true, rows by starts."""
    need = ctypes.c_int64(0)
    sizes = PagedCacheStruct(0, 0, 0, 0, 1, page_size, kv_heads, head_dim, fp8)
    call("ff_attention_paged_workspace", ctypes.byref(sizes), heads, width, batch, starts, t, ctypes.byref(need))
    return need.value


class PagedCache:
    """Keys and values of one layer: ``k``, ``v`` (pages, kv_heads, page_size, head_dim), bf16
    or, ``dtype=torch.float8_e4m3fn``, e4m3 codes with ``k_scale``, ``v_scale`` (pages,
    kv_heads, page_size) uint8, the biased exponent of a token's scale in each head:
    value = code * 2^(byte - 127), NaN where the byte is 255. ``write`` makes bytes from 27 to 247; ``attend``
    may take values under smaller ones, below 2^-91 all of them, as zeros. ``head_dim`` is 64 or 128, ``page_size`` a power of
    two, 16 to 4096. Pages begin as zeros; which sequence a page belongs to is the
    caller's to say, and sequences may share the pages of a common prefix.

    A position past the table's reach, and one whose table entry is outside [0, pages),
    holds nothing: it is not written, reads as zeros and is not attended to."""

    def __init__(self, pages, page_size, kv_heads, head_dim, dtype=BF16, device=None):
        assert dtype in (BF16, E4M3), dtype
        assert head_dim in (64, 128), head_dim
        assert 16 <= page_size <= 4096 and page_size & (page_size - 1) == 0, page_size
        assert 0 < pages < 1 << 31 and 0 < kv_heads <= 65535, (pages, kv_heads)
        device = torch.device("cuda" if device is None else device)
        assert device.type == "cuda", device
        self.pages, self.page_size, self.kv_heads, self.head_dim, self.dtype = pages, page_size, kv_heads, head_dim, dtype
        shape = (pages, kv_heads, page_size, head_dim)
        k, v = (torch.zeros(shape, device=device, dtype=torch.uint8 if dtype == E4M3 else BF16).view(dtype) for _ in range(2))
        scales = (None, None)
        if dtype == E4M3:
            scales = tuple(torch.zeros(shape[:3], device=device, dtype=torch.uint8) for _ in range(2))
        self._hold(k, v, *scales)

    def _hold(self, k, v, k_scale, v_scale):
        self._tensors = (k, v, k_scale, v_scale)
        self._device = k.get_device()
        self._struct = PagedCacheStruct(*(0 if x is None else x.data_ptr() for x in self._tensors), self.pages,
                                        self.page_size, self.kv_heads, self.head_dim, k_scale is not None)
        self._c = ctypes.addressof(self._struct)
        self._sizes = (self.page_size, self.kv_heads, self.head_dim, k_scale is not None)

    # the pages are filled in place; the tensors stay the same
    k = property(lambda self: self._tensors[0])
    v = property(lambda self: self._tensors[1])
    k_scale = property(lambda self: self._tensors[2])
    v_scale = property(lambda self: self._tensors[3])

    def _rows(self, t, table, lengths, starts, *rows):
        """Checks what the calls share (and that ``rows`` are on the cache's device, the current
        one); the arguments as the C entry points take them."""
        assert table.dim() == 2 and table.dtype == I32 and table.is_contiguous(), (table.shape, table.dtype)
        batch, width = table.shape
        assert 0 < batch <= 65536 and 0 < width and width * self.page_size <= _POSITIONS and t <= _ROWS, (batch, width, t)
        assert lengths.shape == (batch,) and lengths.dtype == I32 and lengths.is_contiguous(), lengths.shape
        if starts is None:
            assert t == batch, f"{t} rows for {batch} sequences of one row: starts is missing"
            rows += (table, lengths)
            first = 0
        else:
            assert starts.shape == (batch + 1,) and starts.dtype == I32 and starts.is_contiguous(), starts.shape
            rows += (table, lengths, starts)
            first = starts.data_ptr()
        here = self._device
        for x in rows:
            assert x.get_device() == here >= 0, f"tensor on {x.device}, the cache on {self.k.device}"
        assert torch._C._cuda_getDevice() == here, f"the cache is on GPU {here}, which is not the current one"
        return table.data_ptr(), width, lengths.data_ptr(), first, batch

    def write(self, k, v, table, lengths, starts=None):
        """Put k, v (T, kv_heads, head_dim) bf16 (any strides) at their sequences' last
        positions. bf16 pages keep the values; FP8 pages e4m3(x / 2^e), 2^e the smallest power of two, e in
        [-100, 120], for which the largest finite magnitude of the token's row in its head is
        at most 448 * 2^e (and nothing past 240 * 2^120, which bf16 does not hold). NaN and
        infinities become NaN and leave the rest of their row as it is. Rows behind the last sequence
        are not written. The rows of one call have different places: where two name the same one (sequences
        that share the page of a position that both write), what ends there may be pieces of both, and a
        code under the other row's scale."""
        assert k.dim() == 3 and k.shape == v.shape and k.dtype == v.dtype == BF16, (k.shape, v.shape, k.dtype, v.dtype)
        t, hk, d = k.shape
        assert hk == self.kv_heads and d == self.head_dim, (k.shape, self.kv_heads, self.head_dim)
        rows = self._rows(t, table, lengths, starts, k, v)
        ks, vs = k.stride(), v.stride()
        if ks[2] != 1:
            k = k.contiguous()
            ks = k.stride()
        if vs[2] != 1:
            v = v.contiguous()
            vs = v.stride()
        entry("ff_cache_write")(k.data_ptr(), ks[0], ks[1], v.data_ptr(), vs[0], vs[1], self._c, *rows, t, stream())

    def read(self, table, lengths, starts=None, rows=None):
        """(k, v), each (rows, kv_heads, head_dim) bf16, of the sequences' last positions; an FP8
        cache's values are exact in bf16. ``rows`` (default: one per sequence) is T, a host
        number. Rows behind the last sequence, and positions that hold nothing, are zero."""
        t = table.shape[0] if rows is None else rows
        assert t >= 0 and (rows is not None or starts is None), "rows is missing"
        args = self._rows(t, table, lengths, starts)
        k = table.new_empty(t, self.kv_heads, self.head_dim, dtype=BF16)
        v = torch.empty_like(k)
        entry("ff_cache_read")(self._c, *args, k.data_ptr(), v.data_ptr(), t, stream())
        return k, v

    def attend_workspace(self, t, heads, width, batch, starts):
        """Bytes of workspace that a call of ``attend`` takes (0: none)."""
        return attend_workspace(*self._sizes, t, heads, width, batch, bool(starts))

    def attend(self, q, table, lengths, starts=None, scale=None):
        """Causal attention of q (T, heads, head_dim) bf16, any strides, heads a multiple of
        kv_heads: row i of a sequence's n rows has position length - n + i and sees the positions up to its
        own (written before, its own among them). Softmax of q . k * ``scale`` (default
        1 / sqrt(head_dim)) with fp32 statistics, weights rounded to bf16 for the product
        with the values, fp32 sums. (T, heads, head_dim) bf16. A row that sees nothing, and
        rows behind the last sequence, are zero; a NaN in a row's query or in a key that it
        sees makes it NaN. Scores are up to 2^30 in size (past it they may become NaN), and
        a row's largest value times the positions that it sees up to 2^127 (past it the sums may become
        infinite); an infinite value that a row sees makes it infinite or NaN."""
        assert q.dim() == 3 and q.dtype == BF16, (q.shape, q.dtype)
        t, heads, d = q.shape
        assert d == self.head_dim and 0 < heads <= 65535 and heads % self.kv_heads == 0, (q.shape, self.kv_heads)
        scale = d ** -0.5 if scale is None else float(scale)
        assert 0 < scale < float("inf"), scale
        rows = self._rows(t, table, lengths, starts, q)
        qs = q.stride()
        if qs[2] != 1:
            q = q.contiguous()
            qs = q.stride()
        y = q.new_empty(t, heads, d)
        need = attend_workspace(*self._sizes, t, heads, rows[1], rows[4], starts is not None)
        ws = q.new_empty(need, dtype=torch.uint8) if need else None
        entry("ff_attention_paged")(q.data_ptr(), qs[0], qs[1], self._c, heads, *rows, y.data_ptr(), t, scale,
                                    0 if ws is None else ws.data_ptr(), need, stream())
        return y


__all__ = ["PagedCache", "attend_workspace"]
