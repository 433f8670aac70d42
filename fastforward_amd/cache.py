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
import functools

import torch

from ._lib import call, entry, stream
from .linear import check_here

BF16, E4M3, I32 = torch.bfloat16, torch.float8_e4m3fn, torch.int32
_ROWS = 1 << 24


@functools.lru_cache(maxsize=1024)
def attend_workspace(heads, kv_heads, head_dim, fp8, page_size, width, batch, t):
    """Bytes of workspace ff_attention_paged needs (0: none)."""
    need = ctypes.c_int64(0)
    call("ff_attention_paged_workspace", heads, kv_heads, head_dim, fp8, page_size, width, batch, t, ctypes.byref(need))
    return need.value


class PagedCache:
    """Keys and values of one layer: ``k``, ``v`` (pages, kv_heads, page_size, head_dim), bf16
    or, ``dtype=torch.float8_e4m3fn``, e4m3 codes with ``k_scale``, ``v_scale`` (pages,
    kv_heads, page_size) uint8, the biased exponent of a token's scale in each head:
    value = code * 2^(byte - 127). ``head_dim`` is 64 or 128, ``page_size`` a power of
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
        self.k, self.v = (torch.zeros(shape, device=device, dtype=torch.uint8 if dtype == E4M3 else BF16).view(dtype)
                          for _ in range(2))
        self.k_scale = self.v_scale = None
        if dtype == E4M3:
            self.k_scale, self.v_scale = (torch.zeros(shape[:3], device=device, dtype=torch.uint8) for _ in range(2))

    def _held(self):
        """The pages as the C entry points take them."""
        ks = vs = 0
        if self.k_scale is not None:
            ks, vs = self.k_scale.data_ptr(), self.v_scale.data_ptr()
        return (self.k.data_ptr(), self.v.data_ptr(), ks, vs, self.pages, self.page_size)

    def _rows(self, t, table, lengths, starts):
        assert table.dim() == 2 and table.dtype == I32 and table.is_contiguous() and table.shape[1] > 0, table.shape
        batch, width = table.shape
        assert 0 < batch <= 65536 and width * self.page_size < 1 << 31 and t <= _ROWS, (batch, width, t)
        assert lengths.shape == (batch,) and lengths.dtype == I32 and lengths.is_contiguous(), lengths.shape
        if starts is None:
            assert t == batch, f"{t} rows for {batch} sequences of one row: starts is missing"
            check_here(self.k, table, lengths)
            return (table.data_ptr(), width, lengths.data_ptr(), 0, batch)
        assert starts.shape == (batch + 1,) and starts.dtype == I32 and starts.is_contiguous(), starts.shape
        check_here(self.k, table, lengths, starts)
        return (table.data_ptr(), width, lengths.data_ptr(), starts.data_ptr(), batch)

    def write(self, k, v, table, lengths, starts=None):
        """Put k, v (T, kv_heads, head_dim) bf16 (any strides) at their sequences' last
        positions. bf16 pages keep the values; FP8 pages e4m3(x / 2^e), 2^e the smallest power of two, e in
        [-100, 120], for which the largest finite magnitude of the token's row in its head
        is at most 448 * 2^e. NaN and infinities become NaN and leave the rest
        of their row as it is. Rows behind the last sequence are not written. The positions of
        one call are different ones: where two rows name one place, either may end there."""
        shape = (k.shape[0], self.kv_heads, self.head_dim)
        assert k.shape == v.shape == shape and k.dtype == v.dtype == BF16, (k.shape, v.shape, k.dtype, v.dtype)
        rows = self._rows(shape[0], table, lengths, starts)
        check_here(k, v)
        if k.stride(2) != 1:
            k = k.contiguous()
        if v.stride(2) != 1:
            v = v.contiguous()
        entry("ff_cache_write")(k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1),
                                *self._held(), self.kv_heads, self.head_dim, self.dtype == E4M3, *rows, shape[0],
                                stream())

    def read(self, table, lengths, starts=None, rows=None):
        """(k, v), each (rows, kv_heads, head_dim) bf16, of the sequences' last positions; an FP8
        cache's values are exact in bf16. ``rows`` (default: one per sequence) is T, a host
        number. Rows behind the last sequence, and positions that hold nothing, are zero."""
        t = table.shape[0] if rows is None else rows
        assert t >= 0 and (rows is None) <= (starts is None), "rows is missing"
        args = self._rows(t, table, lengths, starts)
        k = torch.empty((t, self.kv_heads, self.head_dim), device=table.device, dtype=BF16)
        v = torch.empty_like(k)
        entry("ff_cache_read")(*self._held(), self.kv_heads, self.head_dim, self.dtype == E4M3, *args, k.data_ptr(),
                               v.data_ptr(), t, stream())
        return k, v

    def attend(self, q, table, lengths, starts=None, scale=None):
        """Causal attention of q (T, heads, head_dim) bf16, any strides, heads a multiple of
        kv_heads: row i of a sequence's n rows has position length - n + i and sees the positions up to its
        own (written before, its own among them). Softmax of q . k * ``scale`` (default
        1 / sqrt(head_dim)) with fp32 statistics, weights rounded to bf16 for the product
        with the values, fp32 sums. (T, heads, head_dim) bf16. A row that sees nothing, and
        rows behind the last sequence, are zero."""
        assert q.dim() == 3 and q.dtype == BF16 and q.shape[2] == self.head_dim, (q.shape, q.dtype)
        t, heads, d = q.shape
        hk = self.kv_heads
        assert heads > 0 and heads % hk == 0 and heads <= 65535, (heads, hk)
        scale = d ** -0.5 if scale is None else float(scale)
        assert 0 < scale < float("inf"), scale
        rows = self._rows(t, table, lengths, starts)
        check_here(q)
        if q.stride(2) != 1:
            q = q.contiguous()
        y = q.new_empty((t, heads, d))
        need = attend_workspace(heads, hk, d, self.dtype == E4M3, self.page_size, rows[1], rows[4], t)
        ws = q.new_empty((need,), dtype=torch.uint8) if need else None
        entry("ff_attention_paged")(q.data_ptr(), q.stride(0), q.stride(1), *self._held(), heads, hk, d,
                                    self.dtype == E4M3, *rows, y.data_ptr(), t, scale, 0 if ws is None else ws.data_ptr(),
                                    need, stream())
        return y


__all__ = ["PagedCache", "attend_workspace"]
