// Pieces shared by the paged cache's kernels: where a sequence's positions lie, which
// sequence a row belongs to, and the attention's work list.
//
// A cache has `pages` pages of `ps` tokens (a power of two) of `hk` heads: k and v
// (pages, hk, ps, d), bf16 or e4m3 codes, and for codes a byte per (page, head, token):
// the biased exponent of the row's power-of-two scale, value = code * 2^(byte - 127).
// Position p of sequence b is slot p % ps of page table[b][p / ps]. A position that the
// table does not reach and an entry outside [0, pages) hold nothing: not written, read
// as zeros, not attended to.
#pragma once

#include "ff_common.h"

namespace ff {

// The rows of a call: sequence b has rows [starts[b], starts[b + 1]) of the t rows (one
// row each without starts), its last positions of lengths[b].
struct Rows {
  const int* table;
  const int* lengths;
  const int* starts;  // batch + 1, or null
  int64_t width;      // entries of a table row
  int batch, t, pages, lps;

  __device__ __forceinline__ int begin(int b) const { return !starts ? b : b ? min(max(starts[b], 0), t) : 0; }
  __device__ __forceinline__ int end(int b) const {
    return !starts ? b + 1 : b < batch ? min(max(starts[b + 1], 0), t) : t;
  }
  __device__ __forceinline__ int64_t capacity() const { return width << lps; }
};

// The largest index in [0, n) with at[index] <= x, by a wave; at rises, at[0] <= x. (Some index in [0, n) whatever
// it holds.)
__device__ __forceinline__ int last_upto(const int* at, int n, int x, int lane) {
  int lo = 0;
  while (n > 1) {
    const int step = (n + 63) >> 6, i = lane * step;
    const int c = max(__popcll(__ballot((i < n ? at[lo + i] : 0x7FFFFFFF) <= x)) - 1, 0);
    lo += c * step;
    n = min(step, n - c * step);
  }
  return __builtin_amdgcn_readfirstlane(lo);
}

// Sequences of the N rows row0 .. row0 + N - 1 (a wave's; uniform row0): of[i] = how many
// sequences end at or before row0 + i. batch where the row lies behind the last one.
template <int N>
__device__ __forceinline__ void find_sequences(const Rows& a, int row0, int lane, int (&of)[N]) {
  int b0 = a.starts && a.batch > 64 ? last_upto(a.starts, a.batch + 1, row0, lane) : 0;
#pragma unroll
  for (int i = 0; i < N; ++i) of[i] = a.starts ? b0 : row0 + i;
  if (!a.starts) return;
  for (; b0 < a.batch; b0 += 64) {
    const int end = b0 + lane < a.batch ? a.starts[b0 + lane + 1] : 0x7FFFFFFF;
#pragma unroll
    for (int i = 0; i < N; ++i) of[i] += __popcll(__ballot(end <= row0 + i));
    if (__ballot(end > row0 + N - 1)) break;
  }
}

// Page and slot of row `row` of sequence b; false where there is none.
__device__ __forceinline__ bool find_slot(const Rows& a, int row, int b, int64_t* page, int* slot) {
  if (row >= a.t || b >= a.batch) return false;
  const int64_t pos = (int64_t)a.lengths[b] - a.end(b) + row;
  if (pos < 0 || pos >= a.capacity()) return false;
  const int p = a.table[b * a.width + (pos >> a.lps)];
  *page = p;
  *slot = (int)(pos & ((1 << a.lps) - 1));
  return (unsigned)p < (unsigned)a.pages;
}

// Positions that a table may reach: those of the blocks behind the last one, too, are counted in 32 bits.
constexpr int64_t kMaxPositions = INT32_MAX - 65535;

// Host checks that the entry points share.
inline int check_cache(const char* what, const ff_paged_cache* c) {
  FF_REQUIRE(c, "%s: null pointer", what);
  FF_REQUIRE(c->d == 64 || c->d == 128, "%s: head_dim %lld unsupported (64, 128)", what, (long long)c->d);
  FF_REQUIRE(c->page_size >= 16 && c->page_size <= 4096 && (c->page_size & (c->page_size - 1)) == 0,
             "%s: page_size %lld (a power of two, 16 .. 4096)", what, (long long)c->page_size);
  FF_REQUIRE(c->pages > 0 && c->pages <= INT32_MAX && c->hk > 0 && c->hk <= 65535, "%s: bad sizes pages=%lld hk=%lld",
             what, (long long)c->pages, (long long)c->hk);
  return FF_OK;
}
inline int check_rows(const char* what, const ff_paged_cache* c, const int32_t* table, int64_t width,
                      const int32_t* lengths, const int32_t* starts, int64_t batch, int64_t t) {
  const int st = check_cache(what, c);
  if (st != FF_OK) return st;
  FF_REQUIRE(c->k && c->v && (!c->fp8 || (c->k_scale && c->v_scale)) && table && lengths, "%s: null pointer", what);
  FF_REQUIRE(width > 0 && width <= kMaxPositions / c->page_size && batch > 0 && batch <= 65536 && t > 0 && t <= (1 << 24),
             "%s: bad sizes width=%lld batch=%lld t=%lld", what, (long long)width, (long long)batch, (long long)t);
  FF_REQUIRE(starts || batch == t, "%s: without starts every sequence has one row", what);
  FF_REQUIRE(ff_aligned(c->k, 16) && ff_aligned(c->v, 16) && ff_aligned(c->k_scale, 8) && ff_aligned(c->v_scale, 8),
             "%s: alignment", what);
  return FF_OK;
}
inline Rows rows_of(const ff_paged_cache* c, const int32_t* table, int64_t width, const int32_t* lengths,
                    const int32_t* starts, int64_t batch, int64_t t) {
  return Rows{table, lengths, starts, width, (int)batch, (int)t, (int)c->pages, __builtin_ctzll((uint64_t)c->page_size)};
}

// The float of a scale byte (0 for byte 0, and for 255 an infinity, which is no number times any code).
__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }

}  // namespace ff
