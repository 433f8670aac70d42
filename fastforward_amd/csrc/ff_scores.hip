// Log probabilities of given tokens, entropy and the most likely tokens of rows of
// logits, in one pass over them.
//
// A wave sums relative to a reference c that is one of its logits: over all the others,
// r = sum e^(x - c) and t = sum (x - c) e^(x - c), so that a row's are
//   log p(x) = (x - c) - log1p(r),   entropy = log1p(r) - t / (1 + r).
// c moves to the largest logit where that passes it by 4 ln 2. A token that is all but
// certain is then the reference, the 1 is never added, and what is left of the
// probability keeps its relative precision in 32 bits; a token above c by less
// has a probability of 16 / 17 at most, where there is nothing to lose. Exponents are of base
// 2 until the end.
//
// The most likely tokens: a wave's best 64 so far lie sorted in its lanes, as 64-bit keys of
// (value, lowest index first). A vector of logits is looked at only where one of
// them is above the wave's k-th best, or c's limit: one comparison with the smaller of the
// two. After a look the waves of a row share what bounds the row's k-th best from below, so that
// a wave skips what others have beaten (64 alternatives of 577 rows of 151936 149 -> 115 us, 20 of 512
// fp32 rows 73 -> 66, 5 of 577 60 -> 56; with the best of the waves' own k-th bests 137, 71, 57).
// The lists of waves, then of a row's parts, are joined by sorts over the lanes.
//
// Bound by the logits' bytes, beside ten instructions a logit: a row is read once, 16 bytes a lane
// and load, two loads ahead. 577 rows of 151936 in bf16 39 us (4.5 TB/s), with 5 alternatives 46. Few
// rows are split over workgroups, and a second launch joins their parts (one row 10 and 5 us).
#include "ff_common.h"

using namespace ff;

namespace {

constexpr int kWaves = 8, kThreads = 64 * kWaves;
constexpr int kMaxTop = 64;
// Lists past this length are joined list after list by four waves, shorter ones by two sorts (one row's 64
// parts, the whole call: 20 keys 16 us against 19 list after list, 32 keys 18.5 against 21.5; of 64 keys all
// but the first sort would overflow: 34 us, and 49 by taking the best head 64 times).
constexpr int kLongTop = 32;
// Up to so many alternatives a workgroup begins with the bound that the maxima of its 32 rows of 16 lanes
// give, longer lists with a sort of each wave's lanes (us, maxima and sort, rows of 151936: 577 rows of 20 keys 60 and 65, 64 rows
// of 28 28.5 and 33.6, of 32 36 and 36; one row of 28 16.9 and 17.7, of 32 21.4 and 18.9).
constexpr int kSeedTop = 28;
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;

struct Args {
  const void* x;
  int64_t ld;
  const int64_t* tokens;
  int64_t tok_ts, tok_ns;
  float *logprobs, *entropy, *top_logprobs;
  int* top_ids;
  float* part;          // (rows, parts, 4): c, r, t
  uint64_t* part_keys;  // (rows, parts, top)
  int64_t v;
  int t, n, top, parts;
};

// Keys in the order of (value, lowest index first); 0 is below every value's. NaN is above
// every value, -0 equals 0.
__device__ __forceinline__ uint64_t key_of(float x, uint32_t index) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  const uint32_t k = x != x ? 0xFFFFFFFFu : u >> 31 ? ~u : u | 0x80000000u;
  return (uint64_t)k << 32 | (uint32_t)~index;
}
__device__ __forceinline__ float value_of(uint64_t key) {
  const uint32_t k = (uint32_t)(key >> 32);
  return k == 0xFFFFFFFFu ? __builtin_nanf("") : __uint_as_float(k >> 31 ? k & 0x7FFFFFFFu : ~k);
}

// A row's statistics, or a part's: the reference (-inf: no logit yet), r and t (in base 2).
struct Stats {
  float m, r, t;
};

// What s adds, its reference too, relative to one that is `down` above (in base 2; -inf or so far that
// nothing is left: 0, or NaN where there is one).
__device__ __forceinline__ Stats lowered(const Stats& s, float down) {
  const float e = __builtin_amdgcn_exp2f(down);
  if (!(e > 0.f)) return Stats{s.m, s.r * 0.f, s.t * 0.f};
  return Stats{s.m, e * (1.f + s.r), e * (s.t + down * (1.f + s.r))};
}

// The statistics of all lanes joined: everything relative to the largest reference. (A lane without one
// has r 0, or NaN where it saw one.)
__device__ __forceinline__ Stats joined(Stats s, int lane) {
  const float high = wave_max(s.m);
  const bool first = __builtin_ctzll(__ballot(s.m == high) | 1ull << 63) == lane;
  if (!first && s.m != -INFINITY) s = lowered(s, (s.m - high) * kLog2e);
  return Stats{high, wave_sum(s.r), wave_sum(s.t)};
}

template <int CTRL>
__device__ __forceinline__ uint64_t dpp64(uint64_t v) {
  return (uint64_t)(uint32_t)__builtin_amdgcn_update_dpp((int)(v >> 32), (int)(v >> 32), CTRL, 0xF, 0xF, false) << 32 |
         (uint32_t)__builtin_amdgcn_update_dpp((int)(uint32_t)v, (int)(uint32_t)v, CTRL, 0xF, 0xF, false);
}
__device__ __forceinline__ uint64_t read_lane(uint64_t v, int lane) {
  return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32 |
         (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, lane);
}
__device__ __forceinline__ uint64_t larger(uint64_t a, uint64_t b) { return a > b ? a : b; }

// Puts the uniform key into the wave's falling list (one entry a lane).
__device__ __forceinline__ void insert(uint64_t& list, uint64_t key) {
  // the lane before (wave_shr:1); lane 0 has none, and gets a key above all
  const uint64_t up = (uint64_t)(uint32_t)__builtin_amdgcn_update_dpp(-1, (int)(list >> 32), 0x138, 0xF, 0xF, false) << 32 |
                      (uint32_t)__builtin_amdgcn_update_dpp(-1, (int)(uint32_t)list, 0x138, 0xF, 0xF, false);
  list = key <= list ? list : key > up ? up : key;
}

// A given token's logit; `there` is false where it is none.
struct Token {
  float x;
  bool there;
};
template <typename T>
__device__ __forceinline__ Token token_at(const Args& p, int row, int i) {
  const int64_t id = i < p.n ? p.tokens[row * p.tok_ts + i * p.tok_ns] : -1;
  if (id < 0 || id >= p.v) return Token{0.f, false};
  const T* x = (const T*)p.x + row * p.ld + id;
  return Token{sizeof(T) == 2 ? bf16_to_f32(*(const bf16_t*)x) : *(const float*)x, true};
}

// log p of a logit, and the row's entropy.
struct Answer {
  float m, l, entropy;
  bool odd, none;  // the row holds a NaN or +inf; every token is switched off
  __device__ __forceinline__ explicit Answer(const Stats& s)
      : m(s.m), l(log1pf(s.r)), odd(s.r != s.r || s.t != s.t || s.m == INFINITY), none(s.m == -INFINITY) {
    entropy = odd ? __builtin_nanf("") : none ? 0.f : l - kLn2 * s.t / (1.f + s.r);
  }
  __device__ __forceinline__ float operator()(float x) const {
    return odd ? __builtin_nanf("") : none ? -INFINITY : (x - m) - l;
  }
};

// Writes a row's results, by a whole wave each; `first` is token_at(lane), loaded before.
template <typename T>
__device__ __forceinline__ void finish_tokens(const Args& p, int row, const Stats& s, Token first, int lane) {
  const Answer lp(s);
  for (int i = lane; i < p.n; i += 64) {
    const Token k = i == lane ? first : token_at<T>(p, row, i);
    p.logprobs[(int64_t)row * p.n + i] = k.there ? lp(k.x) : 0.f;
  }
  if (lane == 0) p.entropy[row] = lp.entropy;
}
__device__ __forceinline__ void finish_top(const Args& p, int row, const Stats& s, uint64_t list, int lane) {
  if (lane >= p.top) return;
  p.top_logprobs[(int64_t)row * p.top + lane] = Answer(s)(value_of(list));
  p.top_ids[(int64_t)row * p.top + lane] = (int)~(uint32_t)list;
}

// One step of a bitonic network over the wave: the lanes whose bit `bit` is clear keep the larger
// of their own key and `other`, the others the smaller.
__device__ __forceinline__ uint64_t keep(uint64_t mine, uint64_t other, int lane, int bit) {
  return (mine > other) == ((lane & bit) == 0) ? mine : other;
}
__device__ __forceinline__ uint64_t xor4(uint64_t v) { return dpp64<kDppQuadReverse>(dpp64<kDppHalfMirror>(v)); }
__device__ __forceinline__ uint64_t xor8(uint64_t v) { return dpp64<kDppRowRor8>(v); }
template <bool WIDE>
__device__ __forceinline__ uint64_t xor_rows(uint64_t v, int lane) {  // lane ^ 16, or ^ 32
  const uint32_t h = (uint32_t)(v >> 32), l = (uint32_t)v;
  const auto a = WIDE ? __builtin_amdgcn_permlane32_swap(h, h, false, false) : __builtin_amdgcn_permlane16_swap(h, h, false, false);
  const auto b = WIDE ? __builtin_amdgcn_permlane32_swap(l, l, false, false) : __builtin_amdgcn_permlane16_swap(l, l, false, false);
  const int k = lane & (WIDE ? 32 : 16) ? 0 : 1;
  return (uint64_t)a[k] << 32 | b[k];
}

// The lanes' keys in falling order.
__device__ __forceinline__ uint64_t sorted(uint64_t v, int lane) {
  v = keep(v, dpp64<kDppXor1>(v), lane, 1);
  v = keep(v, dpp64<kDppQuadReverse>(v), lane, 2);
  v = keep(v, dpp64<kDppXor1>(v), lane, 1);
  v = keep(v, dpp64<kDppHalfMirror>(v), lane, 4);
  v = keep(v, dpp64<kDppXor2>(v), lane, 2);
  v = keep(v, dpp64<kDppXor1>(v), lane, 1);
  v = keep(v, dpp64<kDppRowMirror>(v), lane, 8);
#pragma unroll
  for (int size = 16; size <= 64; size *= 2) {
    if (size == 32) v = keep(v, xor_rows<false>(dpp64<kDppRowMirror>(v), lane), lane, 16);
    if (size == 64) {
      v = keep(v, xor_rows<true>(xor_rows<false>(dpp64<kDppRowMirror>(v), lane), lane), lane, 32);
      v = keep(v, xor_rows<false>(v, lane), lane, 16);
    }
    if (size > 16) v = keep(v, xor8(v), lane, 8);
    v = keep(v, xor4(v), lane, 4);
    v = keep(v, dpp64<kDppXor2>(v), lane, 2);
    v = keep(v, dpp64<kDppXor1>(v), lane, 1);
  }
  return v;
}

// The same of 32-bit keys, for each half of the wave.
__device__ __forceinline__ uint32_t keep32(uint32_t mine, uint32_t other, int lane, int bit) {
  return lane & bit ? min(mine, other) : max(mine, other);
}
template <int CTRL>
__device__ __forceinline__ uint32_t dpp32(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, CTRL, 0xF, 0xF, false);
}
template <bool WIDE>
__device__ __forceinline__ uint32_t xor_rows32(uint32_t v, int lane) {
  const auto a = WIDE ? __builtin_amdgcn_permlane32_swap(v, v, false, false) : __builtin_amdgcn_permlane16_swap(v, v, false, false);
  return a[lane & (WIDE ? 32 : 16) ? 0 : 1];
}
__device__ __forceinline__ uint32_t sorted32(uint32_t v, int lane) {
  v = keep32(v, dpp32<kDppXor1>(v), lane, 1);
  v = keep32(v, dpp32<kDppQuadReverse>(v), lane, 2);
  v = keep32(v, dpp32<kDppXor1>(v), lane, 1);
  v = keep32(v, dpp32<kDppHalfMirror>(v), lane, 4);
  v = keep32(v, dpp32<kDppXor2>(v), lane, 2);
  v = keep32(v, dpp32<kDppXor1>(v), lane, 1);
  v = keep32(v, dpp32<kDppRowMirror>(v), lane, 8);
  v = keep32(v, dpp32<kDppQuadReverse>(dpp32<kDppHalfMirror>(v)), lane, 4);
  v = keep32(v, dpp32<kDppXor2>(v), lane, 2);
  v = keep32(v, dpp32<kDppXor1>(v), lane, 1);
  v = keep32(v, xor_rows32<false>(dpp32<kDppRowMirror>(v), lane), lane, 16);
  v = keep32(v, dpp32<kDppRowRor8>(v), lane, 8);
  v = keep32(v, dpp32<kDppQuadReverse>(dpp32<kDppHalfMirror>(v)), lane, 4);
  v = keep32(v, dpp32<kDppXor2>(v), lane, 2);
  v = keep32(v, dpp32<kDppXor1>(v), lane, 1);
  return v;
}

// The best 64 of a falling list and of keys in rising order: the larger of each two is a bitonic sequence.
__device__ __forceinline__ uint64_t merged(uint64_t falling, uint64_t rising, int lane) {
  uint64_t v = larger(falling, rising);
  v = keep(v, xor_rows<true>(v, lane), lane, 32);
  v = keep(v, xor_rows<false>(v, lane), lane, 16);
  v = keep(v, xor8(v), lane, 8);
  v = keep(v, xor4(v), lane, 4);
  v = keep(v, dpp64<kDppXor2>(v), lane, 2);
  return keep(v, dpp64<kDppXor1>(v), lane, 1);
}

// The best of the falling lists [from, to) of `top` keys at `keys` (LDS), by one wave: entry i in lane i.
__device__ __forceinline__ uint64_t best_merged(const uint64_t* keys, int from, int to, int top, int lane) {
  uint64_t v = 0;
  for (int i = from; i < to; ++i) {
    const uint64_t key = 63 - lane < top ? keys[i * top + 63 - lane] : 0;
    if (read_lane(key, 63) > read_lane(v, top - 1)) v = merged(v, key, lane);
  }
  return v;
}

// The best of up to LISTS (8 or 64) lists: their first keys, 64 in all, are sorted at once, and the others
// that beat the top-th of those (2 or 3 for 20 of 64 lists) are sorted in; list after list only where there
// are more than 64 of both. 64 lists of 20: the join of one row's parts 4.6 us against 7.3.
template <int LISTS>
__device__ __forceinline__ uint64_t best_of(const uint64_t* keys, int lists, int top, int lane, uint64_t* pool) {
  constexpr int M = 64 / LISTS;
  uint64_t v = sorted(lane / M < lists && lane % M < top ? keys[lane / M * top + lane % M] : 0, lane);
  if (top <= M) return v;
  const uint64_t least = read_lane(v, top - 1);
  auto entry = [&](int j) { return lane < lists && j < top ? keys[lane * top + j] : 0; };
  uint64_t key = entry(M), hits = __ballot(key > least);
  if (!hits) return v;
  int count = __popcll(__ballot(v != 0 && lane < top));
  if (lane < count) pool[lane] = v;
  for (int j = M + 1; hits; ++j) {
    if (count + __popcll(hits) > 64) return best_merged(keys, 0, lists, top, lane);
    if (key > least) pool[count + __popcll(hits & ((1ull << lane) - 1))] = key;
    count += __popcll(hits);
    key = entry(j);
    hits = __ballot(key > least);
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  return sorted(lane < count ? pool[lane] : 0, lane);
}

// A wave's pass over its logits. Exponents are y = fma(x, log2 e, -yc), yc = c log2 e rounded: one
// instruction, and all weights are relative to 2^yc. The reference's own weight is 2^off,
// off = fma(c, log2 e, -yc), by which the sums are divided at the end. Where |c| is past 2^22 (`huge`), off
// could be more than the exponential can take, and y = (x - c) log2 e.
template <int N>
struct Wave {
  float c = -INFINITY, limit = -INFINITY;  // the reference and where it moves; uniform
  float yc = 0.f, off = 0.f;
  bool huge = false;
  float r = 0.f, t = 0.f;                  // this lane's part of the sums, t of y e
  uint64_t list = 0, least = 0;            // the best keys; the k-th best (uniform)
  float kth = __builtin_nanf("");          // its logit (NaN: there are not k, or it is one)
  float bound = __builtin_nanf("");        // what makes a vector worth a look; NaN: every one is

  template <bool HUGE_C>
  __device__ __forceinline__ void add(float x, bool counts) {
    const float y = fmaxf(HUGE_C ? (x - c) * kLog2e : __builtin_fmaf(x, kLog2e, -yc), -1e6f);
    const float e = counts ? __builtin_amdgcn_exp2f(y) : 0.f;
    r += e;
    t = __builtin_fmaf(e, y, t);
  }

  // Whether N logits of every lane need a look.
  __device__ __forceinline__ bool hot(const float (&x)[N]) const {
    float m = x[0];
#pragma unroll
    for (int i = 1; i < N; ++i) m = __builtin_elementwise_maximum(m, x[i]);  // (NaN if there is one)
    return __ballot(!(m <= bound)) != 0;
  }
  __device__ __forceinline__ void add_all(const float (&x)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) add<false>(x[i], true);
  }

  // The wave's first logits, those of lane l at first + l N. Past the end lanes have -inf. `row`: upper half of
  // a key that at least `top` of the row's (or part's) reach, 0 if there is none.
  __device__ __forceinline__ void begin(const float (&x)[N], int64_t first, int64_t end, int top, int lane, uint32_t row) {
    refer(x, lane);
    if (top) {
      if (row > 0x00800000u && row < 0xFF800000u) {  // a finite one
        raise(row, 0);
        pick(x, first, end, top);
        kth = fmaxf(kth, value_of(least));
      } else {
        seed(x, first, end, top, lane);
        kth = value_of(least);
      }
    }
    set_bound(top);
  }

  // Later ones that need a look, all above the indices of earlier ones.
  __device__ __forceinline__ void look(const float (&x)[N], int64_t first, int64_t end, int top, int lane) {
    float m = x[0];
#pragma unroll
    for (int i = 1; i < N; ++i) m = __builtin_elementwise_maximum(m, x[i]);
    if (huge || __ballot(!(m <= limit))) refer(x, lane);
    else add_all(x);
    if (top) {
      if (__ballot(!(m <= kth))) pick(x, first, end, top);
      kth = fmaxf(kth, value_of(least));
    }
    set_bound(top);
  }

  // Takes over the row's bound: 2 below a key's upper half, so that equal values and both zeros stay above it.
  __device__ __forceinline__ void raise(uint32_t bound_key, int top) {
    const uint32_t k = bound_key - 2;
    const float v = bound_key > 2 ? __uint_as_float(k >> 31 ? k & 0x7FFFFFFFu : ~k) : __builtin_nanf("");
    kth = fmaxf(kth, v);
    set_bound(top);
  }

  __device__ __forceinline__ void set_bound(int top) {
    // (NaN while there is no reference or there are not k)
    bound = huge || c == -INFINITY || (top && kth != kth) ? __builtin_nanf("") : top ? fminf(limit, kth) : limit;
  }

  // Moves the reference where a logit passes its limit, and adds the logits.
  __device__ __forceinline__ void refer(const float (&x)[N], int lane) {
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < N; ++i) m = fmaxf(m, x[i]);
    const float high = wave_max(m);
    bool skip = false;  // this lane holds the new reference
    if (high > limit) {
      const bool big = fabsf(high) > 4194304.f;
      const float y = big ? 0.f : high * kLog2e;
      if (c != -INFINITY) {  // the old one becomes an ordinary logit, lane 0's
        const float down = big || huge ? (c - high) * kLog2e : yc - y, e = __builtin_amdgcn_exp2f(down);
        const float one = lane ? 0.f : __builtin_amdgcn_exp2f(off);
        t = e > 0.f ? e * (t + down * (one + r) + off * one) : t * 0.f;
        r = e > 0.f ? e * (one + r) : r * 0.f;
      }
      c = high;
      huge = big;
      yc = y;
      off = big ? 0.f : __builtin_fmaf(high, kLog2e, -y);
      limit = high + 2.7725887f;
      skip = __builtin_ctzll(__ballot(m == high)) == lane;
    }
    if (c != -INFINITY) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const bool it = skip && x[i] == c;  // one occurrence of it is left out
        skip = skip && !it;
        if (huge) add<true>(x[i], !it);
        else add<false>(x[i], !it);
      }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) r += x[i] != x[i] ? x[i] : 0.f;  // (a NaN always comes here; add's maximum drops it)
  }

  // The first logits: the lanes' best keys at once, then the others that beat the k-th of those.
  __device__ __forceinline__ void seed(const float (&x)[N], int64_t first, int64_t end, int top, int lane) {
    auto key = [&](int i) {
      const int64_t index = first + lane * N + i;
      return index < end ? key_of(x[i], (uint32_t)index) : 0;
    };
    uint64_t best = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) best = larger(best, key(i));
    list = sorted(best, lane);
    least = read_lane(list, top - 1);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const uint64_t k = key(i);
      uint64_t hits = __ballot(k > least && k != best);
      while (hits) {
        put(read_lane(k, __builtin_ctzll(hits)), top);
        hits &= hits - 1;
      }
    }
  }

  // Later ones: a logit equal to the k-th best comes behind it.
  __device__ __forceinline__ void pick(const float (&x)[N], int64_t first, int64_t end, int top) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      uint64_t hits = __ballot(!(x[i] <= kth));
      while (hits) {
        const int src = __builtin_ctzll(hits);
        const int64_t index = first + src * N + i;
        const float v = __uint_as_float(__builtin_amdgcn_readlane((int)__float_as_uint(x[i]), src));
        if (index < end) put(key_of(v, (uint32_t)index), top);
        hits &= hits - 1;
      }
    }
  }

  __device__ __forceinline__ void put(uint64_t key, int top) {
    if (key <= least) return;
    insert(list, key);
    least = read_lane(list, top - 1);
  }

  __device__ __forceinline__ Stats stats() const {
    const float rs = wave_sum(r), ts = wave_sum(t);
    if (c == -INFINITY) return Stats{c, rs, ts};  // no logit, or NaN
    const float w = __builtin_amdgcn_exp2f(-off);
    return Stats{c, rs * w, (ts - off * rs) * w};
  }
};

// The n-th largest of the 8 keys in a row's lanes, which hold them twice.
template <int R>
__device__ __forceinline__ int not_below(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x120 + R, 0xF, 0xF, false) >= v;  // row_ror:R
}
template <int R>
__device__ __forceinline__ uint32_t most_with(uint32_t v) {
  return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x120 + R, 0xF, 0xF, false));
}
__device__ __forceinline__ uint32_t nth_of_8(uint32_t v, int n) {
  const int count = 1 + not_below<1>(v) + not_below<2>(v) + not_below<3>(v) + not_below<4>(v) + not_below<5>(v) +
                    not_below<6>(v) + not_below<7>(v);
  return most_with<1>(most_with<2>(most_with<4>(count >= n ? v : 0)));
}

// W waves a row (or a part of one), kWaves / W rows a workgroup.
template <typename T, int W>
__global__ __launch_bounds__(kThreads, 6) void scores_kernel(Args p, int64_t per, int vec) {
  constexpr int N = 16 / sizeof(T);
  constexpr int64_t STEP = 64 * W * N;
  __shared__ uint64_t keys[W > 1 ? W * kMaxTop : 1];
  __shared__ uint64_t pool[W > 1 ? 64 : 1];
  __shared__ Stats stats[W];
  __shared__ uint32_t row_kth, shown[kWaves], maxima[32];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) % W;
  const int row = W == kWaves ? blockIdx.x / p.parts : blockIdx.x * (kWaves / W) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) / W;
  const int part = W == kWaves ? blockIdx.x % p.parts : 0;
  static_assert(kWaves == 8 && W == kWaves || W == 1, "a workgroup's barriers are one row's");
  if (row >= p.t) return;
  if (W > 1) {
    if (threadIdx.x < kWaves) shown[threadIdx.x] = 0;
    if (threadIdx.x == 0) row_kth = 0;
    __syncthreads();
  }
  // Every wave shows its j-th best; the q-th largest of those, q j >= top, is at most the row's top-th best.
  const int j = (p.top + kWaves - 1) / kWaves, q = p.top ? (p.top + j - 1) / j : 0;
  auto share = [&](const Wave<N>& w) {
    if (W == 1 || !p.top) return;
    __hip_atomic_store(&shown[wave], (uint32_t)(read_lane(w.list, j - 1) >> 32), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    const uint32_t best =
        nth_of_8(__hip_atomic_load(&shown[lane & 7], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP), q);
    if (lane == 0) __hip_atomic_fetch_max(&row_kth, best, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
  };
  const T* x = (const T*)p.x + row * p.ld;
  const int64_t begin = part * per, end = min(begin + per, p.v);
  Wave<N> w;
  auto unpack = [&](const u32x4& v, float (&f)[N]) {
    if constexpr (N == 8) {
      unpack8(v, f);
    } else {
      f[0] = __uint_as_float(v.x), f[1] = __uint_as_float(v.y), f[2] = __uint_as_float(v.z), f[3] = __uint_as_float(v.w);
    }
  };
  // 16 bytes of a lane's logits, -inf past the end
  auto load = [&](int64_t i) {
    u32x4 v;
    if (vec && i + N <= end) {
      v = *reinterpret_cast<const u32x4*>(x + i);
    } else {
      uint32_t word[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (N == 8) {
          const uint32_t lo = i + 2 * e < end ? x[i + 2 * e] : 0xFF80u, hi = i + 2 * e + 1 < end ? x[i + 2 * e + 1] : 0xFF80u;
          word[e] = lo | hi << 16;
        } else {
          word[e] = i + e < end ? __float_as_uint(x[i + e]) : 0xFF800000u;
        }
      }
      v = u32x4{word[0], word[1], word[2], word[3]};
    }
    return v;
  };
  // loads run a vector or two ahead
  int64_t i0 = begin + wave * 64 * N;
  const T* at = x + lane * N;
  const int64_t whole = vec ? end - (STEP + 64 * N) : -1;  // i0 up to which two vectors are whole
  u32x4 next[2];
  auto load_next = [&](int64_t i) {
    if (i <= whole) {
      next[0] = *reinterpret_cast<const u32x4*>(at + i);
      next[1] = *reinterpret_cast<const u32x4*>(at + i + STEP);
    } else if (i < end) {
      next[0] = load(i + lane * N);
    }
  };
  // a row's tokens are its second wave's (its first one's where it is alone)
  const bool whole_row = W == 1 || p.parts == 1;
  Token token = {0.f, false};
  if (whole_row && wave == (W > 1)) token = token_at<T>(p, row, lane);
  float f0[N];
  if (i0 < end) {
    const u32x4 v = load(i0 + lane * N);
    load_next(i0 + STEP);
    unpack(v, f0);
  }
  uint32_t bound0 = 0;
  if (W > 1 && p.top && p.top <= kSeedTop) {
    uint32_t k = 0;
    if (i0 < end) {
      float m = f0[0];
#pragma unroll
      for (int i = 1; i < N; ++i) m = __builtin_elementwise_maximum(m, f0[i]);
      k = (uint32_t)(key_of(m, 0) >> 32);
      k = max(k, dpp32<kDppXor1>(k));
      k = max(k, dpp32<kDppXor2>(k));
      k = max(k, dpp32<kDppHalfMirror>(k));
      k = max(k, dpp32<kDppRowMirror>(k));
    }
    if ((lane & 15) == 0) maxima[wave * 4 + lane / 16] = k;
    __syncthreads();
    bound0 = (uint32_t)__builtin_amdgcn_readlane((int)sorted32(maxima[lane & 31], lane), p.top - 1);
  }
  if (i0 < end) {
    w.begin(f0, i0, end, p.top, lane, bound0);
    share(w);
    i0 += STEP;
  }
  for (; i0 <= whole; i0 += 2 * STEP) {
    uint32_t seen = 0;
    if (W > 1) seen = __hip_atomic_load(&row_kth, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    const u32x4 v[2] = {next[0], next[1]};
    load_next(i0 + 2 * STEP);
    float f[2][N];
    unpack(v[0], f[0]);
    unpack(v[1], f[1]);
    if (W > 1 && p.top) w.raise(seen, p.top);
    const bool hot = w.hot(f[0]) | w.hot(f[1]);
    if (!hot) {
      w.add_all(f[0]);
      w.add_all(f[1]);
    } else {
#pragma unroll 1
      for (int u = 0; u < 2; ++u) {
        float g[N];
#pragma unroll
        for (int e = 0; e < N; ++e) g[e] = u ? f[1][e] : f[0][e];
        w.look(g, i0 + u * STEP, end, p.top, lane);
      }
      share(w);
    }
  }
  for (; i0 < end; i0 += STEP) {
    float f[N];
    unpack(next[0], f);
    if (i0 + STEP < end) next[0] = load(i0 + STEP + lane * N);
    w.look(f, i0, end, p.top, lane);
  }
  Stats s = w.stats();
  uint64_t list = w.list;
  if constexpr (W > 1) {
    if (lane < p.top) keys[wave * p.top + lane] = list;
    if (lane == 0) stats[wave] = s;
    __syncthreads();
    if (wave > 1) return;
    s = joined(lane < W ? stats[lane] : Stats{-INFINITY, 0.f, 0.f}, lane);
    if (wave == 0 && p.top) list = best_of<W>(keys, W, p.top, lane, pool);
  }
  if (whole_row) {
    if (wave == 0) finish_top(p, row, s, list, lane);
    if (wave == (W > 1)) finish_tokens<T>(p, row, s, token, lane);
    return;
  }
  const int64_t to = (int64_t)row * p.parts + part;
  if (wave) {
    if (lane == 0) *reinterpret_cast<f32x4*>(p.part + 4 * to) = f32x4{s.m, s.r, s.t, 0.f};
  } else if (lane < p.top) {
    p.part_keys[to * p.top + lane] = list;
  }
}

// A workgroup per row joins its parts (64 at most): the first wave the lists, the second the tokens.
template <typename T>
__global__ __launch_bounds__(256) void join_kernel(Args p) {
  __shared__ uint64_t keys[64 * kMaxTop];
  __shared__ uint64_t pool[64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row = blockIdx.x;
  const int64_t at = (int64_t)row * p.parts;
  Stats s = {-INFINITY, 0.f, 0.f};
  Token token = {0.f, false};
  if (wave <= 1) {
    if (wave) token = token_at<T>(p, row, lane);
    if (lane < p.parts) {
      const f32x4 q = *reinterpret_cast<const f32x4*>(p.part + 4 * (at + lane));
      s = Stats{q[0], q[1], q[2]};
    }
  }
  for (int i = threadIdx.x; i < p.parts * p.top; i += 256) keys[i] = p.part_keys[at * p.top + i];
  __syncthreads();
  const bool all = p.top > kLongTop;  // every wave merges a quarter of the lists
  if (all) {
    const int from = p.parts * wave / 4, to = p.parts * (wave + 1) / 4;
    const uint64_t list = best_merged(keys, from, to, p.top, lane);
    if (lane < p.top && from < to) keys[from * p.top + lane] = list;  // read by this wave alone so far
    __syncthreads();
  }
  if (wave > 1) return;
  s = joined(s, lane);
  if (wave) {
    finish_tokens<T>(p, row, s, token, lane);
  } else if (all) {
    uint64_t list = 0;
    for (int w = 0; w < 4; ++w)
      if (p.parts * w / 4 < p.parts * (w + 1) / 4)
        list = merged(list, 63 - lane < p.top ? keys[p.parts * w / 4 * p.top + 63 - lane] : 0, lane);
    finish_top(p, row, s, list, lane);
  } else if (p.top) {
    finish_top(p, row, s, best_of<64>(keys, p.parts, p.top, lane, pool), lane);
  }
}

// Parts of a row: enough workgroups for the GPU, 2048 logits a part at least. us, rows of 151936 in bf16 with 20
// alternatives: one in 64 parts 17.6, in 32 17.9, in 16 19.2; 64 rows in 8 parts 24.2, in 4 28.6, in 16 24.7; 16 in
// 32 17.9, in 16 22.2; 200 in 2 39, in 5 35; 256 in 1 35, in 4 35; 400 in 1 46, in 2 57.
int parts_of(int64_t t, int64_t v) {
  const int64_t most = (v + 2047) / 2048;
  int64_t parts = t >= 256 ? 1 : 512 / t;
  if (parts > most) parts = most;
  return (int)(parts > 64 ? 64 : parts < 1 ? 1 : parts);
}

int check(const char* what, int64_t t, int64_t v, int64_t n, int64_t top) {
  FF_REQUIRE(t > 0 && t <= (1 << 24) && v > 0 && v <= INT32_MAX && n >= 0 && n <= 65536 && top >= 0 && top <= kMaxTop && top <= v,
             "%s: bad sizes t=%lld v=%lld n=%lld top=%lld", what, (long long)t, (long long)v, (long long)n,
             (long long)top);
  return FF_OK;
}

}  // namespace

extern "C" int ff_token_scores_workspace(int64_t t, int64_t v, int64_t top, int64_t* bytes) {
  FF_REQUIRE(bytes, "ff_token_scores_workspace: null pointer");
  *bytes = 0;
  if (t == 0) return FF_OK;
  const int st = check("ff_token_scores_workspace", t, v, 0, top);
  if (st != FF_OK) return st;
  const int64_t parts = parts_of(t, v);
  *bytes = parts > 1 ? t * parts * (16 + 8 * top) : 0;
  return FF_OK;
}

extern "C" int ff_token_scores(const void* logits, int f32, int64_t ld, const int64_t* tokens, int64_t tok_ts,
                               int64_t tok_ns, float* logprobs, float* entropy, float* top_logprobs, int32_t* top_ids,
                               int64_t t, int64_t v, int64_t n, int64_t top, void* workspace, int64_t workspace_bytes,
                               ff_stream_t stream) {
  if (t == 0) return FF_OK;
  const int st = check("ff_token_scores", t, v, n, top);
  if (st != FF_OK) return st;
  FF_REQUIRE(logits && entropy && (n == 0 || (tokens && logprobs)) && (top == 0 || (top_logprobs && top_ids)),
             "ff_token_scores: null pointer");
  const int parts = parts_of(t, v);
  const int64_t need = parts > 1 ? t * parts * (16 + 8 * top) : 0;
  FF_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && ff_aligned(workspace, 16)),
             "ff_token_scores: workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)need);
  Args p = {logits, ld, tokens, tok_ts, tok_ns, logprobs, entropy, top_logprobs, top_ids, (float*)workspace,
            (uint64_t*)((char*)workspace + 16 * t * parts), v, (int)t, (int)n, (int)top, parts};
  const int64_t unit = f32 ? 4 : 8, chunks = (v + unit - 1) / unit;
  const int64_t per = (chunks + parts - 1) / parts * unit;
  const int vec = ff_aligned(logits, 16) && ld % unit == 0;
  hipStream_t s = (hipStream_t)stream;
  // A row a wave where there are rows for every SIMD twice and they are short: no lists to join, and one
  // to begin instead of eight. us, a wave and a workgroup a row, 5 alternatives in bf16: 4096 x 8000 27 and 44 (fp32 31
  // and 51), 2048 x 8000 20 and 25, 2048 x 32768 39 and 46 (fp32 60 and 51); 1024 x 8000 19 and 15, 2048 x 65536 61
  // and 63 (fp32 126 and 101).
  if (parts == 1 && t >= 2048 && v <= 32768) {
    const dim3 grid((unsigned)((t + kWaves - 1) / kWaves));
    if (f32) hipLaunchKernelGGL((scores_kernel<float, 1>), grid, dim3(kThreads), 0, s, p, per, vec);
    else hipLaunchKernelGGL((scores_kernel<bf16_t, 1>), grid, dim3(kThreads), 0, s, p, per, vec);
  } else {
    const dim3 grid((unsigned)(t * parts));
    if (f32) hipLaunchKernelGGL((scores_kernel<float, kWaves>), grid, dim3(kThreads), 0, s, p, per, vec);
    else hipLaunchKernelGGL((scores_kernel<bf16_t, kWaves>), grid, dim3(kThreads), 0, s, p, per, vec);
  }
  if (parts > 1) {
    if (f32) hipLaunchKernelGGL((join_kernel<float>), dim3((unsigned)t), dim3(256), 0, s, p);
    else hipLaunchKernelGGL((join_kernel<bf16_t>), dim3((unsigned)t), dim3(256), 0, s, p);
  }
  FF_LAUNCH_CHECK("ff_token_scores");
  return FF_OK;
}
