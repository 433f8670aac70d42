// Log probabilities of given tokens, entropy and the most likely tokens of rows of
// logits, in one pass over them.
//
// Every lane keeps a running maximum m and, of its values x, the sums over all but one
// occurrence of the maximum: r = sum e^(x - m) and t = sum (x - m) e^(x - m). With M, R
// and T of the whole row, log sum e^x = M + log1p(R), so
//   log p(x) = (x - M) - log1p(R),   entropy = log1p(R) - T / (1 + R):
// what is left of a near-certain token's probability keeps its relative precision in 32
// bits, since 1 is never added to it. The exponents are of base 2 until the end.
//
// The most likely tokens: a wave's best 64 so far lie sorted in its lanes, as one
// 64-bit key of (value, lowest index first). A vector of logits enters only where one of
// its values beats the wave's k-th best, which soon is rare. Waves, then parts of a row,
// are joined by taking the best of their lists' heads k times.
//
// Bound by the logits' bytes: a row is read once, 16 bytes a lane and load. Few rows are
// split over workgroups, and a second launch joins their parts.
#include "ff_common.h"

using namespace ff;

namespace {

constexpr int kWaves = 8, kThreads = 64 * kWaves;
constexpr int kMaxTop = 64;
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;

struct Args {
  const void* x;
  int64_t ld;
  const int64_t* tokens;
  int64_t tok_ts, tok_ns;
  float *logprobs, *entropy, *top_logprobs;
  int* top_ids;
  float* part;          // (rows, parts, 4): maximum, r, t, whether a NaN or +inf was seen
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

// A row's statistics (or a part's): m in natural units; r and t as above, t in base 2.
struct Stats {
  float m, r, t;
};

// Joins b into a.
__device__ __forceinline__ void join(Stats& a, const Stats& b) {
  if (b.m == -INFINITY) return;
  if (a.m == -INFINITY) {
    a = b;
    return;
  }
  const bool up = b.m > a.m;
  const float d = -fabsf(a.m - b.m) * kLog2e, e = __builtin_amdgcn_exp2f(d);
  const Stats hi = up ? b : a, lo = up ? a : b;
  // the lower side's 1 + r and its maximum's own share move d down
  a.m = hi.m;
  a.r = hi.r + e * (1.f + lo.r);
  a.t = hi.t + e * (lo.t + d * (1.f + lo.r));
}

__device__ __forceinline__ Stats shuffle_xor(const Stats& s, int mask) {
  return Stats{__shfl_xor(s.m, mask, 64), __shfl_xor(s.r, mask, 64), __shfl_xor(s.t, mask, 64)};
}

__device__ __forceinline__ uint64_t shuffle(uint64_t v, int lane) {
  return (uint64_t)(uint32_t)__shfl((int)(v >> 32), lane, 64) << 32 | (uint32_t)__shfl((int)(uint32_t)v, lane, 64);
}
__device__ __forceinline__ uint64_t read_lane(uint64_t v, int lane) {
  return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32 |
         (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, lane);
}

// Puts the uniform key into the wave's falling list (one entry a lane).
__device__ __forceinline__ void insert(uint64_t& list, uint64_t key, int lane) {
  const uint64_t up = shuffle(list, lane - 1 < 0 ? 0 : lane - 1);
  const bool beats = key > list;
  list = !beats ? list : lane && key > up ? up : key;
}

template <int N>
__device__ __forceinline__ void take(const float (&x)[N], uint32_t index0, Stats& s) {
  float top = x[0];
#pragma unroll
  for (int i = 1; i < N; ++i) top = fmaxf(top, x[i]);
  if (top > s.m) {  // a new maximum: the old one becomes an ordinary value
    if (s.m != -INFINITY) {
      const float d = (s.m - top) * kLog2e, e = __builtin_amdgcn_exp2f(d);
      s.t = e * (s.t + d * (1.f + s.r));
      s.r = e * (1.f + s.r);
    }
    s.m = top;
    bool first = true;  // one occurrence of it is left out
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const bool it = first && x[i] == top;
      first = first && !it;
      const float d = fmaxf((x[i] - top) * kLog2e, -1e6f), e = __builtin_amdgcn_exp2f(d);
      s.r += it ? 0.f : e;
      s.t = __builtin_fmaf(e, d, s.t);
    }
  } else if (s.m != -INFINITY) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float d = fmaxf((x[i] - s.m) * kLog2e, -1e6f), e = __builtin_amdgcn_exp2f(d);
      s.r += e;
      s.t = __builtin_fmaf(e, d, s.t);
    }
  }
}

// The best `top` of `lists` falling lists of `top` keys at `keys` (LDS), by one wave: the
// result's entry i in lane i.
__device__ __forceinline__ uint64_t best_of(const uint64_t* keys, int lists, int top, int lane) {
  uint64_t out = 0;
  // lane l holds the heads of lists l, l + 64, ...; lists <= 64
  int at = 0;
  uint64_t head = lane < lists ? keys[(int64_t)lane * top] : 0;
  for (int i = 0; i < top; ++i) {
    uint64_t best = head;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint64_t other = (uint64_t)(uint32_t)__shfl_xor((int)(best >> 32), o, 64) << 32 |
                             (uint32_t)__shfl_xor((int)(uint32_t)best, o, 64);
      best = best > other ? best : other;
    }
    if (lane == i) out = best;
    if (head == best && best) {  // keys differ, so one lane at most
      ++at;
      head = at < top ? keys[(int64_t)lane * top + at] : 0;
    }
  }
  return out;
}

// Writes a row's results; the whole wave. `odd`: the row holds a NaN or +inf.
template <typename T>
__device__ __forceinline__ void finish(const Args& p, int row, const Stats& s, bool odd, uint64_t list, int lane) {
  const float nan = __builtin_nanf("");
  const bool none = s.m == -INFINITY;  // every token is switched off
  const float l = log1pf(s.r);
  const T* x = (const T*)p.x + row * p.ld;
  for (int i = lane; i < p.n; i += 64) {
    const int64_t id = p.tokens[row * p.tok_ts + i * p.tok_ns];
    float lp = 0.f;  // no token
    if (id >= 0 && id < p.v) {
      const float xi = sizeof(T) == 2 ? bf16_to_f32(((const bf16_t*)x)[id]) : ((const float*)x)[id];
      lp = odd ? nan : none ? -INFINITY : (xi - s.m) - l;
    }
    p.logprobs[(int64_t)row * p.n + i] = lp;
  }
  if (lane == 0) p.entropy[row] = odd ? nan : none ? 0.f : l - kLn2 * s.t / (1.f + s.r);
  if (lane < p.top) {
    const float xi = value_of(list);
    p.top_logprobs[(int64_t)row * p.top + lane] = odd ? nan : none ? -INFINITY : (xi - s.m) - l;
    p.top_ids[(int64_t)row * p.top + lane] = (int)~(uint32_t)list;
  }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void scores_kernel(Args p, int64_t per, int vec) {
  constexpr int N = 16 / sizeof(T);
  __shared__ uint64_t keys[kWaves * kMaxTop];
  __shared__ Stats stats[kWaves];
  __shared__ int odds[kWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int row = blockIdx.x / p.parts, part = blockIdx.x % p.parts;
  const T* x = (const T*)p.x + row * p.ld;
  const int64_t begin = part * per, end = min(begin + per, p.v);
  Stats s = {-INFINITY, 0.f, 0.f};
  bool odd = false;
  uint64_t list = 0, least = 0;  // least: the k-th best so far
  for (int64_t i0 = begin + wave * 64 * N; i0 < end; i0 += kThreads * N) {
    const int64_t i = i0 + lane * N;
    float f[N];
    if (vec && i + N <= end) {
      const u32x4 w = *reinterpret_cast<const u32x4*>(x + i);
      if constexpr (N == 8) {
        unpack8(w, f);
      } else {
        f[0] = __uint_as_float(w.x), f[1] = __uint_as_float(w.y), f[2] = __uint_as_float(w.z), f[3] = __uint_as_float(w.w);
      }
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        f[e] = -INFINITY;
        if (i + e < end) f[e] = N == 8 ? bf16_to_f32(((const bf16_t*)x)[i + e]) : ((const float*)x)[i + e];
      }
    }
#pragma unroll
    for (int e = 0; e < N; ++e) odd |= !(f[e] < INFINITY);
    take<N>(f, (uint32_t)i, s);
    if (p.top) {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const uint64_t key = i + e < end ? key_of(f[e], (uint32_t)(i + e)) : 0;
        uint64_t hits = __ballot(key > least);
        while (hits) {
          const int src = __builtin_ctzll(hits);
          hits &= hits - 1;
          const uint64_t k = read_lane(key, src);
          if (k > least) {
            insert(list, k, lane);
            least = read_lane(list, p.top - 1);
          }
        }
      }
    }
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    // both partners join in the same order, so that they get the same bits
    const Stats other = shuffle_xor(s, o);
    Stats a = lane & o ? other : s;
    join(a, lane & o ? s : other);
    s = a;
  }
  odd = __ballot(odd) != 0;
  if (lane < p.top) keys[wave * p.top + lane] = list;
  if (lane == 0) {
    stats[wave] = s;
    odds[wave] = odd;
  }
  __syncthreads();
  if (wave) return;
  s = stats[0];
  odd = odds[0];
  for (int w = 1; w < kWaves; ++w) {
    join(s, stats[w]);
    odd |= odds[w];
  }
  if (p.top) list = best_of(keys, kWaves, p.top, lane);
  if (p.parts == 1) {
    finish<T>(p, row, s, odd, list, lane);
    return;
  }
  const int64_t at = (int64_t)row * p.parts + part;
  if (lane == 0) *reinterpret_cast<f32x4*>(p.part + 4 * at) = f32x4{s.m, s.r, s.t, odd ? 1.f : 0.f};
  if (lane < p.top) p.part_keys[at * p.top + lane] = list;
}

// A wave per row joins its parts (64 at most).
template <typename T>
__global__ __launch_bounds__(64) void join_kernel(Args p) {
  __shared__ uint64_t keys[64 * kMaxTop];
  const int lane = threadIdx.x, row = blockIdx.x;
  const int64_t at = (int64_t)row * p.parts;
  Stats s = {-INFINITY, 0.f, 0.f};
  bool odd = false;
  if (lane < p.parts) {
    const f32x4 q = *reinterpret_cast<const f32x4*>(p.part + 4 * (at + lane));
    s = Stats{q[0], q[1], q[2]};
    odd = q[3] != 0.f;
  }
  odd = __ballot(odd) != 0;
  for (int i = lane; i < p.parts * p.top; i += 64) keys[i] = p.part_keys[at * p.top + i];
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const Stats other = shuffle_xor(s, o);
    Stats a = lane & o ? other : s;
    join(a, lane & o ? s : other);
    s = a;
  }
  __syncthreads();
  const uint64_t list = p.top ? best_of(keys, p.parts, p.top, lane) : 0;
  finish<T>(p, row, s, odd, list, lane);
}

// Parts of a row: enough workgroups for the GPU, 2048 logits a part at least.
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
  const dim3 grid((unsigned)(t * parts));
  if (f32) hipLaunchKernelGGL((scores_kernel<float>), grid, dim3(kThreads), 0, s, p, per, vec);
  else hipLaunchKernelGGL((scores_kernel<bf16_t>), grid, dim3(kThreads), 0, s, p, per, vec);
  if (parts > 1) {
    if (f32) hipLaunchKernelGGL((join_kernel<float>), dim3((unsigned)t), dim3(64), 0, s, p);
    else hipLaunchKernelGGL((join_kernel<bf16_t>), dim3((unsigned)t), dim3(64), 0, s, p);
  }
  FF_LAUNCH_CHECK("ff_token_scores");
  return FF_OK;
}
