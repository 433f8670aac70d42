// Mixture-of-experts operators for gfx950: routing (the experts of each token and
// their weights) and the chosen experts' products on block-scaled FP8 weights
// (ff_block.h states the format).
//
// y[t] = sum_j w[t, j] D_e (silu(G_e x[t]) * (U_e x[t])), e = ids[t, j]. The rows x
// are quantised per 128 channels as the linear's rows are; the SwiGLU's values go
// into the down products as bf16: each is off by at most 2^-8 of itself, as large a
// rounding as the output's own, so an output is off by 2.3e-3 to 2.5e-3 RMS where the
// output's rounding alone is 1.7e-3. It buys the matrix instructions' bf16 rate: fp32
// values would need two bf16 parts, twice the down products. Quantised a second time, as
// a dense layer of BlockFP8Linear's quantises them, a value next to a border between
// two e4m3 codes would move by 1/16 with the last bit of a sum. Sums stay fp32
// throughout, and their order depends on the shapes alone.
//
// Few (token, expert) pairs: two launches. gate_up: a workgroup per pair and 16
// channels, the row quantised in the workgroup; down: a workgroup per token and 16
// channels, its waves sharing the k steps of all the token's experts, so the
// weighted sum over experts needs no launch of its own.
// More pairs: one launch orders them by expert and quantises the rows, row tiles that
// belong to one expert each run both products, and the down products of a token's experts
// are added by a last launch in the order of the token's list.
#include "ff_block_tile.h"

using namespace ff;

namespace {

constexpr int kThreads = 512, kWaves = kThreads / 64;
constexpr int kMaxExperts = 1024;
constexpr int kInlineCodes = 49152;  // codes of the row that a gate_up workgroup quantises

// ---------------------------------------------------------------- routing

constexpr int kRouteWaves = 4;

template <int CTRL, typename T>
__device__ __forceinline__ T dpp_of(T x) {
  if constexpr (sizeof(T) == 4) {
    return __builtin_bit_cast(
        T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xF, 0xF, false));
  } else {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, 0xF, 0xF, false);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, 0xF, 0xF, false);
    return __builtin_bit_cast(T, (uint64_t)hi << 32 | lo);
  }
}

// The value of lane l ^ D, D 16 or 32: both results of a row swap, of which one is the lane's own.
template <int D>
__device__ __forceinline__ uint32_t swap32(uint32_t x) {
  if constexpr (D == 32) {
    const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return (threadIdx.x & 32) ? r[0] : r[1];
  } else {
    const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    return (threadIdx.x & 16) ? r[0] : r[1];
  }
}
template <int D, typename T>
__device__ __forceinline__ T swap_of(T x) {
  if constexpr (sizeof(T) == 4) {
    return __builtin_bit_cast(T, swap32<D>(__builtin_bit_cast(uint32_t, x)));
  } else {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    return __builtin_bit_cast(T, (uint64_t)swap32<D>((uint32_t)(u >> 32)) << 32 | swap32<D>((uint32_t)u));
  }
}

// f over LPR (16 or 64) lanes, the same bits in each (every step combines a lane with its partner).
template <int LPR, typename T, typename F>
__device__ __forceinline__ T reduce(T v, F&& f) {
  v = f(v, dpp_of<kDppXor1>(v));
  v = f(v, dpp_of<kDppXor2>(v));
  v = f(v, dpp_of<kDppHalfMirror>(v));
  v = f(v, dpp_of<kDppRowMirror>(v));
  if constexpr (LPR == 64) {
    v = f(v, swap_of<16>(v));
    v = f(v, swap_of<32>(v));
  }
  return v;
}

// exp(x) to about 1e-14 of its value: 2^k exp(r), k = rint(x / ln 2), |r| <= ln 2 / 2, and
// the Taylor polynomial of degree 11 (its next term is below 7e-15). r = x - k ln 2 with
// ln 2 = 0x0.b17217f7d1cf79ab.. in two parts, its leading 32 bits and the double nearest
// to the rest: the product with the first is exact, the second's error is below 2^-85.
__device__ __forceinline__ double exp64(double x) {
  if (x < -746.0) return 0.0;
  if (x > 710.0) return __builtin_inf();
  const double k = __builtin_rint(x * 1.4426950408889634);
  double r = __builtin_fma(-k, 0x0.b17217f7p0, x);
  r = __builtin_fma(-k, 0x1.a39ef35793c76p-33, r);
  double p = 1.0 / 39916800;
  constexpr double kInv[11] = {1.0, 1.0, 1.0 / 2, 1.0 / 6, 1.0 / 24, 1.0 / 120, 1.0 / 720, 1.0 / 5040, 1.0 / 40320,
                               1.0 / 362880, 1.0 / 3628800};
#pragma unroll
  for (int i = 10; i >= 0; --i) p = __builtin_fma(p, r, kInv[i]);
  return __builtin_ldexp(p, (int)k);
}

// LPR lanes per row; lane l of them holds experts l, l + LPR, ... Without a bias experts are
// compared by their logits (scores rise with them); with one by score + bias in 64 bits: in 32,
// scores that lie next to each other would change places with the last bit of exp(). Sums and
// weights are 64-bit until their one rounding.
// Bound by instructions, not by its few bytes. 16 lanes for many rows (16387 x 160, top 6,
// softmax over 160, 16 us; 31 with 64 lanes, which spend four times the steps on a row's
// reductions), 64 for few: one row takes 3.9 us, 576 rows of 256 experts in 8 groups 8.1.
template <int LPR, int EPL, bool F32, bool BIAS>
__global__ __launch_bounds__(64 * kRouteWaves) void route_kernel(
    const void* __restrict__ logits, int64_t ld, const float* __restrict__ bias, float* __restrict__ weights,
    int* __restrict__ ids, int64_t t, int experts, int top_k, int sigmoid, int groups, int top_groups, int renormalize,
    double scale) {
  using Key = std::conditional_t<BIAS, double, float>;
  constexpr int kRows = 64 / LPR;  // rows of a wave
  __shared__ Key sc[kRouteWaves * kRows][LPR * EPL];
  __shared__ Key best_of[kRouteWaves * kRows][64];
  const int lane = threadIdx.x & 63, li = lane % LPR, slot = threadIdx.x / LPR;
  const int64_t row = blockIdx.x * (int64_t)(kRouteWaves * kRows) + slot;
  const bool live = row < t;  // rows past the end are worked on as all-off ones: every lane takes part in every step
  const Key kNone = -(Key)__builtin_inf();
  const auto larger = [](auto a, auto b) { return a > b ? a : b; };
  const auto load = [&](int e) {
    if constexpr (F32) return reinterpret_cast<const float*>(logits)[row * ld + e];
    else return bf16_to_f32(reinterpret_cast<const bf16_t*>(logits)[row * ld + e]);
  };
  float l[EPL];
  bool bad = false;
  float top = -__builtin_inff();
#pragma unroll
  for (int v = 0; v < EPL; ++v) {
    const int e = li + LPR * v;
    l[v] = live && e < experts ? load(e) : -__builtin_inff();
    bad |= l[v] != l[v] || (!sigmoid && l[v] == __builtin_inff());
    top = larger(top, l[v]);
  }
  double inv = 0;  // 1 / the softmax's sum
  if (!sigmoid) {
    top = reduce<LPR>(top, larger);
    double sum = 0;
#pragma unroll
    for (int v = 0; v < EPL; ++v)
      if (LPR * v < experts) sum += l[v] == -__builtin_inff() ? 0.0 : exp64((double)l[v] - (double)top);
    sum = reduce<LPR>(sum, [](double a, double b) { return a + b; });
    inv = sum > 0 ? 1.0 / sum : 0.0;
  }
  const auto score = [&](float x) {
    return sigmoid ? 1.0 / (1.0 + exp64(-(double)x)) : exp64((double)x - (double)top) * inv;
  };
  Key c[EPL];  // what experts are compared by; -inf for those switched off
#pragma unroll
  for (int v = 0; v < EPL; ++v) {
    if constexpr (BIAS) {
      const int e = li + LPR * v;
      const double b = e < experts ? (double)bias[e] : 0.0;
      bad |= b != b;
      c[v] = l[v] == -__builtin_inff() ? kNone : score(l[v]) + b;
    } else {
      c[v] = l[v];
    }
  }
  const uint64_t row_lanes = LPR == 64 ? ~0ull : ((1ull << (LPR & 63)) - 1) << (lane - li);
  if (groups > 1) {
    const int per = experts / groups;
#pragma unroll
    for (int v = 0; v < EPL; ++v) sc[slot][li + LPR * v] = c[v];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    int share = 1;  // lanes of a group, a power of two
    while (2 * share * groups <= LPR) share *= 2;
    for (int g0 = 0; g0 < groups; g0 += LPR / share) {
      const int g = g0 + li / share;
      Key best = kNone, second = kNone;
      if (g < groups)
        for (int m = li % share; m < per; m += share) {
          const Key s = sc[slot][g * per + m];
          second = larger(second, s < best ? s : best);
          best = larger(best, s);
        }
      for (int d = 1; d < share; d *= 2) {
        const Key ob = __shfl_xor(best, d), os = __shfl_xor(second, d);
        second = larger(larger(second, os), best < ob ? best : ob);
        best = larger(best, ob);
      }
      if (BIAS && second != kNone) best += second;
      if (g < groups && li % share == 0) best_of[slot][g] = best;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    const Key mine = li < groups ? best_of[slot][li] : kNone;
    int rank = 0;  // groups ahead of this lane's
    for (int o = 0; o < groups; ++o) {
      const Key s = best_of[slot][o];
      rank += s > mine || (s == mine && o < li);
    }
    const uint64_t keep = __ballot(li < groups && rank < top_groups) >> (lane - li);
#pragma unroll
    for (int v = 0; v < EPL; ++v) {
      const int e = li + LPR * v;
      if (e < experts && !(keep >> (e / per) & 1)) c[v] = kNone;
    }
  }
  int mine_id = -1;  // lane j's: the j-th chosen
  for (int j = 0; j < top_k; ++j) {
    Key best = kNone;
#pragma unroll
    for (int v = 0; v < EPL; ++v) best = larger(best, c[v]);
    best = reduce<LPR>(best, larger);
    int id = 1 << 30;  // the lowest expert with that score
#pragma unroll
    for (int v = EPL - 1; v >= 0; --v)
      if (c[v] == best) id = li + LPR * v;
    id = reduce<LPR>(id, [](int a, int b) { return a < b ? a : b; });
#pragma unroll
    for (int v = 0; v < EPL; ++v)
      if (li + LPR * v == id) c[v] = kNone;
    if (li == j && best != kNone) mine_id = id;
  }
  const bool poisoned = (__ballot(bad) & row_lanes) != 0;  // a NaN (or a softmax over +inf) shows in every weight
  double w = live && li < top_k && mine_id >= 0 && !poisoned ? score(load(mine_id)) : 0.0;
  const double total = reduce<LPR>(w, [](double a, double b) { return a + b; });
  if (!live || li >= top_k) return;
  if (renormalize) w = total > 0 ? w / total : 0.0;
  ids[row * top_k + li] = poisoned ? li : mine_id;
  weights[row * top_k + li] = poisoned ? __builtin_nanf("") : (float)(w * scale);
}

// ---------------------------------------------------------------- pairs by expert

// The first `experts` workgroups order the pairs, one expert each: its pairs p = token *
// top_k + slot in rising order to list[off[e] ..), off[e] = pairs of lower experts. Every
// workgroup reads all ids, twice where its expert has pairs, and needs nothing from the
// others: no counters in memory, no order of arrival. That is experts x pairs x 8 bytes at
// most, from L2: 33 MB at 4096 tokens x 8 of 128, and it grows with the tokens alone. ids
// outside [0, experts) are in no list. The other workgroups quantise the rows.
// 4.8 us to 577 tokens, about the shortest a launch takes, 12 us at 4096 tokens x 8.
constexpr int kPlanThreads = 1024, kPlanWaves = kPlanThreads / 64, kPlanBatch = 8;
__global__ __launch_bounds__(kPlanThreads) void plan_kernel(const int* __restrict__ ids, int pairs, int experts,
                                                            int* __restrict__ off, int* __restrict__ list,
                                                            const bf16_t* __restrict__ x, int64_t ldx, int vec,
                                                            int64_t t, int64_t h, int kt_n, uint8_t* __restrict__ q,
                                                            float* __restrict__ qs) {
  if ((int)blockIdx.x >= experts) {
    const int64_t tiles = (t + kPlanThreads / 16 - 1) / (kPlanThreads / 16) * kt_n;
    for (int64_t i = blockIdx.x - experts; i < tiles; i += gridDim.x - experts)
      quant_rows_tile<kPlanThreads / 16>(x, ldx, q, qs, t, h, kt_n, vec, i);
    return;
  }
  __shared__ int below[kPlanWaves], equal[kPlanWaves];
  const int e = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int seg = (pairs + kPlanWaves - 1) / kPlanWaves;
  const int lo = min(pairs, wave * seg), hi = min(pairs, lo + seg);
  int nb = 0, ne = 0;
  for (int i0 = lo; i0 < hi; i0 += 64 * kPlanBatch) {  // the loads of a batch in flight together
    int id[kPlanBatch];
#pragma unroll
    for (int v = 0; v < kPlanBatch; ++v) {
      const int i = i0 + 64 * v + lane;
      id[v] = i < hi ? ids[i] : -1;
    }
#pragma unroll
    for (int v = 0; v < kPlanBatch; ++v) {
      nb += id[v] >= 0 && id[v] < e;
      ne += id[v] == e;
    }
  }
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    nb += __shfl_xor(nb, d);
    ne += __shfl_xor(ne, d);
  }
  if (lane == 0) {
    below[wave] = nb;
    equal[wave] = ne;
  }
  __syncthreads();
  int base = 0, all = 0;
  for (int w = 0; w < kPlanWaves; ++w) {
    base += below[w] + (w < wave ? equal[w] : 0);
    all += below[w] + equal[w];
  }
  if (threadIdx.x == 0) {
    off[e] = base;
    if (e == experts - 1) off[experts] = all;
  }
  if (equal[wave] == 0) return;
  for (int i0 = lo; i0 < hi; i0 += 64 * kPlanBatch) {
    int id[kPlanBatch];
#pragma unroll
    for (int v = 0; v < kPlanBatch; ++v) {
      const int i = i0 + 64 * v + lane;
      id[v] = i < hi ? ids[i] : -1;
    }
#pragma unroll
    for (int v = 0; v < kPlanBatch; ++v) {
      const uint64_t b = __ballot(id[v] == e);
      if (id[v] == e) list[base + __builtin_popcountll(b & ((1ull << lane) - 1))] = i0 + 64 * v + lane;
      base += __builtin_popcountll(b);
    }
  }
}

// ---------------------------------------------------------------- gate/up + SwiGLU

// g / (1 + exp(-g)) to a few units in the last place of fp32 (its bf16 rounding follows):
// exp(-g) = 2^(-g log2 e), the product's rounding error added back to first order, and the
// hardware's exponential and reciprocal (1 ulp each) in place of the library's (some 50
// instructions a value, a fifth of the gate/up tiles' time). Below g = -87.3 exp(-g)
// passes 2^126, its reciprocal is subnormal and comes out as 0: so does the value, whose
// magnitude is under 1.1e-36 there.
__device__ __forceinline__ float silu_fast(float g) {
  constexpr float kLog2e = 1.44269504f, kLog2eLow = 1.92596299e-8f, kLn2 = 0.693147181f;
  const float p = -g * kLog2e;
  const float low = __builtin_fmaf(-g, kLog2e, -p) - g * kLog2eLow;
  float e = __builtin_amdgcn_exp2f(p);
  e = e > 0.f && e < __builtin_inff() ? __builtin_fmaf(e, low * kLn2, e) : e;
  return g * __builtin_amdgcn_rcpf(1.0f + e);
}

__device__ __forceinline__ u32x2 swiglu4(const f32x4& g, const f32x4& u) {
  return pack4_bf16(silu_fast(g[0]) * u[0], silu_fast(g[1]) * u[1], silu_fast(g[2]) * u[2], silu_fast(g[3]) * u[3]);
}

// Adds the waves' sums of slot t (a lane's 4 values of one fragment pair) in wave order.
template <int SLOTS, int WAVES = kWaves>
__device__ __forceinline__ f32x4 sum_waves(const f32x4* red, int t) {
  f32x4 v = red[t];
#pragma unroll
  for (int w = 1; w < WAVES; ++w) v += red[w * SLOTS + t];
  return v;
}

// One pair x 16 channels: gate and up fragment of the channels, k steps shared by the
// waves; the workgroup quantises the token's row. Weights of an expert: gate then up, each
// nf fragments x kt_n k steps; scales (2, nf / 8, kt_n).
// Bound by the weights' bytes and the launch: 8 pairs, h 2048, i 768: 6.2 us for 25 MB.
__global__ __launch_bounds__(kThreads) void gate_up_pair_kernel(
    const bf16_t* __restrict__ x, int64_t ldx, int vec, int64_t h_n, const int* __restrict__ ids,
    const uint8_t* __restrict__ wp, const float* __restrict__ ws, bf16_t* __restrict__ h, int top_k, int experts,
    int kt_n, int nf) {
  constexpr int PF = 4;
  __shared__ __align__(16) uint8_t smem[kInlineCodes + 4 * kInlineCodes / kBlock];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r16 = lane & 15, g = lane >> 4;
  const int pair = blockIdx.x / nf, c = blockIdx.x % nf, e = ids[pair];
  if (e < 0 || e >= experts) return;
  const int64_t matrix = (int64_t)nf * kt_n * 2048;
  const uint8_t* fg = wp + 2 * e * matrix + (int64_t)c * 2048;
  const float* sg = ws + ((int64_t)2 * e * (nf / 8) + c / 8) * kt_n;
  const int64_t sup = (int64_t)(nf / 8) * kt_n;
  float* scales = reinterpret_cast<float*>(smem + kInlineCodes);
  i32x8 wq[PF][2];
  float wsc[PF][2];
  const int mine = (kt_n - wave + kWaves - 1) / kWaves;
  f32x4 acc[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
  for (int b = 0; b < mine || b == 0; b += PF) {
#pragma unroll
    for (int u = 0; u < PF; ++u)
      if (b + u < mine) {
        const int kt = wave + kWaves * (b + u);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          wq[u][j] = load_frag(fg + j * matrix + (int64_t)kt * nf * 2048, lane);
          wsc[u][j] = sg[j * sup + kt];
        }
      }
    if (b == 0) {  // the first weights are in flight meanwhile
      const bf16_t* src = x + (int64_t)(pair / top_k) * ldx;
      for (int kt = threadIdx.x >> 4; kt < kt_n; kt += kThreads / 16) {
        float scale;
        const u32x2 code = quant_group16(src, h_n, kt, r16, vec, &scale);
        *reinterpret_cast<u32x2*>(smem + kt * kBlock + 8 * r16) = code;
        if (r16 == 0) scales[kt] = scale;
      }
      __syncthreads();
    }
#pragma unroll
    for (int u = 0; u < PF; ++u)
      if (b + u < mine) {
        const int kt = wave + kWaves * (b + u);
        const i32x4v* p = reinterpret_cast<const i32x4v*>(smem + kt * kBlock + 32 * g);
        const i32x8 xq = join(p[0], p[1]);
#pragma unroll
        for (int j = 0; j < 2; ++j) fma4(acc[j], mfma_step(wq[u][j], xq), scales[kt] * wsc[u][j]);
      }
  }
  __syncthreads();  // the codes are no longer read
  f32x4* red = reinterpret_cast<f32x4*>(smem);  // every result row is the pair's: one lane of each group keeps it
  if (r16 == 0)
#pragma unroll
    for (int j = 0; j < 2; ++j) red[wave * 8 + 4 * j + g] = acc[j];
  __syncthreads();
  if (threadIdx.x < 4)
    *reinterpret_cast<u32x2*>(h + (int64_t)pair * (16 * nf) + 16 * c + 4 * threadIdx.x) =
        swiglu4(sum_waves<8>(red, threadIdx.x), sum_waves<8>(red, 4 + threadIdx.x));
}

// ---------------------------------------------------------------- down

// This lane's operand of one k step: channels 128 kt + 32 g .. + 31 of a row of h.
__device__ __forceinline__ void load_h(u32x4 (&x)[4], const bf16_t* p) {
#pragma unroll
  for (int u = 0; u < 4; ++u) x[u] = reinterpret_cast<const u32x4*>(p)[u];
}

// One token's y, 16 channels: the k steps of all its experts shared by 16 waves (few
// workgroups: with three steps each, all of 128 x 768 x 8 experts is in flight at once). All
// 16 result rows are the token's (every lane group reads the same row). A slot without an
// expert reads expert 0's weights and is not added (its row of h was not written); every
// id is read before the first use of one, so the loads do not wait for each other.
// 8 pairs, h 2048, i 768: 4.7 us for 12.6 MB, three dependent trips to memory.
constexpr int kDownThreads = 1024, kDownWaves = kDownThreads / 64;
__global__ __launch_bounds__(kDownThreads) void down_pair_kernel(
    const bf16_t* __restrict__ h, const float* __restrict__ weights, const int* __restrict__ ids,
    const uint8_t* __restrict__ wp, const float* __restrict__ ws, bf16_t* __restrict__ y, int64_t ldy, int64_t n,
    int top_k, int experts, int kt_n, int nf) {
  constexpr int PF = 3;
  __shared__ f32x4 red[kDownWaves * 4];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r16 = lane & 15, g = lane >> 4;
  const int f = blockIdx.x % nf, tok = blockIdx.x / nf;
  const int64_t matrix = (int64_t)nf * kt_n * 2048;
  const int64_t nb = (n + kBlock - 1) / kBlock;
  const int steps = top_k * kt_n;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int b = wave; b < steps; b += kDownWaves * PF) {
    int id[PF];
    float wt[PF], s[PF];
    i32x8 wq[PF];
    u32x4 xh[PF][4];
#pragma unroll
    for (int u = 0; u < PF; ++u) {
      const int pair = tok * top_k + min(b + kDownWaves * u, steps - 1) / kt_n;
      id[u] = ids[pair];
      wt[u] = weights[pair];
    }
#pragma unroll
    for (int u = 0; u < PF; ++u) {
      const int at = min(b + kDownWaves * u, steps - 1), pair = tok * top_k + at / kt_n, kt = at % kt_n;
      const bool on = id[u] >= 0 && id[u] < experts && b + kDownWaves * u < steps;
      const int e = on ? id[u] : 0;
      id[u] = on;
      wq[u] = load_frag(wp + e * matrix + ((int64_t)kt * nf + f) * 2048, lane);
      load_h(xh[u], h + ((int64_t)pair * kt_n + kt) * kBlock + 32 * g);
      s[u] = ws[((int64_t)e * nb + f / 8) * kt_n + kt];
    }
#pragma unroll
    for (int u = 0; u < PF; ++u)
      if (id[u]) fma4(acc, mfma_step_bf16(wq[u], xh[u]), wt[u] * s[u]);
  }
  if (r16 == 0) red[wave * 4 + g] = acc;
  __syncthreads();
  if (threadIdx.x < 4) {
    const f32x4 v = sum_waves<4, kDownWaves>(red, threadIdx.x);
    const int64_t c = 16 * (int64_t)f + 4 * threadIdx.x;
    if (c < n) store4_bf16(y + tok * ldy + c, v, n - c);
  }
}

// ---------------------------------------------------------------- row tiles

// BM rows of one expert x 2 CW channels: wave w's fragments alternate gate and up of the
// same 16 channels, so SwiGLU runs on the lane's own sums.
// Few rows an expert: bound by the weights' bytes (48 tokens x 4 of 64 experts, h 2560, i 1024,
// 32-row tiles: 51 us, 5.4 TB/s; 577 x 5 of 60, h 2120, i 1000, 64-row: 56 us, 5.0 TB/s).
// Many (4096 x 8 of 128, h 2048, i 768): 190 us, 1.1 PFLOP/s; the path that loads come back on
// is busy 77 % of the time (40 KB a step and workgroup, 640 clocks against the matrix
// instructions' 512), the matrix unit 32 %. 128 rows a tile take as long: fewer loads, but more
// rows past an expert's end and twice the reads from LDS.
template <int BM, int CW, int P>
__global__ __launch_bounds__(kTileThreads, 2) void gate_up_tile_kernel(
    const uint8_t* __restrict__ q, const float* __restrict__ qs, const int* __restrict__ off,
    const int* __restrict__ list, const uint8_t* __restrict__ wp, const float* __restrict__ ws,
    bf16_t* __restrict__ h, int64_t t_n, int top_k, int experts, int kt_n, int nf, int tiles_n) {
  constexpr int RA = BM / 16, TJ = CW / 16;
  static_assert(TJ % 2 == 0, "gate and up");
  __shared__ __align__(1024) uint8_t smem[tile_smem<BM>()];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r16 = lane & 15, g = lane >> 4;
  ExpertTile at;
  if (!find_tile(off, experts, BM, tiles_n, &at)) return;
  const int e = at.expert, row0 = at.row0, rows = at.rows;
  const int c0 = (at.col * 4 + wave) * (TJ / 2);  // the wave's first 16-channel block
  const int64_t matrix = (int64_t)nf * kt_n * 2048;
  const int64_t nb = nf / 8;
  const float* scale = ws + (2 * e * nb + min(c0, nf - 1) / 8) * kt_n;
  const uint8_t* gate = wp + 2 * e * matrix;
  TileWeights<TJ, 2> w{{gate, gate + matrix}, (uint32_t)matrix, (uint32_t)nf * 2048u, {scale, scale + nb * kt_n}, {}};
#pragma unroll
  for (int j = 0; j < TJ; ++j) w.frag[j] = (uint32_t)(c0 + j / 2) * 2048u;
  const uint32_t kp = (uint32_t)kt_n * kBlock;
  const auto token = [&](int r) { return (uint32_t)(list[row0 + min(r, rows - 1)] / top_k); };
  f32x4 acc[RA][TJ];
  tile_mainloop<BM, CW, 2, P, 1>(
      acc, smem, kt_n, 0, kt_n, q, (uint32_t)t_n * kp, [&](int r) { return token(r) * kp; }, qs, (uint32_t)(4 * t_n) * kt_n,
      token, (uint32_t)(4 * t_n), w);
#pragma unroll
  for (int i = 0; i < RA; ++i) {
    if (16 * i + r16 >= rows) continue;
    bf16_t* out = h + (int64_t)(row0 + 16 * i + r16) * (16 * nf) + 4 * g;
#pragma unroll
    for (int j = 0; j < TJ; j += 2)
      if (c0 + j / 2 < nf) *reinterpret_cast<u32x2*>(out + 16 * (c0 + j / 2)) = swiglu4(acc[i][j], acc[i][j + 1]);
  }
}

// BM rows of one expert x 4 CW channels of the down product; fp32 to part[pair] (as bf16 they
// would save 25 us of 424 at 4096 tokens and cost a rounding of every expert's share).
// Sizes as above: 29 us (5.0 TB/s), 40 us (4.0 TB/s) and 175 us, 0.6 PFLOP/s: 274 MB read, 268
// MB of sums written. Two steps of loads ahead, narrower tiles with three workgroups a CU and
// block scales through vector loads all take the same time.
template <int BM, int CW, int P>
__global__ __launch_bounds__(kTileThreads, 2) void down_tile_kernel(
    const bf16_t* __restrict__ h, const int* __restrict__ off, const int* __restrict__ list,
    const uint8_t* __restrict__ wp, const float* __restrict__ ws, float* __restrict__ part, int64_t ldp, int64_t n,
    int experts, int kt_n, int nf, int tiles_n) {
  constexpr int RA = BM / 16, TJ = CW / 16;
  __shared__ __align__(1024) uint8_t smem[tile_smem_bf16<BM>()];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r16 = lane & 15, g = lane >> 4;
  ExpertTile at;
  if (!find_tile(off, experts, BM, tiles_n, &at)) return;
  const int e = at.expert, row0 = at.row0, rows = at.rows;
  const int f0 = (at.col * 4 + wave) * TJ;
  const int64_t matrix = (int64_t)nf * kt_n * 2048;
  const int64_t nb = (n + kBlock - 1) / kBlock;
  TileWeights<TJ, 1> w{{wp + e * matrix}, (uint32_t)matrix, (uint32_t)nf * 2048u,
                       {ws + (e * nb + min(f0, nf - 1) / 8) * kt_n}, {}};
#pragma unroll
  for (int j = 0; j < TJ; ++j) w.frag[j] = (uint32_t)(f0 + j) * 2048u;
  const uint32_t kp = (uint32_t)kt_n * (2 * kBlock);
  f32x4 acc[RA][TJ];
  tile_mainloop_bf16<BM, CW, P>(acc, smem, kt_n, reinterpret_cast<const uint8_t*>(h) + (int64_t)row0 * kp,
                                (uint32_t)rows * kp, [&](int r) { return (uint32_t)min(r, rows - 1) * kp; }, w);
#pragma unroll
  for (int i = 0; i < RA; ++i) {
    if (16 * i + r16 >= rows) continue;
    float* out = part + (int64_t)list[row0 + 16 * i + r16] * ldp;
#pragma unroll
    for (int j = 0; j < TJ; ++j) {
      const int64_t c = 16 * (int64_t)(f0 + j) + 4 * g;
      if (c < n) *reinterpret_cast<f32x4*>(out + c) = acc[i][j];
    }
  }
}

// y[t] = sum_j w[t, j] part[t top_k + j], slots in order; a slot without an expert adds nothing.
// Bound by memory: 4096 x 8 rows of 2048 in 56 us, 5.1 TB/s, a large copy's rate.
__global__ __launch_bounds__(256) void combine_kernel(const float* __restrict__ part, int64_t ldp,
                                                      const float* __restrict__ weights, const int* __restrict__ ids,
                                                      bf16_t* __restrict__ y, int64_t ldy, int64_t t, int64_t n,
                                                      int top_k, int experts) {
  const int64_t cols = ldp / 4;
  for (int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x; i < t * cols; i += (int64_t)gridDim.x * 256) {
    const int64_t tok = i / cols, c = 4 * (i % cols);
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    for (int j = 0; j < top_k; ++j) {
      const int64_t pair = tok * top_k + j;
      const int e = ids[pair];
      if (e >= 0 && e < experts) fma4(v, *reinterpret_cast<const f32x4*>(part + pair * ldp + c), weights[pair]);
    }
    store4_bf16(y + tok * ldy + c, v, n - c);
  }
}

// ---------------------------------------------------------------- host

struct Shape {
  int64_t t, h, i;
  int top_k, experts;
  int tune = ff_tuning(FF_TUNE_MOE_TILE);  // read once: the workspace's layout and the launches go by the same value
  int64_t pairs() const { return t * top_k; }
  int kth() const { return (int)((h + kBlock - 1) / kBlock); }
  int kti() const { return (int)((i + kBlock - 1) / kBlock); }
  // Up to 32 pairs they are taken one by one (128 experts, 8 a token, h 2048, i 768, us: 4 tokens
  // 36.9 against 40.0 on tiles, 8 tokens 68.8 against 54.0).
  // The row has to fit in LDS and either grid's threads in 32 bits.
  bool by_pair() const {
    return (tune ? tune == 1 : pairs() <= 32) && (int64_t)kth() * kBlock <= kInlineCodes &&
           pairs() * 8 * (kth() > kti() ? kth() : kti()) < (1 << 22);
  }
};

int64_t align256(int64_t b) { return (b + 255) / 256 * 256; }

// Workspace regions, in bytes from its start.
struct Layout {
  int64_t h, off, list, q, qs, part, ldp, total;
  explicit Layout(const Shape& s) {
    const int64_t pairs = s.pairs();
    h = 0;
    total = align256(pairs * s.kti() * kBlock * 2);
    off = list = q = qs = part = 0;
    ldp = (s.h + 3) / 4 * 4;
    if (s.by_pair()) return;
    const auto take = [&](int64_t bytes) {
      const int64_t at = total;
      total += align256(bytes);
      return at;
    };
    off = take((s.experts + 1) * 4);
    list = take(pairs * 4);
    q = take(s.t * s.kth() * kBlock);
    qs = take(s.t * s.kth() * 4);
    part = take(pairs * ldp * 4);
  }
};

// Sizes under which 32-bit offsets hold: one matrix of an expert, with the loads of some
// steps past its end, the rows' codes, and the threads of every grid (32 rows x 64 channels
// a workgroup at the least).
int check_shape(const char* who, int64_t t, int64_t top_k, int64_t experts, int64_t h, int64_t i) {
  constexpr int64_t kMax = 1ll << 32;
  FF_REQUIRE(t >= 0 && top_k > 0 && experts > 0 && experts <= kMaxExperts && h > 0 && i > 0 && h <= (1 << 24) &&
                 i <= (1 << 24) && top_k <= 1024 && t < (1 << 24),
             "%s: bad sizes t=%lld top_k=%lld experts=%lld h=%lld i=%lld", who, (long long)t, (long long)top_k,
             (long long)experts, (long long)h, (long long)i);
  const int64_t hb = (h + kBlock - 1) / kBlock, ib = (i + kBlock - 1) / kBlock;
  FF_REQUIRE(hb * ib * kBlock * kBlock < kMax / 2 && ib * kBlock * (hb + 8) * kBlock < kMax &&
                 hb * kBlock * (ib + 8) * kBlock < kMax && t * (hb + 8) * kBlock < kMax &&
                 (t * top_k / 32 + experts) * ((h > i ? h : i) / 64 + 2) < (1 << 24),
             "%s: bad sizes t=%lld top_k=%lld experts=%lld h=%lld i=%lld", who, (long long)t, (long long)top_k,
             (long long)experts, (long long)h, (long long)i);
  return FF_OK;
}

template <int BM, int CWG, int PG, int CWD, int PD>
void launch_tiles(const Shape& s, uint8_t* w, const Layout& l, const void* gate_up, const float* gate_up_scales,
                  const void* down, const float* down_scales, hipStream_t st) {
  const int tiles = (int)(s.pairs() / BM + (s.pairs() < s.experts ? s.pairs() : s.experts));
  const int nfi = s.kti() * 8, nfh = (int)((s.h + 15) / 16);
  const int* off = (const int*)(w + l.off);
  const int* list = (const int*)(w + l.list);
  const int tg = (nfi + CWG / 8 - 1) / (CWG / 8), td = (nfh + CWD / 4 - 1) / (CWD / 4);
  hipLaunchKernelGGL((gate_up_tile_kernel<BM, CWG, PG>), dim3((unsigned)(tiles * tg)), dim3(kTileThreads), 0, st,
                     w + l.q, (const float*)(w + l.qs), off, list, (const uint8_t*)gate_up, gate_up_scales,
                     (bf16_t*)(w + l.h), s.t, s.top_k, s.experts, s.kth(), nfi, tg);
  hipLaunchKernelGGL((down_tile_kernel<BM, CWD, PD>), dim3((unsigned)(tiles * td)), dim3(kTileThreads), 0, st,
                     (const bf16_t*)(w + l.h), off, list, (const uint8_t*)down, down_scales, (float*)(w + l.part),
                     l.ldp, s.h, s.experts, s.kti(), nfh, td);
}

}  // namespace

extern "C" int ff_moe_route(const void* logits, int logits_f32, int64_t ld, const float* bias, float* weights, int* ids,
                            int64_t t, int64_t experts, int64_t top_k, int sigmoid, int64_t groups, int64_t top_groups,
                            int renormalize, double scale, ff_stream_t stream) {
  FF_REQUIRE(t >= 0 && t < (1ll << 25) && experts > 0 && experts <= kMaxExperts && ld >= 0 && top_k > 0 &&
                 top_k <= 64 && top_k <= experts && groups > 0 && groups <= 64 && experts % groups == 0 &&
                 top_groups > 0 && top_groups <= groups && top_groups * (experts / groups) >= top_k,
             "ff_moe_route: bad sizes t=%lld experts=%lld top_k=%lld groups=%lld top_groups=%lld", (long long)t,
             (long long)experts, (long long)top_k, (long long)groups, (long long)top_groups);
  if (t == 0) return FF_OK;
  FF_REQUIRE(logits && weights && ids, "ff_moe_route: null pointer");
  FF_REQUIRE(ff_aligned(logits, logits_f32 ? 4 : 2), "ff_moe_route: alignment");
  const hipStream_t st = (hipStream_t)stream;
  const auto go = [&](auto LPR_, auto EPL_) {
    constexpr int LPR = decltype(LPR_)::value, EPL = decltype(EPL_)::value, rows = kRouteWaves * 64 / LPR;
    const dim3 grid((unsigned)((t + rows - 1) / rows)), block(64 * kRouteWaves);
    const auto run = [&](auto F32_, auto BIAS_) {
      hipLaunchKernelGGL((route_kernel<LPR, EPL, decltype(F32_)::value, decltype(BIAS_)::value>), grid, block, 0, st,
                         logits, ld, bias, weights, ids, t, (int)experts, (int)top_k, sigmoid, (int)groups,
                         (int)top_groups, renormalize, scale);
    };
    using Yes = std::true_type;
    using No = std::false_type;
    if (logits_f32) bias ? run(Yes{}, Yes{}) : run(Yes{}, No{});
    else bias ? run(No{}, Yes{}) : run(No{}, No{});
  };
  using std::integral_constant;
  using L16 = integral_constant<int, 16>;
  using L64 = integral_constant<int, 64>;
  if (t >= 1024 && experts <= 256 && groups <= 16 && top_k <= 16) {
    if (experts <= 64) go(L16{}, integral_constant<int, 4>{});
    else if (experts <= 128) go(L16{}, integral_constant<int, 8>{});
    else if (experts <= 192) go(L16{}, integral_constant<int, 12>{});
    else go(L16{}, integral_constant<int, 16>{});
  } else if (experts <= 64) {
    go(L64{}, integral_constant<int, 1>{});
  } else if (experts <= 128) {
    go(L64{}, integral_constant<int, 2>{});
  } else if (experts <= 256) {
    go(L64{}, integral_constant<int, 4>{});
  } else if (experts <= 512) {
    go(L64{}, integral_constant<int, 8>{});
  } else {
    go(L64{}, integral_constant<int, 16>{});
  }
  FF_LAUNCH_CHECK("ff_moe_route");
  return FF_OK;
}

extern "C" int ff_moe_experts_workspace(int64_t t, int64_t top_k, int64_t experts, int64_t h, int64_t i,
                                        int64_t* bytes) {
  FF_REQUIRE(bytes, "ff_moe_experts_workspace: null pointer");
  const int rc = check_shape("ff_moe_experts_workspace", t, top_k, experts, h, i);
  if (rc != FF_OK) return rc;
  *bytes = Layout(Shape{t, h, i, (int)top_k, (int)experts}).total;
  return FF_OK;
}

extern "C" int ff_moe_experts(const void* x, int64_t ldx, const float* weights, const int* ids, const void* gate_up,
                              const float* gate_up_scales, const void* down, const float* down_scales, void* y,
                              int64_t ldy, int64_t t, int64_t top_k, int64_t experts, int64_t h, int64_t i,
                              void* workspace, int64_t workspace_bytes, ff_stream_t stream) {
  const int rc = check_shape("ff_moe_experts", t, top_k, experts, h, i);
  if (rc != FF_OK || t == 0) return rc;
  FF_REQUIRE(x && weights && ids && gate_up && gate_up_scales && down && down_scales && y,
             "ff_moe_experts: null pointer");
  FF_REQUIRE(ldx >= 0 && ldy >= h, "ff_moe_experts: bad strides ldx=%lld ldy=%lld", (long long)ldx, (long long)ldy);
  FF_REQUIRE(ff_aligned(x, 2) && ff_aligned(y, 2) && ff_aligned(gate_up, 16) && ff_aligned(down, 16),
             "ff_moe_experts: alignment");
  const Shape s{t, h, i, (int)top_k, (int)experts};
  const Layout l(s);
  FF_REQUIRE(workspace && workspace_bytes >= l.total && ff_aligned(workspace, 256),
             "ff_moe_experts: workspace of %lld bytes needed", (long long)l.total);
  const hipStream_t st = (hipStream_t)stream;
  uint8_t* w = (uint8_t*)workspace;
  const int nfi = s.kti() * 8, nfh = (int)((h + 15) / 16);
  const int vec = ff_aligned(x, 16) && ldx % 8 == 0;
  if (s.by_pair()) {
    hipLaunchKernelGGL(gate_up_pair_kernel, dim3((unsigned)(s.pairs() * nfi)), dim3(kThreads), 0, st, (const bf16_t*)x,
                       ldx, vec, h, ids, (const uint8_t*)gate_up, gate_up_scales, (bf16_t*)(w + l.h), (int)top_k,
                       (int)experts, s.kth(), nfi);
    hipLaunchKernelGGL(down_pair_kernel, dim3((unsigned)(t * nfh)), dim3(kDownThreads), 0, st, (const bf16_t*)(w + l.h),
                       weights, ids, (const uint8_t*)down, down_scales, (bf16_t*)y, ldy, h, (int)top_k, (int)experts,
                       s.kti(), nfh);
    FF_LAUNCH_CHECK("ff_moe_experts");
    return FF_OK;
  }
  const int64_t quant = (t + kPlanThreads / 16 - 1) / (kPlanThreads / 16) * s.kth();
  hipLaunchKernelGGL(plan_kernel, dim3((unsigned)(experts + (quant < (1 << 20) ? quant : (1 << 20)))),
                     dim3(kPlanThreads), 0, st, ids, (int)s.pairs(), (int)experts, (int*)(w + l.off), (int*)(w + l.list),
                     (const bf16_t*)x, ldx, vec, t, h, s.kth(), w + l.q, (float*)(w + l.qs));
  // Rows of an expert on average: with few, tiles of 32 rows (us on 32- and 64-row tiles, 128
  // experts, 8 a token, h 2048, i 768: 8 tokens 54.0 and 61.7, 32 tokens 101 and 111, 128 tokens
  // 122 and 121, 512 tokens 163 and 155, 4096 tokens 581 and 429).
  if (s.tune ? s.tune == 2 : s.pairs() / experts < 8)
    launch_tiles<32, 32, 3, 32, 2>(s, w, l, gate_up, gate_up_scales, down, down_scales, st);
  else
    launch_tiles<64, 64, 3, 64, 1>(s, w, l, gate_up, gate_up_scales, down, down_scales, st);
  const int64_t grid = (t * (l.ldp / 4) + 255) / 256;
  hipLaunchKernelGGL(combine_kernel, dim3((unsigned)(grid < (1 << 20) ? grid : (1 << 20))), dim3(256), 0, st,
                     (const float*)(w + l.part), l.ldp, weights,
                     ids, (bf16_t*)y, ldy, t, h, (int)top_k, (int)experts);
  FF_LAUNCH_CHECK("ff_moe_experts");
  return FF_OK;
}
