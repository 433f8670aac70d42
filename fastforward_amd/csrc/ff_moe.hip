// Mixture-of-experts operators for gfx950: routing (the experts of each token and
// their weights) and the chosen experts' products on block-scaled FP8 weights
// (ff_block.h states the format).
//
// y[t] = sum_j w[t, j] D_e (silu(G_e x[t]) * (U_e x[t])), e = ids[t, j]. The rows x
// are quantised per 128 channels as the linear's rows are; the SwiGLU's values go
// into the down products as bf16 (relative error 2^-9 each, below the output's own
// rounding): quantised again, a value next to a border between two e4m3 codes
// would move by 1/16 with the last bit of a sum. Sums stay fp32 throughout, and
// their order depends on the shapes alone.
//
// Few (token, expert) pairs: two launches. gate_up: a workgroup per pair and 16
// channels, the row quantised in the workgroup; down: a workgroup per token and 16
// channels, its waves sharing the k steps of all the token's experts, so the
// weighted sum over experts needs no launch of its own.
// More pairs: they are ordered by expert (plan), the rows quantised once, and row
// tiles that belong to one expert each run both products; the down products of a
// token's experts are added by a last launch in the order of the token's list.
#include "ff_block.h"

using namespace ff;

namespace {

constexpr int kThreads = 512, kWaves = kThreads / 64;
constexpr int kMaxExperts = 1024;
constexpr int kInlineCodes = 49152;  // codes of the row that a gate_up workgroup quantises

// ---------------------------------------------------------------- routing

constexpr int kRouteRows = 4;  // rows (one wave each) per workgroup

template <int CTRL>
__device__ __forceinline__ double dpp64(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, 0xF, 0xF, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, 0xF, 0xF, false);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

// f over the 64 lanes, the same bits in every lane (each step combines a lane with its partner).
template <typename F>
__device__ __forceinline__ double wave_reduce64(double v, F&& f) {
  v = f(v, dpp64<kDppXor1>(v));
  v = f(v, dpp64<kDppXor2>(v));
  v = f(v, dpp64<kDppHalfMirror>(v));
  v = f(v, dpp64<kDppRowMirror>(v));
  v = f(v, __shfl_xor(v, 16));
  return f(v, __shfl_xor(v, 32));
}

// One wave per row; lane l holds experts l, l + 64, ... Scores, sums and the
// comparisons between experts are 64-bit: in 32 bits, scores that lie next to
// each other change places with the last bit of exp().
template <int EPL, bool F32>
__global__ __launch_bounds__(64 * kRouteRows) void route_kernel(
    const void* __restrict__ logits, int64_t ld, const float* __restrict__ bias, float* __restrict__ weights,
    int* __restrict__ ids, int64_t t, int experts, int top_k, int sigmoid, int groups, int top_groups, int renormalize,
    float scale) {
  __shared__ double sc[kRouteRows][EPL * 64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t row = blockIdx.x * (int64_t)kRouteRows + wave;
  if (row >= t) return;  // waves share nothing: LDS rows are per wave
  const double kNone = -__builtin_inf();
  const auto maximum = [](double a, double b) { return a > b ? a : b; };
  double p[EPL], c[EPL];
  bool bad = false;
  double top = kNone;
#pragma unroll
  for (int v = 0; v < EPL; ++v) {
    const int e = lane + 64 * v;
    float l = -__builtin_inff();
    if (e < experts) {
      if constexpr (F32) l = reinterpret_cast<const float*>(logits)[row * ld + e];
      else l = bf16_to_f32(reinterpret_cast<const bf16_t*>(logits)[row * ld + e]);
    }
    bad |= l != l || (!sigmoid && l == __builtin_inff());
    p[v] = (double)l;
    top = maximum(top, p[v]);
  }
  if (sigmoid) {
#pragma unroll
    for (int v = 0; v < EPL; ++v) {
      c[v] = p[v];
      p[v] = 1.0 / (1.0 + exp(-p[v]));
    }
  } else {
    top = wave_reduce64(top, maximum);
    double sum = 0;
#pragma unroll
    for (int v = 0; v < EPL; ++v) {
      c[v] = p[v];
      p[v] = p[v] == kNone ? 0.0 : exp(p[v] - top);
      sum += p[v];
    }
    sum = wave_reduce64(sum, [](double a, double b) { return a + b; });
#pragma unroll
    for (int v = 0; v < EPL; ++v) p[v] = sum > 0 ? p[v] / sum : 0.0;
  }
  // choice score: -inf for experts that are switched off
#pragma unroll
  for (int v = 0; v < EPL; ++v) {
    const int e = lane + 64 * v;
    const bool off = c[v] == kNone;
    const double b = bias && e < experts ? (double)bias[e] : 0.0;
    bad |= b != b;
    c[v] = off ? kNone : p[v] + b;
  }
  int* out_id = ids + row * top_k;
  float* out_w = weights + row * top_k;
  if (__ballot(bad)) {  // a NaN (or a softmax over +inf) shows in every weight of the row
    for (int j = lane; j < top_k; j += 64) {
      out_id[j] = j;
      out_w[j] = __builtin_nanf("");
    }
    return;
  }
  if (groups > 1) {
    const int per = experts / groups;
#pragma unroll
    for (int v = 0; v < EPL; ++v) sc[wave][lane + 64 * v] = c[v];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    double best = kNone, second = kNone;
    if (lane < groups)
      for (int m = 0; m < per; ++m) {
        const double s = sc[wave][lane * per + m];
        if (s > best) {
          second = best;
          best = s;
        } else if (s > second) {
          second = s;
        }
      }
    if (bias && second != kNone) best += second;
    int rank = 0;  // groups ahead of this lane's
    for (int o = 0; o < groups; ++o) {
      const double s = __shfl(best, o);
      rank += s > best || (s == best && o < lane);
    }
    const uint64_t keep = __ballot(lane < groups && rank < top_groups);
#pragma unroll
    for (int v = 0; v < EPL; ++v) {
      const int e = lane + 64 * v;
      if (e < experts && !(keep >> (e / per) & 1)) c[v] = kNone;
    }
  }
  double total = 0, mine_w = 0;
  int mine_id = -1;
  for (int j = 0; j < top_k; ++j) {
    double best = kNone;
#pragma unroll
    for (int v = 0; v < EPL; ++v) best = maximum(best, c[v]);
    best = wave_reduce64(best, maximum);
    int id = -1;
    double w = 0;
    if (best != kNone) {  // the lowest expert with that score: experts of one v lie below those of the next
#pragma unroll
      for (int v = EPL - 1; v >= 0; --v) {
        const uint64_t hit = __ballot(c[v] == best);
        if (hit) id = 64 * v + __builtin_ctzll(hit);
      }
#pragma unroll
      for (int v = 0; v < EPL; ++v)
        if (id / 64 == v) {
          w = __shfl(p[v], id % 64);
          if (lane == id % 64) c[v] = kNone;
        }
    }
    total += w;
    if (lane == j) {
      mine_w = w;
      mine_id = id;
    }
  }
  if (lane < top_k) {
    if (renormalize) mine_w = total > 0 ? mine_w / total : 0.0;
    out_id[lane] = mine_id;
    out_w[lane] = (float)(mine_w * (double)scale);
  }
}

// ---------------------------------------------------------------- pairs by expert

// One workgroup per expert: pairs p = token * top_k + slot of the expert in rising
// order to list[off[e] ..), off[e] = pairs of lower experts. Every workgroup reads
// all ids (a few hundred KB from L2 at most) and needs nothing from the others: no
// counters in memory, no order of arrival. ids outside [0, experts) are in no list.
constexpr int kPlanThreads = 1024, kPlanWaves = kPlanThreads / 64;
__global__ __launch_bounds__(kPlanThreads) void plan_kernel(const int* __restrict__ ids, int pairs, int experts,
                                                            int* __restrict__ off, int* __restrict__ list) {
  __shared__ int below[kPlanWaves], equal[kPlanWaves];
  const int e = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int seg = (pairs + kPlanWaves - 1) / kPlanWaves;
  const int lo = min(pairs, wave * seg), hi = min(pairs, lo + seg);
  int nb = 0, ne = 0;
  for (int i = lo + lane; i < hi; i += 64) {
    const int id = ids[i];
    nb += id >= 0 && id < e;
    ne += id == e;
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
  for (int i0 = lo; i0 < hi; i0 += 64) {
    const int i = i0 + lane;
    const bool hit = i < hi && ids[i] == e;
    const uint64_t b = __ballot(hit);
    if (hit) list[base + __builtin_popcountll(b & ((1ull << lane) - 1))] = i;
    base += __builtin_popcountll(b);
  }
}

// ---------------------------------------------------------------- gate/up + SwiGLU

// Adds the waves' sums of slot t (a lane's 4 values of one fragment pair) in wave order.
template <int SLOTS>
__device__ __forceinline__ f32x4 sum_waves(const f32x4* red, int t) {
  f32x4 v = red[t];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) v += red[w * SLOTS + t];
  return v;
}

// 16 RI rows of one expert x 16 channels: gate and up fragment of the channels,
// k steps shared by the waves. PAIR: blockIdx.y is the pair itself and the
// workgroup quantises its row. Weights of an expert: gate then up, each nf
// fragments x kt_n k steps; scales (2, nf / 8, kt_n).
template <int RI, bool PAIR>
__global__ __launch_bounds__(kThreads) void gate_up_kernel(
    const bf16_t* __restrict__ x, int64_t ldx, int vec, int64_t h_n, const uint8_t* __restrict__ q,
    const float* __restrict__ qs, const int* __restrict__ ids, const int* __restrict__ off,
    const int* __restrict__ list, const uint8_t* __restrict__ wp, const float* __restrict__ ws,
    bf16_t* __restrict__ h, int64_t t_n, int top_k, int experts, int kt_n, int nf) {
  constexpr int PF = RI == 4 ? 2 : 4;
  constexpr int kLds = PAIR ? kInlineCodes + 4 * kInlineCodes / kBlock : kWaves * RI * 2 * 64 * 16;
  __shared__ __align__(16) uint8_t smem[kLds];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r16 = lane & 15, g = lane >> 4;
  const int c = blockIdx.x % nf, tile = blockIdx.x / nf;
  int e, row0, rows;
  if constexpr (PAIR) {
    row0 = tile;
    rows = 1;
    e = ids[tile];
    if (e < 0 || e >= experts) return;
  } else {
    if (!find_tile(off, experts, 16 * RI, tile, &e, &row0, &rows)) return;
  }
  const int64_t matrix = (int64_t)nf * kt_n * 2048;
  const uint8_t* fg = wp + 2 * e * matrix + (int64_t)c * 2048;
  const float* sg = ws + ((int64_t)2 * e * (nf / 8) + c / 8) * kt_n;
  const int64_t sup = (int64_t)(nf / 8) * kt_n;
  int64_t row[RI];
#pragma unroll
  for (int i = 0; i < RI; ++i) row[i] = PAIR ? 0 : list[row0 + min(16 * i + r16, rows - 1)] / top_k;
  i32x8 wq[PF][2], xq[PF][RI];
  float xs[PF][RI], wsc[PF][2];
  const int mine = (kt_n - wave + kWaves - 1) / kWaves;
  f32x4 acc[RI][2];
#pragma unroll
  for (int i = 0; i < RI; ++i) acc[i][0] = acc[i][1] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int b = 0; b < mine || (PAIR && b == 0); b += PF) {
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
    if constexpr (PAIR) {
      if (b == 0) {
        const bf16_t* src = x + (int64_t)(tile / top_k) * ldx;
        for (int kt = threadIdx.x >> 4; kt < kt_n; kt += kThreads / 16) {
          float scale;
          const u32x2 code = quant_group16(src, h_n, kt, r16, vec, &scale);
          *reinterpret_cast<u32x2*>(smem + kt * kBlock + 8 * r16) = code;
          if (r16 == 0) reinterpret_cast<float*>(smem + kInlineCodes)[kt] = scale;
        }
        __syncthreads();
      }
    }
#pragma unroll
    for (int u = 0; u < PF; ++u)
      if (b + u < mine) {
        const int kt = wave + kWaves * (b + u);
#pragma unroll
        for (int i = 0; i < RI; ++i) {
          const uint8_t* src = PAIR ? smem + kt * kBlock : q + (row[i] * kt_n + kt) * kBlock;
          const i32x4v* p = reinterpret_cast<const i32x4v*>(src + 32 * g);
          xq[u][i] = join(p[0], p[1]);
          xs[u][i] = PAIR ? reinterpret_cast<const float*>(smem + kInlineCodes)[kt] : qs[(int64_t)kt * t_n + row[i]];
        }
      }
#pragma unroll
    for (int u = 0; u < PF; ++u)
      if (b + u < mine) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int i = 0; i < RI; ++i) fma4(acc[i][j], mfma_step(wq[u][j], xq[u][i]), xs[u][i] * wsc[u][j]);
      }
  }
  if constexpr (PAIR) __syncthreads();  // the codes are no longer read
  constexpr int kSlots = RI * 2 * 64;
  f32x4* red = reinterpret_cast<f32x4*>(smem);
#pragma unroll
  for (int i = 0; i < RI; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) red[wave * kSlots + (i * 2 + j) * 64 + lane] = acc[i][j];
  __syncthreads();
  if (threadIdx.x >= RI * 64) return;
  const int i = threadIdx.x >> 6;
  const f32x4 gate = sum_waves<kSlots>(red, i * 128 + lane), up = sum_waves<kSlots>(red, i * 128 + 64 + lane);
  if (16 * i + r16 >= rows) return;
  bf16_t* out = h + (int64_t)(row0 + 16 * i + r16) * (16 * nf) + 16 * c + 4 * g;
  *reinterpret_cast<u32x2*>(out) = pack4_bf16(silu(gate[0]) * up[0], silu(gate[1]) * up[1], silu(gate[2]) * up[2],
                                              silu(gate[3]) * up[3]);
}

// ---------------------------------------------------------------- down

// This lane's operand of one k step: channels 128 kt + 32 g .. + 31 of a row of h.
__device__ __forceinline__ void load_h(u32x4 (&x)[4], const bf16_t* p) {
#pragma unroll
  for (int u = 0; u < 4; ++u) x[u] = reinterpret_cast<const u32x4*>(p)[u];
}

// PAIR: one token's y, 16 channels: the k steps of all its experts shared by the
// waves. All 16 result rows are the token's (every lane group reads the same row).
__global__ __launch_bounds__(kThreads) void down_pair_kernel(
    const bf16_t* __restrict__ h, const float* __restrict__ weights, const int* __restrict__ ids,
    const uint8_t* __restrict__ wp, const float* __restrict__ ws, bf16_t* __restrict__ y, int64_t ldy, int64_t n,
    int top_k, int experts, int kt_n, int nf) {
  constexpr int PF = 4;
  __shared__ f32x4 red[kWaves * 4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r16 = lane & 15, g = lane >> 4;
  const int f = blockIdx.x % nf, tok = blockIdx.x / nf;
  const int64_t matrix = (int64_t)nf * kt_n * 2048;
  const int64_t nb = (n + kBlock - 1) / kBlock;
  const int steps = top_k * kt_n;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int b = wave; b < steps; b += kWaves * PF) {
    i32x8 wq[PF];
    u32x4 xh[PF][4];
    float s[PF];
#pragma unroll
    for (int u = 0; u < PF; ++u) {
      const int at = b + kWaves * u;
      s[u] = 0.f;
      if (at < steps) {
        const int pair = tok * top_k + at / kt_n, kt = at % kt_n;
        const int e = ids[pair];
        if (e >= 0 && e < experts) {
          wq[u] = load_frag(wp + e * matrix + ((int64_t)kt * nf + f) * 2048, lane);
          load_h(xh[u], h + ((int64_t)pair * kt_n + kt) * kBlock + 32 * g);
          s[u] = weights[pair] * ws[((int64_t)e * nb + f / 8) * kt_n + kt];
        }
      }
    }
#pragma unroll
    for (int u = 0; u < PF; ++u) {
      const int at = b + kWaves * u;
      if (at < steps) {
        const int e = ids[tok * top_k + at / kt_n];
        if (e >= 0 && e < experts) fma4(acc, mfma_step_bf16(wq[u], xh[u]), s[u]);
      }
    }
  }
  if (r16 == 0) red[wave * 4 + g] = acc;
  __syncthreads();
  if (threadIdx.x < 4) {
    const f32x4 v = sum_waves<4>(red, threadIdx.x);
    const int64_t c = 16 * (int64_t)f + 4 * threadIdx.x;
    if (c < n) store4_bf16(y + tok * ldy + c, v, n - c);
  }
}

// 16 RI rows of one expert x 16 NJ channels, k steps shared by the waves; fp32
// products to part[pair] (row stride ldp).
template <int RI, int NJ>
__global__ __launch_bounds__(kThreads) void down_kernel(const bf16_t* __restrict__ h, const int* __restrict__ off,
                                                        const int* __restrict__ list, const uint8_t* __restrict__ wp,
                                                        const float* __restrict__ ws, float* __restrict__ part,
                                                        int64_t ldp, int64_t n, int experts, int kt_n, int nf,
                                                        int tiles_n) {
  constexpr int PF = 2;
  constexpr int kSlots = RI * NJ * 64;
  __shared__ f32x4 red[kWaves * kSlots];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r16 = lane & 15, g = lane >> 4;
  const int f0 = blockIdx.x % tiles_n * NJ, tile = blockIdx.x / tiles_n;
  int e, row0, rows;
  if (!find_tile(off, experts, 16 * RI, tile, &e, &row0, &rows)) return;
  const int64_t matrix = (int64_t)nf * kt_n * 2048;
  const int64_t nb = (n + kBlock - 1) / kBlock;
  const int mine = (kt_n - wave + kWaves - 1) / kWaves;
  f32x4 acc[RI][NJ];
#pragma unroll
  for (int i = 0; i < RI; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int b = 0; b < mine; b += PF) {
    i32x8 wq[PF][NJ];
    u32x4 xh[PF][RI][4];
    float s[PF][NJ];
#pragma unroll
    for (int u = 0; u < PF; ++u)
      if (b + u < mine) {
        const int kt = wave + kWaves * (b + u);
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          const int f = min(f0 + j, nf - 1);
          wq[u][j] = load_frag(wp + e * matrix + ((int64_t)kt * nf + f) * 2048, lane);
          s[u][j] = ws[((int64_t)e * nb + f / 8) * kt_n + kt];
        }
#pragma unroll
        for (int i = 0; i < RI; ++i)
          load_h(xh[u][i], h + ((int64_t)(row0 + min(16 * i + r16, rows - 1)) * kt_n + kt) * kBlock + 32 * g);
      }
#pragma unroll
    for (int u = 0; u < PF; ++u)
      if (b + u < mine) {
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
          for (int i = 0; i < RI; ++i) fma4(acc[i][j], mfma_step_bf16(wq[u][j], xh[u][i]), s[u][j]);
      }
  }
#pragma unroll
  for (int i = 0; i < RI; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j) red[wave * kSlots + (i * NJ + j) * 64 + lane] = acc[i][j];
  __syncthreads();
  for (int t = threadIdx.x; t < kSlots; t += kThreads) {
    const f32x4 v = sum_waves<kSlots>(red, t);
    const int l = t & 63, i = t / 64 / NJ, j = t / 64 % NJ;
    const int r = 16 * i + (l & 15);
    const int64_t c = 16 * (int64_t)(f0 + j) + 4 * (l >> 4);
    if (r < rows && c < n) *reinterpret_cast<f32x4*>(part + (int64_t)list[row0 + r] * ldp + c) = v;
  }
}

// y[t] = sum_j w[t, j] part[t top_k + j], slots in order; a slot without an expert adds nothing.
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
  int64_t pairs() const { return t * top_k; }
  int kth() const { return (int)((h + kBlock - 1) / kBlock); }
  int kti() const { return (int)((i + kBlock - 1) / kBlock); }
  // Up to this many pairs they are taken one by one.
  bool by_pair() const { return pairs() <= 64 && (int64_t)kth() * kBlock <= kInlineCodes; }
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

// Bounds under which every grid below stays under 2^32 threads: the row tiles of
// either product (16 rows at least, one more for each expert) times its columns.
int check_shape(const char* who, int64_t t, int64_t top_k, int64_t experts, int64_t h, int64_t i) {
  FF_REQUIRE(t >= 0 && top_k > 0 && experts > 0 && experts <= kMaxExperts && h > 0 && i > 0 && h <= (1 << 24) &&
                 i <= (1 << 24) && top_k <= 1024 && t < (1 << 21) &&
                 (t * top_k / 16 + experts) * ((h > i ? h : i) / 16 + 8) < (1 << 23),
             "%s: bad sizes t=%lld top_k=%lld experts=%lld h=%lld i=%lld", who, (long long)t, (long long)top_k,
             (long long)experts, (long long)h, (long long)i);
  return FF_OK;
}

template <int RI>
void launch_experts(const Shape& s, uint8_t* w, const Layout& l, const void* gate_up, const float* gate_up_scales,
                    const void* down, const float* down_scales, hipStream_t st) {
  const int64_t tiles = s.pairs() / (16 * RI) + (s.pairs() < s.experts ? s.pairs() : s.experts);
  const int nfi = s.kti() * 8, nfh = (int)((s.h + 15) / 16);
  const int* off = (const int*)(w + l.off);
  const int* list = (const int*)(w + l.list);
  hipLaunchKernelGGL((gate_up_kernel<RI, false>), dim3((unsigned)(tiles * nfi)), dim3(kThreads), 0, st, nullptr, 0, 0,
                     s.h, w + l.q, (const float*)(w + l.qs), nullptr, off, list, (const uint8_t*)gate_up,
                     gate_up_scales, (bf16_t*)(w + l.h), s.t, s.top_k, s.experts, s.kth(), nfi);
  constexpr int NJ = 2;
  const int tn = (nfh + NJ - 1) / NJ;
  hipLaunchKernelGGL((down_kernel<RI, NJ>), dim3((unsigned)(tiles * tn)), dim3(kThreads), 0, st,
                     (const bf16_t*)(w + l.h), off, list, (const uint8_t*)down, down_scales, (float*)(w + l.part),
                     l.ldp, s.h, s.experts, s.kti(), nfh, tn);
}

}  // namespace

extern "C" int ff_moe_route(const void* logits, int logits_f32, int64_t ld, const float* bias, float* weights, int* ids,
                            int64_t t, int64_t experts, int64_t top_k, int sigmoid, int64_t groups, int64_t top_groups,
                            int renormalize, float scale, ff_stream_t stream) {
  FF_REQUIRE(t >= 0 && t < (1ll << 31) && experts > 0 && experts <= kMaxExperts && ld >= 0 && top_k > 0 &&
                 top_k <= 64 && top_k <= experts && groups > 0 && groups <= 64 && experts % groups == 0 &&
                 top_groups > 0 && top_groups <= groups && top_groups * (experts / groups) >= top_k,
             "ff_moe_route: bad sizes t=%lld experts=%lld top_k=%lld groups=%lld top_groups=%lld", (long long)t,
             (long long)experts, (long long)top_k, (long long)groups, (long long)top_groups);
  if (t == 0) return FF_OK;
  FF_REQUIRE(logits && weights && ids, "ff_moe_route: null pointer");
  FF_REQUIRE(ff_aligned(logits, logits_f32 ? 4 : 2), "ff_moe_route: alignment");
  const dim3 grid((unsigned)((t + kRouteRows - 1) / kRouteRows)), block(64 * kRouteRows);
  const hipStream_t st = (hipStream_t)stream;
  const auto go = [&](auto EPL_) {
    constexpr int EPL = decltype(EPL_)::value;
    if (logits_f32)
      hipLaunchKernelGGL((route_kernel<EPL, true>), grid, block, 0, st, logits, ld, bias, weights, ids, t, (int)experts,
                         (int)top_k, sigmoid, (int)groups, (int)top_groups, renormalize, scale);
    else
      hipLaunchKernelGGL((route_kernel<EPL, false>), grid, block, 0, st, logits, ld, bias, weights, ids, t,
                         (int)experts, (int)top_k, sigmoid, (int)groups, (int)top_groups, renormalize, scale);
  };
  if (experts <= 64) go(std::integral_constant<int, 1>{});
  else if (experts <= 128) go(std::integral_constant<int, 2>{});
  else if (experts <= 256) go(std::integral_constant<int, 4>{});
  else if (experts <= 512) go(std::integral_constant<int, 8>{});
  else go(std::integral_constant<int, 16>{});
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
    hipLaunchKernelGGL((gate_up_kernel<1, true>), dim3((unsigned)(s.pairs() * nfi)), dim3(kThreads), 0, st,
                       (const bf16_t*)x, ldx, vec, h, nullptr, nullptr, ids, nullptr, nullptr, (const uint8_t*)gate_up,
                       gate_up_scales, (bf16_t*)(w + l.h), t, (int)top_k, (int)experts, s.kth(), nfi);
    hipLaunchKernelGGL(down_pair_kernel, dim3((unsigned)(t * nfh)), dim3(kThreads), 0, st, (const bf16_t*)(w + l.h),
                       weights, ids, (const uint8_t*)down, down_scales, (bf16_t*)y, ldy, h, (int)top_k, (int)experts,
                       s.kti(), nfh);
    FF_LAUNCH_CHECK("ff_moe_experts");
    return FF_OK;
  }
  hipLaunchKernelGGL(plan_kernel, dim3((unsigned)experts), dim3(kPlanThreads), 0, st, ids, (int)s.pairs(), (int)experts,
                     (int*)(w + l.off), (int*)(w + l.list));
  const int rq = quant_rows_block(x, ldx, w + l.q, (float*)(w + l.qs), t, h, st);
  if (rq != FF_OK) return rq;
  const int64_t per = s.pairs() / experts;  // rows of an expert on average
  if (per <= 16) launch_experts<1>(s, w, l, gate_up, gate_up_scales, down, down_scales, st);
  else if (per <= 32) launch_experts<2>(s, w, l, gate_up, gate_up_scales, down, down_scales, st);
  else launch_experts<4>(s, w, l, gate_up, gate_up_scales, down, down_scales, st);
  const int64_t grid = (t * (l.ldp / 4) + 255) / 256;
  hipLaunchKernelGGL(combine_kernel, dim3((unsigned)(grid < (1 << 20) ? grid : (1 << 20))), dim3(256), 0, st,
                     (const float*)(w + l.part), l.ldp, weights,
                     ids, (bf16_t*)y, ldy, t, h, (int)top_k, (int)experts);
  FF_LAUNCH_CHECK("ff_moe_experts");
  return FF_OK;
}
