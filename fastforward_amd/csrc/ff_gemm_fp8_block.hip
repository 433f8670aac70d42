// Block-scaled FP8 linear for gfx950: setup (weight quantisation, packing), the
// row quantiser and the products y = x . W^T (ff_block.h states the format).
//
// Few rows (skinny_kernel): a workgroup of 8 waves owns 16 rows x 16 or 32 weight rows and
// its waves take the k steps in turn (wave w: steps w, w + 8, ..), so that even 4096
// columns make 256 workgroups that read the weights from every channel of memory; their
// sums are added through LDS in wave order. A few short rows are quantised in the same
// launch.
// More rows (tile_kernel): tiles of 32 x 64, 64 x 128 or 128 x 128 (ff_block_tile.h).
#include "ff_block_tile.h"

using namespace ff;

namespace {

constexpr int kSkinnyThreads = 512, kSkinnyWaves = kSkinnyThreads / 64;
constexpr int kRowsMaxCodes = 128 * kBlock;  // codes that the product's own launch quantises

// ---------------------------------------------------------------- setup

// One workgroup per 128 x 128 block: its largest magnitude, then its codes.
__global__ __launch_bounds__(256) void quant_weight_block_kernel(const bf16_t* __restrict__ w, uint8_t* __restrict__ q,
                                                                 float* __restrict__ scales, int64_t n, int64_t k,
                                                                 int kb) {
  __shared__ float red[4];
  const int64_t r0 = (int64_t)(blockIdx.x / kb) * kBlock, c0 = (int64_t)(blockIdx.x % kb) * kBlock;
  const int rows = (int)min((int64_t)kBlock, n - r0), cols = (int)min((int64_t)kBlock, k - c0);
  w += r0 * k + c0;
  float m = 0.f;
  for (int i = threadIdx.x; i < rows * kBlock; i += 256) {
    const int r = i / kBlock, c = i % kBlock;
    if (c < cols) m = fmaxf(m, fabsf(bf16_to_f32(w[r * k + c])));
  }
  m = block_max<4>(m, red);
  const float scale = fmaxf(m, 1e-12f) / 448.0f;
  q += r0 * k + c0;
  for (int i = threadIdx.x; i < rows * kBlock; i += 256) {
    const int r = i / kBlock, c = i % kBlock;
    if (c < cols) q[r * k + c] = (uint8_t)f32_to_e4m3(clamp448(bf16_to_f32(w[r * k + c]) / scale));
  }
  if (threadIdx.x == 0) scales[blockIdx.x] = scale;
}

// One thread per 16 packed bytes.
__global__ __launch_bounds__(256) void pack_block_kernel(const uint8_t* __restrict__ w, uint8_t* __restrict__ p,
                                                         int64_t batch, int64_t n, int64_t k, int64_t nf, int64_t kt_n,
                                                         int aligned) {
  const int64_t total = batch * nf * kt_n * 128;
  for (int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int l = (int)(i & 63), half = (int)(i >> 6) & 1;
    const int64_t f = (i >> 7) % nf, kt = (i >> 7) / nf % kt_n, b = (i >> 7) / nf / kt_n;
    const int64_t row = 16 * f + (l & 15), c = 128 * kt + 32 * (l >> 4) + 16 * half;
    u32x4 v = {0, 0, 0, 0};
    if (row < n) {
      const uint8_t* src = w + (b * n + row) * k + c;
      if (aligned && c + 16 <= k) {
        v = *reinterpret_cast<const u32x4*>(src);
      } else {
        uint32_t d[4] = {0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (c + e < k) d[e / 4] |= (uint32_t)src[e] << (8 * (e % 4));
        v = u32x4{d[0], d[1], d[2], d[3]};
      }
    }
    *reinterpret_cast<u32x4*>(p + 16 * i) = v;
  }
}

__global__ __launch_bounds__(256) void unpack_block_kernel(const uint8_t* __restrict__ p, uint8_t* __restrict__ w,
                                                           int64_t batch, int64_t n, int64_t k, int64_t nf,
                                                           int64_t kt_n) {
  const int64_t total = batch * n * k;
  for (int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t c = i % k, row = i / k % n, b = i / k / n;
    const int64_t kt = c / 128, f = row / 16;
    const int in = (int)(c % 128), l = (in / 32) * 16 + (int)(row % 16);
    w[i] = p[((b * kt_n + kt) * nf + f) * 2048 + (in / 16 % 2) * 1024 + 16 * l + in % 16];
  }
}

// ---------------------------------------------------------------- row quantiser

// 16 lanes a row and 128 channels: the block is read once and kept in registers between its
// maximum and its codes. Bound by memory: 4096 x 25600 in 66 us, 4.8 TB/s (a large copy:
// 5.2); 576 x 4096 3.5 us, about the shortest a launch takes.
__global__ __launch_bounds__(256) void quant_rows_block_kernel(const bf16_t* __restrict__ x, int64_t ldx,
                                                               uint8_t* __restrict__ q, float* __restrict__ scales,
                                                               int64_t rows, int64_t k, int kt_n, int vec) {
  const int64_t tiles = (rows + 15) / 16 * kt_n;
  for (int64_t i = blockIdx.x; i < tiles; i += gridDim.x) quant_rows_tile<16>(x, ldx, q, scales, rows, k, kt_n, vec, i);
}

// ---------------------------------------------------------------- few rows

// INLINE: the workgroup quantises the rows (at most 16) into LDS itself, while its first
// weights are on the way: a launch of its own would take longer than the whole product. Bound
// by the weights' bytes and the launch: 1 x 4096 x 4096 in 4.3 us (16.9 MB at 3.9 TB/s), 8 waves
// with four steps in flight each.
template <int NJ, bool INLINE>
__global__ __launch_bounds__(kSkinnyThreads) void skinny_kernel(
    const bf16_t* __restrict__ x, int64_t ldx, int vec, const uint8_t* __restrict__ q, const float* __restrict__ qs,
    const uint8_t* __restrict__ wp, const float* __restrict__ ws, bf16_t* __restrict__ y, int64_t ldy, int64_t m,
    int64_t n, int64_t k, int kt_n, int nf) {
  constexpr int PF = 4;  // k steps whose loads a wave has in flight
  constexpr int kSums = kSkinnyWaves * NJ * 64 * 16;  // bytes of the waves' sums
  constexpr int kLds = INLINE ? kRowsMaxCodes + 4 * kRowsMaxCodes / kBlock : kSums;
  static_assert(kSums <= kLds, "the sums reuse the codes' LDS");
  __shared__ __align__(16) uint8_t smem[kLds];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r16 = lane & 15, g = lane >> 4;
  const int f0 = blockIdx.x * NJ;
  const int64_t m0 = (int64_t)blockIdx.y * 16, row = min(m0 + r16, m - 1);
  const int mine = (kt_n - wave + kSkinnyWaves - 1) / kSkinnyWaves;  // this wave's k steps

  i32x8 wq[PF][NJ], xq[PF];
  float xs[PF], wsc[PF][NJ];
  const uint8_t* frag[NJ];
  const float* wscale[NJ];
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const int f = min(f0 + j, nf - 1);
    frag[j] = wp + (int64_t)f * 2048;
    wscale[j] = ws + (int64_t)(f / 8) * kt_n;
  }
  auto loadW = [&](int u, int kt) {
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      wq[u][j] = load_frag(frag[j] + (int64_t)kt * nf * 2048, lane);
      wsc[u][j] = wscale[j][kt];
    }
  };
  auto loadX = [&](int u, int kt) {
    const int64_t at = row * kt_n + kt;
    const i32x4v* p = reinterpret_cast<const i32x4v*>((INLINE ? smem : q) + at * kBlock + 32 * g);
    xq[u] = join(p[0], p[1]);
    xs[u] = INLINE ? reinterpret_cast<const float*>(smem + kRowsMaxCodes)[at] : qs[(int64_t)kt * m + row];
  };

  f32x4 acc[NJ];
#pragma unroll
  for (int j = 0; j < NJ; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};

  for (int b = 0; b < mine || (INLINE && b == 0); b += PF) {
#pragma unroll
    for (int u = 0; u < PF; ++u)
      if (b + u < mine) loadW(u, wave + kSkinnyWaves * (b + u));
    if constexpr (INLINE) {
      if (b == 0) {  // the first weights are in flight meanwhile
        for (int i = threadIdx.x >> 4; i < (int)m * kt_n; i += kSkinnyThreads / 16) {
          float scale;
          const u32x2 c = quant_group16(x + i / kt_n * ldx, k, i % kt_n, r16, vec, &scale);
          *reinterpret_cast<u32x2*>(smem + i * kBlock + 8 * r16) = c;
          if (r16 == 0) reinterpret_cast<float*>(smem + kRowsMaxCodes)[i] = scale;
        }
        __syncthreads();
      }
    }
#pragma unroll
    for (int u = 0; u < PF; ++u)
      if (b + u < mine) loadX(u, wave + kSkinnyWaves * (b + u));
#pragma unroll
    for (int u = 0; u < PF; ++u)
      if (b + u < mine) {
#pragma unroll
        for (int j = 0; j < NJ; ++j) fma4(acc[j], mfma_step(wq[u][j], xq[u]), xs[u] * wsc[u][j]);
      }
  }

  if constexpr (INLINE) __syncthreads();  // the codes are no longer read
  f32x4* red = reinterpret_cast<f32x4*>(smem);
#pragma unroll
  for (int j = 0; j < NJ; ++j) red[(wave * NJ + j) * 64 + lane] = acc[j];
  __syncthreads();
  for (int t = threadIdx.x; t < NJ * 64; t += kSkinnyThreads) {
    f32x4 v = red[t];
#pragma unroll
    for (int w = 1; w < kSkinnyWaves; ++w) v += red[w * NJ * 64 + t];
    const int64_t r = m0 + (t & 15), c = 16 * (int64_t)(f0 + t / 64) + 4 * (t % 64 / 16);
    if (r < m && c < n) store4_bf16(y + r * ldy + c, v, n - c);
  }
}

// ---------------------------------------------------------------- many rows

// BM x 4 CW tiles, KG groups of 4 waves that share the k steps of a tile. Tile order: groups
// of 8 row tiles, within a group row tiles fastest, so that the tiles an XCD runs at one
// time share rows and weights.
// 4096 x 5120 x 25600 on 128 x 128 tiles: 535 us, 2.0 PFLOP/s (a library product without block
// scales: 2.8). The matrix unit is busy 52 % of the time: the waves' fragments from LDS (64 KB a
// step and CU, 512 clocks, as long as its matrix instructions), the loads (32 KB, 512 clocks of
// the return path) and the adds (256 clocks) run beside it, not wholly overlapped. One tile of 128 x
// 64 a wave would halve the first, but leaves one wave a SIMD: 1.98 PFLOP/s. Short products
// are a chain of steps on few CUs: 333 x 1152 x 4304 on 32 x 64 tiles in two k groups 8.2 us,
// 576 x 6144 x 4096 24.6 us (240 tiles of 128 x 128).
template <int BM, int CW, int P, int D, int KG, int OCC>
__global__ __launch_bounds__(kTileThreads* KG, OCC) void tile_kernel(
    const uint8_t* __restrict__ q, const float* __restrict__ qs, const uint8_t* __restrict__ wp,
    const float* __restrict__ ws, bf16_t* __restrict__ y, int64_t ldy, int64_t m, int64_t n, int kt_n, int nf,
    int tiles_m, int tiles_n) {
  constexpr int RA = BM / 16, TJ = CW / 16, GM = 8;
  constexpr int kStages = KG * tile_smem<BM>(), kSums = (KG - 1) * kTileThreads * RA * TJ * 16;
  __shared__ __align__(1024) uint8_t smem[kStages > kSums ? kStages : kSums];  // the groups' sums reuse the stages
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r16 = lane & 15, g = lane >> 4, group = wave / 4;
  const int id = xcd_tile(blockIdx.x, tiles_m * tiles_n);
  const int first = id / (GM * tiles_n) * GM, in = id % (GM * tiles_n), gm = min(GM, tiles_m - first);
  const int64_t m0 = (int64_t)(first + in % gm) * BM;
  const int f0 = in / gm * (4 * TJ) + wave % 4 * TJ;
  const int per = (kt_n + KG - 1) / KG, k0 = group * per;
  TileWeights<TJ, 1> w{{wp}, (uint32_t)nf * min(kt_n, k0 + per) * 2048u, (uint32_t)nf * 2048u,
                       {ws + (int64_t)(min(f0, nf - 1) / 8) * kt_n}, {}};
#pragma unroll
  for (int j = 0; j < TJ; ++j) w.frag[j] = (uint32_t)(f0 + j) * 2048u;
  const int rows = (int)min((int64_t)BM, m - m0);
  const uint32_t kp = (uint32_t)kt_n * kBlock;
  f32x4 acc[RA][TJ];
  tile_mainloop<BM, CW, 1, P, D>(
      acc, smem + group * tile_smem<BM>(), kt_n, k0, per, q + m0 * kp, (uint32_t)rows * kp,
      [&](int r) { return (uint32_t)min(r, rows - 1) * kp; }, qs, (uint32_t)(4 * m) * kt_n,
      [&](int r) { return (uint32_t)m0 + min(r, rows - 1); }, (uint32_t)(4 * m), w);
  if constexpr (KG > 1) {  // the groups' sums, added in order
    f32x4* red = reinterpret_cast<f32x4*>(smem);
    __syncthreads();
    if (group > 0) {
#pragma unroll
      for (int i = 0; i < RA; ++i)
#pragma unroll
        for (int j = 0; j < TJ; ++j) red[(i * TJ + j) * (KG - 1) * kTileThreads + threadIdx.x - kTileThreads] = acc[i][j];
    }
    __syncthreads();
    if (group > 0) return;
#pragma unroll
    for (int i = 0; i < RA; ++i)
#pragma unroll
      for (int j = 0; j < TJ; ++j)
#pragma unroll
        for (int o = 0; o < KG - 1; ++o)
          acc[i][j] += red[((i * TJ + j) * (KG - 1) + o) * kTileThreads + threadIdx.x];
  }
#pragma unroll
  for (int i = 0; i < RA; ++i) {
    const int64_t r = m0 + 16 * i + r16;
    if (r >= m) continue;
#pragma unroll
    for (int j = 0; j < TJ; ++j) {
      const int64_t c = 16 * (int64_t)(f0 + j) + 4 * g;
      if (c < n) store4_bf16(y + r * ldy + c, acc[i][j], n - c);
    }
  }
}

inline bool rows_vec(const void* x, int64_t ldx) { return ff_aligned(x, 16) && ldx % 8 == 0; }

// 16 weight rows per workgroup while that leaves at most two workgroups per CU, else 32.
template <bool INLINE>
void launch_skinny(const bf16_t* x, int64_t ldx, const uint8_t* q, const float* qs, const uint8_t* wp, const float* ws,
                   bf16_t* y, int64_t ldy, int64_t m, int64_t n, int64_t k, hipStream_t st) {
  const int nf = (int)((n + 15) / 16), kt_n = (int)((k + kBlock - 1) / kBlock);
  const int64_t tiles_m = (m + 15) / 16;
  const int vec = rows_vec(x, ldx);
  if (tiles_m * nf <= 512)
    hipLaunchKernelGGL((skinny_kernel<1, INLINE>), dim3((unsigned)nf, (unsigned)tiles_m), dim3(kSkinnyThreads), 0, st, x,
                       ldx, vec, q, qs, wp, ws, y, ldy, m, n, k, kt_n, nf);
  else
    hipLaunchKernelGGL((skinny_kernel<2, INLINE>), dim3((unsigned)((nf + 1) / 2), (unsigned)tiles_m),
                       dim3(kSkinnyThreads), 0, st, x, ldx, vec, q, qs, wp, ws, y, ldy, m, n, k, kt_n, nf);
}

template <int BM, int CW, int P, int D, int KG>
void launch_tile(const void* q, const float* qs, const void* packed, const float* ws, void* y, int64_t ldy, int64_t m,
                 int64_t n, int kt_n, int nf, hipStream_t st) {
  const int64_t tm = (m + BM - 1) / BM, tn = (nf + CW / 4 - 1) / (CW / 4);
  hipLaunchKernelGGL((tile_kernel<BM, CW, P, D, KG, 2>), dim3((unsigned)(tm * tn)), dim3(kTileThreads * KG), 0, st,
                     (const uint8_t*)q, qs, (const uint8_t*)packed, ws, (bf16_t*)y, ldy, m, n, kt_n, nf, (int)tm,
                     (int)tn);
}

constexpr int64_t kMaxCodes = 1ll << 31;

}  // namespace

static int quant_rows_block(const void* x, int64_t ldx, void* q, float* scales, int64_t rows, int64_t k,
                            hipStream_t st) {
  const int64_t kt_n = (k + kBlock - 1) / kBlock;
  const int64_t grid = (rows + 15) / 16 * kt_n;
  hipLaunchKernelGGL(quant_rows_block_kernel, dim3((unsigned)(grid < (1 << 20) ? grid : (1 << 20))), dim3(256), 0, st,
                     (const bf16_t*)x, ldx, (uint8_t*)q, scales, rows, k, (int)kt_n, (int)rows_vec(x, ldx));
  FF_LAUNCH_CHECK("quant_rows_fp8_block");
  return FF_OK;
}

extern "C" int ff_quant_weight_fp8_block(const void* w, void* q, float* scales, int64_t n, int64_t k,
                                         ff_stream_t stream) {
  FF_REQUIRE(w && q && scales, "ff_quant_weight_fp8_block: null pointer");
  FF_REQUIRE(n > 0 && k > 0 && n < kMaxCodes && k < kMaxCodes, "ff_quant_weight_fp8_block: bad sizes");
  const int64_t kb = (k + kBlock - 1) / kBlock, nb = (n + kBlock - 1) / kBlock;
  FF_REQUIRE(nb * kb < (1 << 24), "ff_quant_weight_fp8_block: bad sizes");
  hipLaunchKernelGGL(quant_weight_block_kernel, dim3((unsigned)(nb * kb)), dim3(256), 0, (hipStream_t)stream,
                     (const bf16_t*)w, (uint8_t*)q, scales, n, k, (int)kb);
  FF_LAUNCH_CHECK("ff_quant_weight_fp8_block");
  return FF_OK;
}

extern "C" int ff_pack_weight_fp8_block(const void* w, void* packed, int64_t batch, int64_t n, int64_t k, int64_t n_pad,
                                        ff_stream_t stream) {
  FF_REQUIRE(w && packed, "ff_pack_weight_fp8_block: null pointer");
  FF_REQUIRE(batch > 0 && n > 0 && k > 0 && n_pad >= n && n_pad % 16 == 0 && n_pad < kMaxCodes && k < kMaxCodes,
             "ff_pack_weight_fp8_block: bad sizes");
  FF_REQUIRE(ff_aligned(packed, 16), "ff_pack_weight_fp8_block: alignment");
  const int64_t kt_n = (k + kBlock - 1) / kBlock, nf = n_pad / 16;
  const int64_t grid = (batch * nf * kt_n * 128 + 255) / 256;
  hipLaunchKernelGGL(pack_block_kernel, dim3((unsigned)(grid < (1 << 20) ? grid : (1 << 20))), dim3(256), 0,
                     (hipStream_t)stream, (const uint8_t*)w, (uint8_t*)packed, batch, n, k, nf, kt_n,
                     (int)(ff_aligned(w, 16) && k % 16 == 0));
  FF_LAUNCH_CHECK("ff_pack_weight_fp8_block");
  return FF_OK;
}

extern "C" int ff_unpack_weight_fp8_block(const void* packed, void* w, int64_t batch, int64_t n, int64_t k,
                                          int64_t n_pad, ff_stream_t stream) {
  FF_REQUIRE(w && packed, "ff_unpack_weight_fp8_block: null pointer");
  FF_REQUIRE(batch > 0 && n > 0 && k > 0 && n_pad >= n && n_pad % 16 == 0 && n_pad < kMaxCodes && k < kMaxCodes,
             "ff_unpack_weight_fp8_block: bad sizes");
  const int64_t grid = (batch * n * k + 255) / 256;
  hipLaunchKernelGGL(unpack_block_kernel, dim3((unsigned)(grid < (1 << 20) ? grid : (1 << 20))), dim3(256), 0,
                     (hipStream_t)stream, (const uint8_t*)packed, (uint8_t*)w, batch, n, k, n_pad / 16,
                     (k + kBlock - 1) / kBlock);
  FF_LAUNCH_CHECK("ff_unpack_weight_fp8_block");
  return FF_OK;
}

extern "C" int ff_quant_rows_fp8_block(const void* x, int64_t ldx, void* q, float* scales, int64_t rows, int64_t k,
                                       ff_stream_t stream) {
  FF_REQUIRE(rows >= 0 && rows < kMaxCodes && k > 0 && k < kMaxCodes && ldx >= 0, "ff_quant_rows_fp8_block: bad sizes");
  if (rows == 0) return FF_OK;
  FF_REQUIRE(x && q && scales, "ff_quant_rows_fp8_block: null pointer");
  FF_REQUIRE(ff_aligned(x, 2) && ff_aligned(q, 16), "ff_quant_rows_fp8_block: alignment");
  return quant_rows_block(x, ldx, q, scales, rows, k, (hipStream_t)stream);
}

// Sizes under which 32-bit offsets hold: the packed weight, with the loads of some steps past
// its end, the codes of a row tile, the rows' scales, and the threads of a grid.
static int check_gemm(const char* who, const void* packed, const float* ws, const void* y, int64_t ldy, int64_t m,
                      int64_t n, int64_t k) {
  const int64_t n16 = (n + 15) / 16 * 16, kt_n = (k + kBlock - 1) / kBlock;
  FF_REQUIRE(m >= 0 && m < kMaxCodes && n > 0 && k > 0 && n < kMaxCodes && k < (1 << 24) && ldy >= n &&
                 n16 * kt_n * kBlock < kMaxCodes && n16 * (kt_n + 8) * kBlock < 2 * kMaxCodes &&
                 m * kt_n < (1ll << 29) && m * n < (1ll << 38),
             "%s: bad sizes m=%lld n=%lld k=%lld", who, (long long)m, (long long)n, (long long)k);
  if (m == 0) return FF_OK;
  FF_REQUIRE(packed && ws && y, "%s: null pointer", who);
  FF_REQUIRE(ff_aligned(packed, 16) && ff_aligned(y, 2), "%s: alignment", who);
  return FF_OK;
}

// The kernel for quantised rows (us in a graph; columns: few-rows kernel, 32 x 64, 64 x 128,
// 128 x 128 tiles, 128 x 128 with two k groups):
//   m x n x k             few    32 x 64   64 x 128   128 x 128   two groups
//   7 x 4096 x 4096       3.8      6.8       11.9       19.4
//   16 x 2048 x 25600    17.6     26.2       59         99
//   7 x 8192 x 4096       5.9      6.9       12.0       19.4
//   7 x 12288 x 4096     11.5      8.8       12.3       19.5
//   32 x 6144 x 4096     11.5      6.9       12.1       20.0
//   128 x 4096 x 4096    21.9      7.5       12.8       20.6
//   333 x 1152 x 4304    22.5      7.8       13.1       22.8        19.4
//   7 x 19456 x 2560     11.6     12.0        9.8       13.8        13.9
//   176 x 6144 x 4096    70       16.2       13.1       21.4        20.4
//   300 x 4096 x 4096    70       16.4       13.1       20.6        20.2
//   1000 x 2048 x 1024   33       10.0        6.4        9.5        10.9
//   576 x 4096 x 4096             26.8       24.7       21.3        21.5
//   576 x 6144 x 4096   172       40.1       27.5       25.5        23.9
//   1280 x 2560 x 2560                       15.9       16.2        16.8
//   576 x 4096 x 12288            70.7       65.2       52.9        47.6
//   500 x 5120 x 25600                      111        105          88
//   1024 x 6144 x 4096            59.8       35.3       38.0        43.9
//   800 x 6144 x 4096                        33.8       37.6        42.7
//   1000 x 8192 x 4096                       45.4       42.4        46.6
//   576 x 24576 x 4096           140.6       94.5       79.2        89.8
//   1024 x 25600 x 5120 1390     309        179        162
// The larger tile reads less for a product and takes longer for a step. Both large ones take
// about the same time for every 256 tiles (a CU's share of one), the smaller 0.58 of the
// larger's: whichever needs less of it for the whole product. Two k groups put two waves on a
// SIMD where there is one 128 x 128 tile for a CU at most; at 32 k steps the exchange of
// their sums costs what that gains.
static int block_kernel(int64_t m, int64_t n, int64_t kt_n) {
  const int tune = ff_tuning(FF_TUNE_BLOCK_TILE);
  if (tune && m <= 65535 * 16 && m * n < (1ll << 31)) return tune;
  if (m <= 16 && n <= 8192) return 1;
  const auto tiles = [&](int64_t bm, int64_t bn) { return ((m + bm - 1) / bm) * ((n + bn - 1) / bn); };
  const int64_t small = tiles(64, 128), large = tiles(128, 128);
  if (58 * ((small + 255) / 256) > 100 * ((large + 255) / 256)) return large <= 256 && kt_n >= 64 ? 5 : 4;
  return small >= 128 ? 3 : 2;
}

static int gemm_block(const void* q, const float* qs, const void* packed, const float* ws, void* y, int64_t ldy,
                      int64_t m, int64_t n, int64_t k, hipStream_t st) {
  const int nf = (int)((n + 15) / 16), kt_n = (int)((k + kBlock - 1) / kBlock);
  switch (block_kernel(m, n, kt_n)) {
    case 1:
      launch_skinny<false>(nullptr, 0, (const uint8_t*)q, qs, (const uint8_t*)packed, ws, (bf16_t*)y, ldy, m, n, k, st);
      break;
    case 2: launch_tile<32, 16, 4, 2, 2>(q, qs, packed, ws, y, ldy, m, n, kt_n, nf, st); break;
    case 3: launch_tile<64, 32, 3, 1, 1>(q, qs, packed, ws, y, ldy, m, n, kt_n, nf, st); break;
    case 4: launch_tile<128, 32, 3, 1, 1>(q, qs, packed, ws, y, ldy, m, n, kt_n, nf, st); break;
    default: launch_tile<128, 32, 3, 1, 2>(q, qs, packed, ws, y, ldy, m, n, kt_n, nf, st); break;
  }
  FF_LAUNCH_CHECK("ff_gemm_fp8_block");
  return FF_OK;
}

extern "C" int ff_gemm_fp8_block(const void* q, const float* scales, const void* packed, const float* wscales, void* y,
                                 int64_t ldy, int64_t m, int64_t n, int64_t k, ff_stream_t stream) {
  const int rc = check_gemm("ff_gemm_fp8_block", packed, wscales, y, ldy, m, n, k);
  if (rc != FF_OK || m == 0) return rc;
  FF_REQUIRE(q && scales, "ff_gemm_fp8_block: null pointer");
  FF_REQUIRE(ff_aligned(q, 16), "ff_gemm_fp8_block: alignment");
  return gemm_block(q, scales, packed, wscales, y, ldy, m, n, k, (hipStream_t)stream);
}

// Whether m rows of k channels are quantised inside the product's launch. Each workgroup then
// does that work, so it is bounded per CU: 8192 columns are a workgroup or two for each. In a graph,
// weights from memory, us (in the launch / in one of their own): 4 x 4096 x 4096 8.2 / 8.4, 3 x
// 6144 x 4096 10.0 / 10.4, 4 x 4096 x 12288 19.7 / 15.3, 1 x 24576 x 4096 22.0 / 21.5, 2 x 24576 x
// 4096 24.0 / 21.5, 3 x 5120 x 8192 16.3 / 15.5; 6 x 2560 x 2560 6.1 / 6.4. A launch saved is also
// two to three us of the host's.
static bool rows_inline(int64_t m, int64_t n, int64_t k) {
  return m <= 16 && m * ((k + kBlock - 1) / kBlock) * ((n + 8191) / 8192) <= kRowsMaxCodes / kBlock;
}

static int64_t align256(int64_t b) { return (b + 255) / 256 * 256; }

extern "C" int ff_linear_fp8_block_workspace(int64_t m, int64_t n, int64_t k, int64_t* bytes) {
  FF_REQUIRE(bytes, "ff_linear_fp8_block_workspace: null pointer");
  FF_REQUIRE(m >= 0 && n > 0 && k > 0 && m < kMaxCodes && k < kMaxCodes, "ff_linear_fp8_block_workspace: bad sizes");
  const int64_t kt_n = (k + kBlock - 1) / kBlock;
  *bytes = rows_inline(m, n, k) ? 0 : align256(m * kt_n * kBlock) + m * kt_n * 4;
  return FF_OK;
}

extern "C" int ff_linear_fp8_block(const void* x, int64_t ldx, const void* packed, const float* wscales, void* y,
                                   int64_t ldy, int64_t m, int64_t n, int64_t k, void* workspace,
                                   int64_t workspace_bytes, ff_stream_t stream) {
  const int rc = check_gemm("ff_linear_fp8_block", packed, wscales, y, ldy, m, n, k);
  if (rc != FF_OK || m == 0) return rc;
  FF_REQUIRE(x, "ff_linear_fp8_block: null pointer");
  FF_REQUIRE(ff_aligned(x, 2) && ldx >= 0, "ff_linear_fp8_block: alignment");
  const hipStream_t st = (hipStream_t)stream;
  if (rows_inline(m, n, k)) {
    launch_skinny<true>((const bf16_t*)x, ldx, nullptr, nullptr, (const uint8_t*)packed, wscales, (bf16_t*)y, ldy, m,
                           n, k, st);
    FF_LAUNCH_CHECK("ff_linear_fp8_block");
    return FF_OK;
  }
  const int64_t codes = align256(m * ((k + kBlock - 1) / kBlock) * kBlock);
  int64_t need = 0;
  ff_linear_fp8_block_workspace(m, n, k, &need);
  FF_REQUIRE(workspace && workspace_bytes >= need && ff_aligned(workspace, 16),
             "ff_linear_fp8_block: workspace of %lld bytes needed", (long long)need);
  float* scales = (float*)((uint8_t*)workspace + codes);
  const int rq = quant_rows_block(x, ldx, workspace, scales, m, k, st);
  if (rq != FF_OK) return rq;
  return gemm_block(workspace, scales, packed, wscales, y, ldy, m, n, k, st);
}
