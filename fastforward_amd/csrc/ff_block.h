// Pieces shared by the block-scaled FP8 kernels: the row quantiser, the matrix
// instructions on fragment-packed e4m3 weights and the lookup of an expert's rows.
//
// Block-scaled FP8: a weight (n, k) is e4m3 codes with one fp32 scale for every
// 128 x 128 block (the last block of either side may be partial); a row of
// activations is e4m3 codes with one fp32 scale for every 128 channels. One
// v_mfma_f32_16x16x128_f8f6f4 sums exactly the 128 products that share a pair of
// scales, so a product of a k step is that instruction on a zero accumulator,
// followed by one fused multiply-add per value into the fp32 running sum.
//
// Packed weights (ff_pack_weight_fp8_block): rows padded to 16 (or more) and k to
// 128 with zero codes; fragment (f, kt) of rows [16 f, 16 f + 16) and k
// [128 kt, 128 kt + 128) is the 2048 bytes at (kt * NF + f) * 2048, NF the padded
// rows / 16; lane l = 16 g + r holds row 16 f + r, k 128 kt + 32 g .. + 15 at 16 l
// and + 16 .. + 31 at 1024 + 16 l (the layout of ff_pack_weight_fp8).
#pragma once

#include "ff_common.h"

namespace ff {

constexpr int kBlock = 128;  // rows and channels that share a scale

// Scale and codes of 8 of the 128 channels [128 kt, 128 kt + 128) of a bf16 row of
// k channels, lane s of 16 consecutive lanes holding channels 8 s .. + 7 (zeros
// past k): scale = max(amax, 1e-12) / 448, code = e4m3(x / scale), both quotients
// correctly rounded fp32. vec: the row may be read 16 bytes at a time. A NaN
// keeps its code and is not in amax; an infinity makes the scale infinite, its own code
// NaN and the block's other codes 0.
__device__ __forceinline__ u32x2 quant_group16(const bf16_t* __restrict__ row, int64_t k, int kt, int s, bool vec,
                                               float* scale) {
  const int64_t c = (int64_t)kt * kBlock + 8 * s;
  float v[8];
  if (vec && c + 8 <= k) {
    unpack8(*reinterpret_cast<const u32x4*>(row + c), v);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = c + e < k ? bf16_to_f32(row[c + e]) : 0.f;
  }
  float a = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) a = fmaxf(a, fabsf(v[e]));
  a = fmaxf(a, dpp<kDppXor1>(a));
  a = fmaxf(a, dpp<kDppXor2>(a));
  a = fmaxf(a, dpp<kDppHalfMirror>(a));
  a = fmaxf(a, dpp<kDppRowMirror>(a));
  const float sc = fmaxf(a, 1e-12f) / 448.0f;
  *scale = sc;
  // an infinite divisor would make the quotient's correction 0 * inf; with 0 in its place
  // and the reciprocal 0 the quotients are x * 0
  return quant8(v, sc == __builtin_inff() ? 0.0f : sc, 1.0f / sc);
}

// Codes q (rows, 128 kt_n) and scales (kt_n, rows) of ROWS rows x 128 channels by 16 ROWS
// threads, tile `i` of (rows / ROWS rounded up) x kt_n, channel blocks fastest. Scales have
// channel blocks slowest: the lanes of a product's row tile read neighbouring ones, and a
// tile's are whole 64-byte lines here.
template <int ROWS>
__device__ __forceinline__ void quant_rows_tile(const bf16_t* __restrict__ x, int64_t ldx, uint8_t* __restrict__ q,
                                                float* __restrict__ scales, int64_t rows, int64_t k, int kt_n, int vec,
                                                int64_t i) {
  const int s = threadIdx.x & 15;
  const int64_t row = i / kt_n * ROWS + (threadIdx.x >> 4);
  const int kt = (int)(i % kt_n);
  if (row >= rows) return;
  float scale;
  const u32x2 c = quant_group16(x + row * ldx, k, kt, s, vec, &scale);
  *reinterpret_cast<u32x2*>(q + (row * kt_n + kt) * kBlock + 8 * s) = c;
  if (s == 0) scales[(int64_t)kt * rows + row] = scale;
}

// The 128 products of one k step, from zero.
__device__ __forceinline__ f32x4 mfma_step(const i32x8& w, const i32x8& x) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
}

__device__ __forceinline__ i32x8 join(const i32x4v& lo, const i32x4v& hi) {
  return i32x8{lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
}

// Fragment at p (2048 bytes) of this lane.
__device__ __forceinline__ i32x8 load_frag(const uint8_t* p, int lane) {
  return join(*reinterpret_cast<const i32x4v*>(p + 16 * lane), *reinterpret_cast<const i32x4v*>(p + 1024 + 16 * lane));
}

// 8 e4m3 codes (two dwords) as bf16: exact, every e4m3 value is a bf16 value.
__device__ __forceinline__ bf16x8 e4m3_to_bf16x8(uint32_t a, uint32_t b) {
  const bf16x2_t p0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, false);
  const bf16x2_t p1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, true);
  const bf16x2_t p2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, false);
  const bf16x2_t p3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, true);
  return bf16x8{p0.x, p0.y, p1.x, p1.y, p2.x, p2.y, p3.x, p3.y};
}

// The same k step with bf16 activations: e4m3 weights converted in registers and
// four v_mfma_f32_16x16x32_bf16, instruction q taking channels 32 g + 8 q .. + 7
// of every lane group g (x[q] holds those of the lane's row).
__device__ __forceinline__ f32x4 mfma_step_bf16(const i32x8& w, const u32x4 (&x)[4]) {
  f32x4 t = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int q = 0; q < 4; ++q)
    t = __builtin_amdgcn_mfma_f32_16x16x32_bf16(e4m3_to_bf16x8((uint32_t)w[2 * q], (uint32_t)w[2 * q + 1]),
                                                __builtin_bit_cast(bf16x8, x[q]), t, 0, 0, 0);
  return t;
}

__device__ __forceinline__ void fma4(f32x4& acc, const f32x4& t, float s) {
#pragma unroll
  for (int e = 0; e < 4; ++e) acc[e] = __builtin_fmaf(t[e], s, acc[e]);
}

// bf16 of 4 consecutive values of which the first `left` exist.
__device__ __forceinline__ void store4_bf16(bf16_t* p, const f32x4& v, int64_t left) {
  if (left >= 4 && ((uintptr_t)p & 7) == 0) {
    *reinterpret_cast<u32x2*>(p) = pack4_bf16(v[0], v[1], v[2], v[3]);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < left) p[e] = (bf16_t)f32_to_bf16(v[e]);
  }
}

// Inclusive prefix sum over the 64 lanes (row shifts, then the row totals broadcast on).
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);  // row_shr:1
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // row_bcast:15 into rows 1 and 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);  // row_bcast:31 into rows 2 and 3
  return v;
}

// Logical tile of workgroup b of n: consecutive workgroups go to the 8 XCDs in turn, so
// that each XCD (one L2) takes a contiguous run of tiles.
__device__ __forceinline__ int xcd_tile(int b, int n) {
  const int xcd = b & 7, q = n >> 3, r = n & 7;
  return xcd * q + min(xcd, r) + (b >> 3);
}

// This workgroup's tile of a product whose rows are ordered by expert, [off[e], off[e +
// 1]) the rows of expert e: expert, first row, rows and column tile. Row tiles have bm
// rows, every expert's rows starting one of their own, tiles_n column tiles each (fastest).
// The grid holds the most workgroups that any choice of experts can need; those past the
// actual number get false, and the others share the tiles over the XCDs (dealt out over the
// whole grid, the unused ones would all fall to the last XCDs). Uniform results.
struct ExpertTile {
  int expert, row0, rows, col;
};
__device__ __forceinline__ bool find_tile(const int* __restrict__ off, int experts, int bm, int tiles_n,
                                          ExpertTile* out) {
  const int lane = threadIdx.x & 63;
  int total = 0;
  for (int e0 = 0; e0 < experts; e0 += 64) {
    const int e = min(e0 + lane, experts);
    total += (off[min(e + 1, experts)] - off[e] + bm - 1) / bm;
  }
  total = __builtin_amdgcn_readlane(wave_scan(total), 63) * tiles_n;
  if ((int)blockIdx.x >= total) return false;
  const int id = xcd_tile(blockIdx.x, total), tile = id / tiles_n;  // of a list with columns fastest: the right expert
  int base = 0;
  for (int e0 = 0; e0 < experts; e0 += 64) {
    const int e = min(e0 + lane, experts);
    const int lo = off[e], hi = off[min(e + 1, experts)];
    const int n = (hi - lo + bm - 1) / bm;
    const int sum = wave_scan(n), first = base + sum - n;
    const uint64_t hit = __ballot(tile >= first && tile < first + n);
    if (hit) {
      const int src = __builtin_ctzll(hit);
      const int l = __builtin_amdgcn_readlane(lo, src), tiles = __builtin_amdgcn_readlane(n, src);
      const int in = id - __builtin_amdgcn_readlane(first, src) * tiles_n, at = in % tiles * bm;
      out->expert = e0 + src;
      out->row0 = l + at;
      out->rows = min(bm, __builtin_amdgcn_readlane(hi, src) - l - at);
      out->col = in / tiles;
      return true;
    }
    base += __builtin_amdgcn_readlane(sum, 63);
  }
  return false;
}

}  // namespace ff
