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
// keeps its code; a row's infinity makes the scale infinite and its own code NaN.
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
  return quant8(v, sc, 1.0f / sc);
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

// Expert, first row and rows of row tile `tile` (bm rows each, every expert's rows
// starting a tile of their own) among experts whose rows are [off[e], off[e + 1]).
// False past the last tile. Every lane of a wave calls it and gets the result.
__device__ __forceinline__ bool find_tile(const int* __restrict__ off, int experts, int bm, int tile, int* expert,
                                          int* row0, int* rows) {
  const int lane = threadIdx.x & 63;
  int base = 0;
  for (int e0 = 0; e0 < experts; e0 += 64) {
    const int e = e0 + lane;
    const int lo = e < experts ? off[e] : 0, hi = e < experts ? off[e + 1] : 0;
    const int n = (hi - lo + bm - 1) / bm;
    int sum = n;  // inclusive prefix sum over the lanes
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int up = __shfl_up(sum, d);
      if (lane >= d) sum += up;
    }
    const int first = base + sum - n;
    const uint64_t hit = __ballot(tile >= first && tile < first + n);
    if (hit) {
      const int src = __builtin_ctzll(hit);
      const int f = __shfl(first, src), l = __shfl(lo, src), h = __shfl(hi, src);
      *expert = e0 + src;
      *row0 = l + (tile - f) * bm;
      *rows = min(bm, h - *row0);
      return true;
    }
    base += __shfl(sum, 63);
  }
  return false;
}

// Launch of the row quantiser (defined with the linear): q (rows, 128 ceil(k / 128))
// 16-byte aligned, scales (ceil(k / 128), rows).
int quant_rows_block(const void* x, int64_t ldx, void* q, float* scales, int64_t rows, int64_t k, hipStream_t st);

}  // namespace ff
