// Paged key/value cache: new rows written into their sequences' pages, rows read back.
//
// FP8 pages hold e4m3 codes with one power of two per (token, head): 2^e with the
// smallest e for which the row's largest finite value is at most 448 * 2^e. e4m3 is a
// floating-point format, so its relative step does not depend on the scale, and a
// power of two costs at most one of its 15 binades. In return multiplying by it
// is exact, a stored value is a bf16 value, and the conversion instruction applies it
// for nothing when a cache is read.
#include "ff_cache.h"

using namespace ff;

namespace {

constexpr int kLowest = -100, kHighest = 120;  // e; 2^-100 times the smallest code is far from fp32's subnormals

struct Pages {
  uint8_t* k;
  uint8_t* v;
  uint8_t* ks;  // scale bytes (FP8)
  uint8_t* vs;
};

// Largest finite magnitude's e for the row that LPR lanes hold, 8 values each.
template <int LPR>
__device__ __forceinline__ int row_exponent(const float (&x)[8]) {
  float a = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float m = fabsf(x[i]);
    a = fmaxf(a, m < __builtin_inff() ? m : 0.f);
  }
  a = fmaxf(a, dpp<kDppXor1>(a));
  a = fmaxf(a, dpp<kDppXor2>(a));
  a = fmaxf(a, dpp<kDppHalfMirror>(a));
  if (LPR == 16) a = fmaxf(a, dpp<kDppRowMirror>(a));
  // a = 1.m 2^(E - 127), at most 448 2^e = 1.75 2^(e + 8); 0x60 is the 7-bit fraction of 1.75
  const uint32_t bits = __float_as_uint(a);
  const int e = (int)(bits >> 23) - 127 - 8 + (((bits >> 16) & 0x7F) > 0x60);
  return min(max(e, kLowest), kHighest);
}

__device__ __forceinline__ void load8(const bf16_t* p, bool vec, float (&x)[8]) {
  if (vec) {
    unpack8(*reinterpret_cast<const u32x4*>(p), x);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = bf16_to_f32(p[i]);
  }
}

// LPR lanes write one row of D values at row `at` of the pages.
template <int D, bool FP8>
__device__ __forceinline__ void write_row(const float (&x)[8], uint8_t* pages, uint8_t* scales, int64_t at, int j) {
  if (!FP8) {
    *reinterpret_cast<u32x4*>(pages + (at * D + 8 * j) * 2) = pack8(x);
    return;
  }
  const int e = row_exponent<D / 8>(x);
  const float inv = __uint_as_float((uint32_t)(127 - e) << 23);
  const float most = e == kHighest ? 240.f : 448.f;  // 256 * 2^120 is no bf16 value any more
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
    y[i] = fabsf(x[i]) < __builtin_inff() ? __builtin_amdgcn_fmed3f(x[i] * inv, -most, most) : __builtin_nanf("");
  *reinterpret_cast<u32x2*>(pages + at * D + 8 * j) = u32x2{e4m3x4(y[0], y[1], y[2], y[3]), e4m3x4(y[4], y[5], y[6], y[7])};
  if (j == 0) scales[at] = (uint8_t)(127 + e);
}

// A workgroup takes neighbouring tokens of one head; heads are the grid's fastest axis, so that with 8 heads
// (or a divisor) the workgroups of one XCD fill the same pages' lines and its L2 joins the scale bytes of
// neighbouring tokens (32782 tokens, 8 heads of 128: 39.6 us against 42.7 with the tokens fastest).
__device__ __forceinline__ int block_of() { return (int)(blockIdx.z * gridDim.y + blockIdx.y); }

// A wave writes 512 / D neighbouring tokens, D / 8 lanes each for keys and values. Bound by memory: 16 bytes a
// lane and tensor are in flight while the sequence, its length and the page are looked up. Two tokens a lane are
// slower in bf16 (46 us against 43) and even in codes.
template <int D, bool FP8>
__global__ __launch_bounds__(256) void cache_write_kernel(Rows a, Pages c, const bf16_t* __restrict__ k, int64_t k_ts,
                                                          int64_t k_hs, const bf16_t* __restrict__ v, int64_t v_ts,
                                                          int64_t v_hs, int hk, int vec) {
  constexpr int LPR = D / 8, TPW = 64 / LPR;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, j = lane % LPR;
  const int row0 = (block_of() * 4 + wave) * TPW, row = row0 + lane / LPR;
  const int head = blockIdx.x;
  const int64_t src = min(row, a.t - 1);
  float x[8], y[8];
  load8(k + src * k_ts + head * k_hs + 8 * j, vec & 1, x);
  load8(v + src * v_ts + head * v_hs + 8 * j, vec & 2, y);
  int of[TPW];
  find_sequences<TPW>(a, row0, lane, of);
  int b = of[0];
#pragma unroll
  for (int i = 1; i < TPW; ++i) b = lane / LPR == i ? of[i] : b;
  int64_t page;
  int slot;
  if (!find_slot(a, row, b, &page, &slot)) return;
  const int64_t at = ((page * hk + head) << a.lps) + slot;
  write_row<D, FP8>(x, c.k, c.ks, at, j);
  write_row<D, FP8>(y, c.v, c.vs, at, j);
}

using Words4 = uint32_t __attribute__((ext_vector_type(4)));
__device__ __forceinline__ void store_once(bf16_t* p, u32x4 x) {
  __builtin_nontemporal_store(Words4{x.x, x.y, x.z, x.w}, reinterpret_cast<Words4*>(p));
}

template <int D, bool FP8>
__device__ __forceinline__ u32x4 read_row(const uint8_t* pages, const uint8_t* scales, int64_t at, int j) {
  if (!FP8) return *reinterpret_cast<const u32x4*>(pages + (at * D + 8 * j) * 2);
  const u32x2 q = *reinterpret_cast<const u32x2*>(pages + at * D + 8 * j);
  const float s = scale_of(scales[at]);
  u32x4 r;
  r.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q.x, s, false));
  r.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q.x, s, true));
  r.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q.y, s, false));
  r.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q.y, s, true));
  return r;
}

constexpr int kReadRows = 2;  // tokens a lane of the read

// The same shape with two tokens a lane, for the three dependent loads before a row's address is known leave less
// in flight; rows that are nowhere come out zero. The outputs are written past the L2, where they would only
// push out the pages: 48 sequences of about 500 codes 28 us against 36 with one token and 37 with ordinary
// stores, 48782 positions of codes (224 MB) 38 against 44.
template <int D, bool FP8>
__global__ __launch_bounds__(256) void cache_read_kernel(Rows a, Pages c, bf16_t* __restrict__ k,
                                                         bf16_t* __restrict__ v, int hk) {
  constexpr int LPR = D / 8, TPW = 64 / LPR;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, j = lane % LPR;
  const int row0 = (block_of() * 4 + wave) * TPW * kReadRows, row = row0 + lane / LPR;
  const int head = blockIdx.x;
  int of[TPW * kReadRows];
  find_sequences<TPW * kReadRows>(a, row0, lane, of);
  u32x4 x[kReadRows], y[kReadRows];
#pragma unroll
  for (int n = 0; n < kReadRows; ++n) {
    int b = of[n * TPW];
#pragma unroll
    for (int i = 1; i < TPW; ++i) b = lane / LPR == i ? of[n * TPW + i] : b;
    x[n] = y[n] = u32x4{0, 0, 0, 0};
    int64_t page;
    int slot;
    if (find_slot(a, row + n * TPW, b, &page, &slot)) {
      const int64_t at = ((page * hk + head) << a.lps) + slot;
      x[n] = read_row<D, FP8>(c.k, c.ks, at, j);
      y[n] = read_row<D, FP8>(c.v, c.vs, at, j);
    }
  }
#pragma unroll
  for (int n = 0; n < kReadRows; ++n) {
    if (row + n * TPW >= a.t) return;
    const int64_t to = ((int64_t)(row + n * TPW) * hk + head) * D + 8 * j;
    store_once(k + to, x[n]);
    store_once(v + to, y[n]);
  }
}

// hk x ceil(t / per) workgroups; the second axis runs on into the third past its limit.
dim3 grid_of(const ff_paged_cache* c, int64_t t, int64_t rows) {
  const int64_t per = 4 * rows * 512 / c->d, blocks = (t + per - 1) / per, y = blocks < 65535 ? blocks : 65535;
  return dim3((unsigned)c->hk, (unsigned)y, (unsigned)((blocks + y - 1) / y));
}

Pages pages_of(const ff_paged_cache* c) {
  return Pages{(uint8_t*)c->k, (uint8_t*)c->v, (uint8_t*)c->k_scale, (uint8_t*)c->v_scale};
}

}  // namespace

extern "C" int ff_cache_write(const void* k, int64_t k_ts, int64_t k_hs, const void* v, int64_t v_ts, int64_t v_hs,
                              const ff_paged_cache* cache, const int32_t* table, int64_t width, const int32_t* lengths,
                              const int32_t* starts, int64_t batch, int64_t t, ff_stream_t stream) {
  if (t == 0) return FF_OK;
  const int st = check_rows("ff_cache_write", cache, table, width, lengths, starts, batch, t);
  if (st != FF_OK) return st;
  FF_REQUIRE(k && v, "ff_cache_write: null pointer");
  const Rows a = rows_of(cache, table, width, lengths, starts, batch, t);
  const int vec = (ff_aligned(k, 16) && k_ts % 8 == 0 && k_hs % 8 == 0) |
                  (ff_aligned(v, 16) && v_ts % 8 == 0 && v_hs % 8 == 0) << 1;
  const dim3 grid = grid_of(cache, t, 1);
#define FF_WRITE(DIM, F8)                                                                                    \
  if (cache->d == DIM && (cache->fp8 != 0) == F8)                                                            \
    hipLaunchKernelGGL((cache_write_kernel<DIM, F8>), grid, dim3(256), 0, (hipStream_t)stream, a,            \
                       pages_of(cache), (const bf16_t*)k, k_ts, k_hs, (const bf16_t*)v, v_ts, v_hs, (int)cache->hk, vec);
  FF_WRITE(64, false) FF_WRITE(64, true) FF_WRITE(128, false) FF_WRITE(128, true)
#undef FF_WRITE
  FF_LAUNCH_CHECK("ff_cache_write");
  return FF_OK;
}

extern "C" int ff_cache_read(const ff_paged_cache* cache, const int32_t* table, int64_t width, const int32_t* lengths,
                             const int32_t* starts, int64_t batch, void* k, void* v, int64_t t, ff_stream_t stream) {
  if (t == 0) return FF_OK;
  const int st = check_rows("ff_cache_read", cache, table, width, lengths, starts, batch, t);
  if (st != FF_OK) return st;
  FF_REQUIRE(k && v && ff_aligned(k, 16) && ff_aligned(v, 16), "ff_cache_read: output");
  const Rows a = rows_of(cache, table, width, lengths, starts, batch, t);
  const dim3 grid = grid_of(cache, t, kReadRows);
#define FF_READ(DIM, F8)                                                                          \
  if (cache->d == DIM && (cache->fp8 != 0) == F8)                                                 \
    hipLaunchKernelGGL((cache_read_kernel<DIM, F8>), grid, dim3(256), 0, (hipStream_t)stream, a,  \
                       pages_of(cache), (bf16_t*)k, (bf16_t*)v, (int)cache->hk);
  FF_READ(64, false) FF_READ(64, true) FF_READ(128, false) FF_READ(128, true)
#undef FF_READ
  FF_LAUNCH_CHECK("ff_cache_read");
  return FF_OK;
}
