// Causal grouped-query attention of each sequence's last tokens over a paged cache.
//
// Query i of a sequence's n new tokens has position L - n + i of its L and sees the
// positions up to its own: o = sum_j p_j v_j, p = softmax_j(scale q . k_j), exact
// softmax statistics in fp32 over 64-key blocks with a running maximum.
//
// Rows. A tile holds rows (query, head of the group) of one sequence and one key head,
// query-major, so that a group of any size fills tiles and a decode token is the tile of
// its group's heads. Products run as S^T = K Q^T and O^T = V^T P^T on
// v_mfma_f32_16x16x32_bf16: a lane's accumulators belong to one row, and P^T leaves the
// scores in the operand layout of the second product (lane group g of 16 lanes holds
// keys 8 g .. 8 g + 7 of a 32-key chunk in both). V is stored as tokens are, and comes
// out of LDS transposed (ds_read_b64_tr_b16 / _b8).
//
// FP8 pages: codes become bf16 in registers, exactly (a power of two scales a row): a
// key's scale is the conversion's own operand, a value's is multiplied into its P before
// that is rounded to bf16. P in bf16 is off by half a step at most, 2^-8 of it, as the
// output's own rounding; its sum is kept unrounded.
#include <float.h>
#include <limits.h>

#include "ff_block.h"
#include "ff_cache.h"

using namespace ff;

namespace {

typedef short s16x4 __attribute__((ext_vector_type(4)));

struct Args {
  Rows a;
  const bf16_t* q;
  int64_t q_ts, q_hs;
  const uint8_t *k, *v, *ks, *vs;
  bf16_t* y;
  float* part_o;   // (slots, hk, BM, D) unnormalised sums of split tiles
  float2* part_s;  // (slots, hk, BM) their reference (log2) and denominator
  int* plan;       // the list of many sequences, or null
  int2* part_of;   // (rows) where a row (token, head) begins there, and its splits (1: it is done)
  int hk, group, lbm;  // BM = 1 << lbm rows a tile
  int least, budget;  // 64-key blocks are dealt so that about so many items per head come out; 0: no tile is split
  int slots;   // items of split tiles, per head, that the workspace holds
  float c2;    // scale * log2(e)
};

__device__ __forceinline__ f32x4 mfma_bf16(const bf16x8& a, const u32x4& b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// ------------------------------------------------------------------ the work list
//
// Every sequence's rows make ceil(rows / BM) tiles, and every tile is split into as many
// key ranges as its sequence's blocks take chunks. A chunk is the share of all blocks
// that gives `budget` items, `least` blocks at least. All workgroups compute the
// same list from the lengths (of more than 64 sequences a launch writes it); a sequence's last tiles, which see the most keys, come first.
// A split's rows go to the workspace, where the items of split tiles have slots in the list's order, with a
// note for each row where its splits are. Rows behind the last sequence are a sequence without keys.

struct Seq {
  int row0, n;    // first row (token) and rows
  int len;        // its positions
  int keys;       // of which the table reaches so many
  int tiles, blocks;
};

// (loads first, whatever b is, so that those of several calls are in flight together)
__device__ __forceinline__ Seq seq_of(const Args& p, int b) {
  const int batch = p.a.starts ? p.a.batch : p.a.t, in = min(b, batch - 1);
  const int len = p.a.lengths[in];
  const int begin = p.a.begin(min(b, batch)), end = p.a.end(min(b, batch));
  const bool one = b < batch, rest = b == batch && p.a.starts;
  Seq s;
  s.row0 = one || rest ? begin : 0;
  s.n = one ? max(end - begin, 0) : rest ? p.a.t - begin : 0;
  s.len = one ? max(len, -(1 << 30)) : 0;  // (a length below 0 sees nothing, however far)
  s.keys = one ? max(0, (int)min((int64_t)len, p.a.capacity())) : 0;
  s.tiles = (int)(((int64_t)s.n * p.group + (1 << p.lbm) - 1) >> p.lbm);
  s.blocks = s.n ? (s.keys + 63) >> 6 : 0;
  return s;
}

__device__ __forceinline__ int splits_of(int blocks, int chunk) {
  return max(1, blocks / chunk + (blocks % chunk != 0));
}

struct Item {
  Seq s;
  int seq, tile, split, splits;
  int slot;  // of a split tile's item
};

// Slots of a sequence with `splits` splits a tile. A split sequence has more blocks than a chunk, so that
// its splits are fewer than twice blocks / chunk, and all of them fewer than twice the budget.
__device__ __forceinline__ int slots_of(const Seq& s, int splits) { return splits > 1 ? s.tiles * splits : 0; }

// The chunk: the share of all blocks that gives `budget` items, or as many more as keep the items within it
// (one round of the GPU's workgroups; a few of a second would take as long). Where the tiles alone are more
// than that, only sequences past their share are split. sum(f): f over all sequences.
template <class Sum>
__device__ __forceinline__ int chunk_of(const Args& p, Sum sum) {
  if (!p.budget) return INT_MAX;
  const int total = sum([](const Seq& s) { return s.tiles * s.blocks; });
  const int tiles = sum([](const Seq& s) { return s.tiles; });
  int chunk = max(p.least, (int)(((int64_t)total + p.budget - 1) / p.budget));
  for (int i = 0; i < 3 && tiles < p.budget; ++i) {
    const int items = sum([=](const Seq& s) { return s.tiles * splits_of(s.blocks, chunk); });
    if (items <= p.budget) break;
    chunk = (int)min((int64_t)INT_MAX, ((int64_t)chunk * items + p.budget - 1) / p.budget);
  }
  return chunk;
}

// Sequences for a lane each, the rows behind the last one among them.
__host__ __device__ inline bool fit_lanes(int64_t batch, bool starts) { return batch + starts <= 64; }

// The list of more sequences than a wave has lanes, by one workgroup in a launch of its own: plan[0] the chunk,
// plan[1 + b] the first item of sequence b (b = batch: of the rows behind the last; batch + 1: all items),
// plan[3 + batch + b] its first slot. With every workgroup reading all lengths instead, decode of 256 sequences of 500 positions took 134 us (102 so), 1024
// sequences of 3 tokens over 200 positions 427 (208).
__global__ __launch_bounds__(1024) void plan_kernel(Args p) {
  __shared__ int part[16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // The workgroup's sum of v, and how much of it lies before the thread's own.
  auto scan = [&](int v, int* before) {
    const int upto = wave_scan(v);
    __syncthreads();
    if (lane == 63) part[wave] = upto;
    __syncthreads();
    int sum = 0;
    *before = upto - v;
#pragma unroll
    for (int w = 0; w < 16; ++w) {
      *before += w < wave ? part[w] : 0;
      sum += part[w];
    }
    return sum;
  };
  int before;
  const int chunk = chunk_of(p, [&](auto f) {
    int v = 0;
    for (int b = threadIdx.x; b <= p.a.batch; b += 1024) v += f(seq_of(p, b));
    return scan(v, &before);
  });
  if (threadIdx.x == 0) p.plan[0] = chunk;
  int base = 0, slots = 0;
  for (int b0 = 0; b0 <= p.a.batch; b0 += 1024) {
    const int b = b0 + threadIdx.x;
    const bool in = b <= p.a.batch;
    const Seq s = seq_of(p, b);
    const int splits = splits_of(s.blocks, chunk);
    const int n = scan(in ? s.tiles * splits : 0, &before);
    if (in) p.plan[1 + b] = base + before;
    base += n;
    const int m = scan(in ? slots_of(s, splits) : 0, &before);
    if (in) p.plan[3 + p.a.batch + b] = slots + before;
    slots += m;
  }
  if (threadIdx.x == 0) p.plan[2 + p.a.batch] = base;
}

// Item `id` of the list.
__device__ __forceinline__ bool find_item(const Args& p, int lane, int id, Item* out) {
  Seq s;
  int chunk, first, slot;
  if (p.plan) {
    const int* starts = p.plan + 1;
    const int lo = last_upto(starts, p.a.batch + 2, id, lane);  // the last one that begins at or before the item
    if (lo > p.a.batch) return false;
    chunk = __builtin_amdgcn_readfirstlane(p.plan[0]);
    first = __builtin_amdgcn_readfirstlane(starts[lo]);
    slot = __builtin_amdgcn_readfirstlane(starts[p.a.batch + 2 + lo]);
    s = seq_of(p, lo);
    out->seq = lo;
    lane = 0;
  } else {
    s = seq_of(p, lane);
    chunk = chunk_of(p, [&](auto f) { return __builtin_amdgcn_readlane(wave_scan(f(s)), 63); });
    const int splits = splits_of(s.blocks, chunk), n = s.tiles * splits, upto = wave_scan(n);
    const int m = slots_of(s, splits), slots = wave_scan(m);
    const uint64_t hit = __ballot(id >= upto - n && id < upto);
    if (!hit) return false;
    lane = __builtin_ctzll(hit);
    first = __builtin_amdgcn_readlane(upto - n, lane);
    slot = __builtin_amdgcn_readlane(slots - m, lane);
    out->seq = lane;
  }
  out->s = {__builtin_amdgcn_readlane(s.row0, lane), __builtin_amdgcn_readlane(s.n, lane),
            __builtin_amdgcn_readlane(s.len, lane),  __builtin_amdgcn_readlane(s.keys, lane),
            __builtin_amdgcn_readlane(s.tiles, lane), __builtin_amdgcn_readlane(s.blocks, lane)};
  out->splits = splits_of(out->s.blocks, chunk);
  const int in = id - first;
  if (in < 0 || in >= out->s.tiles * out->splits) return false;  // (counts of starts that do not rise may pass 32 bits)
  out->tile = out->s.tiles - 1 - in / out->splits;
  out->split = in % out->splits;
  out->slot = slot + in;
  // (and so may those of slots, without which an item of a split tile does nothing)
  return out->splits == 1 || (unsigned)out->slot < (unsigned)p.slots;
}

// ------------------------------------------------------------------ pieces of a block

// 16-byte chunk at which chunk c of a value row of RB bytes is kept in LDS: the rows that
// a transposed read takes together (see below) fall on different banks.
template <int RB, bool FP8>
__device__ __forceinline__ int v_swizzle(int row) {
  if (FP8) return RB == 128 ? (row >> 1) & 7 : (row >> 2) & 3;
  return RB == 256 ? 2 * ((row & 3) | ((row >> 1) & 4)) : 2 * (((row >> 1) & 1) | ((row >> 2) & 2));
}

// The same address, of which the compiler does not know that it is: fragments read at one and
// at the other are not kept in registers between the two.
__device__ __forceinline__ uint32_t another(uint32_t lds) {
  asm volatile("" : "+s"(lds));
  return lds;
}

__device__ __forceinline__ s16x4 read_tr16(uint32_t lds, int offset = 0) {
  typedef __attribute__((address_space(3))) uint8_t* Bytes;
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)((Bytes)(uintptr_t)lds + offset));
}
__device__ __forceinline__ i32x2v read_tr8(uint32_t lds) {
  return __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) i32x2v*)(uintptr_t)lds);
}

// V^T fragment of chunk c, dims 16 dt ..: lane (r16, g) gets keys 32 c + 8 g .. + 7 of dim
// 16 dt + r16. 16 lanes read 4 keys x 32 bytes (bf16) or 8 keys x 16 bytes (codes) and
// receive them transposed.
template <int D, bool FP8>
__device__ __forceinline__ bf16x8 v_fragment(uint32_t lds, int c, int dt, int r16, int g) {
  constexpr int RB = FP8 ? D : 2 * D;
  if constexpr (FP8) {
    const int row = 32 * c + 8 * g + (r16 >> 1);
    const i32x2v q = read_tr8(lds + row * RB + 16 * (dt ^ v_swizzle<RB, FP8>(row)) + 8 * (r16 & 1));
    return e4m3_to_bf16x8((uint32_t)q.x, (uint32_t)q.y);
  } else {
    s16x4 h[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = 32 * c + 8 * g + 4 * i + (r16 >> 2);
      const int chunk = (2 * dt + ((r16 >> 1) & 1)) ^ v_swizzle<RB, FP8>(row);
      h[i] = read_tr16(lds + row * RB + 16 * chunk + 8 * (r16 & 1));
    }
    typedef short s16x8 __attribute__((ext_vector_type(8)));
    return __builtin_bit_cast(bf16x8, (s16x8)__builtin_shufflevector(h[0], h[1], 0, 1, 2, 3, 4, 5, 6, 7));
  }
}

// The dims that k step st of q . k takes for lane group g: where 16 bytes of a key row
// are 16 codes they serve two steps.
template <bool FP8>
__device__ __forceinline__ int step_dim(int st, int g) {
  return FP8 ? 64 * (st >> 1) + 16 * g + 8 * (st & 1) : 32 * st + 8 * g;
}

__device__ __forceinline__ bf16x8 e4m3_to_bf16x8(uint32_t a, uint32_t b, float s) {
  const bf16x2_t p0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, s, false);
  const bf16x2_t p1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, s, true);
  const bf16x2_t p2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, s, false);
  const bf16x2_t p3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, s, true);
  return bf16x8{p0.x, p0.y, p1.x, p1.y, p2.x, p2.y, p3.x, p3.y};
}

// lds_dma16 from a uniform base: lane l's 16 bytes at base + offset.
__device__ __forceinline__ void lds_dma16_at(const uint8_t* base, uint32_t offset, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(offset), "s"(base), "s"(lds)
               : "memory", "m0");
}

// The reference of a row that sees a key is at least this, also where its scores are NaN or -inf. A reference of
// -inf is a row that sees nothing, which alone is zero: the others divide by their sum, be it 0 or NaN.
constexpr float kLeast = -FLT_MAX;
__device__ __forceinline__ float inverse_sum(float m, float sum) { return m == -INFINITY ? 0.f : 1.0f / sum; }

// This wave's LDS reads and writes are done (no other wave uses the memory).
__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory"); }

// One block of the running softmax. s[2 c + tt][r] is q . k of key 32 c + 8 g + 4 tt + r;
// vis: the block's keys that this lane's row sees (`masked`: not all of them, in some
// lane). m is the reference, the maximum of q . k times c2 = scale log2 e, rounded: all
// weights are relative to that very number. P^T of chunk c goes to pf[c], times the keys'
// value scales (FP8).
template <bool FP8>
__device__ __forceinline__ float softmax_block(f32x4 (&s)[4], bool masked, uint64_t vis, int g, float c2,
                                               const u32x2 (&vsc)[2], float& m, float& den, u32x4 (&pf)[2]) {
  if (masked) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t bits = (uint32_t)(vis >> (32 * (i >> 1) + 8 * g)) >> (4 * (i & 1));
#pragma unroll
      for (int r = 0; r < 4; ++r) s[i][r] = bits >> r & 1 ? s[i][r] : -INFINITY;
    }
  }
  float top = s[0][0];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) top = __builtin_elementwise_maximum(top, s[i][r]);
  const float mnew = fmaxf(m, fmaxf(max_rows(top) * c2, masked && !vis ? -INFINITY : kLeast));  // (drops NaN)
  const float mref = mnew == -INFINITY ? 0.f : mnew;
  const float alpha = __builtin_amdgcn_exp2f(m - mref);
  float psum = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      s[i][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i][r], c2, -mref));
      psum += s[i][r];
    }
  den = den * alpha + psum;
  m = mnew;
  if constexpr (FP8) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) s[i][r] *= scale_of((i & 1 ? vsc[i >> 1].y : vsc[i >> 1].x) >> (8 * r) & 0xFF);
  }
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    pf[c].x = pack_bf16x2(s[2 * c][0], s[2 * c][1]);
    pf[c].y = pack_bf16x2(s[2 * c][2], s[2 * c][3]);
    pf[c].z = pack_bf16x2(s[2 * c + 1][0], s[2 * c + 1][1]);
    pf[c].w = pack_bf16x2(s[2 * c + 1][2], s[2 * c + 1][3]);
  }
  return alpha;
}

// Whether a block's values (all of them in LDS, those that are not there as zeros) hold an
// infinity or a NaN: their sum by the matrix unit says so.
template <int D, bool FP8>
__device__ __forceinline__ bool values_odd(uint32_t lds, int r16, int g) {
  const u32x4 ones = {0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u};
  f32x4 t = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int c = 0; c < 2; ++c)
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt) t = mfma_bf16(v_fragment<D, FP8>(lds, c, dt, r16, g), ones, t);
  bool odd = false;
#pragma unroll
  for (int r = 0; r < 4; ++r) odd |= !(fabsf(t[r]) < INFINITY);
  return __ballot(odd) != 0;
}

// A fragment with zeros in place of infinities and NaN.
__device__ __forceinline__ bf16x8 finite_only(const bf16x8& v) {
  u32x4 w = __builtin_bit_cast(u32x4, v);
  uint32_t* x = &w.x;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t lo = (x[i] & 0x7F80u) == 0x7F80u ? 0u : 0xFFFFu, hi = (x[i] & 0x7F800000u) == 0x7F800000u ? 0u : 0xFFFF0000u;
    x[i] &= lo | hi;
  }
  return __builtin_bit_cast(bf16x8, w);
}

// 4 values of a bf16 row, what is finite as 0.
__device__ __forceinline__ f32x4 odd_only(const u32x2& w) {
  const f32x4 v = {bf16_to_f32(w.x & 0xFFFF), __uint_as_float(w.x & 0xFFFF0000u), bf16_to_f32(w.y & 0xFFFF),
                   __uint_as_float(w.y & 0xFFFF0000u)};
  f32x4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = fabsf(v[i]) < INFINITY ? 0.f : v[i];
  return r;
}

// Bits 0 .. last of a block's 64 keys (none where last < 0).
__device__ __forceinline__ uint64_t keys_to(int last) {
  return last < 0 ? 0 : last >= 63 ? ~0ull : (2ull << last) - 1;
}

// ------------------------------------------------------------------ few rows
//
// One workgroup per item: a 16-row tile, its key blocks dealt to the waves, each with a
// running softmax of its own; the waves are joined in LDS. Keys go from memory straight
// into the operand registers, values by DMA into the wave's own LDS: no barrier until
// the end. Bound by the cache's bytes: 131072 FP8 positions of 8 heads of 128 (271 MB) 52 us, 48
// sequences of about 3000 in bf16 (597 MB) 122 us, 5.2 and 4.9 TB/s. Blocks of 64 keys keep 32 KB of
// a wave in flight; a CU takes in 64 bytes a clock, so that one row's cache is dealt to all of them.
constexpr int kFewWaves = 4;     // two workgroups a CU
constexpr int kDecodeWaves = 8;  // a workgroup a CU, no splits

template <int D, bool FP8, int NW, bool DECODE>
__global__ __launch_bounds__(64 * NW, NW == 4 ? 2 : 1) void few_rows_kernel(Args p) {
  constexpr int RB = FP8 ? D : 2 * D, KST = D / 32, DTN = D / 16, KL = RB / 64;  // KL: 16-byte loads of a key row
  constexpr int PI = 16 * RB / 1024;                                            // value DMAs of 16 keys
  constexpr int SLAB = 64 * RB, LDO = D + 4;
  constexpr int JOIN = NW * 16 * (LDO + 2) * 4;
  __shared__ __align__(1024) uint8_t smem[NW * SLAB > JOIN ? NW * SLAB : JOIN];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r16 = lane & 15, g = lane >> 4;
  const int head = (int)blockIdx.x % p.hk, id = (int)blockIdx.x / p.hk;
  Item it;
  if (DECODE || (!p.a.starts && !p.budget)) {  // one row a sequence and no splits: the list is known without the lengths
    const int tiles = (p.group + 15) >> 4;
    it.seq = __builtin_amdgcn_readfirstlane(id / tiles);
    it.tile = id - it.seq * tiles;
    it.split = 0;
    it.splits = 1;
    if (it.seq >= p.a.t) return;
    const Seq s = seq_of(p, it.seq);
    it.s = {it.seq, 1, __builtin_amdgcn_readfirstlane(s.len), __builtin_amdgcn_readfirstlane(s.keys), tiles,
            __builtin_amdgcn_readfirstlane(s.blocks)};
  } else {
    if (!find_item(p, lane, id, &it)) return;
  }
  const int64_t page_rows = (int64_t)p.hk << p.a.lps, head_rows = (int64_t)head << p.a.lps;
  const int in_page = (1 << p.a.lps) - 1;
  const int* table = p.a.table + (int64_t)min(it.seq, p.a.batch - 1) * p.a.width;
  // table entry of the lane's key of block b
  auto entry_of = [&](int b) { return table[min((int64_t)((64 * b + lane) >> p.a.lps), p.a.width - 1)]; };
  int ahead = DECODE ? entry_of(wave) : 0;

  const int row = it.tile * 16 + r16, rows = it.s.n * p.group;
  const bool real = row < rows;
  const int query = DECODE ? 0 : (real ? row : rows - 1) / p.group;
  const int hq = head * p.group + (real ? row : rows - 1) - query * p.group;
  u32x4 qf[KST];
  const bf16_t* qp = p.q + (it.s.row0 + query) * p.q_ts + hq * p.q_hs;
#pragma unroll
  for (int st = 0; st < KST; ++st) {
    const bf16_t* src = qp + step_dim<FP8>(st, g);
    if (((uintptr_t)p.q & 15) == 0 && ((p.q_ts | p.q_hs) & 7) == 0) {
      qf[st] = *reinterpret_cast<const u32x4*>(src);
    } else {
      float x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = bf16_to_f32(src[i]);
      qf[st] = pack8(x);
    }
  }
  const int pos = real ? it.s.len - it.s.n + query : -1;
  // one past the tile's last position
  const int kend = min(it.s.keys, DECODE ? it.s.len : it.s.len - it.s.n + min(rows - 1, it.tile * 16 + 15) / p.group + 1);
  const int nb = max(0, kend + 63) >> 6, per = DECODE ? nb : (nb + it.splits - 1) / it.splits;
  const int b_end = min(nb, (it.split + 1) * per), b_first = it.split * per + wave;
  if (!DECODE) ahead = entry_of(b_first);

  f32x4 o[DTN];
#pragma unroll
  for (int dt = 0; dt < DTN; ++dt) o[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, den = 0.f;
  const uint32_t lds = lds_addr(smem) + wave * SLAB;
  uint32_t v_from[PI];  // where a lane's 16 bytes lie among 16 keys' values, for the i-th DMA of them
#pragma unroll
  for (int i = 0; i < PI; ++i) {
    const int key = i * (1024 / RB) + lane / (RB / 16);
    v_from[i] = key * RB + 16 * (lane % (RB / 16) ^ v_swizzle<RB, FP8>(key)) - i * 1024;
  }

  for (int b = b_first; b < b_end; b += NW) {
    const int kb = 64 * b;
    // the lane's key of the block: its page, and whether there is one
    const int entry = ahead;
    ahead = entry_of(b + NW);
    const bool there = kb + lane < kend && (unsigned)entry < (unsigned)p.a.pages;
    const uint64_t ok = __ballot(there);
    // row of the pages' (page, head, slot) that holds the first of 16 keys: a uniform one
    auto first = [&](int j) {
      return __builtin_amdgcn_readlane(there ? entry : 0, 16 * j) * page_rows + head_rows + ((kb + 16 * j) & in_page);
    };
    const int64_t f0 = first(0), f1 = first(1), f2 = first(2), f3 = first(3);
    u32x4 kf[4][KL];
    float ksc[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // key 32 (i / 2) + 8 (r16 / 4) + 4 (i % 2) + r16 % 4
      const int64_t at = (r16 & 8 ? (i < 2 ? f1 : f3) : (i < 2 ? f0 : f2)) + 2 * (r16 & 4) + 4 * (i & 1) + (r16 & 3);
#pragma unroll
      for (int j = 0; j < KL; ++j) kf[i][j] = *reinterpret_cast<const u32x4*>(p.k + at * RB + 64 * j + 16 * g);
      if (FP8) ksc[i] = scale_of(p.ks[at]);
    }
    u32x2 vsc[2];
    if (FP8) {
      vsc[0] = *reinterpret_cast<const u32x2*>(p.vs + (g & 2 ? f1 : f0) + 8 * (g & 1));
      vsc[1] = *reinterpret_cast<const u32x2*>(p.vs + (g & 2 ? f3 : f2) + 8 * (g & 1));
    }
    wait_lds();
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < PI; ++i)
        lds_dma16_at(p.v + (j == 0 ? f0 : j == 1 ? f1 : j == 2 ? f2 : f3) * RB + i * 1024, v_from[i],
                     lds + (j * PI + i) * 1024);
    __builtin_amdgcn_sched_barrier(0);  // all of the block's loads before the first wait for one
    f32x4 s[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int st = 0; st < KST; ++st) {
        bf16x8 k;
        if constexpr (FP8) {
          const u32x4 c = kf[i][st >> 1];
          k = st & 1 ? e4m3_to_bf16x8(c.z, c.w, ksc[i]) : e4m3_to_bf16x8(c.x, c.y, ksc[i]);
        } else {
          k = __builtin_bit_cast(bf16x8, kf[i][st]);
        }
        s[i] = mfma_bf16(k, qf[st], s[i]);
      }
    }
    const uint64_t vis = ok & keys_to(pos - kb);
    const bool masked = __ballot(vis != ~0ull) != 0;
    if (FP8 && masked) {  // a scale byte of a key that the row does not see may be anything, and 0 times it not 0
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const uint32_t bits = (uint32_t)(vis >> (32 * c + 8 * g));
        vsc[c].x &= ((bits & 15) * 0x204081u & 0x01010101u) * 255u;
        vsc[c].y &= ((bits >> 4 & 15) * 0x204081u & 0x01010101u) * 255u;
      }
    }
    u32x4 pf[2];
    const float alpha = softmax_block<FP8>(s, masked, vis, g, p.c2, vsc, m, den, pf);
#pragma unroll
    for (int dt = 0; dt < DTN; ++dt) o[dt] = o[dt] * alpha;
    wait_vmcnt<0>();
    wait_lds();
    if (ok != ~0ull) {  // values that are not there may be anything, and 0 times it not 0
      if (!(ok >> lane & 1)) {
#pragma unroll
        for (int j = 0; j < RB / 16; ++j)
          *reinterpret_cast<u32x4*>(smem + wave * SLAB + lane * RB + 16 * j) = u32x4{0, 0, 0, 0};
      }
      wait_lds();
    }
    // Where the tile's rows see different keys, one that a row does not see may be odd, and 0 times
    // its value not 0: the product takes the finite values, and a row adds the odd ones it sees.
    if (__ballot(real && vis != ok) && values_odd<D, FP8>(another(lds), r16, g)) {
      const uint32_t lds1 = another(lds);
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int dt = 0; dt < DTN; ++dt)
          o[dt] = mfma_bf16(finite_only(v_fragment<D, FP8>(lds1, c, dt, r16, g)), pf[c], o[dt]);
#pragma unroll 1
      for (int key = 0; key < 64; ++key) {
        const uint8_t* at = smem + wave * SLAB + key * RB;
#pragma unroll
        for (int dt = 0; dt < DTN; ++dt) {
          f32x4 x;
          const int place = v_swizzle<RB, FP8>(key);
          if constexpr (FP8) {  // the only odd code is NaN
            const uint32_t w = *reinterpret_cast<const uint32_t*>(at + 16 * (dt ^ place) + 4 * g);
#pragma unroll
            for (int r = 0; r < 4; ++r) x[r] = (w >> (8 * r) & 0x7F) == 0x7F ? __builtin_nanf("") : 0.f;
          } else {
            x = odd_only(*reinterpret_cast<const u32x2*>(at + 16 * ((2 * dt + (g >> 1)) ^ place) + 8 * (g & 1)));
          }
          if (vis >> key & 1) o[dt] = o[dt] + x;
        }
      }
      continue;
    }
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int dt = 0; dt < DTN; ++dt) o[dt] = mfma_bf16(v_fragment<D, FP8>(lds, c, dt, r16, g), pf[c], o[dt]);
  }
  den = sum_rows(den);

  // join the waves
  float* so = reinterpret_cast<float*>(smem);
  float* sm = so + NW * 16 * LDO;
  float* sd = sm + NW * 16;
  __syncthreads();
  if (real) {
#pragma unroll
    for (int dt = 0; dt < DTN; ++dt) *reinterpret_cast<f32x4*>(so + (wave * 16 + r16) * LDO + 16 * dt + 4 * g) = o[dt];
  }
  if (g == 0) {
    sm[wave * 16 + r16] = m;
    sd[wave * 16 + r16] = den;
  }
  __syncthreads();
  const int here = min(rows - it.tile * 16, 16);  // rows of the tile
  for (int e = threadIdx.x; e < here * (D / 4); e += 64 * NW) {
    const int r = e / (D / 4), d0 = e % (D / 4) * 4;
    float mx = -INFINITY;
#pragma unroll
    for (int w = 0; w < NW; ++w) mx = fmaxf(mx, sm[w * 16 + r]);
    const float mref = mx == -INFINITY ? 0.f : mx;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float wt = __builtin_amdgcn_exp2f(sm[w * 16 + r] - mref);
      sum += sd[w * 16 + r] * wt;
      fma4(acc, *reinterpret_cast<const f32x4*>(so + (w * 16 + r) * LDO + d0), wt);
    }
    const int rr = it.tile * 16 + r, query = DECODE ? 0 : rr / p.group;
    const int64_t to = (int64_t)(it.s.row0 + query) * (p.hk * p.group) + head * p.group + rr - query * p.group;
    if (it.splits == 1) {
      const float inv = inverse_sum(mx, sum);
      *reinterpret_cast<u32x2*>(p.y + to * D + d0) = pack4_bf16(acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv);
      if (!DECODE && p.budget && d0 == 0) p.part_of[to] = int2{0, 1};
    } else {
      const int64_t at = ((int64_t)it.slot * p.hk + head) * 16 + r;
      *reinterpret_cast<f32x4*>(p.part_o + at * D + d0) = acc;
      if (d0 == 0) p.part_s[at] = float2{mx, sum};
      if (d0 == 0 && it.split == 0) p.part_of[to] = int2{(int)at, it.splits};
    }
  }
}

// ------------------------------------------------------------------ many rows
//
// One workgroup per item: NW waves of 32 rows each share the item's 64-key blocks, which
// pass through LDS in three stages (bf16 pages by DMA; codes through registers, where they
// become scaled bf16, in two). v_mfma_f32_32x32x16_bf16: a lane's scores and sums
// belong to one row, and 16 of a 32-key tile's scores are the two operand
// registers of the second product. The reference moves only where a score passes it, and
// then to 2^8 times that score: P is 1 at most and mostly near 2^-8, which costs nothing in a
// floating-point format, and the sums are rescaled in few blocks only. Bound by the matrix instructions with the softmax beside
// them: 2048 tokens over 32748 positions, 32 / 8 heads of 128, 1.03 ms (1.03 PFLOP/s; the products alone 1.13
// in a copy of the kernel; 16 x 16 x 32 tiles a wave 5.35 ms, four waves of 32 rows 1.06, of 64 1.48). 64 dims
// have half the products for the same exponentials: 0.60 ms, 0.88 PFLOP/s.
// (DMA in two stages where 32 rows a wave leave room for two workgroups a CU.)
//
// LDS rows are bf16 (RB = 2 D bytes); 16-byte chunk c of key k is kept at chunk
// c ^ k_place(k) (keys: the 16 keys that a fragment read takes together fall on different
// banks), c ^ v_place(k) (values: 4 keys x 64 bytes do).
typedef float f32x16 __attribute__((ext_vector_type(16)));

template <int D>
__device__ __forceinline__ int k_place(int key) {
  return D == 128 ? key & 15 : (key >> 1) & 7;
}
template <int D>
__device__ __forceinline__ int v_place(int key) {
  return D == 128 ? 4 * (key & 3) : 4 * ((key >> 1) & 1);
}

__device__ __forceinline__ f32x16 mfma32(const bf16x8& a, const u32x4& b, const f32x16& c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// V^T fragment of 16 keys from 16 c, dims 32 dt ..: lane 32 h + r gets keys 16 c + 8 h .. + 7 of
// dim 32 dt + r.
template <int D>
__device__ __forceinline__ bf16x8 v_fragment32(uint32_t lds, int c, int dt, int lane) {
  // the lane's address for dims 32 dt .., to which keys add a constant
  const int key = 8 * (lane >> 5) + ((lane >> 2) & 3);
  const int chunk = (4 * dt + 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1)) ^ v_place<D>(key);
  const uint32_t at = lds + key * 2 * D + 16 * chunk + 8 * (lane & 1);
  s16x4 v[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) v[i] = read_tr16(at, (16 * c + 4 * i) * 2 * D);
  typedef short s16x8 __attribute__((ext_vector_type(8)));
  return __builtin_bit_cast(bf16x8, (s16x8)__builtin_shufflevector(v[0], v[1], 0, 1, 2, 3, 4, 5, 6, 7));
}

__device__ __forceinline__ float max_halves(float x) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ float sum_halves(float x) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

// values_odd on this kernel's fragments.
template <int D>
__device__ __forceinline__ bool values_odd32(uint32_t lds, int lane) {
  const u32x4 ones = {0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u};
  f32x16 t = {};
#pragma unroll
  for (int c = 0; c < 4; ++c)
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt) {
      t = mfma32(v_fragment32<D>(lds, c, dt, lane), ones, t);
      __builtin_amdgcn_sched_barrier(0);
    }
  bool odd = false;
#pragma unroll
  for (int r = 0; r < 16; ++r) odd |= !(fabsf(t[r]) < INFINITY);
  return __ballot(odd) != 0;
}

template <int D, bool FP8, int NW>
__global__ __launch_bounds__(64 * NW, NW == 4 ? 2 : 1) void many_rows_kernel(Args p) {
  constexpr int RB = 2 * D, KST = D / 16, DTN = D / 32;
  constexpr int NS = FP8 || NW == 4 ? 2 : 3, HALF = 64 * RB, STAGE = 2 * HALF;
  constexpr int TASKS = 8 / NW;      // of the 8 16-key groups of a block's keys and values, a wave's
  constexpr int PI = 16 * RB / 1024; // DMAs of a group
  __shared__ __align__(1024) uint8_t smem[NS * STAGE];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r32 = lane & 31, h = lane >> 5;
  const int head = (int)blockIdx.x % p.hk, id = (int)blockIdx.x / p.hk;
  Item it;
  if (!find_item(p, lane, id, &it)) return;
  const int rows = it.s.n * p.group, row0 = (it.tile << p.lbm) + wave * 32;
  const int shift = it.s.len - it.s.n;  // position of query 0
  const int kend = min(it.s.keys, shift + min(rows - 1, ((it.tile + 1) << p.lbm) - 1) / p.group + 1);
  const int nb = max(0, kend + 63) >> 6, per = (nb + it.splits - 1) / it.splits;
  const int b0 = it.split * per, b1 = min(nb, b0 + per);

  // keys that some row of the wave sees, and that all the tile's rows see
  const int some = row0 < rows ? shift + min(rows - 1, row0 + 31) / p.group + 1 : 0;
  const int all = shift + (it.tile << p.lbm) / p.group + 1;

  u32x4 qf[KST];
  const int row = row0 + r32, real = min(row, rows - 1);
  const int pos = row < rows ? shift + row / p.group : -1;
  const bf16_t* qp = p.q + (it.s.row0 + real / p.group) * p.q_ts + (head * p.group + real % p.group) * p.q_hs + 8 * h;
  const bool vec = ((uintptr_t)p.q & 15) == 0 && ((p.q_ts | p.q_hs) & 7) == 0;
#pragma unroll
  for (int st = 0; st < KST; ++st) {
    if (vec) {
      qf[st] = *reinterpret_cast<const u32x4*>(qp + 16 * st);
    } else {
      float x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = bf16_to_f32(qp[16 * st + i]);
      qf[st] = pack8(x);
    }
  }
  // waited for here, not behind the first blocks' loads
#pragma unroll
  for (int st = 0; st < KST; ++st)
    asm volatile("" : : "v"(qf[st].x), "v"(qf[st].y), "v"(qf[st].z), "v"(qf[st].w));

  f32x16 o[DTN];
  float m = -INFINITY, den = 0.f;
#pragma unroll
  for (int dt = 0; dt < DTN; ++dt) o[dt] = f32x16{};

  // The table is read through the scalar cache: a vector load would be waited for together
  // with the blocks' DMAs.
  typedef const __attribute__((address_space(4))) int* ConstInts;
  const ConstInts table =
      (ConstInts)(uintptr_t)(p.a.table + (int64_t)min(it.seq, p.a.batch - 1) * p.a.width);
  const uint32_t lds0 = lds_addr(smem);
  const int in_page = (1 << p.a.lps) - 1;
  // A block's table entries, one for each 16 keys; read a block ahead of their use.
  struct Entries {
    int e[4];
  };
  auto entries = [&](int b) {
    Entries n;
#pragma unroll
    for (int j = 0; j < 4; ++j) n.e[j] = table[min((int64_t)((64 * b + 16 * j) >> p.a.lps), p.a.width - 1)];
    return n;
  };
  auto page_there = [&](int e) { return (unsigned)e < (unsigned)p.a.pages; };
  auto keys_there = [&](int b, const Entries& n) {
    uint64_t ok = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) ok |= page_there(n.e[j]) ? 0xFFFFull << (16 * j) : 0;
    return ok & keys_to(kend - 1 - 64 * b);
  };
  // Row of the pages' (page, head, slot) of the first of 16 keys (uniform).
  auto first_row = [&](int b, int grp, const Entries& n) {
    const int e = grp == 0 ? n.e[0] : grp == 1 ? n.e[1] : grp == 2 ? n.e[2] : n.e[3];
    return (((int64_t)(page_there(e) ? e : 0) * p.hk + head) << p.a.lps) + ((64 * b + 16 * grp) & in_page);
  };

  // One block into LDS. bf16: DMA of this wave's groups. Codes: into registers (load), and later
  // scaled to LDS (store).
  constexpr int CK = D / 16, CH = FP8 ? 2 * CK / NW : 1;  // 16-code chunks of a key, of a thread
  u32x4 code[CH];
  uint32_t byte[CH];
  uint32_t k_from[FP8 ? 1 : PI], v_from;  // where a lane's 16 bytes lie among a group's keys (i-th DMA), values (first)
  if constexpr (!FP8) {
#pragma unroll
    for (int i = 0; i < PI; ++i) {
      const int off = i * 1024 + lane * 16, key = off / RB, chunk = off % RB / 16;
      k_from[i] = key * RB + 16 * (chunk ^ k_place<D>(key)) - i * 1024;
      if (i == 0) v_from = key * RB + 16 * (chunk ^ v_place<D>(key));  // v_place repeats every 1024 bytes
    }
  }
  auto issue = [&](int b, int buf, const Entries& n) {
#pragma unroll
    for (int j = 0; j < TASKS; ++j) {
      const int task = wave + j * NW, grp = task & 3;
      const bool values = task >> 2;
      const uint8_t* src = (values ? p.v : p.k) + first_row(b, grp, n) * RB;
      const uint32_t dst = lds0 + buf * STAGE + values * HALF + grp * 16 * RB;
#pragma unroll
      for (int i = 0; i < PI; ++i)
        lds_dma16_at(src + i * 1024, values ? v_from : k_from[i], dst + i * 1024);
    }
  };
  auto load = [&](int b, const Entries& n) {
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int c0 = (i * NW + wave) * 64;  // the wave's first chunk; all of them are of one 16-key group
      const int key0 = c0 / CK & 63, key = key0 + lane / CK;
      const bool values = c0 >= 64 * CK;
      const int64_t at = first_row(b, key0 >> 4, n) + (key & 15);
      code[i] = *reinterpret_cast<const u32x4*>((values ? p.v : p.k) + at * D + 16 * (lane % CK));
      byte[i] = (values ? p.vs : p.ks)[at];
    }
  };
  auto store = [&](int buf, uint64_t there) {
    if (there != ~0ull) {  // nothing is read as zero (waits for the loads here alone)
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        const bool it = there >> (((i * NW + wave) * 64 / CK & 63) + lane / CK) & 1;
        code[i] = it ? code[i] : u32x4{0, 0, 0, 0};
        byte[i] = it ? byte[i] : 0;
      }
    }
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int c0 = (i * NW + wave) * 64, key = (c0 / CK & 63) + lane / CK, chunk = 2 * (lane % CK);
      const bool values = c0 >= 64 * CK;
      const int place = values ? v_place<D>(key) : k_place<D>(key);
      uint8_t* to = smem + buf * STAGE + values * HALF + key * RB;
      const float s = scale_of(byte[i]);
      *reinterpret_cast<bf16x8*>(to + 16 * (chunk ^ place)) = e4m3_to_bf16x8(code[i].x, code[i].y, s);
      *reinterpret_cast<bf16x8*>(to + 16 * ((chunk + 1) ^ place)) = e4m3_to_bf16x8(code[i].z, code[i].w, s);
    }
  };

  // Zeros in place of a block's infinite values and NaN.
  auto scrub = [&](int buf) {
    barrier_lds();
    for (int e = threadIdx.x; e < HALF / 16; e += 64 * NW) {
      bf16x8* at = reinterpret_cast<bf16x8*>(smem + buf * STAGE + HALF + 16 * e);
      *at = finite_only(*at);
    }
    barrier_lds();
  };

  // The keys of blocks b, b + 1 (and b + 2) that are there, and the entries of the one after.
  uint64_t ok = 0, ok1 = 0, ok2 = 0;
  Entries ahead = entries(b0);
  if (b0 < b1) {
    ok = keys_there(b0, ahead);
    if constexpr (FP8) {
      load(b0, ahead);
      store(0, ok);
    } else {
      issue(b0, 0, ahead);
    }
    ahead = entries(b0 + 1);
  }
  if (b0 + 1 < b1) {
    ok1 = keys_there(b0 + 1, ahead);
    if constexpr (FP8) load(b0 + 1, ahead);
    else if (NS == 3) issue(b0 + 1, 1, ahead);
    if (FP8 || NS == 3) ahead = entries(b0 + 2);
  }
  for (int b = b0; b < b1; ++b, ok = ok1, ok1 = ok2) {
    const int kb = 64 * b, buf = (b - b0) % NS;
    if constexpr (FP8) {
      barrier_lds();  // block b is there for every wave, block b - 1 no longer read
      if (b + 1 < b1) store(buf ^ 1, ok1);
    } else {
      if (NS == 3 && b + 1 < b1) wait_vmcnt<TASKS * PI>();
      else wait_vmcnt<0>();
      barrier_lds();
    }
    constexpr int AHEAD = FP8 || NS == 3 ? 2 : 1;
    if (b + AHEAD < b1) {
      if constexpr (FP8) load(b + 2, ahead);
      else issue(b + AHEAD, (b - b0 + AHEAD) % NS, ahead);
      (AHEAD == 2 ? ok2 : ok1) = keys_there(b + AHEAD, ahead);
      ahead = entries(b + AHEAD + 1);
    }
    const uint32_t lds = lds0 + buf * STAGE;
    if (!FP8 && ok != ~0ull) {  // values that are not there may be anything, and 0 times it not 0
      for (int e = threadIdx.x; e < HALF / 16; e += 64 * NW)
        if (!(ok >> (e * 16 / RB) & 1)) *reinterpret_cast<u32x4*>(smem + buf * STAGE + HALF + 16 * e) = u32x4{0, 0, 0, 0};
      barrier_lds();
    }
    // Where the tile's rows see different keys, one that a row does not see may have odd values, and
    // 0 times them is not 0: a row adds the odd ones that it sees, and the product takes the
    // finite ones. The same for all waves.
    const bool odd = !(ok == ~0ull && kb + 64 <= all) && values_odd32<D>(another(lds + HALF), lane);
    if (kb >= some) {
      if (odd) scrub(buf);
      continue;
    }

    // matrix row r32 of key tile kt is key 32 kt + 16 (r32 / 16) + 8 (r32 / 4 % 2) + 4 (r32 / 8 % 2) + r32 % 4
    const int key = (r32 & 16) + ((r32 & 4) << 1) + ((r32 & 8) >> 1) + (r32 & 3);
    auto k_fragment = [&](int kt, int st) {
      return *reinterpret_cast<const bf16x8*>(smem + buf * STAGE + (32 * kt + key) * RB +
                                              16 * ((2 * st + h) ^ k_place<D>(key)));
    };
    f32x16 s[2] = {};
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int st = 0; st < KST; ++st) s[kt] = mfma32(k_fragment(kt, st), qf[st], s[kt]);
    u32x4 pf[4];
    float least = kLeast;
    const bool full = ok == ~0ull && kb + 64 <= all;
    if (!full) {
      asm volatile("");  // a branch: as selects the masks would be computed for every block
      const uint64_t vis = ok & keys_to(pos - kb);
      least = vis ? kLeast : -INFINITY;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const uint32_t bits = (uint32_t)(vis >> (16 * c + 8 * h));
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int i = 8 * (c & 1) + e;
          s[c >> 1][i] = bits >> e & 1 ? s[c >> 1][i] : -INFINITY;
        }
      }
    }
    float top = s[0][0];
#pragma unroll
    for (int i = 1; i < 32; ++i) top = __builtin_elementwise_maximum(top, s[i >> 4][i & 15]);
    top = fmaxf(max_halves(top) * p.c2, least);  // (drops NaN)
    if (__ballot(top > m)) {
      const float mnew = top > m ? top + 8.f : m, mref = mnew == -INFINITY ? 0.f : mnew;
      const float alpha = __builtin_amdgcn_exp2f(m - mref);
      m = mnew;
      den *= alpha;
#pragma unroll
      for (int dt = 0; dt < DTN; ++dt) o[dt] = o[dt] * alpha;
    }
    const float mref = m == -INFINITY ? 0.f : m;
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[c >> 1][8 * (c & 1) + e], p.c2, -mref));
        sum[e & 3] += x[e];
      }
      pf[c] = pack8(x);
    }
    den += (sum[0] + sum[1]) + (sum[2] + sum[3]);
    if (odd) {
#pragma unroll 1
      for (int key = 0; key < 64; ++key) {
        const uint8_t* at = smem + buf * STAGE + HALF + key * RB + 8 * h;
#pragma unroll
        for (int i = 0; i < 4 * DTN; ++i) {
          const f32x4 x = odd_only(*reinterpret_cast<const u32x2*>(at + 16 * (i ^ v_place<D>(key))));
#pragma unroll
          for (int e = 0; e < 4; ++e)
            o[i >> 2][4 * (i & 3) + e] += (ok & keys_to(pos - kb)) >> key & 1 ? x[e] : 0.f;
        }
      }
      scrub(buf);
    }
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int dt = 0; dt < DTN; ++dt) o[dt] = mfma32(v_fragment32<D>(lds + HALF, c, dt, lane), pf[c], o[dt]);
  }

  // lane (h, r32) holds dims 32 dt + 8 a + 4 h .. + 3 of its row
  const float sum = sum_halves(den);
  if (row >= rows) return;
  const int64_t to = (int64_t)(it.s.row0 + row / p.group) * (p.hk * p.group) + head * p.group + row % p.group;
  if (it.splits == 1) {
    const float inv = inverse_sum(m, sum);
#pragma unroll
    for (int i = 0; i < 4 * DTN; ++i) {
      const f32x16& x = o[i >> 2];
      const int a = 4 * (i & 3);
      *reinterpret_cast<u32x2*>(p.y + to * D + 8 * i + 4 * h) =
          pack4_bf16(x[a] * inv, x[a + 1] * inv, x[a + 2] * inv, x[a + 3] * inv);
    }
    if (p.budget && h == 0) p.part_of[to] = int2{0, 1};
  } else {
    const int64_t at = (((int64_t)it.slot * p.hk + head) << p.lbm) + (row - (it.tile << p.lbm));
#pragma unroll
    for (int i = 0; i < 4 * DTN; ++i) {
      const f32x16& x = o[i >> 2];
      const int a = 4 * (i & 3);
      *reinterpret_cast<f32x4*>(p.part_o + at * D + 8 * i + 4 * h) = f32x4{x[a], x[a + 1], x[a + 2], x[a + 3]};
    }
    if (h == 0) p.part_s[at] = float2{m, sum};
    if (h == 0 && it.split == 0) p.part_of[to] = int2{(int)at, it.splits};
  }
}

// ------------------------------------------------------------------ joining split tiles

// A row (token, head) is joined by GROUPS groups of D / 4 lanes, 4 dims a lane, each group taking
// every GROUPS-th split with a running reference of its own. Few rows: 256 threads a row, so
// that a long list of splits is short for each; many rows: a group a row. Rows of unsplit
// tiles are there already.
template <int D, bool WIDE>
__global__ __launch_bounds__(256) void join_kernel(Args p) {
  constexpr int LPR = D / 4, PER = 64 / LPR, GROUPS = WIDE ? 4 * PER : 1;
  __shared__ f32x4 parts[WIDE ? 256 : 1];
  __shared__ float2 stats[WIDE ? GROUPS : 1];
  const int group = threadIdx.x / LPR, dim = threadIdx.x % LPR * 4;
  const int row = WIDE ? blockIdx.x : (int)blockIdx.x * 4 * PER + group;
  if (row >= p.a.t * p.hk * p.group) return;
  const int2 of = p.part_of[row];
  const int64_t at0 = of.x;
  const int splits = of.y;
  const int64_t step = (int64_t)p.hk << p.lbm;  // from a split's row to the next one's
  // (starts that do not rise leave rows that no tile has)
  if (splits <= 1 || at0 < 0 || at0 + (splits - 1) * step >= ((int64_t)p.slots * p.hk) << p.lbm) return;
  float m = -INFINITY, sum = 0.f;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int i0 = WIDE ? group : 0; i0 < splits; i0 += 4 * GROUPS) {
    float2 st[4];
    f32x4 o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool there = i0 + i * GROUPS < splits;
      const int64_t at = at0 + (there ? i0 + i * GROUPS : i0) * step;
      st[i] = p.part_s[at];
      o[i] = *reinterpret_cast<const f32x4*>(p.part_o + at * D + dim);
      if (!there) st[i] = float2{-INFINITY, 0.f};
    }
    const float mnew = fmaxf(fmaxf(m, fmaxf(st[0].x, st[1].x)), fmaxf(st[2].x, st[3].x));
    const float mref = mnew == -INFINITY ? 0.f : mnew;
    const float alpha = __builtin_amdgcn_exp2f(m - mref);
    sum *= alpha;
    acc = acc * alpha;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // (a split without keys, and one read twice in place of none, count for nothing)
      const float w = __builtin_amdgcn_exp2f(st[i].x - mref);
      if (st[i].x != -INFINITY) {
        sum = __builtin_fmaf(st[i].y, w, sum);
        fma4(acc, o[i], w);
      }
    }
    m = mnew;
  }
  if (WIDE) {
    parts[threadIdx.x] = acc;
    if (dim == 0) stats[group] = float2{m, sum};
    __syncthreads();
    if (group) return;
    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < GROUPS; ++i) mx = fmaxf(mx, stats[i].x);
    const float mref = mx == -INFINITY ? 0.f : mx;
    m = mx;
    acc = f32x4{0.f, 0.f, 0.f, 0.f};
    sum = 0.f;
#pragma unroll
    for (int i = 0; i < GROUPS; ++i) {
      const float w = __builtin_amdgcn_exp2f(stats[i].x - mref);
      sum = __builtin_fmaf(stats[i].y, w, sum);
      fma4(acc, parts[i * LPR + threadIdx.x], w);
    }
  }
  const float inv = inverse_sum(m, sum);
  *reinterpret_cast<u32x2*>(p.y + (int64_t)row * D + dim) =
      pack4_bf16(acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv);
}

// ------------------------------------------------------------------ host

struct Plan {
  int kind;  // 0: few rows; 1, 2: many rows on 4 and 8 waves
  bool decode;
  int lbm, least, budget;
  int64_t items, slots;  // per key head
  bool listed;    // a launch writes the list
};

// 256-row tiles (one workgroup of 8 waves a CU) against 128-row ones (two or three of 4): half the loads
// of keys and values, coarser work. Ahead where there is a tile for every CU and the table may hold
// eight times the new tokens or more, so that tiles are equally long; at 128 dims also where there are two
// tiles a CU; for codes at 128 dims (two workgroups a CU leave them short of registers) where the
// table may hold four times the new tokens. us, 256 against 128 rows, 32 / 8 heads: 2048 tokens over 30700
// positions 1021 and 1060 (64 dims 636 and 705), over 4000 196 and 181, 4096 over none 153 and 157 (64
// dims 107 and 93); codes: 512 over 4000 59 and 64, 4096 over none 159 and 186, 2048 over none 76 and 72.
bool wide_tiles(int64_t rows, int64_t t, int64_t batch, int64_t hk, int64_t d, int fp8, int64_t capacity) {
  const int64_t all = rows * hk, depth = capacity * batch;
  if (all >= 65536 && depth >= 8 * t) return true;
  if (d == 64) return false;
  return all >= 131072 || (fp8 && all >= 16384 && depth >= 4 * t);
}

// The sizes of the call are all that the host knows: a table that reaches further than the sequences has their
// kernel, splits and join chosen for what it may hold (one token over 577 positions 11 us, 13.6 with a table of 8192;
// 61 tokens over 176 9.6 and 15).
Plan plan_of(int64_t t, int64_t batch, bool starts, int64_t hk, int64_t group, int64_t d, int fp8, int64_t capacity) {
  const int64_t rows = t * group;
  const int force = ff_tuning(FF_TUNE_PAGED_ROWS);
  Plan p = {};
  // 16-row tiles read the cache once a tile, and a wave has a block of its own: ahead where every
  // sequence is one tile, and while the (tile, block) pairs that the table can hold are about as many as
  // the GPU's waves (2048; twice that for codes, whose way through registers to LDS makes the large tiles slower
  // to begin). us, 16-row against 128-row tiles, 32 / 8 heads: 40 tokens over 1000 positions (1360 pairs) 17.3 and
  // 19.3, 100 over 1000 (3600) 23.4 and 22.3, 100 over 4000 (13000) 54.1 and 29.5, 8 sequences of 16 over 500 (2304)
  // 23.1 and 23.1, over 1000 (4352) 32.7 and 23.2; codes: 100 over 1000 18.6 and 24.8, 8 of 40 over 500 (5760)
  // 33.6 and 29.5, 100 over 4000 33.5 and 34.4.
  const int64_t pairs = (rows / 16 + batch) * hk * ((capacity + 63) / 64);
  if (force) p.kind = force - 1;
  else if (rows <= 16 * batch || pairs <= (fp8 ? 5120 : 2560)) p.kind = 0;
  else p.kind = wide_tiles(rows, t, batch, hk, d, fp8, capacity) ? 2 : 1;
  // One row a sequence, a table of up to 768 positions, a CU for each tile: one launch. A CU takes in 64 bytes a
  // clock at most, so that longer caches are better shared by several and joined. us, one launch and splits, 32 / 8
  // heads of 128: 320 positions 9.1 and 13.7, 577 11.2 and 13.9, 768 11.8 and 13.7, 1024 15.3 and 14.0, 1500 20.6 and
  // 13.9; codes 768 9.3 and 13.5, 1024 10.3 and 13.6, 1500 12.8 and 13.5; 32 sequences of 577 16.1 and 21.2.
  const int64_t decode = (group + 15) / 16 * t;
  if (p.kind == 0 && !starts && capacity <= 768 && decode * hk <= 256) {
    p.decode = true;
    p.lbm = 4;
    p.items = decode;
    return p;
  }
  p.lbm = p.kind == 0 ? 4 : p.kind == 1 ? 7 : 8;
  p.least = p.kind == 0 ? kFewWaves : 8;
  // workgroups that the GPU holds at once: 256 CUs, by registers and LDS
  const int64_t workgroups = 256 * (p.kind == 0 ? 2 : p.kind == 1 ? (d == 64 ? 3 : 2) : (d == 64 && !fp8 ? 2 : 1));
  const int64_t tiles = (rows >> p.lbm) + batch + 1;
  const int64_t budget = workgroups / hk > 0 ? workgroups / hk : 1;
  // No splits where a sequence's keys are one chunk whatever its length is, nor where the tiles are many
  // (one sequence: as many as workgroups; more: twice as many, for sequences that are about equally long).
  if ((capacity + 63) / 64 > p.least && (rows >> p.lbm) < (batch == 1 ? 1 : 2) * budget) p.budget = (int)budget;
  // More sequences than a wave's lanes are split in 16-row tiles all the same where one may be far longer than a
  // workgroup's share, with starts and without. 1024 sequences of 100 positions, one of 60000 among them, 179 us
  // (without splits 794, by starts 808); what that costs where they are equal: 1024 rows over 200 positions each by
  // starts 204 us against 199, 3 rows each 226 against 218, 200 rows beside 1000 of one prompt 498 against 492.
  if (p.kind == 0 && !fit_lanes(batch, starts) && capacity > 4096) p.budget = (int)budget;
  p.items = tiles + p.budget;
  p.slots = 2 * p.budget < p.items ? 2 * p.budget : p.items;  // (1536, or 2 hk, for all heads: their rows fit 32 bits)
  // (no list: 16-row tiles of one row a sequence that are not split)
  p.listed = !fit_lanes(batch, starts) && (starts || p.budget || p.kind);
  return p;
}

int threads_of(const Plan& p) { return 64 * (p.decode ? kDecodeWaves : p.kind == 2 ? 8 : 4); }

// Rows (token, head) of a workgroup of the join. us, one and 8 or 16: one token over 131072 positions (32 rows, 64
// splits) 101 and 120; from 512 rows on they are even; 6 chunks of about 300 tokens of 20 heads 78 and 56.
int64_t join_rows(int64_t t, int64_t hq, int64_t d) { return t * hq <= 2048 ? 1 : 1024 / d; }

// A launch has fewer than 2^32 threads; past that it would fail between others that do not.
int check_launches(const char* what, const Plan& p, int64_t t, int64_t hq, int64_t hk, int64_t d) {
  const int64_t per = join_rows(t, hq, d);
  FF_REQUIRE(p.items * hk <= (int64_t)UINT32_MAX / threads_of(p) &&
                 (!p.budget || (t * hq + per - 1) / per <= (int64_t)UINT32_MAX / 256),
             "%s: too large a call (%lld workgroups)", what, (long long)(p.items * hk));
  return FF_OK;
}

// (sizes of the cache and the rows are checked already)
int check_sizes(const char* what, const ff_paged_cache* c, int64_t hq, int64_t width, int64_t batch, int64_t t) {
  FF_REQUIRE(hq > 0 && hq <= 65535 && hq % c->hk == 0, "%s: bad sizes hq=%lld hk=%lld", what, (long long)hq,
             (long long)c->hk);
  const int64_t tiles = t * (hq / c->hk) / 16 + batch + 1;
  FF_REQUIRE(tiles * ((width * c->page_size + 63) / 64) <= INT32_MAX && (tiles + 768) * c->hk <= INT32_MAX &&
                 t * hq <= INT32_MAX,
             "%s: too large a call (rows x positions)", what);
  return FF_OK;
}

// Partial sums, their statistics, the rows' notes; the list.
int64_t parts_bytes(const Plan& p, int64_t t, int64_t hq, int64_t hk, int64_t d) {
  return p.budget ? ((p.slots * hk) << p.lbm) * (d * 4 + 8) + t * hq * 8 : 0;
}
int64_t workspace_of(const Plan& p, int64_t t, int64_t hq, int64_t hk, int64_t d, int64_t batch) {
  return parts_bytes(p, t, hq, hk, d) + (p.listed ? (2 * batch + 4) * 4 : 0);
}

}  // namespace

extern "C" int ff_attention_paged_workspace(const ff_paged_cache* cache, int64_t hq, int64_t width, int64_t batch,
                                            int starts, int64_t t, int64_t* bytes) {
  FF_REQUIRE(bytes, "ff_attention_paged_workspace: null pointer");
  *bytes = 0;
  if (t == 0) return FF_OK;
  int st = check_cache("ff_attention_paged_workspace", cache);
  if (st != FF_OK) return st;
  FF_REQUIRE(width > 0 && width <= kMaxPositions / cache->page_size && batch > 0 && batch <= 65536 && t > 0 && t <= (1 << 24),
             "ff_attention_paged_workspace: bad sizes width=%lld batch=%lld t=%lld", (long long)width, (long long)batch,
             (long long)t);
  st = check_sizes("ff_attention_paged_workspace", cache, hq, width, batch, t);
  if (st != FF_OK) return st;
  const Plan plan =
      plan_of(t, batch, starts, cache->hk, hq / cache->hk, cache->d, cache->fp8 != 0, width * cache->page_size);
  st = check_launches("ff_attention_paged_workspace", plan, t, hq, cache->hk, cache->d);
  if (st != FF_OK) return st;
  *bytes = workspace_of(plan, t, hq, cache->hk, cache->d, batch);
  return FF_OK;
}

extern "C" int ff_attention_paged(const void* q, int64_t q_ts, int64_t q_hs, const ff_paged_cache* cache, int64_t hq,
                                  const int32_t* table, int64_t width, const int32_t* lengths, const int32_t* starts,
                                  int64_t batch, void* y, int64_t t, float scale, void* workspace,
                                  int64_t workspace_bytes, ff_stream_t stream) {
  if (t == 0) return FF_OK;
  int st = check_rows("ff_attention_paged", cache, table, width, lengths, starts, batch, t);
  if (st != FF_OK) return st;
  st = check_sizes("ff_attention_paged", cache, hq, width, batch, t);
  if (st != FF_OK) return st;
  FF_REQUIRE(q && y, "ff_attention_paged: null pointer");
  FF_REQUIRE(scale > 0.f && scale < __builtin_inff(), "ff_attention_paged: scale %g", (double)scale);
  FF_REQUIRE(ff_aligned(y, 16), "ff_attention_paged: alignment");
  const int64_t hk = cache->hk, d = cache->d;
  const bool fp8 = cache->fp8 != 0;
  const Plan plan = plan_of(t, batch, starts != nullptr, hk, hq / hk, d, fp8, width * cache->page_size);
  st = check_launches("ff_attention_paged", plan, t, hq, hk, d);
  if (st != FF_OK) return st;
  const int64_t need = workspace_of(plan, t, hq, hk, d, batch);
  FF_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && ff_aligned(workspace, 16)),
             "ff_attention_paged: workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)need);
  Args p;
  p.a = rows_of(cache, table, width, lengths, starts, batch, t);
  p.q = (const bf16_t*)q;
  p.q_ts = q_ts;
  p.q_hs = q_hs;
  p.k = (const uint8_t*)cache->k;
  p.v = (const uint8_t*)cache->v;
  p.ks = (const uint8_t*)cache->k_scale;
  p.vs = (const uint8_t*)cache->v_scale;
  p.y = (bf16_t*)y;
  p.part_o = (float*)workspace;
  p.part_s = (float2*)((char*)workspace + ((plan.slots * hk) << plan.lbm) * d * 4);
  p.part_of = (int2*)(p.part_s + ((plan.slots * hk) << plan.lbm));
  p.plan = plan.listed ? (int*)((char*)workspace + parts_bytes(plan, t, hq, hk, d)) : nullptr;
  p.hk = (int)hk;
  p.group = (int)(hq / hk);
  p.lbm = plan.lbm;
  p.least = plan.least;
  p.budget = plan.budget;
  p.slots = (int)plan.slots;
  p.c2 = (float)((double)scale * 1.4426950408889634);
  const dim3 grid((unsigned)(plan.items * hk));
  const int64_t per = join_rows(t, hq, d);
  const bool wide = per == 1;
  const dim3 join((unsigned)((t * hq + per - 1) / per));
  hipStream_t s = (hipStream_t)stream;
  if (plan.listed) hipLaunchKernelGGL(plan_kernel, dim3(1), dim3(1024), 0, s, p);
  const dim3 block((unsigned)threads_of(plan));
#define FF_PAGED(DIM, F8)                                                                                          \
  if (d == DIM && fp8 == F8) {                                                                              \
    if (plan.decode) hipLaunchKernelGGL((few_rows_kernel<DIM, F8, kDecodeWaves, true>), grid, block, 0, s, p);     \
    else if (plan.kind == 0) hipLaunchKernelGGL((few_rows_kernel<DIM, F8, kFewWaves, false>), grid, block, 0, s, p); \
    else if (plan.kind == 1) hipLaunchKernelGGL((many_rows_kernel<DIM, F8, 4>), grid, block, 0, s, p);             \
    else hipLaunchKernelGGL((many_rows_kernel<DIM, F8, 8>), grid, block, 0, s, p);                                 \
    if (plan.budget && wide) hipLaunchKernelGGL((join_kernel<DIM, true>), join, dim3(256), 0, s, p);               \
    else if (plan.budget) hipLaunchKernelGGL((join_kernel<DIM, false>), join, dim3(256), 0, s, p);                 \
  }
  FF_PAGED(64, false) FF_PAGED(64, true) FF_PAGED(128, false) FF_PAGED(128, true)
#undef FF_PAGED
  FF_LAUNCH_CHECK("ff_attention_paged");
  return FF_OK;
}
