// Main loops of the block-scaled FP8 products on tiles of many rows (ff_block.h
// states the format and the packed layout).
//
// A workgroup of 4 waves owns BM rows x 4 CW weight rows; wave w owns all BM rows x
// CW of the weight rows. Activations go global -> registers -> LDS,
// weight fragments straight from memory into the operand registers of the one wave
// that uses them (a fragment is two contiguous 1 KB reads). P: k steps of weights and
// of activations in flight in registers.
// The weight fragment is the first operand, so lane 16 g + r of accumulator (i, j)
// holds row 16 i + r, weight rows 16 j + 4 g .. + 3.
#pragma once

#include "ff_block.h"

namespace ff {

constexpr int kTileThreads = 256;

// The weights a wave multiplies its tile's rows with. base, bytes: the packed weight; frag[j]:
// byte offset of fragment row j at k step 0 (uniform), `stride` bytes for the next k step;
// reads past the last fragment stay in the weight or give zeros (their sums are not stored).
// scale[s]: block scales of the fragments j with j % NS == s, one per k step; base[s],
// likewise, the packed weight itself.
template <int TJ, int NS>
struct TileWeights {
  const uint8_t* base[NS];
  uint32_t bytes, stride;
  const float* scale[NS];
  uint32_t frag[TJ];
};

// LDS of the three stages: codes, then the rows' scales and a place for values that are none.
template <int BM>
constexpr int tile_smem() {
  return 3 * (BM * (kBlock + 4) + 16);
}

// acc = rows . weights^T with e4m3 rows. abase, abytes: the rows' codes; aoff(r): byte offset of
// row r of the tile at k step 0 (rows past the end take a valid one); sbase, sbytes (below 2^31):
// the rows' scales; soff(r): index of row r's at k step 0, the next step's sstride bytes on.
// A step of 128 channels is one matrix instruction per 16 x 16 products on a zero
// accumulator and four fused multiply-adds into the running sums, which stay in ordinary
// registers: the adds of one instruction's result run while the next instruction does.
// k0, steps: the k steps [k0, k0 + steps) of the row's kt_n; every wave of the workgroup
// calls it with the same number. P, D: slots of weights and of activations in flight.
template <int BM, int CW, int NS, int P, int D, typename AOff, typename SOff>
__device__ __forceinline__ void tile_mainloop(f32x4 (&acc)[BM / 16][CW / 16], uint8_t* smem, int kt_n, int k0, int steps,
                                              const uint8_t* abase, uint32_t abytes, AOff&& aoff, const float* sbase,
                                              uint32_t sbytes, SOff&& soff, uint32_t sstride,
                                              const TileWeights<CW / 16, NS>& w) {
  constexpr int RA = BM / 16, TJ = CW / 16;
  constexpr int NA = BM * 8 / kTileThreads;  // 16-byte chunks of a stage per thread
  static_assert(NA * kTileThreads == BM * 8 && BM <= kTileThreads, "whole rounds of chunks");
  static_assert(P >= 2 && D < P && P % D == 0, "slots");
  constexpr int STAGE = BM * kBlock;
  constexpr int ALL = RA * TJ, LAG = ALL >= 4 ? 3 : 1, RING = LAG + 1;
  static_assert(ALL % RING == 0, "a step's results take the places of the last step's");
  const int tid = threadIdx.x % kTileThreads, lane = tid & 63, r16 = lane & 15, g = lane >> 4;
  uint8_t* sc_lds = smem + 3 * STAGE;

  __amdgpu_buffer_rsrc_t rW[NS];
#pragma unroll
  for (int s = 0; s < NS; ++s) rW[s] = make_rsrc(w.base[s], w.bytes);
  i32x8 wq[P][TJ];
  uint32_t wat = k0 * w.stride;  // offset of the next weights' k step
  auto loadW = [&](int slot, int j) {
    wq[slot][j] = join(bload16(rW[j % NS], 16 * lane, w.frag[j] + wat),
                       bload16(rW[j % NS], 1024 + 16 * lane, w.frag[j] + wat));
  };
  // Block scales: lane l has those of step l of CHUNK steps (zeros past the last); the next
  // chunk's are loaded a chunk ahead. As vector loads: scalar ones return in no order with LDS
  // reads, and waiting for them would drain those.
  constexpr int CHUNK = 64 / P * P;
  __amdgpu_buffer_rsrc_t rWS[NS];
#pragma unroll
  for (int s = 0; s < NS; ++s) rWS[s] = make_rsrc(w.scale[s], 4 * kt_n);
  uint32_t wsc[NS], wsn[NS];
  auto loadWS = [&](uint32_t (&to)[NS], int k) {
#pragma unroll
    for (int s = 0; s < NS; ++s) to[s] = bload4(rWS[s], 4 * lane, 4 * (k0 + k));
  };
  loadWS(wsc, 0);

  // LDS stage: 1 KB blocks of 8 rows, chunk c of row r at slot c ^ (r % 8) ^ (r / 8 % 2): the
  // 16 rows x 2 chunks of a fragment read fall on distinct banks per 8 and 16 lanes.
  const __amdgpu_buffer_rsrc_t rA = make_rsrc(abase, abytes);
  uint32_t asrc[NA];
  int adst[NA];
#pragma unroll
  for (int i = 0; i < NA; ++i) {
    const int c = tid + kTileThreads * i, row = c >> 3, ch = c & 7;
    asrc[i] = aoff(row) + 16 * ch;
    adst[i] = (row >> 3) * 1024 + 128 * (row & 7) + 16 * (ch ^ (row & 7) ^ ((row >> 3) & 1));
  }
  const __amdgpu_buffer_rsrc_t rS = make_rsrc(sbase, sbytes);
  // A wave takes the scales of BM / 4 rows, its other lanes an offset out of range: no branch in
  // the loop, and no line is asked for twice.
  const int srow = tid / 64 * (BM / 4) + lane;
  const uint32_t ssrc = lane < BM / 4 ? 4 * soff(srow) : 0x80000000u;
  constexpr int SSTAGE = 4 * BM + 16;
  const int sdst = lane < BM / 4 ? 4 * srow : 4 * BM;
  i32x4v ast[D][NA];
  uint32_t sst[D];
  int ak = min(k0, kt_n - 1);  // k step of the next activations
  auto loadA = [&](int slot) {
#pragma unroll
    for (int i = 0; i < NA; ++i) ast[slot][i] = bload16(rA, asrc[i], (uint32_t)ak * kBlock);
    sst[slot] = bload4(rS, ssrc, (uint32_t)ak * sstride);
    ak = ak + 1 == kt_n ? 0 : ak + 1;
  };
  auto writeA = [&](int slot, int stage) {
#pragma unroll
    for (int i = 0; i < NA; ++i) *reinterpret_cast<i32x4v*>(smem + stage * STAGE + adst[i]) = ast[slot][i];
    *reinterpret_cast<uint32_t*>(sc_lds + stage * SSTAGE + sdst) = sst[slot];
  };
  const int frag = 128 * (r16 & 7) + 1024 * (r16 >> 3);
  const int sw = (r16 & 7) ^ (r16 >> 3);
  const int c0 = frag + 16 * ((2 * g) ^ sw), c1 = frag + 16 * ((2 * g + 1) ^ sw);
  i32x8 xq[RA];
  float xs[RA];
  auto readA = [&](int stage, int i) {
    const uint8_t* st = smem + stage * STAGE + 2048 * i;
    xq[i] = join(*reinterpret_cast<const i32x4v*>(st + c0), *reinterpret_cast<const i32x4v*>(st + c1));
    xs[i] = *reinterpret_cast<const float*>(sc_lds + stage * SSTAGE + 64 * i + 4 * r16);
  };
#pragma unroll
  for (int i = 0; i < RA; ++i)
#pragma unroll
    for (int j = 0; j < TJ; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  // The prologue's loads are issued in the loop's order (a step's activations, then its
  // weights): the compiler's wait counts in the loop hold for both ways into it.
  loadA(0);
  writeA(0, 0);
  loadA(0);
  writeA(0, 1);
  static_for<0, P - 1>([&](auto P_) {
    constexpr int p = decltype(P_)::value;
    if constexpr (p >= P - 1 - D) {
      loadA((p - (P - 1 - D)) % D);
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int j = 0; j < TJ; ++j) loadW(p, j);
    wat += w.stride;
    __builtin_amdgcn_sched_barrier(0);
  });
  __syncthreads();
#pragma unroll
  for (int i = 0; i < RA; ++i) readA(0, i);

  // Step kt reads stage kt + 1 (row block by row block, each once its products of this step
  // are issued, so the reads run under all of the step) and writes stage kt + 2, whose buffer
  // held step kt - 1: every wave had read that before the barrier of step kt - 1. The one
  // barrier, after the first row block, is behind the last step's writes of stage kt + 1.
  int rd = 1;  // stage kt + 1
  f32x4 t[RING];  // the last results, and the scales of those not yet added
  float sp[LAG];
#pragma unroll
  for (int n = 0; n < RING; ++n) t[n] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int n = 0; n < LAG; ++n) sp[n] = 0.f;
  auto step = [&](int u, int at) {  // at: the step's place in its chunk
    const int wr = rd == 2 ? 0 : rd + 1;
    float ws[NS];
#pragma unroll
    for (int v = 0; v < NS; ++v) ws[v] = __uint_as_float(__builtin_amdgcn_readlane(wsc[v], at));
    // Instruction n = i TJ + j is followed by the adds of instruction n - LAG, the first LAG
    // of a step by those of the last step's last. A result is there some 40 clocks after its
    // instruction's start. In a bare loop of these instructions and adds, without loads, LDS
    // or barriers, the matrix unit is busy 83 % of the time with LAG 3 (one wave a SIMD; 89 %
    // with two), 69 and 86 % with 2, 44 and 76 % with 1. In the whole loop it is 22 % with one
    // wave (576 x 6144 x 4096) and 52 % with two (4096 x 5120 x 25600): the rest waits.
    float s[RA][NS];
    static_for<0, ALL>([&](auto N_) {
      constexpr int n = decltype(N_)::value, i = n / TJ, j = n % TJ;
      t[n % RING] = mfma_step(wq[u][j], xq[i]);
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (n >= LAG) {
        constexpr int d = n - LAG;
        fma4(acc[d / TJ][d % TJ], t[d % RING], s[d / TJ][d % TJ % NS]);
      } else {
        constexpr int d = ALL - LAG + n;
        fma4(acc[d / TJ][d % TJ], t[d % RING], sp[n]);
      }
      if constexpr (j < NS) s[i][j] = xs[i] * ws[j];
      if constexpr (n == TJ - 1) {
        __syncthreads();
        writeA(u % D, wr);
        loadA(u % D);
      }
      if constexpr (n % RA == RA / 2) loadW((u + P - 1) % P, n / RA);
      if constexpr (j == TJ - 1) readA(rd, i);
      __builtin_amdgcn_sched_barrier(0);
    });
#pragma unroll
    for (int n = 0; n < LAG; ++n) sp[n] = s[(ALL - LAG + n) / TJ][(ALL - LAG + n) % TJ % NS];
    wat += w.stride;
    rd = wr;
  };
  // Whole rounds of P steps: a way out of the loop, or past some of its loads, inside a round
  // would cost every round the wait counts of the shorter way. The weights of steps past the
  // last lie past their end (w.bytes), where loads give zeros; the activations are the row's
  // own, so a NaN stays in its row.
  for (int c = 0; c < steps; c += CHUNK) {
    loadWS(wsn, c + CHUNK);
    const int n = min(CHUNK, steps - c);
    for (int at = 0; at < n; at += P)
      static_for<0, P>([&](auto U_) { step(decltype(U_)::value, at + decltype(U_)::value); });
#pragma unroll
    for (int s = 0; s < NS; ++s) wsc[s] = wsn[s];
  }
#pragma unroll
  for (int n = 0; n < LAG; ++n) fma4(acc[(ALL - LAG + n) / TJ][(ALL - LAG + n) % TJ], t[(ALL - LAG + n) % RING], sp[n]);
}

// The same with bf16 rows: the e4m3 weights become bf16 in registers (exact) and a step of
// 128 channels is four v_mfma_f32_16x16x32_bf16 per 16 x 16 products.
template <int BM>
constexpr int tile_smem_bf16() {
  return 2 * BM * kBlock * 2;
}

template <int BM, int CW, int P, typename AOff>
__device__ __forceinline__ void tile_mainloop_bf16(f32x4 (&acc)[BM / 16][CW / 16], uint8_t* smem, int kt_n,
                                                   const uint8_t* abase, uint32_t abytes, AOff&& aoff,
                                                   const TileWeights<CW / 16, 1>& w) {
  constexpr int RA = BM / 16, TJ = CW / 16;
  constexpr int NA = BM * 16 / kTileThreads;
  static_assert(NA * kTileThreads == BM * 16, "whole rounds of chunks");
  static_assert(P == 1 || P % 2 == 0, "the two LDS stages alternate");
  constexpr int STAGE = BM * kBlock * 2;
  const int tid = threadIdx.x, lane = tid & 63, r16 = lane & 15, g = lane >> 4;

  const __amdgpu_buffer_rsrc_t rW = make_rsrc(w.base[0], w.bytes);
  i32x8 wq[P][TJ];
  uint32_t wat = 0;
  auto loadW = [&](int slot, int j) {
    wq[slot][j] = join(bload16(rW, 16 * lane, w.frag[j] + wat), bload16(rW, 1024 + 16 * lane, w.frag[j] + wat));
  };

  // LDS stage: 256 bytes a row, chunk c of row r at slot c ^ key(r). The hardware serves 16
  // lanes at a time, of one lane group g or (rows 0-3 and 12-15, rows 4-11) of g and g + 1:
  // with row quarters 0, 1, 2, 3 keyed 0, 2, 3, 1 both sets of 16 chunks are distinct banks.
  const auto key = [](int r) {
    const int hi = r >> 2 & 3;
    return (r & 3) | ((hi ^ hi >> 1) & 1) << 3 | (hi >> 1) << 2;
  };
  const __amdgpu_buffer_rsrc_t rA = make_rsrc(abase, abytes);
  uint32_t asrc[NA];
  int adst[NA];
#pragma unroll
  for (int i = 0; i < NA; ++i) {
    const int c = tid + kTileThreads * i, row = c >> 4, ch = c & 15;
    asrc[i] = aoff(row) + 16 * ch;
    adst[i] = row * 256 + 16 * (ch ^ key(row));
  }
  i32x4v ast[P][NA];
  int ak = 0;
  auto loadA = [&](int slot) {
#pragma unroll
    for (int i = 0; i < NA; ++i) ast[slot][i] = bload16(rA, asrc[i], (uint32_t)ak * (2 * kBlock));
    ak = ak + 1 == kt_n ? 0 : ak + 1;
  };
  auto writeA = [&](int slot, int buf) {
#pragma unroll
    for (int i = 0; i < NA; ++i) *reinterpret_cast<i32x4v*>(smem + buf * STAGE + adst[i]) = ast[slot][i];
  };
  u32x4 xh[RA][4];
  const uint8_t* xsrc[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) xsrc[q] = smem + r16 * 256 + 16 * ((4 * g + q) ^ key(r16));
  auto readA = [&](int buf, int i, int q) {
    xh[i][q] = *reinterpret_cast<const u32x4*>(xsrc[q] + buf * STAGE + i * 4096);
  };
#pragma unroll
  for (int i = 0; i < RA; ++i)
#pragma unroll
    for (int j = 0; j < TJ; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  // The prologue's loads are issued in the loop's order (a step's activations, then its
  // weights): the compiler's wait counts in the loop hold for both ways into it.
  loadA(0);
  writeA(0, 0);
  static_for<0, P>([&](auto P_) {
    constexpr int p = decltype(P_)::value;
    loadA((1 + p) % P);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < TJ; ++j) loadW(p, j);
    wat += w.stride;
    __builtin_amdgcn_sched_barrier(0);
  });
  float ws = w.scale[0][0];
  __syncthreads();
#pragma unroll
  for (int q = 0; q < 4; ++q)
#pragma unroll
    for (int i = 0; i < RA; ++i) readA(0, i, q);

  auto step = [&](int kt, int u, int buf) {
    // the other stage last held the step before, read by every wave before the last barrier
    writeA((u + 1) % P, buf ^ 1);
    loadA((u + 1) % P);
    __builtin_amdgcn_sched_barrier(0);
    const float s = ws;
    ws = w.scale[0][min(kt + 1, kt_n - 1)];
    static_for<0, TJ>([&](auto J_) {
      constexpr int j = decltype(J_)::value;
      if constexpr (j == TJ - 1) __syncthreads();  // the next stage is written
      f32x4 t[RA];
#pragma unroll
      for (int i = 0; i < RA; ++i) t[i] = f32x4{0.f, 0.f, 0.f, 0.f};
      static_for<0, 4>([&](auto Q_) {
        constexpr int q = decltype(Q_)::value;
        const bf16x8 wb = e4m3_to_bf16x8((uint32_t)wq[u][j][2 * q], (uint32_t)wq[u][j][2 * q + 1]);
#pragma unroll
        for (int i = 0; i < RA; ++i) {
          t[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wb, __builtin_bit_cast(bf16x8, xh[i][q]), t[i], 0, 0, 0);
          if constexpr (j == TJ - 1) readA(buf ^ 1, i, q);
        }
      });
      loadW(u, j);
      __builtin_amdgcn_sched_barrier(0);  // the loads keep this order
#pragma unroll
      for (int i = 0; i < RA; ++i) fma4(acc[i][j], t[i], s);
    });
    wat += w.stride;
  };
  if constexpr (P == 1) {
    for (int kt = 0; kt < kt_n; ++kt) step(kt, 0, kt & 1);
  } else {
    for (int kt = 0; kt < kt_n; kt += P)
      static_for<0, P>([&](auto U_) {
        constexpr int u = decltype(U_)::value;
        step(kt + u, u, u & 1);
      });
  }
}

}  // namespace ff
