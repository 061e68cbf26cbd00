// Tiled matrix products of the feed-forward operators on gfx950's matrix instructions: one kernel
// template over the element type, the layout of each operand and the epilogue.
//
//   D[m][n] = sum_k A(m, k) B(n, k)
//
// Byte geometry. Everything is counted in 16-byte chunks, so one address plan serves 8-bit
// integers, bf16 and fp32: a K-step is 128 bytes of a row, a fragment is one chunk a lane
// (16 bytes = 16 int8 / 8 bf16 / 4 fp32 values of k), a 64-byte half K-step is one
// mfma_i32_16x16x64_i8, one mfma_f32_16x16x32_bf16 or four mfma_f32_16x16x4_f32.
//
// Operand layouts.
//   ROW: k runs along memory. LDS tile [rows][128 B]; chunk c of row r sits at chunk slot
//        c ^ (r & 7), so the 8 rows that a b128 read takes at a time touch all 32 banks once.
//   COL: k is the row index (weights of an input gradient, both operands of a weight gradient).
//        LDS tile [KS rows][tile columns], read as transposed fragments
//        (ds_read_b64_tr_b16; fp32: four b32 reads), slots swizzled by swz_col() below.
// Global -> LDS by LDS-DMA (16 bytes a lane, no registers); the swizzle is in the source address
// a lane picks, the LDS side is written in order.
//
// The matrix instruction's A operand is the N side and its B operand the M side: a lane then holds
// 4 consecutive n of one row m.
//
// Ends: rows / columns past the last are clamped to the last (their results are not stored); k
// past the end reads a page of zeros on BOTH sides (a NaN times zero would not vanish).
#pragma once
#include <algorithm>

#include "hgk_conv.h"
#include "hgk_philox.h"

namespace hgk {

enum GemmType { G_F32 = 0, G_BF16 = 1, G_I8 = 2 };
enum GemmLayout { L_ROW = 0, L_COL = 1 };
enum GemmEpi {
  E_SLAB = 0,   // fp32 partial sums of one k range to slab[split][batch][M][N]
  E_OUT = 1,    // rounded to T: plain, bias, scales, dropout, residual
  E_GATED = 2,  // a(g) u, the N tile holding gate columns and up columns
  E_GATED_BWD = 3  // dg, du from dh and the recomputed g, u
};
enum { kActSilu = HGK_ACT_SILU, kActGelu = HGK_ACT_GELU, kActRelu = HGK_ACT_RELU, kActSigmoid = HGK_ACT_SIGMOID };

template <int DT>
struct GT;
template <>
struct GT<G_F32> {
  typedef float elem;
  typedef f32x4 acc;
  static constexpr int es = 4;
};
template <>
struct GT<G_BF16> {
  typedef bf16_t elem;
  typedef f32x4 acc;
  static constexpr int es = 2;
};
typedef int i32x4 __attribute__((ext_vector_type(4)));
template <>
struct GT<G_I8> {
  typedef int8_t elem;
  typedef i32x4 acc;
  static constexpr int es = 1;
};

// one fragment pair: 64 bytes of k
template <int DT>
__device__ __forceinline__ typename GT<DT>::acc mma(i32x4 a, i32x4 b, typename GT<DT>::acc c) {
  if constexpr (DT == G_I8) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
  } else if constexpr (DT == G_BF16) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      c = __builtin_amdgcn_mfma_f32_16x16x4f32(__int_as_float(a[i]), __int_as_float(b[i]), c, 0, 0, 0);
    return c;
  }
}

struct GemmArgs {
  // operand bases; p1 is the second one of a two-part launch: E_GATED*: the up weights (N side);
  // two k segments: both sides' second segment; two batches: the M side's second batch
  const char *m0, *m1, *n0, *n1;
  long ldm, ldn;      // row pitch in bytes
  int M, N;           // output rows / columns (of one part)
  int km, kn;         // k extent per segment: ROW side in chunk-padded elements, COL side in rows
  int spseg, nseg;    // K-steps per segment, segments
  int tiles_m, tiles_n, batch, splits;
  // epilogue
  void* out;          // rows of N, like res and dh
  void* out1;         // second batch's / du
  float* slab;
  const void* res;    // residual
  const void* dh;     // E_GATED_BWD: incoming gradient
  int npad;           // E_GATED_BWD: columns [N, npad) of dg / du are written as zero
  const float *row_scale, *col_scale, *col_scale1, *bias;
  float alpha;        // E_OUT: factor of the sum
  int act, vec;       // vec: N % 8 == 0, rows are read and written in groups of 8
  int drop;           // apply `d`
  DropArgs d;
};

static __device__ __attribute__((aligned(64))) char g_zero_page[64];

// ---- activations: value and slope. `FAST`: bf16 results (hardware exponential and reciprocal,
// 1 ulp of fp32, against a half step of 2^-9); fp32 results take the full-precision functions ----
template <bool FAST>
__device__ __forceinline__ float sigmoid_f(float g) {
  if (FAST) return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(g * -1.44269504f));
  return 1.f / (1.f + expf(-g));
}
template <bool FAST>
__device__ __forceinline__ float act_f(int act, float g) {
  if (act == kActSilu) return g * sigmoid_f<FAST>(g);
  if (act == kActGelu) return 0.5f * g * erfcf(g * -0.70710678f);
  if (act == kActRelu) return g > 0.f || g != g ? g : 0.f;
  return sigmoid_f<FAST>(g);
}
// a(g) and a'(g)
template <bool FAST>
__device__ __forceinline__ void act_slope(int act, float g, float& a, float& s) {
  if (act == kActSilu) {
    const float q = sigmoid_f<FAST>(g);
    a = g * q;
    s = q + a * (1.f - q);
  } else if (act == kActGelu) {
    const float h = 0.5f * erfcf(g * -0.70710678f);
    const float e = FAST ? __builtin_amdgcn_exp2f(g * g * -0.72134752f) : expf(-0.5f * g * g);
    a = g * h;
    s = h + g * 0.39894228f * e;
  } else if (act == kActRelu) {
    a = g > 0.f || g != g ? g : 0.f;
    s = g > 0.f ? 1.f : 0.f;
  } else {
    const float q = sigmoid_f<FAST>(g);
    a = q;
    s = q * (1.f - q);
  }
}

// 8 consecutive elements of a row as they lie in memory (16 bytes of bf16, 32 of fp32)
template <typename T>
struct Raw8 {
  uint4 v[sizeof(T) / 2];
};
template <typename T>
__device__ __forceinline__ Raw8<T> load_raw8(const T* p) {
  Raw8<T> r;
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) r.v[i] = reinterpret_cast<const uint4*>(p)[i];
  return r;
}
template <typename T>
__device__ __forceinline__ void unpack_raw8(const Raw8<T>& r, float* f) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 2; ++i) unpack16<float>(__builtin_bit_cast(float4, r.v[i]), f + 4 * i);
  } else {
    unpack16<bf16_t>(r.v[0], f);
  }
}
// elements n .. n + 7 of a row of N; vec: N % 8 == 0 (a group lies inside or outside as a whole)
template <typename T>
__device__ __forceinline__ void load8(const T* p, int n, int N, bool vec, float* f) {
  if (vec) {
    unpack_raw8<T>(load_raw8<T>(p + n), f);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = n + e < N ? to_f(p[n + e]) : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, int n, int N, bool vec, const float* f) {
  if (vec) {
    if constexpr (sizeof(T) == 4) {
      store16<float>(p + n, pack16<float>(f));
      store16<float>(p + n + 4, pack16<float>(f + 4));
    } else {
      store16<bf16_t>(p + n, pack16<bf16_t>(f));
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (n + e < N) p[n + e] = from_f<T>(f[e]);
  }
}
// dropout of the 8 outputs of one group of row m
__device__ __forceinline__ void drop8(const GemmArgs& a, int m, int n, float* f, uint64_t off) {
  const uint64_t gid = (uint64_t)m * ((a.N + 7) >> 3) + (n >> 3);
  const uint32_t k = drop_mask8(gid, off, a.d.seed, a.d.thr);
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = (k >> e) & 1u ? f[e] * a.d.scale : 0.f;
}

// COL tiles: the rows that one half-wave reads together (8 lg + 0 .. 3 of two lane groups) land on
// distinct 32-byte positions; fp32 reads 4 lg + i of two lane groups, 64 bytes apart
template <int DT>
__device__ __forceinline__ int swz_col(int p) {
  if constexpr (DT == G_BF16) return ((p & 3) | (((p >> 3) & 1) << 2)) << 1;
  return ((p >> 2) & 1) << 2;
}

// T: type of outputs, residual and dh
template <int DT, typename T, int LM, int LN, int BM, int BN, int WM, int WN, int EPI, int MINW>
__global__ __launch_bounds__(WM * WN * 64) __attribute__((amdgpu_waves_per_eu(MINW)))
void gemm_kernel(GemmArgs a) {
  constexpr int NW = WM * WN, es = GT<DT>::es;
  constexpr int KS = 128 / es;               // k per step
  constexpr bool DUAL = EPI == E_GATED || EPI == E_GATED_BWD;
  constexpr int PM = BM * 128, PN = BN * 128, SB = PM + PN;  // LDS bytes of a stage
  constexpr int DM = BM / 8 / NW, DN = BN / 8 / NW;          // 1-KB DMAs of a wave per stage
  static_assert(BM % (8 * NW) == 0 && BN % (8 * NW) == 0, "whole DMAs per wave");
  static_assert(LM == L_ROW || BM * es >= 256, "COL swizzle needs 16 chunks a row");
  static_assert(LN == L_ROW || BN * es >= 256, "COL swizzle needs 16 chunks a row");
  static_assert(DT != G_I8 || (LM == L_ROW && LN == L_ROW), "8-bit operands are ROW");
  constexpr int WTM = BM / WM, WTN = BN / WN, FM = WTM / 16, FN = WTN / 16;
  static_assert(!DUAL || FN % 2 == 0, "gate and up halves");
  __shared__ __attribute__((aligned(16))) char lds[2 * SB];

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int lr = lane & 15, lg = lane >> 4;
  const int wm = wave / WN, wn = wave % WN;

  // ---- workgroup -> tile. One XCD takes a contiguous run of tiles (its L2 then holds their
  // panels), walked in bands of 8 tile rows ----
  const long tiles = (long)a.tiles_m * a.tiles_n;
  long l = xcd_slot(blockIdx.x, gridDim.x);
  const int split = (int)(l / (tiles * a.batch));
  l -= split * (tiles * a.batch);
  const int bat = (int)(l / tiles);
  l -= bat * tiles;
  const long band = l / (8l * a.tiles_n);
  const int bh = min(8, a.tiles_m - (int)band * 8);
  const int within = (int)(l - band * 8 * a.tiles_n);
  const int m0 = ((int)band * 8 + within % bh) * BM;
  const int n0 = (within / bh) * (DUAL ? BN / 2 : BN);
  // K-steps of this split
  const int steps = a.spseg * a.nseg;
  const int s0 = (int)((long)split * steps / a.splits), s1 = (int)((long)(split + 1) * steps / a.splits);

  // ---- DMA sources ----
  const char* pm[DM];
  const char* pn[DN];
  const int seg0 = s0 / a.spseg, kin0 = s0 - seg0 * a.spseg;
  const char* bm = (a.batch > 1 ? bat : seg0) ? a.m1 : a.m0;
  const char* bn = (!DUAL && a.nseg > 1 && seg0) ? a.n1 : a.n0;
  const int rchunk = (lane & 7) ^ ((lane >> 3) & 7);  // ROW: chunk of every DMA of this lane
  constexpr int CM = BM * es / 16, CN = BN * es / 16;  // COL: chunks per LDS row
  auto colrow = [&](int d, int C) { return ((d * NW + wave) * 64 + lane) / C; };
#pragma unroll
  for (int d = 0; d < DM; ++d) {
    if (LM == L_ROW) {
      const int r = min(m0 + (d * NW + wave) * 8 + (lane >> 3), a.M - 1);
      pm[d] = bm + r * a.ldm + (long)kin0 * 128 + rchunk * 16;
    } else {
      const int p = colrow(d, CM);
      const int c = (((d * NW + wave) * 64 + lane) % CM) ^ swz_col<DT>(p);
      const int col = min(m0 * es + c * 16, (a.M * es - 1) & ~15);
      pm[d] = bm + ((long)kin0 * KS + p) * a.ldm + col;
    }
  }
#pragma unroll
  for (int d = 0; d < DN; ++d) {
    if (LN == L_ROW) {
      int r = (d * NW + wave) * 8 + (lane >> 3);
      const char* b = bn;
      if (DUAL) {
        if (r >= BN / 2) {
          b = a.n1;
          r -= BN / 2;
        }
      }
      r = min(n0 + r, a.N - 1);
      pn[d] = b + r * a.ldn + (long)kin0 * 128 + rchunk * 16;
    } else {
      const int p = colrow(d, CN);
      const int c = (((d * NW + wave) * 64 + lane) % CN) ^ swz_col<DT>(p);
      const int col = min(n0 * es + c * 16, (a.N * es - 1) & ~15);
      pn[d] = bn + ((long)kin0 * KS + p) * a.ldn + col;
    }
  }
  const bool tail_m = a.km % KS != 0, tail_n = a.kn % KS != 0;
  int kin = kin0;
  auto issue = [&](int slot) __attribute__((always_inline)) {
    char* sb = lds + slot * SB;
    const bool last = kin + 1 == a.spseg;
    if (last && (tail_m || tail_n)) {
      // the zero page stands in for k past the end
#pragma unroll
      for (int d = 0; d < DM; ++d) {
        const bool ok = LM == L_ROW ? kin * 128 + rchunk * 16 < a.km * es
                                    : kin * KS + colrow(d, CM) < a.km;
        dma16(ok ? pm[d] : g_zero_page, sb + (d * NW + wave) * 1024);
      }
#pragma unroll
      for (int d = 0; d < DN; ++d) {
        const bool ok = LN == L_ROW ? kin * 128 + rchunk * 16 < a.kn * es
                                    : kin * KS + colrow(d, CN) < a.kn;
        dma16(ok ? pn[d] : g_zero_page, sb + PM + (d * NW + wave) * 1024);
      }
    } else {
#pragma unroll
      for (int d = 0; d < DM; ++d) dma16(pm[d], sb + (d * NW + wave) * 1024);
#pragma unroll
      for (int d = 0; d < DN; ++d) dma16(pn[d], sb + PM + (d * NW + wave) * 1024);
    }
    ++kin;
    long im = LM == L_ROW ? 128 : (long)KS * a.ldm, in = LN == L_ROW ? 128 : (long)KS * a.ldn;
    if (a.nseg > 1 && last) {  // on to the second segment
      im += (a.m1 - a.m0) - (LM == L_ROW ? (long)a.spseg * 128 : (long)a.spseg * KS * a.ldm);
      in += (a.n1 - a.n0) - (LN == L_ROW ? (long)a.spseg * 128 : (long)a.spseg * KS * a.ldn);
      kin = 0;
    }
#pragma unroll
    for (int d = 0; d < DM; ++d) pm[d] += im;
#pragma unroll
    for (int d = 0; d < DN; ++d) pn[d] += in;
  };

  // ---- fragment offsets within a stage ----
  // ROW: row + lr, chunk lg + 4 s at slot ^ (row & 7) (tile rows are multiples of 8 apart)
  const int x0 = (lg ^ (lr & 7)) << 4, x1 = ((lg + 4) ^ (lr & 7)) << 4;
  auto rown = [&](int f) {
    return DUAL ? (f < FN / 2 ? wn * (WTN / 2) + f * 16 : BN / 2 + wn * (WTN / 2) + (f - FN / 2) * 16)
                : wn * WTN + f * 16;
  };
  auto frag_row = [&](const char* t, int row, int s) __attribute__((always_inline)) {
    return *reinterpret_cast<const i32x4*>(t + (row + lr) * 128 + (s ? x1 : x0));
  };
  typedef short s16x8 __attribute__((ext_vector_type(8)));
  auto frag_col = [&](const char* t, int pitch, int col, int s) __attribute__((always_inline)) -> i32x4 {
    if constexpr (DT == G_BF16) {
      const int p = 32 * s + 8 * lg + (lr >> 2), c = col + 4 * (lr & 3);
      const char* q = t + p * pitch + (((c >> 3) ^ swz_col<DT>(p)) << 4) + (c & 7) * 2;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(q));
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (__attribute__((address_space(3))) s16x4*)(q + 4 * pitch));
      const s16x8 v = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
      return __builtin_bit_cast(i32x4, v);
    } else {
      i32x4 v;
      const int c = col + lr;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int p = 16 * s + 4 * lg + i;
        v[i] = *reinterpret_cast<const int*>(t + p * pitch + (((c >> 2) ^ swz_col<DT>(p)) << 4) + (c & 3) * 4);
      }
      return v;
    }
  };

  typename GT<DT>::acc acc[FN][FM];
#pragma unroll
  for (int i = 0; i < FN; ++i)
#pragma unroll
    for (int j = 0; j < FM; ++j) acc[i][j] = typename GT<DT>::acc{0, 0, 0, 0};

  if (s0 < s1) issue(0);
#pragma unroll 1
  for (int s = s0; s < s1; ++s) {
    // this wave's DMAs of step s have landed, and after the barrier every wave's; the other slot's
    // last reads were consumed by the matrix instructions before it
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    const int slot = (s - s0) & 1;
    if (s + 1 < s1) issue(slot ^ 1);
    const char* tm = lds + slot * SB;
    const char* tn = tm + PM;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      i32x4 fm[FM], fn[FN];
#pragma unroll
      for (int j = 0; j < FN; ++j)
        fn[j] = LN == L_ROW ? frag_row(tn, rown(j), h) : frag_col(tn, BN * es, rown(j), h);
#pragma unroll
      for (int i = 0; i < FM; ++i)
        fm[i] = LM == L_ROW ? frag_row(tm, wm * WTM + i * 16, h) : frag_col(tm, BM * es, wm * WTM + i * 16, h);
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[j][i] = mma<DT>(fn[j], fm[i], acc[j][i]);
    }
  }

  // ---- epilogue. The sums go through LDS 16 rows of a wave at a time, so that a lane gets 8
  // consecutive columns of one row (a dropout group, a 16-byte vector of bf16): rows are then
  // read and written in whole lines. Stored from the fragment layout (8 bytes a lane, 16 rows an
  // instruction) the 256-wide tile of a [32768][1024] result took 45 us a tile. ----
  constexpr bool FAST = sizeof(T) == 2;
  constexpr int CW = DUAL ? WTN / 2 : WTN;          // output columns of a wave
  constexpr int GP = CW / 8, RP = 64 / GP, NP = 16 / RP, PITCH = CW + 4;
  static_assert(GP >= 4 && NP >= 1, "wave tile");
  constexpr int PARTS = DUAL ? 2 : 1;
  static_assert(NW * PARTS * 16 * PITCH * 4 <= 2 * SB, "scratch fits the stages");
  __syncthreads();
  float* scr = reinterpret_cast<float*>(lds) + wave * (PARTS * 16 * PITCH);
  const int cg = lane % GP, r0 = lane / GP;
  const int n = n0 + wn * CW + cg * 8, mw = m0 + wm * WTM + r0;
  const bool in_n = n < (EPI == E_GATED_BWD ? a.npad : a.N);
  const bool vec = a.vec != 0;
  const uint64_t off = EPI == E_OUT && a.drop ? drop_offset(a.d) : 0;
  float cs0[8], cs1[8], bias[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int c = min(n + e, a.N - 1);
    if constexpr (DT == G_I8) {
      cs0[e] = a.col_scale[c];
      cs1[e] = DUAL ? a.col_scale1[c] : 0.f;
    }
    if constexpr (EPI == E_OUT) bias[e] = a.bias ? a.bias[c] : 0.f;
  }
  // what a row brings along, loaded one fragment row ahead
  const T* side = EPI == E_GATED_BWD ? (const T*)a.dh : EPI == E_OUT ? (const T*)a.res : nullptr;
  Raw8<T> sv[NP];
  float rs[NP];
  auto ahead = [&](int i) __attribute__((always_inline)) {
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      const int m = min(mw + i * 16 + p * RP, a.M - 1);
      if constexpr (DT == G_I8) rs[p] = a.row_scale[m];
      if constexpr (EPI == E_GATED_BWD || EPI == E_OUT) {
        if (side && vec && n < a.N) sv[p] = load_raw8<T>(side + (long)m * a.N + n);
      }
    }
  };
  ahead(0);
#pragma unroll
  for (int i = 0; i < FM; ++i) {
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      const int part = DUAL ? j / (FN / 2) : 0, jc = DUAL ? j % (FN / 2) : j;
      *reinterpret_cast<typename GT<DT>::acc*>(scr + (part * 16 + lr) * PITCH + jc * 16 + lg * 4) = acc[j][i];
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // this wave's own rows: no barrier
    float f[NP][8], u[NP][8], q[NP][8];
#pragma unroll
    for (int p = 0; p < NP; ++p) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const auto v = *reinterpret_cast<const typename GT<DT>::acc*>(scr + (r0 + p * RP) * PITCH + cg * 8 + 4 * h);
#pragma unroll
        for (int e = 0; e < 4; ++e) f[p][4 * h + e] = (float)v[e];
        if constexpr (DUAL) {
          const auto w = *reinterpret_cast<const typename GT<DT>::acc*>(scr + (16 + r0 + p * RP) * PITCH + cg * 8 + 4 * h);
#pragma unroll
          for (int e = 0; e < 4; ++e) u[p][4 * h + e] = (float)w[e];
        }
      }
      if constexpr (DT == G_I8) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          f[p][e] = f[p][e] * rs[p] * cs0[e];
          if constexpr (DUAL) u[p][e] = u[p][e] * rs[p] * cs1[e];
        }
      }
      if constexpr (EPI == E_GATED_BWD || EPI == E_OUT) {
        if (side) {
          if (vec) unpack_raw8<T>(sv[p], q[p]);
          else if (n < a.N) load8<T>(side + (long)min(mw + i * 16 + p * RP, a.M - 1) * a.N, n, a.N, false, q[p]);
        }
      }
    }
    if (i + 1 < FM) ahead(i + 1);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // read before the next rows overwrite
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      const int m = mw + i * 16 + p * RP;
      if (m >= a.M || !in_n) continue;
      if constexpr (EPI == E_GATED) {
#pragma unroll
        for (int e = 0; e < 8; ++e) f[p][e] = act_f<FAST>(a.act, f[p][e]) * u[p][e];
        store8<T>((T*)a.out + (long)m * a.N, n, a.N, vec, f[p]);
      } else if constexpr (EPI == E_GATED_BWD) {
        float dg[8], du[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float av, sl;
          act_slope<FAST>(a.act, f[p][e], av, sl);
          dg[e] = n + e < a.N ? q[p][e] * u[p][e] * sl : 0.f;
          du[e] = n + e < a.N ? q[p][e] * av : 0.f;
        }
        store8<T>((T*)a.out + (long)m * a.npad, n, a.npad, true, dg);
        store8<T>((T*)a.out1 + (long)m * a.npad, n, a.npad, true, du);
      } else if constexpr (EPI == E_SLAB) {
        store8<float>(a.slab + (((long)split * a.batch + bat) * a.M + m) * a.N, n, a.N, vec, f[p]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) f[p][e] = fmaf(f[p][e], a.alpha, bias[e]);
        if (a.drop) drop8(a, m, n, f[p], off);
        if (side) {
#pragma unroll
          for (int e = 0; e < 8; ++e) f[p][e] += q[p][e];
        }
        store8<T>((T*)(bat ? a.out1 : a.out) + (long)m * a.N, n, a.N, vec, f[p]);
      }
    }
  }
}

// ---- few rows (M <= 16 MT): the weights stream once from memory into fragments, no LDS tiles ----
// A workgroup owns 16 output columns (gated: 16 gate and 16 up), its 8 waves take every 8th K-step
// of 128 bytes, the partial sums meet in LDS in wave order. Bound by the weights' bytes: one
// column group of 16 rows x 128 bytes per load pair, M rows of x from the caches.
template <int DT, typename T, int MT, bool DUAL>
__global__ __launch_bounds__(512) void skinny_kernel(GemmArgs a) {
  constexpr int es = GT<DT>::es, P = DUAL ? 2 : 1, NW = 8;
  typedef typename GT<DT>::acc acc_t;
  __shared__ acc_t red[NW][P * MT][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lr = lane & 15, lg = lane >> 4;
  const int n0 = blockIdx.x * 16;
  const char* w[P];
  w[0] = a.n0 + (long)min(n0 + lr, a.N - 1) * a.ldn;
  if (DUAL) w[P - 1] = a.n1 + (long)min(n0 + lr, a.N - 1) * a.ldn;
  const char* x[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) x[i] = a.m0 + (long)min(i * 16 + lr, a.M - 1) * a.ldm;
  acc_t acc[P][MT];
#pragma unroll
  for (int p = 0; p < P; ++p)
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[p][i] = acc_t{0, 0, 0, 0};
  const int kb = a.km * es;
#pragma unroll 2
  for (int s = wave; s < a.spseg; s += NW) {
    i32x4 wv[2][P], xv[2][MT];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int k = s * 128 + h * 64 + lg * 16;
      const bool ok = k < kb;
#pragma unroll
      for (int p = 0; p < P; ++p) wv[h][p] = *reinterpret_cast<const i32x4*>(ok ? w[p] + k : g_zero_page);
#pragma unroll
      for (int i = 0; i < MT; ++i) xv[h][i] = *reinterpret_cast<const i32x4*>(ok ? x[i] + k : g_zero_page);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int p = 0; p < P; ++p)
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[p][i] = mma<DT>(wv[h][p], xv[h][i], acc[p][i]);
  }
#pragma unroll
  for (int p = 0; p < P; ++p)
#pragma unroll
    for (int i = 0; i < MT; ++i) red[wave][p * MT + i][lane] = acc[p][i];
  __syncthreads();
  if (wave >= MT) return;
  const int m = wave * 16 + lr, n = n0 + lg * 4;
  if (m >= a.M || n >= a.N) return;
  float f[P][4];
#pragma unroll
  for (int p = 0; p < P; ++p) {
    acc_t t = red[0][p * MT + wave][lane];
#pragma unroll
    for (int q = 1; q < NW; ++q) t += red[q][p * MT + wave][lane];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      f[p][e] = (float)t[e];
      if constexpr (DT == G_I8)
        f[p][e] = f[p][e] * a.row_scale[m] * (p ? a.col_scale1 : a.col_scale)[min(n + e, a.N - 1)];
    }
  }
  const uint32_t keep = !DUAL && a.drop ? drop_mask8((uint64_t)m * ((a.N + 7) >> 3) + (n >> 3), drop_offset(a.d),
                                                     a.d.seed, a.d.thr) >> (n & 4) : 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (n + e >= a.N) break;
    const long at = (long)m * a.N + n + e;
    float v = f[0][e];
    if constexpr (DUAL) {
      v = act_f<sizeof(T) == 2>(a.act, v) * f[P - 1][e];
    } else {
      if (a.bias) v += a.bias[n + e];
      if (a.drop) v = (keep >> e) & 1u ? v * a.d.scale : 0.f;
      if (a.res) v += to_f(((const T*)a.res)[at]);
    }
    ((T*)a.out)[at] = from_f<T>(v);
  }
}

// sum of the k ranges' partial sums in their order, then the epilogue of E_OUT
template <typename T>
__global__ __launch_bounds__(256) void gemm_join_kernel(GemmArgs a) {
  const int n8 = (a.N + 7) >> 3;
  const long t = (long)blockIdx.x * 256 + threadIdx.x;
  if (t >= (long)a.batch * a.M * n8) return;
  const int n = (int)(t % n8) * 8;
  const long bm = t / n8;  // batch * M + m
  const int bat = (int)(bm / a.M), m = (int)(bm - (long)bat * a.M);
  const long pitch = (long)a.batch * a.M * a.N;
  const float* s = a.slab + bm * a.N;
  const bool vec = a.vec != 0;
  float f[8] = {};
#pragma unroll 4
  for (int k = 0; k < a.splits; ++k) {
    float q[8];
    load8<float>(s + k * pitch, n, a.N, vec, q);
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] += q[e];
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = f[e] * a.alpha + (a.bias && n + e < a.N ? a.bias[n + e] : 0.f);
  if (a.drop) drop8(a, m, n, f, drop_offset(a.d));
  if (a.res) {
    float q[8];
    load8<T>((const T*)a.res + (long)m * a.N, n, a.N, vec, q);
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] += q[e];
  }
  store8<T>((T*)(bat ? a.out1 : a.out) + (long)m * a.N, n, a.N, vec, f);
}

// rows of K elements -> rows of Kp (16-byte multiple), the rest zero. E: unsigned type of es bytes
template <typename E>
__global__ __launch_bounds__(256) void pad_rows_kernel(const E* __restrict__ src, E* __restrict__ dst,
                                                       long rows, int K, int Kp) {
  constexpr int V = 16 / sizeof(E);
  const long t = (long)blockIdx.x * 256 + threadIdx.x;
  const int cp = Kp / V;
  const long r = t / cp;
  if (r >= rows) return;
  const int c0 = (int)(t - r * cp) * V;
  E v[V];
#pragma unroll
  for (int e = 0; e < V; ++e) v[e] = c0 + e < K ? src[r * K + c0 + e] : E(0);
  *reinterpret_cast<uint4*>(dst + r * Kp + c0) = *reinterpret_cast<const uint4*>(v);
}
static __global__ __launch_bounds__(256) void zero_kernel(uint32_t* p, long words) {
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < words; i += (long)gridDim.x * 256) p[i] = 0;
}

// ---- host side ----
// hgk_dropout.hip
int dropout_mask(hipStream_t st, int dtype, const void* dy, void* dz, long rows, int C, const DropArgs& d);

static inline long up_to(long n, long q) { return (n + q - 1) / q * q; }
// workgroups a launch is split up to along k: two 4-wave workgroups a CU
static constexpr int kFillGroups = 512;

template <typename E>
static inline void launch_pad(hipStream_t st, const void* src, void* dst, long rows, int K, int Kp) {
  const long n = rows * (Kp * (long)sizeof(E) / 16);
  hipLaunchKernelGGL((pad_rows_kernel<E>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st,
                     (const E*)src, (E*)dst, rows, K, Kp);
}

// ---- tile size and split of a product ----
struct GemmPlan {
  bool big;  // 256-row / column tiles
  int tiles_m, tiles_n, splits;
  long slab;  // bytes
};
// per: a gated tile holds 2 x tile / 2 columns. wide: the type has 256-wide tiles
static inline GemmPlan plan_gemm(bool wide, long M, long N, int per, int steps, int batch, bool can_split) {
  GemmPlan p;
  const long big = ((M + 255) / 256) * ((N + 256 / per - 1) / (256 / per)) * batch;
  const long asked = route(HGK_ROUTE_FFN_TILE);
  p.big = wide && (asked ? asked == 256 : big >= 256);
  const int b = p.big ? 256 : 128;
  p.tiles_m = (int)((M + b - 1) / b);
  p.tiles_n = (int)((N + b / per - 1) / (b / per));
  const long tiles = (long)p.tiles_m * p.tiles_n * batch;
  p.splits = 1;
  if (can_split && tiles * 2 <= (p.big ? 256 : kFillGroups))
    p.splits = (int)std::max(1l, std::min<long>((p.big ? 256 : kFillGroups) / tiles, steps / 4));
  p.slab = p.splits > 1 ? (long)p.splits * batch * M * N * 4 : 0;
  return p;
}

// what a launch needs before its kernel is chosen
static inline GemmArgs gemm_args() {
  GemmArgs a;
  memset((void*)&a, 0, sizeof(a));
  a.alpha = 1.f;
  a.nseg = a.batch = a.splits = 1;
  return a;
}

}  // namespace hgk
