// Tiled matrix products of the feed-forward operators on gfx950's matrix instructions: one kernel
// template over the element type, the layout of each operand and the epilogue.
//
//   D[m][n] = sum_k A(m, k) B(n, k)
//
// Byte geometry. Everything is counted in 16-byte chunks, so one address plan serves 8-bit
// integers, bf16 and fp32: a K-step is 128 bytes of a row (a whole cache line), a fragment is one
// chunk a lane (16 bytes = 16 int8 / 8 bf16 / 4 fp32 values of k), and a half step's fragment pair
// is one mfma_i32_16x16x64_i8, one mfma_f32_16x16x32_bf16 or four mfma_f32_16x16x4_f32.
//
// Operand layouts.
//   ROW: k runs along memory. LDS tile [rows][128 B]; chunk c of row r sits at slot c ^ s(r), s(r) = r & 7
//        on the M side and (r & 3) | (r >> 3 & 1) << 2 on the N side (below), so the 8 rows that a
//        b128 read takes at a time touch all banks once.
//   COL: k is the row index (weights of an input gradient, both operands of a weight gradient).
//        LDS tile [KS rows][tile columns], read as transposed fragments
//        (ds_read_b64_tr_b16; fp32: four b32 reads), slots swizzled by swz_col() below.
// Global -> LDS by LDS-DMA (16 bytes a lane, no registers); the swizzle is in the source address
// a lane picks, the LDS side is written in order.
//
// Pipeline. The tiles of the two sides of each K-step are units M0 N0 M1 N1 .. in a ring of five
// LDS slots. In the first half of step P the unit M(P + 2) is sent for, the second half's fragments
// are read and the first half's products run; then one barrier says that step P + 1 has landed and
// step P is in registers; in the second half N(P + 2) is sent for (into M(P)'s slot), the next
// step's first fragments are read and the second half's products run. Each unit is on its way
// for two to three half steps. Lines are asked for whole: with 64-byte K-steps, four slots of both
// sides and a barrier each, the address units took twice as many requests and an
// 8192 x 4096 x 8192 product ran at 1227 TFLOP/s (1651 with the DMAs left out).
//
// The matrix instruction's A operand is the N side and its B operand the M side: a lane then holds 4
// consecutive rows of the N side for one row m. The N side's rows are dealt to the fragments so that
// a pair of them gives a lane 8 CONSECUTIVE columns of row m: row i of fragment 2 G + o is column
// 32 G + 8 (i / 4) + 4 o + i % 4. 8 columns are a dropout group and 16 bytes of bf16; four lanes fill
// 64 bytes of a row, and the epilogue works from registers. (Through LDS, in whole lines, the
// epilogue of a [32768][2048] result from K = 256 took 13 us of 60.)
//
// Ends: rows / columns past the last are clamped to the last (their results are not stored); k
// past the end reads a page of zeros on BOTH sides (a NaN times zero would not vanish).
#pragma once
#include <algorithm>
#include <type_traits>

#include "hgk_conv.h"
#include "hgk_philox.h"

namespace hgk {

enum GemmType { G_F32 = 0, G_BF16 = 1, G_I8 = 2 };
enum GemmLayout { L_ROW = 0, L_COL = 1 };
enum GemmEpi {
  E_SLAB = 0,   // fp32 partial sums of one k range to slab[split][batch][M][N up to a multiple of 8]
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

// dma16 (hgk_conv.h) from a wave-uniform base and a 32-bit offset a lane
__device__ __forceinline__ void dma16s(const char* base, uint32_t off, char* lds_wave_base) {
  const uint32_t l = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds_wave_base;
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
               ::"s"(__builtin_amdgcn_readfirstlane(l)), "v"(off), "s"(base)
               : "memory", "m0");
}

// ---- activations: value and slope. `FAST`: bf16 results (hardware exponential and reciprocal,
// 1 ulp of fp32, against a half step of 2^-8); fp32 results take the full-precision functions ----
template <bool FAST>
__device__ __forceinline__ float sigmoid_f(float g) {
  if (FAST) return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(g * -1.44269504f));
  return 1.f / (1.f + expf(-g));
}
// Phi(g), the normal distribution's integral, and e = exp(-g^2 / 2). FAST: with x = |g| / sqrt 2, erfc(x) exp(x^2)
// as t P(t), t = 1 / (1 + 0.4125 x), a third of erfcf's instructions. P is fitted (least squares, reweighted
// until its largest error is least, x up to 9.6) to be off by at most 2e-7 of 1 AND by at most 5.7e-5 of Phi itself,
// evaluated in fp32: where gelu is small it still has bf16's digits.
template <bool FAST>
__device__ __forceinline__ float phi_f(float g, float& e) {
  if (!FAST) {
    e = expf(-0.5f * g * g);
    return 0.5f * erfcf(g * -0.70710678f);
  }
  const float x = fabsf(g) * 0.70710678f;
  const float t = __builtin_amdgcn_rcpf(fmaf(0.4125f, x, 1.f));
  e = __builtin_amdgcn_exp2f(x * x * -1.44269504f);
  float p = fmaf(-0.17424254f, t, 0.5463044f);
  p = fmaf(p, t, -0.15833175f);
  p = fmaf(p, t, 0.3448905f);
  p = fmaf(p, t, 0.20665284f);
  p = fmaf(p, t, 0.2347265f);
  const float q = 0.5f * p * t * e;  // Phi(-|g|)
  return g < 0.f ? q : 1.f - q;
}
template <int ACT, bool FAST>
__device__ __forceinline__ float act_f(float g) {
  if (ACT == kActSilu) return g * sigmoid_f<FAST>(g);
  if (ACT == kActGelu) {
    float e;
    return g * phi_f<FAST>(g, e);
  }
  if (ACT == kActRelu) return g > 0.f || g != g ? g : 0.f;
  return sigmoid_f<FAST>(g);
}
// a(g) and a'(g)
template <int ACT, bool FAST>
__device__ __forceinline__ void act_slope(float g, float& a, float& s) {
  if (ACT == kActSilu) {
    const float q = sigmoid_f<FAST>(g);
    a = g * q;
    s = q + a * (1.f - q);
  } else if (ACT == kActGelu) {
    float e;
    const float h = phi_f<FAST>(g, e);
    a = g * h;
    s = h + g * 0.39894228f * e;
  } else if (ACT == kActRelu) {
    a = g > 0.f || g != g ? g : 0.f;
    s = g > 0.f ? 1.f : 0.f;
  } else {
    // from exp(-|g|): 1 - q would leave nothing of the slope where q is next to 1
    const float e = FAST ? __builtin_amdgcn_exp2f(fabsf(g) * -1.44269504f) : expf(-fabsf(g));
    const float q = FAST ? __builtin_amdgcn_rcpf(1.f + e) : 1.f / (1.f + e);
    a = g < 0.f ? e * q : q;
    s = e * q * q;
  }
}
// f(constant) for the activation that `act` names: one branch, not one an element
template <typename F>
__device__ __forceinline__ void with_act(int act, F&& f) {
  if (act == kActSilu) f(std::integral_constant<int, kActSilu>());
  else if (act == kActGelu) f(std::integral_constant<int, kActGelu>());
  else if (act == kActRelu) f(std::integral_constant<int, kActRelu>());
  else f(std::integral_constant<int, kActSigmoid>());
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
// a + b that no product before it is fused into: the kernels of the 8-bit products round alike, so a row's
// result does not depend on the rows beside it
__device__ __forceinline__ float plus(float a, float b) {
#pragma clang fp contract(off)
  return a + b;
}
// dropout of the 8 outputs of one group of row m
__device__ __forceinline__ void drop8(const GemmArgs& a, int m, int n, float* f, uint64_t off) {
  const uint64_t gid = (uint64_t)m * ((a.N + 7) >> 3) + (n >> 3);
  const uint32_t k = drop_mask8(gid, off, a.d.seed, a.d.thr);
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = (k >> e) & 1u ? f[e] * a.d.scale : 0.f;
}

// COL tiles of CH chunks a row. A half-wave's transposed read takes 8 bytes of each of 8 rows (8 lg +
// 0 .. 3 of two lane groups) and 4 places; its 32 pieces should cover a 256-byte window of the banks.
//   M side: the 4 places are 32 bytes of a row: the rows differ in chunk bits 1 .. 3.
//   N side: place q is column 8 q + 4 (o ^ q & 1), half a chunk, the halves alternating with q: two
//   places share a half and differ in chunk bit 1, the rows in bits 0, 2 and 3. (Odd lane groups
//   then hold their 8 columns' halves the other way round; the epilogue swaps them.)
// Rows of 8 chunks: two fill the window, one bit less. fp32 reads single values: rows 4 lg + i of two
// lane groups, 64 contiguous bytes of each (M) or four chunks two apart (N).
template <int DT, int CH, bool NSIDE>
__device__ __forceinline__ int swz_col(int p) {
  if constexpr (DT == G_BF16 && !NSIDE) {
    if constexpr (CH >= 16) return ((p & 3) | (((p >> 3) & 1) << 2)) << 1;
    return (((p >> 1) & 1) | (((p >> 3) & 1) << 1)) << 1;
  } else if constexpr (DT == G_BF16) {
    if constexpr (CH >= 16) return (p & 1) | (((p >> 1) & 1) << 2) | (((p >> 3) & 1) << 3);
    return ((p >> 1) & 1) | (((p >> 3) & 1) << 2);
  }
  return ((p >> 2) & 1) << (NSIDE ? 0 : 2);
}

// T: type of outputs, residual and dh
template <int DT, typename T, int LM, int LN, int BT, int WM, int WN, int EPI>
__global__ __launch_bounds__(WM * WN * 64) __attribute__((amdgpu_waves_per_eu(2)))
void gemm_kernel(GemmArgs a) {
  constexpr int NW = WM * WN, es = GT<DT>::es, BM = BT, BN = BT;
  constexpr int KS = 128 / es;               // k per step
  constexpr bool DUAL = EPI == E_GATED || EPI == E_GATED_BWD;
  constexpr int UB = BT * 128;               // LDS bytes of a unit
  constexpr int D = BT / 8 / NW;             // 1-KB DMAs of a wave per unit
  static_assert(BT % (8 * NW) == 0, "whole DMAs per wave");
  static_assert(DT != G_I8 || (LM == L_ROW && LN == L_ROW), "8-bit operands are ROW");
  constexpr int WTM = BM / WM, WTN = BN / WN, FM = WTM / 16, FN = WTN / 16;
  static_assert(FN % (DUAL ? 4 : 2) == 0 && NW % 2 == 0, "pairs of N fragments, of gate and of up columns");
  __shared__ __attribute__((aligned(16))) char lds[5 * UB];

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
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

  // ---- DMA sources: a base that moves with the steps and an offset a lane (host: 256 rows of an
  // operand are less than 4 GB) ----
  const int seg0 = s0 / a.spseg;
  const long stepm = LM == L_ROW ? 128 : (long)KS * a.ldm, stepn = LN == L_ROW ? 128 : (long)KS * a.ldn;
  int kinm = s0 - seg0 * a.spseg, kinn = kinm;
  const char* bm = ((a.batch > 1 ? bat : seg0) ? a.m1 : a.m0) + kinm * stepm;
  const char* bn = (!DUAL && a.nseg > 1 && seg0 ? a.n1 : a.n0) + kinn * stepn;
  if (LM == L_ROW) bm += (long)m0 * a.ldm;
  if (LN == L_ROW) bn += (long)n0 * a.ldn;
  const char* bu = bn;  // E_GATED*: the up weights
  if (DUAL) bu += a.n1 - a.n0;
  const long jumpm = (a.m1 - a.m0) - a.spseg * stepm, jumpn = (a.n1 - a.n0) - a.spseg * stepn;
  uint32_t om[D], on[D];
  // ROW: chunk of every DMA of this lane (a DMA's 8 rows start at a multiple of 8, N: at odd or even
  // multiples with the wave)
  const int rchm = (lane & 7) ^ ((lane >> 3) & 7), rchn = (lane & 7) ^ (((lane >> 3) & 3) | ((wave & 1) << 2));
  constexpr int CH = BT * es / 16;                    // COL: chunks per LDS row
  auto colrow = [&](int d) { return ((d * NW + wave) * 64 + lane) / CH; };
#pragma unroll
  for (int d = 0; d < D; ++d) {
    const int row = (d * NW + wave) * 8 + (lane >> 3), p = colrow(d);
    const int c = ((d * NW + wave) * 64 + lane) % CH;
    const int cm = c ^ swz_col<DT, CH, false>(p), cn = c ^ swz_col<DT, CH, true>(p);
    if (LM == L_ROW) om[d] = (uint32_t)min(row, a.M - 1 - m0) * (uint32_t)a.ldm + rchm * 16;
    else om[d] = (uint32_t)p * (uint32_t)a.ldm + min(m0 * es + cm * 16, (a.M * es - 1) & ~15);
    // gated: the first half of the tile's rows are gate rows, the second up rows
    if (LN == L_ROW) on[d] = (uint32_t)min(DUAL ? row % (BN / 2) : row, a.N - 1 - n0) * (uint32_t)a.ldn + rchn * 16;
    else on[d] = (uint32_t)p * (uint32_t)a.ldn + min(n0 * es + cn * 16, (a.N * es - 1) & ~15);
  }
  static_assert(!DUAL || BN / 2 % (8 * NW) == 0, "DMA d of every wave brings gate rows or up rows");
  const bool tail_m = a.km % KS != 0, tail_n = a.kn % KS != 0;
  // DMA d of the M (N) side's next unit into a slot. TAIL: a segment's last step, where the zero page
  // stands in for k past the end
  auto dma = [&](auto nside, auto tail, int d, int slot) __attribute__((always_inline)) {
    constexpr bool NS = decltype(nside)::value, TAIL = decltype(tail)::value;
    char* to = lds + slot * UB + (d * NW + wave) * 1024;
    const char* base = NS ? (DUAL && d * NW * 8 >= BN / 2 ? bu : bn) : bm;
    const uint32_t off = NS ? on[d] : om[d];
    if constexpr (TAIL) {
      const int k = NS ? a.kn : a.km, kin = NS ? kinn : kinm;
      const bool ok = (NS ? LN : LM) == L_ROW ? kin * 128 + (NS ? rchn : rchm) * 16 < k * es : kin * KS + colrow(d) < k;
      dma16(ok ? base + off : g_zero_page, to);
    } else {
      dma16s(base, off, to);
    }
  };
  auto is_tail = [&](auto nside) {
    constexpr bool NS = decltype(nside)::value;
    return (NS ? tail_n : tail_m) && (NS ? kinn : kinm) + 1 == a.spseg;
  };
  auto advance = [&](auto nside) __attribute__((always_inline)) {
    constexpr bool NS = decltype(nside)::value;
    int& kin = NS ? kinn : kinm;
    long by = NS ? stepn : stepm;
    if (!DUAL) {  // past a segment's end: on to the second one
      const bool over = kin + 1 == a.spseg && a.nseg > 1;
      by += over ? (NS ? jumpn : jumpm) : 0;
      kin = over ? 0 : kin + 1;
    } else {
      ++kin;
    }
    (NS ? bn : bm) += by;
    if (DUAL && NS) bu += by;
  };
  const std::false_type side_m;
  const std::true_type side_n;
  auto send = [&](auto nside, int slot) __attribute__((always_inline)) {
    if (is_tail(nside)) {
#pragma unroll
      for (int d = 0; d < D; ++d) dma(nside, std::true_type(), d, slot);
    } else {
#pragma unroll
      for (int d = 0; d < D; ++d) dma(nside, std::false_type(), d, slot);
    }
    advance(nside);
  };

  // ---- fragments of a step ----
  const int x0 = (lg ^ (lr & 7)) << 4, x1 = ((lg + 4) ^ (lr & 7)) << 4;  // ROW: s(row) is lr & 7 on both sides
  const int rm = (wm * WTM + lr) * 128, rn = (8 * (lr >> 2) + (lr & 3)) * 128;
  // first column of N fragment f's group of 32
  auto coln = [&](int f) {
    return DUAL ? (f < FN / 2 ? wn * (WTN / 2) + f / 2 * 32 : BN / 2 + wn * (WTN / 2) + (f - FN / 2) / 2 * 32)
                : wn * WTN + f / 2 * 32;
  };
  typedef short s16x8 __attribute__((ext_vector_type(8)));
  // 4 k values (fp32: one) of the fragment's 16 columns; N side: group `col`, half `o`
  auto frag_col = [&](auto nside, const char* t, int col, int o, int h) __attribute__((always_inline)) -> i32x4 {
    constexpr bool NS = decltype(nside)::value;
    constexpr int pitch = CH * 16;
    if constexpr (DT == G_BF16) {
      const int p = 32 * h + 8 * lg + (lr >> 2), q = lr & 3;
      const int c = col + (NS ? 8 * q + 4 * (o ^ (q & 1)) : 4 * q);
      const char* at = t + p * pitch + (((c >> 3) ^ swz_col<DT, CH, NS>(p)) << 4) + (c & 7) * 2;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(at));
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (__attribute__((address_space(3))) s16x4*)(at + 4 * pitch));
      const s16x8 v = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
      return __builtin_bit_cast(i32x4, v);
    } else {
      i32x4 v;
      const int c = col + (NS ? 8 * (lr >> 2) + 4 * o + (lr & 3) : lr);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int p = 16 * h + 4 * lg + i;
        v[i] = *reinterpret_cast<const int*>(t + p * pitch + (((c >> 2) ^ swz_col<DT, CH, NS>(p)) << 4) + (c & 3) * 4);
      }
      return v;
    }
  };
  struct Frags {
    i32x4 m[FM], n[FN];
  };
  // fragment r of half h of a step: the N side's first
  auto read1 = [&](int um, int un, int h, Frags& f, int r) __attribute__((always_inline)) {
    const char* tm = lds + um * UB;
    const char* tn = lds + un * UB;
    if (r < FN) {
      f.n[r % FN] = LN == L_ROW ? *reinterpret_cast<const i32x4*>(tn + (coln(r) + 4 * (r & 1)) * 128 + rn + (h ? x1 : x0))
                                : frag_col(side_n, tn, coln(r), r & 1, h);
    } else {
      const int i = r - FN;
      f.m[i % FM] = LM == L_ROW ? *reinterpret_cast<const i32x4*>(tm + i * 16 * 128 + rm + (h ? x1 : x0))
                                : frag_col(side_m, tm, wm * WTM + i * 16, 0, h);
    }
  };

  typename GT<DT>::acc acc[FN][FM];
#pragma unroll
  for (int i = 0; i < FN; ++i)
#pragma unroll
    for (int j = 0; j < FM; ++j) acc[i][j] = typename GT<DT>::acc{0, 0, 0, 0};

  const int np = s1 - s0;
  send(side_m, 0);
  send(side_n, 1);
  if (np > 1) {
    send(side_m, 2);
    send(side_n, 3);
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * D) : "memory");  // step 0 has landed
  } else {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  }
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  Frags fa, fb;
#pragma unroll
  for (int r = 0; r < FN + FM; ++r) read1(0, 1, 0, fa, r);
  auto wrap = [](int slot) { return slot >= 5 ? slot - 5 : slot; };
  // half a step in FM parts: each takes its share of the DMAs and of the next half's fragment reads
  // along with the products of one fragment row. All DMAs first hold every wave behind the barrier
  // until the address unit has taken them; a branch around each DMA takes longer than the other
  // wave's share of matrix instructions lasts.
  // PLAIN: the DMAs are neither missing nor a segment's last
  auto half = [&](auto is_plain, auto nside, bool more, int to, int um, int un, int h, const Frags& cur,
                  Frags& nxt) __attribute__((always_inline)) {
    constexpr bool PLAIN = decltype(is_plain)::value;
    const bool last = !PLAIN && is_tail(nside);
#pragma unroll
    for (int i = 0; i < FM; ++i) {
#pragma unroll
      for (int r = (FN + FM) * i / FM; r < (FN + FM) * (i + 1) / FM; ++r) read1(um, un, h, nxt, r);
#pragma unroll
      for (int j = 0; j < FN; ++j) acc[j][i] = mma<DT>(cur.n[j], cur.m[i], acc[j][i]);
      // the parts stay as they are written, and no product is carried past the next barrier
#pragma unroll
      for (int j = 0; j < FN; ++j) asm volatile("" : "+v"(acc[j][i]));
#pragma unroll
      for (int d = D * i / FM; d < D * (i + 1) / FM; ++d) {
        if (PLAIN) {
          dma(nside, std::false_type(), d, to);
        } else if (more) {
          if (last) dma(nside, std::true_type(), d, to);
          else dma(nside, std::false_type(), d, to);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    if (PLAIN || more) advance(nside);
  };
  int s = 0;  // slot of M(P)
  auto step = [&](auto is_plain, bool more) __attribute__((always_inline)) {
    half(is_plain, side_m, more, wrap(s + 4), s, wrap(s + 1), 1, fa, fb);
    // step P + 1 has landed (M(P + 2) may be on its way), step P is in registers: of every wave
    // after the barrier
    if (decltype(is_plain)::value || more) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(D) : "memory");
    else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    // past the last step the fragments are whatever the slots hold, and unused
    half(is_plain, side_n, more, s, wrap(s + 2), wrap(s + 3), 0, fb, fa);
    s = wrap(s + 2);
  };
  const bool tails = tail_m || tail_n;
#pragma unroll 1
  for (int P = 0; P < np; ++P) {
    // a run of steps without a branch, up to one that sends a segment's last step or nothing
    int lim = np - 2;
    if (tails) lim = min(lim, P + a.spseg - 1 - kinm);
#pragma unroll 1
    for (; P < lim; ++P) step(std::true_type(), true);
    step(std::false_type(), P + 2 < np);
  }

  // ---- epilogue: a lane holds groups of 8 columns of row m, a pair of fragments each ----
  constexpr bool FAST = sizeof(T) == 2;
  constexpr int NG = DUAL ? FN / 4 : FN / 2;  // groups of a row
  const bool vec = a.vec != 0;
  const uint64_t off = EPI == E_OUT && a.drop ? drop_offset(a.d) : 0;
  const int nw = n0 + wn * (DUAL ? WTN / 2 : WTN) + 8 * lg, mw = m0 + wm * WTM + lr;
  const T* side = EPI == E_GATED_BWD ? (const T*)a.dh : EPI == E_OUT ? (const T*)a.res : nullptr;
  const bool swapped = LN == L_COL && DT == G_BF16 && (lg & 1);
  auto group = [&](int g, int i, float* f) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const auto x = acc[2 * g][i][e], y = acc[2 * g + 1][i][e];
      f[e] = (float)(swapped ? y : x);
      f[4 + e] = (float)(swapped ? x : y);
    }
  };
  // two groups at a time, one line of bf16: its halves are stored one after the other
  constexpr int GS = NG > 1 ? 2 : 1;
#pragma unroll
  for (int g0 = 0; g0 < NG; g0 += GS) {
    float cs0[GS][8], cs1[GS][8], bias[GS][8];
#pragma unroll
    for (int k = 0; k < GS; ++k)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int c = min(nw + 32 * (g0 + k) + e, a.N - 1);
        if constexpr (DT == G_I8) {
          cs0[k][e] = a.col_scale[c];
          cs1[k][e] = DUAL ? a.col_scale1[c] : 0.f;
        }
        if constexpr (EPI == E_OUT) bias[k][e] = a.bias ? a.bias[c] : 0.f;
      }
    // what the rows bring along
    Raw8<T> sv[FM][GS];
    float rs[FM];
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      const int m = min(mw + i * 16, a.M - 1);
      if constexpr (DT == G_I8) rs[i] = a.row_scale[m];
      if constexpr (EPI == E_GATED_BWD || EPI == E_OUT) {
#pragma unroll
        for (int k = 0; k < GS; ++k) {
          const int n = nw + 32 * (g0 + k);
          if (side && vec && n < a.N) sv[i][k] = load_raw8<T>(side + (long)m * a.N + n);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      const int m = mw + i * 16;
      if (m >= a.M) continue;
      float dg[GS][8], du[GS][8];  // E_GATED_BWD
#pragma unroll
      for (int k = 0; k < GS; ++k) {
        const int n = nw + 32 * (g0 + k);
        if (n >= (EPI == E_GATED_BWD ? a.npad : a.N)) continue;
        float f[8], u[8], q[8];
        group(g0 + k, i, f);
        if constexpr (DUAL) group(NG + g0 + k, i, u);
        if constexpr (DT == G_I8) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            f[e] = f[e] * rs[i] * cs0[k][e];
            if constexpr (DUAL) u[e] = u[e] * rs[i] * cs1[k][e];
          }
        }
        if constexpr (EPI == E_GATED_BWD || EPI == E_OUT) {
          if (side) {
            if (vec) unpack_raw8<T>(sv[i][k], q);
            else load8<T>(side + (long)m * a.N, n, a.N, false, q);
          }
        }
        if constexpr (EPI == E_GATED) {
          with_act(a.act, [&](auto A) __attribute__((always_inline)) {
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = act_f<decltype(A)::value, FAST>(f[e]) * u[e];
          });
          store8<T>((T*)a.out + (long)m * a.N, n, a.N, vec, f);
        } else if constexpr (EPI == E_GATED_BWD) {
          with_act(a.act, [&](auto A) __attribute__((always_inline)) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              float av, sl;
              act_slope<decltype(A)::value, FAST>(f[e], av, sl);
              dg[k][e] = q[e] * u[e] * sl;
              du[k][e] = q[e] * av;
            }
          });
          if (!vec) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (n + e >= a.N) dg[k][e] = du[k][e] = 0.f;
          }
        } else if constexpr (EPI == E_SLAB) {
          store8<float>(a.slab + (((long)split * a.batch + bat) * a.M + m) * ((a.N + 7) & ~7), n, a.N, true, f);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) f[e] = fmaf(f[e], a.alpha, bias[k][e]);
          if (a.drop) drop8(a, m, n, f, off);
          if (side) {
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] += q[e];
          }
          store8<T>((T*)(bat ? a.out1 : a.out) + (long)m * a.N, n, a.N, vec, f);
        }
      }
      if constexpr (EPI == E_GATED_BWD) {
#pragma unroll
        for (int k = 0; k < 2 * GS; ++k) {
          const int n = nw + 32 * (g0 + k % GS);
          if (n < a.npad)
            store8<T>((T*)(k < GS ? a.out : a.out1) + (long)m * a.npad, n, a.npad, true, k < GS ? dg[k % GS] : du[k % GS]);
        }
      }
    }
  }
}

// ---- quantising: s = max |v| / 127, q = rint(v / s) ----
struct QuantScale {
  float sc, inv;
  bool none, plain;
};
// m: the largest magnitude's bits (magnitudes compare like their bits, infinities and NaN above all
// numbers); returns the scale that is stored
__device__ __forceinline__ float quant_scale(uint32_t m, QuantScale& z) {
  const bool odd = m >= 0x7f800000u;  // an infinity or a NaN
  z.sc = __uint_as_float(m) / 127.f;
  z.none = odd || z.sc == 0.f;
  z.inv = 1.f / z.sc;
  z.plain = z.sc >= 1e-30f && z.sc <= 1e30f;
  return odd ? __int_as_float(0x7fc00000) : z.sc;
}
// The low byte of b[e] is rint(v[e] / sc), v / sc correctly rounded as the definition's quotient of two fp32
// values is: from the correctly rounded reciprocal, one fused step makes the product faithful (within a
// unit in the last place) and the next one exact (Markstein, 1990). Where sc or its reciprocal leaves
// the normal numbers: the division itself. Adding 1.5 2^23 rounds to a whole number.
template <int V>
__device__ __forceinline__ void quant_bytes(const float* v, const QuantScale& z, uint32_t* b) {
  if (z.plain) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      float t = v[e] * z.inv;
      t = fmaf(fmaf(-t, z.sc, v[e]), z.inv, t);
      t = fmaf(fmaf(-t, z.sc, v[e]), z.inv, t);
      b[e] = __float_as_uint(t + 12582912.f);
    }
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e)
      b[e] = z.none ? 0 : (uint32_t)(int)fminf(fmaxf(rintf(v[e] / z.sc), -127.f), 127.f);
  }
}
__device__ __forceinline__ uint32_t pack_bytes(const uint32_t* b) {
  return (b[0] & 0xffu) | (b[1] & 0xffu) << 8 | (b[2] & 0xffu) << 16 | b[3] << 24;
}
template <int V>
__device__ __forceinline__ uint32_t max_bits(const float* v, uint32_t m) {
#pragma unroll
  for (int e = 0; e < V; ++e) m = max(m, __float_as_uint(v[e]) & 0x7fffffffu);
  return m;
}
// Largest magnitude of the chunks first, first + step .. of a row of nc 16-byte chunks, over the wave
template <typename T>
__device__ __forceinline__ uint32_t row_max(const T* row, int first, int step, int nc) {
  constexpr int V = Vec16<T>::N;
  uint32_t m = 0;
  for (int c = first; c < nc; c += step) {
    float f[V];
    unpack16<T>(load16(row + (long)c * V), f);
    m = max_bits<V>(f, m);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, o, 64));
  return m;
}
// those chunks in bytes (from the cache)
template <typename T>
__device__ __forceinline__ void row_bytes(const T* row, int8_t* q, const QuantScale& z, int first, int step, int nc) {
  constexpr int V = Vec16<T>::N;
  for (int c = first; c < nc; c += step) {
    float f[V];
    uint32_t b[V];
    unpack16<T>(load16(row + (long)c * V), f);
    quant_bytes<V>(f, z, b);
#pragma unroll
    for (int e = 0; e < V; e += 4) *reinterpret_cast<uint32_t*>(q + (long)c * V + e) = pack_bytes(b + e);
  }
}

// ---- few rows (M <= 16 MT): the weights stream once from memory into fragments, no LDS tiles ----
// A workgroup owns 16 output columns (gated: 16 gate and 16 up), its 8 waves take every 8th K-step
// of 128 bytes, the partial sums meet in LDS in wave order. Bound by the weights' bytes: one
// column group of 16 rows x 128 bytes per load pair, M rows of x from the caches.
// QUANT (8-bit integers, M <= kQuantRows, M K <= kQuantBytes): x is T, and every workgroup quantises its few
// rows into LDS itself, in place of a launch and a trip through memory. All eight waves share them (one wave a
// row: 1 x 8192 -> 1024 in 11.9 us, so 7.7).
static constexpr int kQuantRows = 16, kQuantBytes = 32768;
template <int DT, typename T, int MT, bool DUAL, bool QUANT = false>
__global__ __launch_bounds__(512) void skinny_kernel(GemmArgs a) {
  constexpr int es = GT<DT>::es, P = DUAL ? 2 : 1, NW = 8;
  typedef typename GT<DT>::acc acc_t;
  __shared__ acc_t red[NW][P * MT][64];
  __shared__ __attribute__((aligned(16))) int8_t xq[QUANT ? kQuantBytes : 16];
  __shared__ float xs[QUANT ? kQuantRows : 1];
  __shared__ uint32_t xm[QUANT ? kQuantRows : 1][NW];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lr = lane & 15, lg = lane >> 4;
  const int n0 = blockIdx.x * 16;
  const char* w[P];
  w[0] = a.n0 + (long)min(n0 + lr, a.N - 1) * a.ldn;
  if (DUAL) w[P - 1] = a.n1 + (long)min(n0 + lr, a.N - 1) * a.ldn;
  const char* x[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) x[i] = a.m0 + (long)min(i * 16 + lr, a.M - 1) * a.ldm;
  if constexpr (QUANT) {
    // W waves a row, so that the eight share few rows evenly
    const int W = a.M == 1 ? 8 : a.M == 2 ? 4 : a.M <= 4 ? 2 : 1, part = wave & (W - 1);
    const int first = part * 64 + lane, nc = a.km / Vec16<T>::N;
    for (int r = wave / W; r < a.M; r += NW / W) {
      const uint32_t m = row_max<T>((const T*)a.m0 + (long)r * a.km, first, W * 64, nc);
      if (lane == 0) xm[r][part] = m;
    }
    __syncthreads();
    for (int r = wave / W; r < a.M; r += NW / W) {
      uint32_t m = xm[r][0];
      for (int i = 1; i < W; ++i) m = max(m, xm[r][i]);
      QuantScale z;
      const float sc = quant_scale(m, z);
      row_bytes<T>((const T*)a.m0 + (long)r * a.km, xq + r * a.km, z, first, W * 64, nc);
      if (part == 0 && lane == 0) xs[r] = sc;
    }
    __syncthreads();
  }
  acc_t acc[P][MT];
#pragma unroll
  for (int p = 0; p < P; ++p)
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[p][i] = acc_t{0, 0, 0, 0};
  const int kb = a.km * es, steps = (kb + 127) / 128;
#pragma unroll 2
  for (int s = wave; s < steps; s += NW) {
    i32x4 wv[2][P], xv[2][MT];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int k = s * 128 + h * 64 + lg * 16;
      const bool ok = k < kb;
#pragma unroll
      for (int p = 0; p < P; ++p) wv[h][p] = *reinterpret_cast<const i32x4*>(ok ? w[p] + k : g_zero_page);
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        if constexpr (QUANT) {
          xv[h][i] = ok ? *reinterpret_cast<const i32x4*>(xq + min(lr, a.M - 1) * a.km + k) : i32x4{0, 0, 0, 0};
        } else {
          xv[h][i] = *reinterpret_cast<const i32x4*>(ok ? x[i] + k : g_zero_page);
        }
      }
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
        f[p][e] = f[p][e] * (QUANT ? xs[QUANT ? m : 0] : a.row_scale[m]) * (p ? a.col_scale1 : a.col_scale)[min(n + e, a.N - 1)];
    }
  }
  if constexpr (DUAL) {
    with_act(a.act, [&](auto A) __attribute__((always_inline)) {
#pragma unroll
      for (int e = 0; e < 4; ++e) f[0][e] = act_f<decltype(A)::value, sizeof(T) == 2>(f[0][e]) * f[P - 1][e];
    });
  }
  const uint32_t keep = !DUAL && a.drop ? drop_mask8((uint64_t)m * ((a.N + 7) >> 3) + (n >> 3), drop_offset(a.d),
                                                     a.d.seed, a.d.thr) >> (n & 4) : 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (n + e >= a.N) break;
    const long at = (long)m * a.N + n + e;
    float v = f[0][e];
    if constexpr (!DUAL) {
      if (a.bias) v = plus(v, a.bias[n + e]);
      if (a.drop) v = (keep >> e) & 1u ? v * a.d.scale : 0.f;
      if (a.res) v = plus(v, to_f(((const T*)a.res)[at]));
    }
    ((T*)a.out)[at] = from_f<T>(v);
  }
}

// sum of the k ranges' partial sums in their order, then the epilogue of E_OUT
template <typename T>
__global__ __launch_bounds__(64) void gemm_join_kernel(GemmArgs a) {
  const int n8 = (a.N + 7) >> 3;
  const long t = (long)blockIdx.x * 64 + threadIdx.x;
  if (t >= (long)a.batch * a.M * n8) return;
  const int n = (int)(t % n8) * 8;
  const long bm = t / n8;  // batch * M + m
  const int bat = (int)(bm / a.M), m = (int)(bm - (long)bat * a.M);
  const long pitch = (long)a.batch * a.M * (n8 * 8);
  const float* s = a.slab + bm * (n8 * 8);
  const bool vec = a.vec != 0;
  float f[8] = {};
#pragma unroll 4
  for (int k = 0; k < a.splits; ++k) {
    float q[8];
    load8<float>(s + k * pitch, n, a.N, true, q);
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

// Up to three tensors at once: rows of K elements -> rows of Kp (whole 16-byte chunks), the rest zero; the
// one with `drop` set also through a dropout mask (unscaled). E: unsigned type of an element. Rows are
// read in words of `unit` bytes, the largest that both their pitch and their start allow.
struct PadJob {
  const char* src;
  char* dst;
  long rows, first;  // first: chunks of the jobs before
  int K, Kp, unit, drop;
};
struct PadArgs {
  PadJob j[3];
  int n;
  long chunks;
  DropArgs d;
};
template <typename E>
__global__ __launch_bounds__(256) void pad_rows_kernel(PadArgs a) {
  constexpr int V = 16 / sizeof(E);
  const long t = (long)blockIdx.x * 256 + threadIdx.x;
  if (t >= a.chunks) return;
  const int k = a.n > 2 && t >= a.j[2].first ? 2 : a.n > 1 && t >= a.j[1].first ? 1 : 0;
  const PadJob& j = a.j[k];
  const int cp = j.Kp / V;
  const long l = t - j.first;
  const long r = a.chunks >> 32 ? l / cp : (long)((uint32_t)l / (uint32_t)cp);
  const int c0 = (int)(l - r * cp) * V;
  const char* src = j.src + (r * j.K + c0) * (long)sizeof(E);
  const int left = (j.K - c0) * (int)sizeof(E);  // bytes of the row from here on
  uint4 v = make_uint4(0, 0, 0, 0);
  auto take = [&](auto word) __attribute__((always_inline)) {
    typedef decltype(word) W;
    W w[16 / sizeof(W)];
#pragma unroll
    for (int e = 0; e < (int)(16 / sizeof(W)); ++e)
      w[e] = (e + 1) * (int)sizeof(W) <= left ? reinterpret_cast<const W*>(src)[e] : W(0);
    memcpy(&v, w, 16);
  };
  if (j.unit >= 8) take(uint64_t());
  else if (j.unit == 4) take(uint32_t());
  else if (sizeof(E) == 2 || j.unit == 2) take(uint16_t());
  else take(uint8_t());
  if (j.drop) {
    E e[V];
    memcpy(e, &v, 16);
    const uint32_t m = drop_mask8((uint64_t)r * ((j.K + 7) >> 3) + (c0 >> 3), drop_offset(a.d), a.d.seed, a.d.thr) >> (c0 & 7);
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (!((m >> i) & 1u)) e[i] = 0;
    memcpy(&v, e, 16);
  }
  reinterpret_cast<uint4*>(j.dst)[l] = v;
}
static __global__ __launch_bounds__(256) void zero_kernel(uint32_t* p, long words) {
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < words; i += (long)gridDim.x * 256) p[i] = 0;
}

// ---- host side ----
// hgk_dropout.hip
int dropout_mask(hipStream_t st, int dtype, const void* dy, void* dz, long rows, int C, const DropArgs& d);

// hgk_gated_rows.hip: the gated product of many rows of few channels
bool gated_rows_ok(int dtype, long M, int C, int F, bool bwd);
int gated_rows_fwd(hipStream_t st, const void* x, const void* wg, const void* wu, void* h, long M, int C, int F, int act);
int gated_rows_bwd(hipStream_t st, const void* x, const void* wg, const void* wu, const void* dh, void* dg, void* du,
                   void* dx, long M, int C, int F, int act);

// hgk_linear_rows.hip: dz and dx of many rows of few output channels
bool linear_rows_ok(int dtype, long M, int K, int N, bool drop);
int linear_rows_bwd(hipStream_t st, const void* dy, const void* w, void* dz, void* dx, long M, int K, int N,
                    const DropArgs& d);

#define HGK_CHECK_WORKSPACE(what, workspace, bytes, need) \
  HGK_CHECK_ARG((bytes) >= (need) && ((workspace) || (need) == 0), what ": workspace of %zu bytes is too small", (size_t)(bytes))

static inline long up_to(long n, long q) { return (n + q - 1) / q * q; }

// collects the rows to pad, then one launch
struct Pads {
  PadArgs a;
  Pads() {
    a.n = 0;
    a.chunks = 0;
    a.d = DropArgs();
  }
  void add(const void* src, void* dst, long rows, int K, int Kp, int es, const DropArgs* drop = nullptr) {
    PadJob& j = a.j[a.n++];
    j.src = (const char*)src;
    j.dst = (char*)dst;
    j.rows = rows;
    j.K = K;
    j.Kp = Kp;
    j.first = a.chunks;
    const long bits = (long)K * es | (long)(uintptr_t)src;
    j.unit = bits % 8 == 0 ? 8 : bits % 4 == 0 ? 4 : bits % 2 == 0 ? 2 : 1;
    j.drop = drop != nullptr;
    if (drop) a.d = *drop;
    a.chunks += rows * ((long)Kp * es / 16);
  }
  template <typename E>
  int launch(hipStream_t st) {
    if (!a.n) return HGK_OK;
    HGK_CHECK_THREADS("padded rows", (a.chunks + 255) / 256, 256);
    hipLaunchKernelGGL((pad_rows_kernel<E>), dim3((unsigned)((a.chunks + 255) / 256)), dim3(256), 0, st, a);
    HGK_LAUNCH_CHECK();
    return HGK_OK;
  }
};

// ---- tile size and split of a product ----
struct GemmPlan {
  int tile;  // rows and columns
  int tiles_m, tiles_n, splits;
  long slab;  // bytes
};
// per: a gated tile holds 2 x (columns / 2) columns. dt: GemmType. steps: K-steps of 128 bytes.
//
// The tile and the split are those of the least estimated time. A K-step of a 256-wide tile takes
// 1.5 us of a CU in bf16 (1467 TFLOP/s over the chip at 8192 x 4096 x 8192); per unit of work a
// 128-wide tile takes 1.3 times that (1147), a 64-wide one 2 to 3 times (502 .. 704): its waves read
// twice to four times the fragments per product. fp32's matrix instructions are 16 times slower and
// hide all of that. A CU with one or two workgroups waits for memory instead: 0.16 us and 0.8 of its
// products a step. A round ends with its epilogue, 4 us of a 256-wide tile. Against the tile stand the
// rounds: tiles are dealt to 256 CUs whole. Splitting k costs the partial sums' way to memory and back
// (4.6 TB/s) and a second launch (4.7 us). The constants of waiting and splitting are fitted to weight
// gradients of 64 x 256 .. 2048 x 512 over 2000 .. 131072 rows. Measured over 28 of those, every tile and 1 to 128
// splits: what they choose is 3 % slower on average than the best of each (256 x 1024 over 32768 rows: 32 us in
// 16 splits of 128-wide tiles, 40 in 64-wide ones), 26 % at worst (the same over 131072 rows: 115 us for 92 of 64
// splits of 256-wide tiles).
static inline GemmPlan plan_gemm(int dt, long M, long N, int per, int steps, int batch, bool can_split) {
  GemmPlan best;
  double least = 1e30;
  const long asked = route(HGK_ROUTE_FFN_TILE);
  for (int b = dt == G_F32 ? 128 : 256; b >= 64; b /= 2) {
    if ((asked == 64 || asked == 128 || (asked == 256 && dt != G_F32)) && asked != b) continue;
    GemmPlan p;
    p.tile = b;
    p.tiles_m = (int)((M + b - 1) / b);
    p.tiles_n = (int)((N + b / per - 1) / (b / per));
    const long n = (long)p.tiles_m * p.tiles_n * batch;
    const double slow = dt == G_F32 ? (b == 128 ? 1.0 : 1.1) : b == 256 ? 1.0 : b == 128 ? 1.3 : 2.4;
    const double step = (dt == G_F32 ? 12.0 : dt == G_I8 ? 1.1 : 1.5) * b * b / 65536 * slow;
    const long slots = 256l * (b == 256 ? 1 : b == 128 ? 2 : 4);
    for (int split = 1; split <= 64; split *= 2) {
      if (split > 1 && (!can_split || n * split > slots || steps / split < 4)) break;
      const double rounds = (double)((n * split + 255) / 256), each = (double)((steps + split - 1) / split);
      double t = std::max(rounds * step, 0.16 + 0.8 * step) * each + rounds * 4.0 * b * b / 65536;
      if (split > 1) t += 4.7 + 8.0 * split * batch * M * N / 4.6e6;
      if (t < least) {
        least = t;
        best = p;
        best.splits = split;
      }
    }
  }
  best.slab = best.splits > 1 ? best.splits * batch * M * up_to(N, 8) * 4 : 0;
  return best;
}

// what a launch needs before its kernel is chosen
static inline GemmArgs gemm_args() {
  GemmArgs a;
  memset((void*)&a, 0, sizeof(a));
  a.alpha = 1.f;
  a.nseg = a.batch = a.splits = 1;
  return a;
}

template <int DT, typename T, int LM, int LN, int EPI>
static int run_tiles(hipStream_t st, GemmArgs& a, const GemmPlan& p) {
  a.tiles_m = p.tiles_m;
  a.tiles_n = p.tiles_n;
  HGK_CHECK_THREADS("product", (long)a.tiles_m * a.tiles_n * a.batch * a.splits, p.tile == 256 ? 512 : 256);
  const dim3 grid((unsigned)((long)a.tiles_m * a.tiles_n * a.batch * a.splits));
  if constexpr (DT != G_F32) {
    if (p.tile == 256) {
      hipLaunchKernelGGL((gemm_kernel<DT, T, LM, LN, 256, 4, 2, EPI>), grid, dim3(512), 0, st, a);
      HGK_LAUNCH_CHECK();
      return HGK_OK;
    }
  }
  if (p.tile == 128) hipLaunchKernelGGL((gemm_kernel<DT, T, LM, LN, 128, 2, 2, EPI>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((gemm_kernel<DT, T, LM, LN, 64, 4, 1, EPI>), grid, dim3(256), 0, st, a);
  HGK_LAUNCH_CHECK();
  return HGK_OK;
}

}  // namespace hgk
