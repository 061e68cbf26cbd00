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
// 4 consecutive n of one row m, which an epilogue loads and stores as one vector.
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
  void* out;
  void* out1;         // second batch's / du
  float* slab;
  long ldo;           // elements per output row
  const void* res;    // residual, rows of ldo
  const void* dh;     // E_GATED_BWD: incoming gradient, rows of N
  int npad;           // E_GATED_BWD: columns [N, npad) of dg / du are written as zero
  const float *row_scale, *col_scale, *col_scale1, *bias;
  float alpha;        // E_OUT: factor of the sum
  int act, vec;       // vec: out / res / dh rows may be accessed in vectors of 4
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

// 4 consecutive elements of a row, n .. n + 3, those past N skipped
template <typename T>
__device__ __forceinline__ void load4(const T* p, int n, int N, bool vec, float* f) {
  if (vec && n + 4 <= N) {
    if constexpr (sizeof(T) == 4) {
      const float4 v = *reinterpret_cast<const float4*>(p + n);
      f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
    } else {
      const uint2 v = *reinterpret_cast<const uint2*>(p + n);
      f[0] = __uint_as_float(v.x << 16); f[1] = __uint_as_float(v.x & 0xffff0000u);
      f[2] = __uint_as_float(v.y << 16); f[3] = __uint_as_float(v.y & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = n + e < N ? to_f(p[n + e]) : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void store4(T* p, int n, int N, bool vec, const float* f) {
  if (vec && n + 4 <= N) {
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<float4*>(p + n) = make_float4(f[0], f[1], f[2], f[3]);
    } else {
      bf16x2_t a = {(__bf16)f[0], (__bf16)f[1]}, b = {(__bf16)f[2], (__bf16)f[3]};
      *reinterpret_cast<uint2*>(p + n) =
          make_uint2(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b));
    }
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (n + e < N) p[n + e] = from_f<T>(f[e]);
  }
}

// factor, bias, dropout and residual of 4 consecutive outputs n .. n + 3 of row m, and the store
template <typename T>
__device__ __forceinline__ void finish4(const GemmArgs& a, void* out, int m, int n, float* f, uint64_t off) {
#pragma unroll
  for (int e = 0; e < 4; ++e) f[e] *= a.alpha;
  if (a.bias) {
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] += n + e < a.N ? a.bias[n + e] : 0.f;
  }
  if (a.drop) {
    const uint64_t gid = (uint64_t)m * ((a.N + 7) >> 3) + (n >> 3);
    const uint32_t k = drop_mask8(gid, off, a.d.seed, a.d.thr) >> (n & 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = (k >> e) & 1u ? f[e] * a.d.scale : 0.f;
  }
  if (a.res) {
    float q[4];
    load4<T>((const T*)a.res + (long)m * a.ldo, n, a.N, a.vec, q);
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] += q[e];
  }
  store4<T>((T*)out + (long)m * a.ldo, n, a.N, a.vec, f);
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

  // ---- epilogue: a lane holds n .. n + 3 of row m ----
  constexpr bool FAST = sizeof(T) == 2;
  const uint64_t off = EPI == E_OUT && a.drop ? drop_offset(a.d) : 0;
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    const int m = m0 + wm * WTM + i * 16 + lr;
    if (m >= a.M) continue;
    float rs = 1.f;
    if constexpr (DT == G_I8) rs = a.row_scale[m];
    if constexpr (DUAL) {
#pragma unroll
      for (int j = 0; j < FN / 2; ++j) {
        const int n = n0 + wn * (WTN / 2) + j * 16 + lg * 4;
        float g[4], u[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          g[e] = (float)acc[j][i][e];
          u[e] = (float)acc[j + FN / 2][i][e];
          if constexpr (DT == G_I8) {
            const int nn = min(n + e, a.N - 1);
            g[e] = g[e] * rs * a.col_scale[nn];
            u[e] = u[e] * rs * a.col_scale1[nn];
          }
        }
        if constexpr (EPI == E_GATED) {
          if (n >= a.N) continue;
#pragma unroll
          for (int e = 0; e < 4; ++e) g[e] = act_f<FAST>(a.act, g[e]) * u[e];
          store4<T>((T*)a.out + (long)m * a.ldo, n, a.N, a.vec, g);
        } else {
          if (n >= a.npad) continue;  // dg / du rows are npad long: always vectors
          float d[4], dg[4], du[4];
          load4<T>((const T*)a.dh + (long)m * a.N, n, a.N, a.vec, d);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float av, sv;
            act_slope<FAST>(a.act, g[e], av, sv);
            dg[e] = n + e < a.N ? d[e] * u[e] * sv : 0.f;
            du[e] = n + e < a.N ? d[e] * av : 0.f;
          }
          store4<T>((T*)a.out + (long)m * a.npad, n, a.npad, true, dg);
          store4<T>((T*)a.out1 + (long)m * a.npad, n, a.npad, true, du);
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < FN; ++j) {
        const int n = n0 + wn * WTN + j * 16 + lg * 4;
        if (n >= a.N) continue;
        float f[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) f[e] = (float)acc[j][i][e];
        if constexpr (EPI == E_SLAB) {
          float* s = a.slab + (((long)split * a.batch + bat) * a.M + m) * a.N;
          store4<float>(s, n, a.N, (a.N & 3) == 0, f);
        } else {
          if constexpr (DT == G_I8) {
#pragma unroll
            for (int e = 0; e < 4; ++e) f[e] = f[e] * rs * a.col_scale[min(n + e, a.N - 1)];
          }
          finish4<T>(a, bat ? a.out1 : a.out, m, n, f, off);
        }
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
  if constexpr (DUAL) {
#pragma unroll
    for (int e = 0; e < 4; ++e) f[0][e] = act_f<sizeof(T) == 2>(a.act, f[0][e]) * f[P - 1][e];
    store4<T>((T*)a.out + (long)m * a.ldo, n, a.N, a.vec, f[0]);
  } else {
    finish4<T>(a, a.out, m, n, f[0], a.drop ? drop_offset(a.d) : 0);
  }
}

// sum of the k ranges' partial sums in their order, then the epilogue of E_OUT
template <typename T>
__global__ __launch_bounds__(256) void gemm_join_kernel(GemmArgs a) {
  const int n4 = (a.N + 3) >> 2;
  const long t = (long)blockIdx.x * 256 + threadIdx.x;
  if (t >= (long)a.batch * a.M * n4) return;
  const int n = (int)(t % n4) * 4;
  const long bm = t / n4;  // batch * M + m
  const int bat = (int)(bm / a.M), m = (int)(bm - (long)bat * a.M);
  const long pitch = (long)a.batch * a.M * a.N;
  const float* s = a.slab + bm * a.N;
  float f[4] = {0.f, 0.f, 0.f, 0.f};
  for (int k = 0; k < a.splits; ++k) {
    float q[4];
    load4<float>(s + k * pitch, n, a.N, (a.N & 3) == 0, q);
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] += q[e];
  }
  finish4<T>(a, bat ? a.out1 : a.out, m, n, f, a.drop ? drop_offset(a.d) : 0);
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

// what a launch needs before its kernel is chosen
static inline GemmArgs gemm_args() {
  GemmArgs a;
  memset((void*)&a, 0, sizeof(a));
  a.alpha = 1.f;
  a.nseg = a.batch = a.splits = 1;
  return a;
}

}  // namespace hgk
