// The gated product of wide maps of few channels (bf16: the pixel levels), forward (C <= 128), and its
// backward up to dg, du AND dx (C <= 256), one pass over the rows each.
//
// The hidden width F is walked in chunks of 32: a wave holds 16 rows of x in registers for all of it, the
// chunk's 32 gate and 32 up rows of the weights stand in LDS (a ring of four, LDS-DMA), and per chunk
//   g, u = x Wg^T, x Wu^T          (the chunk's columns, 8 consecutive of one row a lane)
//   forward:   h = a(g) u, stored
//   backward:  dg = dh u a'(g), du = dh a(g), rounded to bf16 and stored for the weight gradients;
//              dx += dg Wg + du Wu: what a lane holds of dg and du IS the matrix instruction's operand
//              (row = lane % 16, k = 8 (lane / 16) ..), and the weights are the same LDS tile, read as
//              transposed fragments. dg and du are not read back for dx.
// Against the tiled products (hgk_gemm.h), which at K = C <= 256 spend half of their time between the
// products of one tile and the next: two waves share a SIMD, half a chunk apart, and the activations and
// stores of one run beside the products of the other all the way. What bounds it: LDS reads (each wave reads
// the whole chunk for its rows) at C = 256, the stores of h, dg and du at C <= 128. Hence waves of 32 rows in
// the forward of many rows, which read half as much a row; the backward of 256 channels has no registers
// for that (dx alone takes 128 more), and of 128 it gains nothing (210 / 215 us with dW at 131072 rows).
//
// Measured, us, rows here / best tile (F = 4 C; f forward, b backward up to dx; at C > 128 f in waves of 32 rows):
//   C    M = 16384          24576              32768              65536              131072
//   64   f 7.9/6.4 b 11/17  f 8.7/9.4 b 12/24  f 9.4/10 b 13/27   f 14/17            f 21/31
//   128  f 15/11   b 27/32  f 15/18   b 29/40  f 17/19  b 32/49   f 28/36            f 47/66 (waves of 16: 53)
//   192           b 52/49   f 38/29   b 53/67  f 38/31  b 57/82   f 47/58            f 94/111
//   256           b 65/63   f 49/34   b 66/91  f 50/44  b 84/121  f 67/84            f 145/187
// (forward at C = 256 and 49152 rows 58/65, at 80000 rows 105/105; C = 192: 41/47 and 78/73; C = 128 in waves of 32 and
// of 16 rows: 25 and 17 at 32768, 27 and 28 at 65536, 37 and 36 at 80000, 75 and 85 at 200000.) A workgroup takes
// 128 or 256 rows, so 16384 are half of the card's CUs or less. Hence gated_rows_ok() and kTwoGroups.
#include "hgk_gemm.h"

namespace hgk {

struct RowsArgs {
  const bf16_t *x, *wg, *wu, *dh;
  bf16_t *h, *dg, *du, *dx;  // dg / du: null when no weight gradient is wanted
  int M, C, F, act;
};

// NK: 32-channel K-steps, C <= 32 NK. RW: groups of 16 rows of a wave
template <int NK, bool BWD, int ACT, int RW>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2)))
void gated_rows_kernel(RowsArgs a) {
  constexpr int PITCH = NK * 64, SLOT = 64 * PITCH, ND = NK / 2;  // LDS row and chunk bytes; DMAs of a wave
  constexpr int DP = 2, DB = 3;  // fragments are read this many K-steps (pairs) ahead: an LDS read under load takes
                                 // longer than the 4 (2) matrix instructions between
  static_assert(NK >= 2 && NK <= 8 && NK % 2 == 0, "channels");
  static_assert(RW == 1 || !BWD, "the backward takes one group");
  __shared__ __attribute__((aligned(16))) char lds[4 * SLOT];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lr = lane & 15, lg = lane >> 4;
  const int m0 = (blockIdx.x * 8 + wave) * (16 * RW) + lr;  // of group i: + 16 i
  const int nc = (a.F + 31) / 32;

  // ---- weights: row r of a part (gate, up) has its 16-byte chunk c at slot c ^ s(r), s(r) = (r & 3) |
  // (r >> 3 & 1) << 2: the 8 rows of a b128 read of fragment rows 8 (i / 4) + 4 o + i % 4 differ, and so do
  // the 8 rows of a half-wave's transposed read ----
  const char* wp[ND];
  long wstep[ND];
  int wrow[ND];  // row of the part
#pragma unroll
  for (int d = 0; d < ND; ++d) {
    const int at = (d * 8 + wave) * 1024 + lane * 16;
    const int row = at / PITCH, r = row & 31, c = ((at % PITCH) >> 4) ^ ((r & 3) | (((r >> 3) & 1) << 2));
    const bool in = c * 8 < a.C;  // channels past the last read zeros
    wp[d] = in ? (const char*)((row >> 5 ? a.wu : a.wg) + (long)r * a.C + c * 8) : g_zero_page;
    wstep[d] = in ? 64l * a.C : 0;
    wrow[d] = r;
  }
  auto send = [&](int chunk, int slot) __attribute__((always_inline)) {
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      const bool in = chunk * 32 + wrow[d] < a.F;  // rows past the last are zeros: nothing times them
      dma16(in ? wp[d] : g_zero_page, lds + slot * SLOT + (d * 8 + wave) * 1024);
      wp[d] += wstep[d];
    }
  };
  send(0, 0);
  if (nc > 1) send(1, 1);

  i32x4 xf[RW][NK];
#pragma unroll
  for (int i = 0; i < RW; ++i)
#pragma unroll
    for (int k = 0; k < NK; ++k) {
      const int c = k * 32 + lg * 8;
      const long m = min(m0 + 16 * i, a.M - 1);
      xf[i][k] = c < a.C ? *reinterpret_cast<const i32x4*>(a.x + m * a.C + c) : i32x4{0, 0, 0, 0};
    }
  uint4 dhv;  // past the last column: the last group again, unused
  const bf16_t* dhp = BWD ? a.dh + (long)min(m0, a.M - 1) * a.F : nullptr;
  auto load_dh = [&](int chunk) __attribute__((always_inline)) { dhv = load16(dhp + min(chunk * 32 + lg * 8, a.F - 8)); };
  if (BWD) load_dh(0);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");

  // fragment offsets within a chunk
  const int rb = (8 * (lr >> 2) + (lr & 3)) * PITCH;
  const int x0 = rb + ((lg ^ (lr & 7)) << 4), x1 = rb + (((4 + lg) ^ (lr & 7)) << 4);
  // transposed: k rows 8 lg + lr / 4 (+ 4), place q = lr % 4. Place q of pair G is the 8-column chunk A (q & 1) +
  // B (q >> 1) + G, of which fragment o takes half o ^ (q >> 1): the two places of a half differ in a chunk
  // bit that s() does not touch, so a half-wave's 32 pieces cover all banks (NK = 2: in two turns)
  constexpr int PA = NK == 2 ? 4 : 8, PB = NK == 8 ? 16 : NK == 4 ? 4 : 2;
  const int q = lr & 3, ts = (lr >> 2) | ((lg & 1) << 2);
  const int tc = PA * (q & 1) + PB * (q >> 1), tr = (8 * lg + (lr >> 2)) * PITCH;

  f32x4 acc[BWD ? NK : 1][2];
#pragma unroll
  for (int g = 0; g < (BWD ? NK : 1); ++g) acc[g][0] = acc[g][1] = f32x4{0.f, 0.f, 0.f, 0.f};

  f32x4 p[RW][4];  // the chunk's g (halves 0, 1) and u
  auto products = [&](int c) __attribute__((always_inline)) {
    const char* w = lds + (c & 3) * SLOT;
    i32x4 wf[DP + 1][4];  // gate o = 0, 1, up o = 0, 1 of a K-step and of the DP next
    auto read = [&](int k) __attribute__((always_inline)) {
      const char* t = w + (k & 1 ? x1 : x0) + (k >> 1) * 128;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        wf[k % (DP + 1)][j] = *reinterpret_cast<const i32x4*>(t + ((j >> 1) * 32 + (j & 1) * 4) * PITCH);
    };
#pragma unroll
    for (int i = 0; i < RW; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) p[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < DP && k < NK; ++k) read(k);
#pragma unroll
    for (int k = 0; k < NK; ++k) {
      if (k + DP < NK) read(k + DP);
#pragma unroll
      for (int i = 0; i < RW; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) p[i][j] = mma<G_BF16>(wf[k % (DP + 1)][j], xf[i][k], p[i][j]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  uint4 b0, b1;
  auto finish = [&](int c) __attribute__((always_inline)) {
    const int f0 = c * 32 + lg * 8;
    const bool f_in = f0 < a.F;
    // dh of this chunk, and what this wave sent for of the chunk after the one in the products
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    float dh[8];
    if (BWD) unpack16<bf16_t>(dhv, dh);
#pragma unroll
    for (int i = 0; i < RW; ++i) {
      const int m = m0 + 16 * i;
      float v0[8], v1[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float g = p[i][e >> 2][e & 3], u = p[i][2 + (e >> 2)][e & 3];
        if constexpr (BWD) {
          float av, sl;
          act_slope<ACT, true>(g, av, sl);
          v0[e] = f_in ? dh[e] * u * sl : 0.f;
          v1[e] = f_in ? dh[e] * av : 0.f;
        } else {
          v0[e] = act_f<ACT, true>(g) * u;
        }
      }
      b0 = pack16<bf16_t>(v0);
      if constexpr (!BWD) {
        if (m < a.M && f_in) store16(a.h + (long)m * a.F + f0, b0);
      } else {
        b1 = pack16<bf16_t>(v1);
        if (a.dg && m < a.M && f_in) {
          store16(a.dg + (long)m * a.F + f0, b0);
          store16(a.du + (long)m * a.F + f0, b1);
        }
        load_dh(min(c + 1, nc - 1));
      }
    }
  };
  auto back = [&](int c) __attribute__((always_inline)) {
    if constexpr (BWD) {
      const char* w = lds + (c & 3) * SLOT;
      typedef short s16x8 __attribute__((ext_vector_type(8)));
      constexpr int NF = 2 * NK;  // pairs of fragments: gate part, up part
      i32x4 tf[DB + 1][2];
      auto read_t = [&](int i) __attribute__((always_inline)) {
#pragma unroll
        for (int o = 0; o < 2; ++o) {
          const char* t = w + (i / NK) * 32 * PITCH + tr + (((tc + i % NK) ^ ts) << 4) + (o ^ (q >> 1)) * 8;
          const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(t));
          const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (__attribute__((address_space(3))) s16x4*)(t + 4 * PITCH));
          const s16x8 f = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
          tf[i % (DB + 1)][o] = __builtin_bit_cast(i32x4, f);
        }
      };
      const i32x4 bg = __builtin_bit_cast(i32x4, b0), bu = __builtin_bit_cast(i32x4, b1);
#pragma unroll
      for (int i = 0; i < DB && i < NF; ++i) read_t(i);
#pragma unroll
      for (int i = 0; i < NF; ++i) {
        if (i + DB < NF) read_t(i + DB);
#pragma unroll
        for (int o = 0; o < 2; ++o) acc[i % NK][o] = mma<G_BF16>(tf[i % (DB + 1)][o], i < NK ? bg : bu, acc[i % NK][o]);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  };
  auto meet = [&]() __attribute__((always_inline)) {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  // Two waves share a SIMD. The second four run half a chunk behind, so that one wave's activations stand beside
  // the other's products. Iteration c ends when everybody has read chunk c - 1 for the last time (its slot
  // is chunk c + 3's) and chunk c + 1 has landed: it was sent for in iteration c - 1, and every wave
  // waited for its own share in iteration c.
  if (wave < 4) {
#pragma unroll 1
    for (int c = 0; c < nc; ++c) {
      products(c);
      finish(c);
      if (c + 2 < nc) send(c + 2, (c + 2) & 3);
      back(c);
      meet();
    }
    meet();
  } else {
    if (2 < nc) send(2, 2);
    products(0);
    meet();
#pragma unroll 1
    for (int c = 1; c < nc; ++c) {
      finish(c - 1);
      if (c + 2 < nc) send(c + 2, (c + 2) & 3);
      back(c - 1);
      products(c);
      meet();
    }
    finish(nc - 1);
    back(nc - 1);
    meet();
  }
  if constexpr (BWD) {
    if (m0 >= a.M) return;
    const bool swapped = lg >> 1;
#pragma unroll
    for (int g = 0; g < NK; ++g) {
      const int n = (PA * (lg & 1) + PB * (lg >> 1) + g) * 8;
      if (n >= a.C) continue;
      float f[8];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        f[e] = swapped ? acc[g][1][e] : acc[g][0][e];
        f[4 + e] = swapped ? acc[g][0][e] : acc[g][1][e];
      }
      store16(a.dx + (long)m0 * a.C + n, pack16<bf16_t>(f));
    }
  }
}

static constexpr int kTwoGroups = 98304;  // rows
bool gated_rows_ok(int dtype, long M, int C, int F, bool bwd) {
  if (dtype != HGK_BF16 || C % 8 != 0 || F % 8 != 0 || route(HGK_ROUTE_FFN_TILE)) return false;
  if (C <= 128) return M >= (bwd ? 16384 : 24576);
  return C <= 256 && M >= (bwd ? 24576 : 49152);
}

template <int NK, bool BWD, int ACT, int RW>
static int launch_rows_as(hipStream_t st, const RowsArgs& a) {
  constexpr int rows = 128 * RW;
  HGK_CHECK_THREADS("gated", ((long)a.M + rows - 1) / rows, 512);
  hipLaunchKernelGGL((gated_rows_kernel<NK, BWD, ACT, RW>), dim3((unsigned)((a.M + rows - 1) / rows)), dim3(512), 0, st, a);
  HGK_LAUNCH_CHECK();
  return HGK_OK;
}
template <bool BWD, int ACT>
static int launch_rows_act(hipStream_t st, const RowsArgs& a) {
  if (a.C <= 64) return launch_rows_as<2, BWD, ACT, 1>(st, a);
  if constexpr (BWD) return a.C <= 128 ? launch_rows_as<4, true, ACT, 1>(st, a) : launch_rows_as<8, true, ACT, 1>(st, a);
  else if (a.C > 128) return launch_rows_as<8, false, ACT, 2>(st, a);
  else if (a.M >= kTwoGroups) return launch_rows_as<4, false, ACT, 2>(st, a);
  else return launch_rows_as<4, false, ACT, 1>(st, a);
}
template <bool BWD>
static int launch_rows(hipStream_t st, const RowsArgs& a) {
  if (a.act == kActSilu) return launch_rows_act<BWD, kActSilu>(st, a);
  if (a.act == kActGelu) return launch_rows_act<BWD, kActGelu>(st, a);
  if (a.act == kActRelu) return launch_rows_act<BWD, kActRelu>(st, a);
  return launch_rows_act<BWD, kActSigmoid>(st, a);
}

int gated_rows_fwd(hipStream_t st, const void* x, const void* wg, const void* wu, void* h, long M, int C, int F,
                   int act) {
  RowsArgs a = {(const bf16_t*)x, (const bf16_t*)wg, (const bf16_t*)wu, nullptr, (bf16_t*)h, nullptr, nullptr, nullptr,
                (int)M, C, F, act};
  return launch_rows<false>(st, a);
}
int gated_rows_bwd(hipStream_t st, const void* x, const void* wg, const void* wu, const void* dh, void* dg, void* du,
                   void* dx, long M, int C, int F, int act) {
  RowsArgs a = {(const bf16_t*)x, (const bf16_t*)wg, (const bf16_t*)wu, (const bf16_t*)dh, nullptr, (bf16_t*)dg,
                (bf16_t*)du, (bf16_t*)dx, (int)M, C, F, act};
  return launch_rows<true>(st, a);
}

}  // namespace hgk
