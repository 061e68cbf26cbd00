// The input gradient of the product with dropout over wide maps of few output channels (bf16, N <= 256: the
// pixel levels), one pass over the rows:
//   dz = kept ? dy : 0  (stored for the weight gradient),   dx = s dz W
// A wave holds 16 rows of dz in registers, masked as they are read (a lane's 8 channels of a K-step are one
// group of the mask), and the width of dx is walked in chunks of 64 columns, whose N x 64 weights stand in
// LDS (a ring of three, LDS-DMA) and are read as transposed fragments. Against the tiled product this
// spares the launch that writes dz and its read.
//
// Measured, us, here / best tile (the tile with the launch that writes dz; K = 4 N; N > 128: waves of 16 rows, from
// 49152 rows on of 32, which read half as much LDS a row):
//   N     M = 16384    24576      32768      49152      65536      131072
//   64    6.4/10.6     6.8/12     7.2/14     10/19      12/21      17/39         dropped
//         5.8/7.3      6.1/8.6    6.5/9.2    9.7/12     11/13      17/25         p = 0
//   128   12/15        13/21      13/22      18/31      19/40      36/64         dropped
//         10.7/10.2    12/14      13/14      18/23      20/25      34/47         p = 0
//   192   21/22        22/30      23/36      34/46      35/57      68/103        dropped
//         19/15        21/22      23/25      30/35      31/45      61/81         p = 0
//   256   27/26        27/37      30/45      42/60      46/75      104/142       dropped
//         26/17        26/27      30/33      39/49      43/62      97/134        p = 0
// and at 40000 rows, 313 workgroups of 128 one a CU, with nothing dropped 37/29 (192) and 47/42 (256); waves of 16
// rows at 49152: 43 (192) and 53 (256), dropped. 80000 rows, 313 workgroups of 256: 63/68, 80/93, p = 0 55/54, 73/76.
// Hence linear_rows_ok() and kTwoGroups. At N = 256 and 131072 rows: 402 MB at 3.9 TB/s.
#include "hgk_gemm.h"

namespace hgk {

struct LinearRowsArgs {
  const bf16_t *dy, *w;
  bf16_t *dz, *dx;  // dz: null when the weight gradient is not wanted or nothing is dropped
  int M, N, K;
  float alpha;
  int drop;
  DropArgs d;
};

// NK: 32-channel steps of the contraction, N <= 32 NK. RW: groups of 16 rows of a wave
template <int NK, int RW>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2)))
void linear_rows_kernel(LinearRowsArgs a) {
  constexpr int SLOT = NK * 32 * 128, ND = NK / 2, DP = 2;  // DMAs of a wave; fragments are read DP steps ahead
  static_assert(NK >= 2 && NK <= 8 && NK % 2 == 0, "channels");
  __shared__ __attribute__((aligned(16))) char lds[3 * SLOT];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lr = lane & 15, lg = lane >> 4;
  const int m0 = (blockIdx.x * 8 + wave) * (16 * RW) + lr;  // of group i: + 16 i
  auto row_of = [&](int i) __attribute__((always_inline)) { return (long)min(m0 + 16 * i, a.M - 1); };
  const int nc = (a.K + 63) / 64;

  // weights: 8 chunks of 16 bytes of row n, swizzled as gemm_kernel's N side (tiles of 64 columns)
  const char* wp[ND];
  int wstep[ND], wcol[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) {
    const int at = (d * 8 + wave) * 1024 + lane * 16;
    const int n = at >> 7, c = ((at & 127) >> 4) ^ swz_col<G_BF16, 8, true>(n);
    const bool in = n < a.N;  // rows past the last are zeros, like dz's channels
    wp[d] = in ? (const char*)(a.w + (long)n * a.K + c * 8) : g_zero_page;
    wstep[d] = in ? 128 : 0;
    wcol[d] = c * 8;
  }
  auto send = [&](int chunk, int slot) __attribute__((always_inline)) {
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      const bool in = chunk * 64 + wcol[d] < a.K;  // columns past the last: not stored
      dma16(in ? wp[d] : g_zero_page, lds + slot * SLOT + (d * 8 + wave) * 1024);
      wp[d] += wstep[d];
    }
  };
  send(0, 0);
  if (nc > 1) send(1, 1);

  uint4 z[RW][NK];
#pragma unroll
  for (int i = 0; i < RW; ++i)
#pragma unroll
    for (int k = 0; k < NK; ++k) {
      const int c = k * 32 + lg * 8;
      z[i][k] = c < a.N ? load16(a.dy + row_of(i) * a.N + c) : make_uint4(0, 0, 0, 0);
    }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the first chunks have landed
  if (a.drop) {
    const uint64_t off = drop_offset(a.d);
#pragma unroll
    for (int i = 0; i < RW; ++i)
#pragma unroll
      for (int k = 0; k < NK; ++k) {
        const int c = k * 32 + lg * 8;
        const uint32_t keep = drop_mask8((uint64_t)row_of(i) * (a.N >> 3) + (c >> 3), off, a.d.seed, a.d.thr);
        uint32_t* v = &z[i][k].x;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          v[e] &= ((keep >> (2 * e)) & 1u ? 0xffffu : 0u) | ((keep >> (2 * e + 1)) & 1u ? 0xffff0000u : 0u);
        if (a.dz && m0 + 16 * i < a.M && c < a.N) store16(a.dz + row_of(i) * a.N + c, z[i][k]);
      }
  }
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");

  // place q of a fragment pair is 8 columns, of which fragment o takes half o ^ (q & 1)
  const int q = lr & 3, sw = swz_col<G_BF16, 8, true>(8 * lg + (lr >> 2));
  const int row = (8 * lg + (lr >> 2)) * 128;
  typedef short s16x8 __attribute__((ext_vector_type(8)));
  int slot = 0;
#pragma unroll 1
  for (int c = 0; c < nc; ++c) {
    const char* t = lds + slot * SLOT + row;
    f32x4 acc[RW][4];
    i32x4 wf[DP + 1][4];
    auto read = [&](int k) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const char* at = t + k * 32 * 128 + (((4 * (j >> 1) + q) ^ sw) << 4) + ((j & 1) ^ (q & 1)) * 8;
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(at));
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) s16x4*)(at + 4 * 128));
        const s16x8 f = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        wf[k % (DP + 1)][j] = __builtin_bit_cast(i32x4, f);
      }
    };
#pragma unroll
    for (int i = 0; i < RW; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < DP && k < NK; ++k) read(k);
#pragma unroll
    for (int k = 0; k < NK; ++k) {
      if (k + DP < NK) read(k + DP);
#pragma unroll
      for (int i = 0; i < RW; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          acc[i][j] = mma<G_BF16>(wf[k % (DP + 1)][j], __builtin_bit_cast(i32x4, z[i][k]), acc[i][j]);
      __builtin_amdgcn_sched_barrier(0);
    }
    // this wave's share of chunk c + 1 has landed (and its stores of a chunk ago are done); chunk c + 2 goes where
    // c - 1 was, which everybody has read
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (c + 2 < nc) send(c + 2, slot == 0 ? 2 : slot - 1);
    const bool swapped = lg & 1;
#pragma unroll
    for (int i = 0; i < RW; ++i)
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const int n = c * 64 + 32 * g + 8 * lg;
        float f[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = acc[i][2 * g][e] * a.alpha, y = acc[i][2 * g + 1][e] * a.alpha;
          f[e] = swapped ? y : x;
          f[4 + e] = swapped ? x : y;
        }
        if (m0 + 16 * i < a.M && n < a.K) store16(a.dx + row_of(i) * a.K + n, pack16<bf16_t>(f));
      }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    slot = slot == 2 ? 0 : slot + 1;
  }
}

static constexpr int kTwoGroups = 49152;  // rows from which waves take 32 (N > 128)
bool linear_rows_ok(int dtype, long M, int K, int N, bool drop) {
  if (dtype != HGK_BF16 || N % 8 != 0 || K % 8 != 0 || route(HGK_ROUTE_FFN_TILE)) return false;
  if (N <= 128) return M >= 16384;
  return N <= 256 && M >= (drop ? 24576 : kTwoGroups);
}

template <int NK, int RW>
static int launch_as(hipStream_t st, const LinearRowsArgs& a) {
  constexpr int rows = 128 * RW;
  HGK_CHECK_THREADS("linear", ((long)a.M + rows - 1) / rows, 512);
  hipLaunchKernelGGL((linear_rows_kernel<NK, RW>), dim3((unsigned)((a.M + rows - 1) / rows)), dim3(512), 0, st, a);
  HGK_LAUNCH_CHECK();
  return HGK_OK;
}
int linear_rows_bwd(hipStream_t st, const void* dy, const void* w, void* dz, void* dx, long M, int K, int N,
                    const DropArgs& d) {
  LinearRowsArgs a;
  a.dy = (const bf16_t*)dy;
  a.w = (const bf16_t*)w;
  a.dz = (bf16_t*)dz;
  a.dx = (bf16_t*)dx;
  a.M = (int)M;
  a.N = N;
  a.K = K;
  a.drop = d.thr != 0;
  a.alpha = a.drop ? d.scale : 1.f;
  a.d = d;
  if (N <= 64) return launch_as<2, 1>(st, a);
  if (N <= 128) return launch_as<4, 1>(st, a);
  if (M < kTwoGroups) return launch_as<8, 1>(st, a);
  return launch_as<8, 2>(st, a);
}

}  // namespace hgk
