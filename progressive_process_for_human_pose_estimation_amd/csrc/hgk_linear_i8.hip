// Products in 8-bit integers with one scale for each row of the activations (token, pixel) and one
// for each output channel, how the block's products are served:
//   s_m = max_k |x[m][k]| / 127 (fp32),  q[m][k] = rint(x[m][k] / s_m)
//   y[m][n] = s_m w_n sum_k q[m][k] wq[n][k] (+ b[n]);   gated: a(G) U of two such products
// The sums are exact: int32 accumulators (K <= 2^17 keeps |sum| < 2^31). A sum is then rounded to fp32
// (none below 2^24, K = 1040) and multiplied by the two scales in fp32: three roundings of 2^-24, a share of
// 2^-14 of the one to bf16. 64-bit products would run at a small part of the epilogue's rate.
// v_mfma_i32_16x16x64_i8 runs at twice the bf16 rate and the weights are half its bytes.
#include "hgk_gemm.h"

namespace hgk {

static constexpr int kI8MaxK = 1 << 17;

// L lanes a row (64 / L rows a wave, so that short rows fill the wave), NCH 16-byte chunks a lane held in
// registers: the row is read once. NCH == 0: two passes, the second from the cache. VEC false: rows not on
// 16-byte borders, single elements. Bound by memory: 2 bytes in and 1 out an element of bf16.
template <typename T, int L, int NCH, bool VEC>
__global__ __launch_bounds__(256) void quant_rows_kernel(const T* __restrict__ x, int8_t* __restrict__ q,
                                                         float* __restrict__ s, long rows, int K, int Kp) {
  constexpr int V = VEC ? Vec16<T>::N : 1;
  const int lane = threadIdx.x % L;
  const long r = ((long)blockIdx.x * 256 + threadIdx.x) / L;
  if (r >= rows) return;
  const T* row = x + r * K;
  int8_t* qrow = q + r * Kp;
  float f[NCH ? NCH : 1][V];
  auto load = [&](int c, float* v) __attribute__((always_inline)) {
    if constexpr (VEC) unpack16<T>(load16(row + c * V), v);
    else v[0] = to_f(row[c]);
  };
  const int nc = K / V;  // VEC: K % V == 0
  uint32_t m = 0;
  auto scan = [&](const float* v) __attribute__((always_inline)) { m = max_bits<V>(v, m); };
  if constexpr (NCH > 0) {
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const int c = lane + i * L;
      if (c < nc) load(c, f[i]);
      else
        for (int e = 0; e < V; ++e) f[i][e] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < NCH; ++i) scan(f[i]);
  } else {
    for (int c = lane; c < nc; c += L) {
      load(c, f[0]);
      scan(f[0]);
    }
  }
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, o, L));
  QuantScale z;
  const float sc = quant_scale(m, z);
  if (lane == 0) s[r] = sc;
  auto put = [&](int c, const float* v) __attribute__((always_inline)) {
    uint32_t b[V];
    quant_bytes<V>(v, z, b);
    if constexpr (VEC && V == 8) *reinterpret_cast<uint2*>(qrow + c * 8) = make_uint2(pack_bytes(b), pack_bytes(b + 4));
    else if constexpr (VEC) *reinterpret_cast<uint32_t*>(qrow + c * 4) = pack_bytes(b);
    else qrow[c] = (int8_t)b[0];
  };
  if constexpr (NCH > 0) {
#pragma unroll
    for (int i = 0; i < NCH; ++i)
      if (lane + i * L < nc) put(lane + i * L, f[i]);
  } else {
    for (int c = lane; c < nc; c += L) {
      load(c, f[0]);
      put(c, f[0]);
    }
  }
  for (int c = K + lane; c < Kp; c += L) qrow[c] = 0;
}

// long rows (K > 4096 of bf16, 2048 of fp32): a workgroup a row, in two passes, the second from the cache
template <typename T>
__global__ __launch_bounds__(256) void quant_long_kernel(const T* __restrict__ x, int8_t* __restrict__ q,
                                                         float* __restrict__ s, int K, int Kp) {
  __shared__ uint32_t xm[4];
  const long r = blockIdx.x;
  const int tid = threadIdx.x, nc = K / Vec16<T>::N;
  const uint32_t part = row_max<T>(x + r * K, tid, 256, nc);
  if ((tid & 63) == 0) xm[tid >> 6] = part;
  __syncthreads();
  QuantScale z;
  const float sc = quant_scale(max(max(xm[0], xm[1]), max(xm[2], xm[3])), z);
  row_bytes<T>(x + r * K, q + r * Kp, z, tid, 256, nc);
  if (tid == 0) s[r] = sc;
  for (int c = K + tid; c < Kp; c += 256) q[r * Kp + c] = 0;
}

template <typename T, bool VEC>
static void launch_quant_as(hipStream_t st, const T* x, int8_t* q, float* s, long rows, int K, int Kp) {
  const int nc = VEC ? K / Vec16<T>::N : K;
  const dim3 blk(256);
  // in runs of rows: a launch holds less than 2^32 threads
  auto runs = [&](int threads, auto&& launch) {
    const long most = (1l << 31) / threads;
    for (long r = 0; r < rows; r += most) launch(x + r * K, q + r * Kp, s + r, std::min(most, rows - r));
  };
#define HGK_QUANT(L, NCH)                                                                                              \
  runs(L, [&](const T* xr, int8_t* qr, float* sr, long n) {                                                            \
    hipLaunchKernelGGL((quant_rows_kernel<T, L, NCH, VEC>), dim3((unsigned)((n * L + 255) / 256)), blk, 0, st, xr, qr, \
                       sr, n, K, Kp);                                                                                  \
  })
  if (nc <= 8) HGK_QUANT(8, 1);
  else if (nc <= 16) HGK_QUANT(16, 1);
  else if (nc <= 32) HGK_QUANT(16, 2);
  else if (nc <= 64) HGK_QUANT(32, 2);
  else if (nc <= 128) HGK_QUANT(64, 2);
  else if (nc <= 256) HGK_QUANT(64, 4);
  else if (nc <= 512) HGK_QUANT(64, 8);
  else if constexpr (VEC)
    runs(256, [&](const T* xr, int8_t* qr, float* sr, long n) {
      hipLaunchKernelGGL((quant_long_kernel<T>), dim3((unsigned)n), blk, 0, st, xr, qr, sr, K, Kp);
    });
  else HGK_QUANT(64, 0);
#undef HGK_QUANT
}

template <typename T>
static void launch_quant(hipStream_t st, const void* x, int8_t* q, float* s, long rows, int K, int Kp) {
  constexpr int V = Vec16<T>::N;
  // quantised rows are written in words of V: q and its pitch have to allow them
  if (K % V == 0 && Kp % V == 0 && ((uintptr_t)x & 15) == 0 && ((uintptr_t)q & 7) == 0)
    launch_quant_as<T, true>(st, (const T*)x, q, s, rows, K, Kp);
  else
    launch_quant_as<T, false>(st, (const T*)x, q, s, rows, K, Kp);
}

// ---- few channels (K <= 256, N <= 256: the pointwise products of the pixel levels) ----
// A wave keeps its 64 columns of the weights in registers, a workgroup of 4 waves walks 32-row tiles: a
// tile's rows are read once as T, quantised in registers (8 lanes a row) and written to LDS as bytes, so
// the quantised rows never go through memory: 4 bytes an element of x and y in all. The next tile is on
// its way from memory while this one's products run. Two workgroups a CU: the quantising and the
// epilogue of one (18 us of VALU at 131072 x 256 x 256) run beside the memory of the other; one
// workgroup of 8 waves with the weights in LDS took 45 us, one phase after the other.
static constexpr int kMapK = 256, kMapN = 256, kMapRows = 32, kMapGroups = 512;
template <typename T>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2)))
void i8_map_kernel(GemmArgs a, int tiles) {
  constexpr int V = Vec16<T>::N, NC = kMapK / V / 8;  // 16-byte chunks of a lane
  __shared__ __attribute__((aligned(16))) char lx[2][kMapRows * kMapK];
  __shared__ float ls[2][kMapRows];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, lr = lane & 15, lg = lane >> 4;
  const int K = a.km;
  i32x4 w[4][4];
#pragma unroll
  for (int h = 0; h < 4; ++h)
#pragma unroll
    for (int j = 0; j < 4; ++j) {  // the order of the N rows as in gemm_kernel
      const int n = min(wave * 64 + (j >> 1) * 32 + 8 * (lr >> 2) + 4 * (j & 1) + (lr & 3), a.N - 1);
      const int k = h * 64 + lg * 16;
      w[h][j] = k < K ? *reinterpret_cast<const i32x4*>(a.n0 + (long)n * K + k) : i32x4{0, 0, 0, 0};
    }
  const int qr = tid >> 3, ql = tid & 7;
  typename Vec16<T>::type xv[NC];
  auto load = [&](int tile) __attribute__((always_inline)) {
    const T* row = (const T*)a.m0 + min((long)tile * kMapRows + qr, (long)a.M - 1) * K;
#pragma unroll
    for (int j = 0; j < NC; ++j)
      if ((ql + 8 * j) * V < K) xv[j] = load16(row + (ql + 8 * j) * V);
  };
  auto quantise = [&](int buf) __attribute__((always_inline)) {
    uint32_t m = 0;
    float f[V];
#pragma unroll
    for (int j = 0; j < NC; ++j) {
      if ((ql + 8 * j) * V < K) {
        unpack16<T>(xv[j], f);
        m = max_bits<V>(f, m);
      }
    }
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, o, 8));
    QuantScale z;
    const float sc = quant_scale(m, z);
    if (ql == 0) ls[buf][qr] = sc;
#pragma unroll
    for (int j = 0; j < NC; ++j) {
      const int at = (ql + 8 * j) * V;  // byte in the row; past K: zero
      uint32_t b[V];
#pragma unroll
      for (int e = 0; e < V; ++e) b[e] = 0;
      if (at < K) {
        unpack16<T>(xv[j], f);
        quant_bytes<V>(f, z, b);
      }
      // byte chunk c of row r sits at slot c ^ (r & 7) of its group of 8: the 8 rows of a b128 read differ
      char* p = lx[buf] + qr * kMapK + (((at >> 4) ^ (qr & 7)) << 4) + (at & 15);
#pragma unroll
      for (int e = 0; e < V; e += 4) *reinterpret_cast<uint32_t*>(p + e) = pack_bytes(b + e);
    }
  };
  int tile = blockIdx.x, buf = 0;
  if (tile < tiles) load(tile);
#pragma unroll 1
  for (; tile < tiles; tile += gridDim.x, buf ^= 1) {  // the whole workgroup
    quantise(buf);
    __syncthreads();  // also: every wave is done with this buffer's last tile but one
    if (tile + (int)gridDim.x < tiles) load(tile + gridDim.x);
    if (wave * 64 >= a.N) continue;  // a wave without columns quantises only
    i32x4 acc[4][2];
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i) acc[j][i] = i32x4{0, 0, 0, 0};
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      if (h * 64 >= K) break;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const i32x4 x = *reinterpret_cast<const i32x4*>(lx[buf] + (i * 16 + lr) * kMapK + (((h * 4 + lg) ^ (lr & 7)) << 4));
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[j][i] = mma<G_I8>(w[h][j], x, acc[j][i]);
      }
    }
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const int n = wave * 64 + 32 * g + 8 * lg;
      if (n >= a.N) continue;
      float cs[8], bias[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int c = min(n + e, a.N - 1);
        cs[e] = a.col_scale[c];
        bias[e] = a.bias ? a.bias[c] : 0.f;
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = i * 16 + lr;
        const long m = (long)tile * kMapRows + r;
        if (m >= a.M) continue;
        const float rs = ls[buf][r];
        float f[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = plus((float)acc[2 * g + (e >> 2)][i][e & 3] * rs * cs[e], bias[e]);
        if (a.res) {
          float q[8];
          load8<T>((const T*)a.res + m * a.N, n, a.N, a.vec, q);
#pragma unroll
          for (int e = 0; e < 8; ++e) f[e] = plus(f[e], q[e]);
        }
        store8<T>((T*)a.out + m * a.N, n, a.N, a.vec, f);
      }
    }
  }
}

// Which kernel a call takes, and what it needs. Measured, us, this way / the other:
//   rows quantised by the product's workgroups / by a launch of their own at a row 16 longer (bf16): 1 x 32768 ->
//     1024 22.6 / 27.5, 2 x 16384 13.8 / 15.1, 3 x 5456 7.5 / 8.4, 4 x 4096 -> 2048 6.9 / 7.6, 8 x 2048 -> 4096 6.1 /
//     7.4, 16 x 1024 6.1 / 6.1. Twice as much was slower: 8 x 4096 10.9 / 8.4, 16 x 2048 8.4 / 7.6.
//   few channels: the map kernel / the best of quantising launch + tiles (256 x 256 bf16): 5.8 / 6.7 at 65 rows, 6.6
//     / 9.4 at 8192, 13.7 / 19.9 at 32768, 35 / 46 at 131072; fp32 6.4 / 6.6, 8.1 / 10, 19 / 21, 64 / 65 (256 ->
//     64 in fp32 at 131072 the other way: 46 / 40). Up to 64 rows against the weight-streaming kernel: 5.8 / 6.2
//     in bf16, 6.4 / 6.0 in fp32 at 64, 5.6 / 5.2 and 6.2 / 5.0 at 17.
//   weight-streaming / tiles (bf16, gated 1024 -> 4096): 8.6 at 64 rows / 8.4 at 65; linear 4096 -> 1024 17 / 18.
enum I8Way { W_FEW_FUSED, W_FEW, W_MAP, W_TILES };
static I8Way i8_way(long M, int K, int N, bool gated) {
  if (M <= kQuantRows && M * K <= (M <= 2 ? kQuantBytes : kQuantBytes / 2) && K % 16 == 0) return W_FEW_FUSED;
  if (M <= 64) return W_FEW;
  if (!gated && K <= kMapK && K % 16 == 0 && N <= kMapN && !route(HGK_ROUTE_FFN_TILE)) return W_MAP;
  return W_TILES;
}

struct I8Ws {
  long q, s, w0, w1, total;
  int Kp;
  bool pad;
};
static I8Ws i8_ws(long M, int K, int N, bool gated) {
  I8Ws w;
  w.Kp = (int)up_to(K, 16);
  w.pad = w.Kp != K;
  w.q = w.s = w.w0 = w.w1 = w.total = 0;
  const I8Way way = i8_way(M, K, N, gated);
  if (way == W_FEW_FUSED || way == W_MAP) return w;
  long at = 0;
  auto take = [&](long b) {
    const long o = at;
    at += up_to(b, 256);
    return o;
  };
  w.q = take(M * w.Kp);
  w.s = take(M * 4);
  w.w0 = w.pad ? take((long)N * w.Kp) : 0;
  w.w1 = w.pad && gated ? take((long)N * w.Kp) : 0;
  w.total = at;
  return w;
}

template <typename T, bool GATED>
static int linear_i8(hipStream_t st, const void* x, const void* w0, const float* s0, const void* w1,
                     const float* s1, const float* bias, const void* res, void* y, long M, int K, int N, int act,
                     char* ws) {
  const I8Ws w = i8_ws(M, K, N, GATED);
  const I8Way way = i8_way(M, K, N, GATED);
  GemmArgs a = gemm_args();
  a.n0 = (const char*)w0;
  a.n1 = (const char*)w1;
  a.ldm = a.ldn = w.Kp;
  a.M = (int)M;
  a.N = N;
  a.km = a.kn = w.Kp;
  a.spseg = (w.Kp + 127) / 128;
  a.out = y;
  a.col_scale = s0;
  a.col_scale1 = s1;
  a.bias = bias;
  a.res = res;
  a.act = act;
  a.vec = N % 8 == 0;
  if (way == W_FEW_FUSED || way == W_MAP) {
    a.m0 = (const char*)x;
    if (way == W_MAP) {
      const int tiles = (int)((M + kMapRows - 1) / kMapRows);
      hipLaunchKernelGGL((i8_map_kernel<T>), dim3(std::min(tiles, kMapGroups)), dim3(256), 0, st, a, tiles);
    } else {
      hipLaunchKernelGGL((skinny_kernel<G_I8, T, 1, GATED, true>), dim3((unsigned)((N + 15) / 16)), dim3(512), 0, st, a);
    }
    HGK_LAUNCH_CHECK();
    return HGK_OK;
  }
  launch_quant<T>(st, x, (int8_t*)(ws + w.q), (float*)(ws + w.s), M, K, w.Kp);
  HGK_LAUNCH_CHECK();
  a.m0 = ws + w.q;
  a.row_scale = (const float*)(ws + w.s);
  if (w.pad) {
    Pads p;
    p.add(w0, ws + w.w0, N, K, w.Kp, 1);
    a.n0 = ws + w.w0;
    if (GATED) {
      p.add(w1, ws + w.w1, N, K, w.Kp, 1);
      a.n1 = ws + w.w1;
    }
    if (int rc = p.launch<uint8_t>(st)) return rc;
  }
  constexpr int EPI = GATED ? E_GATED : E_OUT, per = GATED ? 2 : 1;
  if (way == W_FEW) {
    const dim3 grid((unsigned)((N + 15) / 16));
    if (M <= 16) hipLaunchKernelGGL((skinny_kernel<G_I8, T, 1, GATED>), grid, dim3(512), 0, st, a);
    else if (M <= 32) hipLaunchKernelGGL((skinny_kernel<G_I8, T, 2, GATED>), grid, dim3(512), 0, st, a);
    else hipLaunchKernelGGL((skinny_kernel<G_I8, T, 4, GATED>), grid, dim3(512), 0, st, a);
  } else {
    return run_tiles<G_I8, T, L_ROW, L_ROW, EPI>(st, a, plan_gemm(G_I8, M, N, per, a.spseg, 1, false));
  }
  HGK_LAUNCH_CHECK();
  return HGK_OK;
}

static bool al16(const void* p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace hgk

using namespace hgk;

extern "C" {

int hgk_quantize_rows_i8(hgk_stream_t stream, int dtype, const void* x, void* q, float* scale, long rows,
                         int K) {
  HGK_CHECK_ARG(rows >= 0 && rows <= (1l << 30) && K >= 1 && K <= kI8MaxK, "quantize: bad sizes (%ld rows of %d)", rows, K);
  if (rows == 0) return HGK_OK;
  HGK_CHECK_ARG(x && q && scale, "quantize: null pointer");
  HGK_DISPATCH_DTYPE(dtype, T, {
    launch_quant<T>((hipStream_t)stream, x, (int8_t*)q, scale, rows, K, K);
    HGK_LAUNCH_CHECK();
    return HGK_OK;
  });
}

size_t hgk_linear_i8_workspace(long M, int K, int N, int gated) {
  if (M <= 0 || K <= 0 || N <= 0) return 0;
  return (size_t)i8_ws(M, K, N, gated != 0).total;
}

int hgk_linear_i8(hgk_stream_t stream, int dtype, const void* x, const void* wq, const float* wscale,
                  const float* bias, const void* res, void* y, long M, int K, int N, void* workspace, size_t ws_bytes) {
  HGK_CHECK_ARG(M >= 0 && M <= (1l << 30) && K >= 1 && K <= kI8MaxK && N >= 1 && N <= (1 << 24),
                "linear_i8: bad sizes (%ld, %d, %d)", M, K, N);
  if (M == 0) return HGK_OK;
  HGK_CHECK_ARG(x && wq && wscale && y, "linear_i8: null pointer");
  HGK_CHECK_ARG(al16(x) && al16(wq) && al16(res) && al16(y) && al16(workspace), "linear_i8: pointers must be 16-byte aligned");
  HGK_CHECK_WORKSPACE("linear_i8", workspace, ws_bytes, hgk_linear_i8_workspace(M, K, N, 0));
  HGK_DISPATCH_DTYPE(dtype, T, return (linear_i8<T, false>((hipStream_t)stream, x, wq, wscale, nullptr, nullptr,
                                                           bias, res, y, M, K, N, 0, (char*)workspace)));
}

int hgk_gated_i8(hgk_stream_t stream, int dtype, const void* x, const void* wqg, const float* sg,
                 const void* wqu, const float* su, void* h, long M, int C, int F, int act, void* workspace,
                 size_t ws_bytes) {
  HGK_CHECK_ARG(M >= 0 && M <= (1l << 30) && C >= 1 && C <= kI8MaxK && F >= 1 && F <= (1 << 24),
                "gated_i8: bad sizes (%ld, %d, %d)", M, C, F);
  HGK_CHECK_ARG(act >= 0 && act < HGK_ACT_COUNT, "gated_i8: unknown activation %d", act);
  if (M == 0) return HGK_OK;
  HGK_CHECK_ARG(x && wqg && sg && wqu && su && h, "gated_i8: null pointer");
  HGK_CHECK_ARG(al16(x) && al16(wqg) && al16(wqu) && al16(h) && al16(workspace), "gated_i8: pointers must be 16-byte aligned");
  HGK_CHECK_WORKSPACE("gated_i8", workspace, ws_bytes, hgk_linear_i8_workspace(M, C, F, 1));
  HGK_DISPATCH_DTYPE(dtype, T, return (linear_i8<T, true>((hipStream_t)stream, x, wqg, sg, wqu, su, nullptr, nullptr, h,
                                                          M, C, F, act, (char*)workspace)));
}
}
