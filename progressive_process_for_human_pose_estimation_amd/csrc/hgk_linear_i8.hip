// Products in 8-bit integers with one scale for each row of the activations (token, pixel) and one
// for each output channel, how the block's products are served:
//   s_m = max_k |x[m][k]| / 127 (fp32),  q[m][k] = rint(x[m][k] / s_m)
//   y[m][n] = s_m w_n sum_k q[m][k] wq[n][k] (+ b[n]);   gated: a(G) U of two such products
// The sums are exact: int32 accumulators (K <= 2^17 keeps |sum| < 2^31), scaled once in fp32.
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
  // magnitudes compare like their bits, infinities and NaN above all numbers
  uint32_t m = 0;
  auto scan = [&](const float* v) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < V; ++e) m = max(m, __float_as_uint(v[e]) & 0x7fffffffu);
  };
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
  const bool odd = m >= 0x7f800000u;  // an infinity or a NaN
  const float sc = __uint_as_float(m) / 127.f;
  const bool none = odd || sc == 0.f;
  if (lane == 0) s[r] = odd ? __int_as_float(0x7fc00000) : sc;
  // v / sc correctly rounded, the quotient of two fp32 values that the definition rounds to a whole step: from
  // the correctly rounded reciprocal, one fused step makes the product faithful (within a unit in the last
  // place) and the next one exact (Markstein, 1990). Where sc or its reciprocal leaves the normal numbers: the
  // division itself. Adding 1.5 2^23 rounds to a whole number, whose low byte is the result.
  const float inv = 1.f / sc;
  const bool plain = sc >= 1e-30f && sc <= 1e30f;
  auto put = [&](int c, const float* v) __attribute__((always_inline)) {
    uint32_t b[V];
    if (plain) {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        float t = v[e] * inv;
        t = fmaf(fmaf(-t, sc, v[e]), inv, t);
        t = fmaf(fmaf(-t, sc, v[e]), inv, t);
        b[e] = __float_as_uint(t + 12582912.f);
      }
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e)
        b[e] = none ? 0 : (uint32_t)(int)fminf(fmaxf(rintf(v[e] / sc), -127.f), 127.f);
    }
    if constexpr (VEC) {
      uint32_t w[V / 4];
#pragma unroll
      for (int e = 0; e < V; e += 4)
        w[e / 4] = (b[e] & 0xffu) | (b[e + 1] & 0xffu) << 8 | (b[e + 2] & 0xffu) << 16 | b[e + 3] << 24;
      if constexpr (V == 8) *reinterpret_cast<uint2*>(qrow + c * 8) = make_uint2(w[0], w[1]);
      else *reinterpret_cast<uint32_t*>(qrow + c * 4) = w[0];
    } else {
      qrow[c] = (int8_t)b[0];
    }
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

template <typename T, bool VEC>
static void launch_quant_as(hipStream_t st, const T* x, int8_t* q, float* s, long rows, int K, int Kp) {
  const int nc = VEC ? K / Vec16<T>::N : K;
  const dim3 blk(256);
  auto grid = [&](int L) { return dim3((unsigned)((rows * L + 255) / 256)); };
#define HGK_QUANT(L, NCH) \
  hipLaunchKernelGGL((quant_rows_kernel<T, L, NCH, VEC>), grid(L), blk, 0, st, x, q, s, rows, K, Kp)
  if (nc <= 8) HGK_QUANT(8, 1);
  else if (nc <= 16) HGK_QUANT(16, 1);
  else if (nc <= 32) HGK_QUANT(16, 2);
  else if (nc <= 64) HGK_QUANT(32, 2);
  else if (nc <= 128) HGK_QUANT(64, 2);
  else if (nc <= 256) HGK_QUANT(64, 4);
  else if (nc <= 512) HGK_QUANT(64, 8);
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

struct I8Ws {
  long q, s, w0, w1, total;
  int Kp;
  bool pad;
};
static I8Ws i8_ws(long M, int K, int N, bool gated) {
  I8Ws w;
  w.Kp = (int)up_to(K, 16);
  w.pad = w.Kp != K;
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
  launch_quant<T>(st, x, (int8_t*)(ws + w.q), (float*)(ws + w.s), M, K, w.Kp);
  HGK_LAUNCH_CHECK();
  if (w.pad) {
    Pads p;
    p.add(w0, ws + w.w0, N, K, w.Kp, 1);
    if (GATED) p.add(w1, ws + w.w1, N, K, w.Kp, 1);
    p.launch<uint8_t>(st);
    HGK_LAUNCH_CHECK();
  }
  GemmArgs a = gemm_args();
  a.m0 = ws + w.q;
  a.n0 = w.pad ? ws + w.w0 : (const char*)w0;
  a.n1 = w.pad ? ws + w.w1 : (const char*)w1;
  a.ldm = a.ldn = w.Kp;
  a.M = (int)M;
  a.N = N;
  a.km = a.kn = w.Kp;
  a.spseg = (w.Kp + 127) / 128;
  a.out = y;
  a.row_scale = (const float*)(ws + w.s);
  a.col_scale = s0;
  a.col_scale1 = s1;
  a.bias = bias;
  a.res = res;
  a.act = act;
  a.vec = N % 8 == 0;
  constexpr int EPI = GATED ? E_GATED : E_OUT, per = GATED ? 2 : 1;
  if (M <= 64) {
    const dim3 grid((unsigned)((N + 15) / 16));
    if (M <= 16) hipLaunchKernelGGL((skinny_kernel<G_I8, T, 1, GATED>), grid, dim3(512), 0, st, a);
    else if (M <= 32) hipLaunchKernelGGL((skinny_kernel<G_I8, T, 2, GATED>), grid, dim3(512), 0, st, a);
    else hipLaunchKernelGGL((skinny_kernel<G_I8, T, 4, GATED>), grid, dim3(512), 0, st, a);
  } else {
    run_tiles<G_I8, T, L_ROW, L_ROW, EPI>(st, a, plan_gemm(G_I8, M, N, per, a.spseg, 1, false));
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
  HGK_CHECK_ARG(x && wq && wscale && y && workspace, "linear_i8: null pointer");
  HGK_CHECK_ARG(al16(x) && al16(wq) && al16(res) && al16(y) && al16(workspace), "linear_i8: pointers must be 16-byte aligned");
  HGK_CHECK_ARG(ws_bytes >= hgk_linear_i8_workspace(M, K, N, 0), "linear_i8: workspace of %zu bytes is too small", ws_bytes);
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
  HGK_CHECK_ARG(x && wqg && sg && wqu && su && h && workspace, "gated_i8: null pointer");
  HGK_CHECK_ARG(al16(x) && al16(wqg) && al16(wqu) && al16(h) && al16(workspace), "gated_i8: pointers must be 16-byte aligned");
  HGK_CHECK_ARG(ws_bytes >= hgk_linear_i8_workspace(M, C, F, 1), "gated_i8: workspace of %zu bytes is too small", ws_bytes);
  HGK_DISPATCH_DTYPE(dtype, T, return (linear_i8<T, true>((hipStream_t)stream, x, wqg, sg, wqu, su, nullptr, nullptr, h,
                                                          M, C, F, act, (char*)workspace)));
}
}
