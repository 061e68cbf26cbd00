// The feed-forward block's products over rows of channels (pixels of an NHWC map), forward and
// backward, on the tiled matrix kernel of hgk_gemm.h.
//
//   gated:   h = a(x Wg^T) * (x Wu^T)                     both products in one pass over x
//   linear:  y = res + D(h Wd^T)                          dropout (hgk_philox.h) and skip in the epilogue
//
// Backward of the gated product, from dh: g and u are computed AGAIN (a third of the step's
// products more), not kept: kept in bf16 they would add a rounding of up to 2^-8 to dg and du before
// the rounding that the matrix instructions need anyway, kept in fp32 they are 8 bytes an element of h
// to write and read. dg = dh u a'(g) and du = dh a(g) are rounded to the operands' type, in workspace:
// the matrix instructions take no other (fp32 ones run at a tenth of the rate). With that the three
// gradients of a bf16 call are off by 0.0023 of their norm, 0.0017 if dg and du stayed fp32. dx = dg Wg + du Wu is ONE product whose k runs over both; dWg = dg^T x and
// dWu = du^T x are one launch of two batches.
// Backward of the linear: dz = kept ? dy : 0 is exact in any type, the factor 1 / (1 - p) goes to
// the fp32 sums in the epilogues.
#include "hgk_gemm.h"

namespace hgk {

// T: type of the result (partial sums are fp32 whatever it is)
template <int DT, typename T, int LM, int LN>
static int run_product(hipStream_t st, GemmArgs& a, const GemmPlan& p, char* slab) {
  a.splits = p.splits;
  a.slab = (float*)slab;
  if (p.splits > 1) {
    if (int rc = run_tiles<DT, std::conditional_t<DT == G_F32, float, bf16_t>, LM, LN, E_SLAB>(st, a, p)) return rc;
    const long n = (long)a.batch * a.M * ((a.N + 7) / 8);
    hipLaunchKernelGGL((gemm_join_kernel<T>), dim3((unsigned)((n + 63) / 64)), dim3(64), 0, st, a);
    HGK_LAUNCH_CHECK();
    return HGK_OK;
  }
  return run_tiles<DT, T, LM, LN, E_OUT>(st, a, p);
}

// Up to this many rows stream the weights (skinny_kernel), more take tiles. The linear's tiles can split k, so
// they take over early. Measured, us, rows / tiles: bf16 gated 1024 -> 4096: 6.1 at 32, 6.9 at 33 / 6.4; linear
// 4096 -> 1024: 9.4 at 16, 10.5 at 17 / 9.0 (1024 -> 256: 4.2, 4.6, 5.3 at 32 / 6.8); fp32 gated: 17.7 at 64 /
// 22.1, linear 16.6 at 16, 23.7 at 32 / 16.3.
template <typename T>
static constexpr int skinny_rows(bool dual) {
  return !dual ? 16 : sizeof(T) == 2 ? 32 : 64;
}
template <int DT, typename T, bool DUAL>
static void run_skinny(hipStream_t st, const GemmArgs& a) {
  constexpr int most = skinny_rows<T>(DUAL);
  const dim3 grid((unsigned)((a.N + 15) / 16));
  if (a.M <= 16) hipLaunchKernelGGL((skinny_kernel<DT, T, 1, DUAL>), grid, dim3(512), 0, st, a);
  if constexpr (most > 16) {
    if (a.M > 16 && a.M <= 32) hipLaunchKernelGGL((skinny_kernel<DT, T, 2, DUAL>), grid, dim3(512), 0, st, a);
  }
  if constexpr (most > 32) {
    if (a.M > 32) hipLaunchKernelGGL((skinny_kernel<DT, T, 4, DUAL>), grid, dim3(512), 0, st, a);
  }
}

template <typename T>
struct TypeOf;
template <>
struct TypeOf<float> {
  static constexpr int dt = G_F32;
  typedef uint32_t raw;
};
template <>
struct TypeOf<bf16_t> {
  static constexpr int dt = G_BF16;
  typedef uint16_t raw;
};

// a weight gradient: T, or fp32
template <int DT, typename T>
static int run_wgrad(hipStream_t st, GemmArgs& a, const GemmPlan& p, char* slab, bool f32) {
  if constexpr (sizeof(T) == 2) {
    if (f32) return run_product<DT, float, L_COL, L_COL>(st, a, p, slab);
  }
  return run_product<DT, T, L_COL, L_COL>(st, a, p, slab);
}

static inline int es_of(int dtype) { return dtype == HGK_BF16 ? 2 : 4; }

// which gradients a backward computes, from hgk.h's HGK_BWD_*
struct Wanted {
  bool dx, dw;
};
static inline Wanted wanted(int backward) { return {backward != HGK_BWD_DW, backward != HGK_BWD_DX}; }
static inline int wanted_code(bool dx, bool dw) { return dx && dw ? HGK_BWD_ALL : dx ? HGK_BWD_DX : HGK_BWD_DW; }

// workspace layout: offsets of the parts, each on a 256-byte border
struct Carve {
  long at = 0;
  long take(long bytes) {
    const long o = at;
    at += up_to(bytes, 256);
    return o;
  }
};

struct GatedWs {
  long x, wg, wu, dg, du, slab, total;
  int Cp, Fp;
  bool pad, rows;
  GemmPlan dx, dw;
};
static GatedWs gated_ws(int dtype, long M, int C, int F, int bwd) {
  GatedWs w;
  const int es = es_of(dtype), q = 16 / es, ks = 128 / es;
  w.Cp = (int)up_to(C, q);
  w.Fp = (int)up_to(F, 8);
  w.pad = w.Cp != C;
  Carve c;
  w.x = w.wg = w.wu = w.dg = w.du = w.slab = 0;
  if (w.pad) {
    w.x = c.take(M * w.Cp * es);
    w.wg = c.take((long)F * w.Cp * es);
    w.wu = c.take((long)F * w.Cp * es);
  }
  w.rows = false;
  if (bwd) {
    const Wanted want = wanted(bwd);
    w.rows = want.dx && gated_rows_ok(dtype, M, C, F, true);
    if (!w.rows || want.dw) {  // the row kernel stores dg and du for the weight gradients alone
      w.dg = c.take(M * w.Fp * es);
      w.du = c.take(M * w.Fp * es);
    }
    w.dx = plan_gemm(dtype == HGK_BF16 ? G_BF16 : G_F32, M, C, 1, 2 * (int)((F + ks - 1) / ks), 1, true);
    w.dw = plan_gemm(dtype == HGK_BF16 ? G_BF16 : G_F32, F, C, 1, (int)((M + ks - 1) / ks), 2, true);
    w.slab = c.take(std::max(want.dx && !w.rows ? w.dx.slab : 0, want.dw ? w.dw.slab : 0));
  }
  w.total = c.at;
  return w;
}

static bool al16(const void* p) { return ((uintptr_t)p & 15) == 0; }

#define HGK_CHECK_ROWS(what, M, A, B)                                                              \
  HGK_CHECK_ARG((M) >= 0 && (M) <= (1l << 30) && (A) >= 1 && (A) <= (1 << 21) && (B) >= 1 &&       \
                    (B) <= (1 << 21),                                                              \
                what ": bad sizes (%ld rows, %d, %d)", (long)(M), (int)(A), (int)(B))

template <typename T>
static int gated_operands(hipStream_t st, GemmArgs& a, const GatedWs& w, char* ws, const void* x,
                           const void* wg, const void* wu, long M, int C, int F) {
  typedef typename TypeOf<T>::raw raw;
  if (w.pad) {
    Pads p;
    p.add(x, ws + w.x, M, C, w.Cp, sizeof(T));
    p.add(wg, ws + w.wg, F, C, w.Cp, sizeof(T));
    p.add(wu, ws + w.wu, F, C, w.Cp, sizeof(T));
    if (int rc = p.launch<raw>(st)) return rc;
  }
  a.m0 = a.m1 = w.pad ? ws + w.x : (const char*)x;
  a.n0 = w.pad ? ws + w.wg : (const char*)wg;
  a.n1 = w.pad ? ws + w.wu : (const char*)wu;
  a.ldm = a.ldn = (long)w.Cp * sizeof(T);
  a.M = (int)M;
  a.N = F;
  a.km = a.kn = w.Cp;
  a.spseg = (int)up_to((long)w.Cp * sizeof(T), 128) / 128;
  return HGK_OK;
}

template <typename T>
static int gated_fwd(hipStream_t st, const void* x, const void* wg, const void* wu, void* h, long M,
                     int C, int F, int act, char* ws, int dtype) {
  constexpr int DT = TypeOf<T>::dt;
  if (gated_rows_ok(dtype, M, C, F, false)) return gated_rows_fwd(st, x, wg, wu, h, M, C, F, act);
  const GatedWs w = gated_ws(dtype, M, C, F, 0);
  GemmArgs a = gemm_args();
  if (int rc = gated_operands<T>(st, a, w, ws, x, wg, wu, M, C, F)) return rc;
  a.out = h;
  a.act = act;
  a.vec = F % 8 == 0;
  if (M <= skinny_rows<T>(true)) {
    run_skinny<DT, T, true>(st, a);
    HGK_LAUNCH_CHECK();
    return HGK_OK;
  }
  const GemmPlan p = plan_gemm(dtype == HGK_BF16 ? G_BF16 : G_F32, M, F, 2, a.spseg, 1, false);
  return run_tiles<DT, T, L_ROW, L_ROW, E_GATED>(st, a, p);
}

template <typename T>
static int gated_bwd(hipStream_t st, const void* x, const void* wg, const void* wu, const void* dh,
                     void* dx, void* dwg, void* dwu, long M, int C, int F, int act, char* ws,
                     int dtype, bool f32_wgrad) {
  constexpr int DT = TypeOf<T>::dt;
  constexpr int es = sizeof(T), ks = 128 / es;
  const GatedWs w = gated_ws(dtype, M, C, F, wanted_code(dx, dwg));
  GemmArgs a = gemm_args();
  if (int rc = gated_operands<T>(st, a, w, ws, x, wg, wu, M, C, F)) return rc;
  const char *xp = a.m0, *wgp = a.n0, *wup = a.n1;
  if (w.rows) {  // Fp is F, Cp is C
    if (int rc = gated_rows_bwd(st, x, wg, wu, dh, dwg ? ws + w.dg : nullptr, ws + w.du, dx, M, C, F, act)) return rc;
  } else {
    a.dh = dh;
    a.out = ws + w.dg;
    a.out1 = ws + w.du;
    a.npad = w.Fp;
    a.act = act;
    a.vec = F % 8 == 0;
    const GemmPlan p = plan_gemm(dtype == HGK_BF16 ? G_BF16 : G_F32, M, F, 2, a.spseg, 1, false);
    if (int rc = run_tiles<DT, T, L_ROW, L_ROW, E_GATED_BWD>(st, a, p)) return rc;
  }
  if (dx && !w.rows) {
    GemmArgs b = gemm_args();
    b.m0 = ws + w.dg;
    b.m1 = ws + w.du;
    b.ldm = (long)w.Fp * es;
    b.n0 = wgp;
    b.n1 = wup;
    b.ldn = (long)w.Cp * es;
    b.M = (int)M;
    b.N = C;
    b.km = w.Fp;
    b.kn = F;
    b.spseg = (F + ks - 1) / ks;
    b.nseg = 2;
    b.out = dx;
    b.vec = C % 8 == 0;
    if (int rc = run_product<DT, T, L_ROW, L_COL>(st, b, w.dx, ws + w.slab)) return rc;
  }
  if (dwg) {
    GemmArgs b = gemm_args();
    b.m0 = ws + w.dg;
    b.m1 = ws + w.du;
    b.ldm = (long)w.Fp * es;
    b.n0 = b.n1 = xp;
    b.ldn = (long)w.Cp * es;
    b.M = F;
    b.N = C;
    b.km = b.kn = (int)M;
    b.spseg = (int)((M + ks - 1) / ks);
    b.batch = 2;
    b.out = dwg;
    b.out1 = dwu;
    b.vec = C % 8 == 0;
    if (int rc = run_wgrad<DT, T>(st, b, w.dw, ws + w.slab, f32_wgrad)) return rc;
  }
  return HGK_OK;
}

// ---- linear with dropout and residual ----
struct LinearWs {
  long x, w, dz, slab, total;
  int Kp, Np;
  bool pad_k, pad_n, rows;
  GemmPlan fwd, dx, dw;
};
static LinearWs linear_ws(int dtype, long M, int K, int N, bool drop, int bwd) {
  LinearWs w;
  const int es = es_of(dtype), q = 16 / es, ks = 128 / es;
  w.Kp = (int)up_to(K, q);
  w.Np = (int)up_to(N, q);
  w.pad_k = w.Kp != K;
  w.pad_n = w.Np != N;
  Carve c;
  const Wanted want = wanted(bwd);
  w.x = w.w = w.dz = w.slab = 0;
  if (w.pad_k && (!bwd || want.dw)) w.x = c.take(M * w.Kp * es);
  if (w.pad_k && (!bwd || want.dx)) w.w = c.take((long)N * w.Kp * es);
  w.rows = false;
  w.fwd = plan_gemm(dtype == HGK_BF16 ? G_BF16 : G_F32, M, N, 1, (int)((w.Kp + ks - 1) / ks), 1, true);
  if (bwd) {
    w.rows = want.dx && linear_rows_ok(dtype, M, K, N, drop);
    // the row kernel stores dz for the weight gradient alone
    if ((drop || w.pad_n) && (!w.rows || want.dw)) w.dz = c.take(M * w.Np * es);
    w.dx = plan_gemm(dtype == HGK_BF16 ? G_BF16 : G_F32, M, K, 1, (N + ks - 1) / ks, 1, true);
    w.dw = plan_gemm(dtype == HGK_BF16 ? G_BF16 : G_F32, N, K, 1, (int)((M + ks - 1) / ks), 1, true);
    w.slab = c.take(std::max(want.dx && !w.rows ? w.dx.slab : 0, want.dw ? w.dw.slab : 0));
  } else {
    w.slab = c.take(M <= skinny_rows<float>(false) ? 0 : w.fwd.slab);  // the same for every type
  }
  w.total = c.at;
  return w;
}

template <typename T>
static int linear_fwd(hipStream_t st, const void* x, const void* wt, const void* res, void* y, long M,
                      int K, int N, const DropArgs& d, char* ws, int dtype) {
  constexpr int DT = TypeOf<T>::dt;
  typedef typename TypeOf<T>::raw raw;
  const LinearWs w = linear_ws(dtype, M, K, N, d.thr != 0, 0);
  if (w.pad_k) {
    Pads p;
    p.add(x, ws + w.x, M, K, w.Kp, sizeof(T));
    p.add(wt, ws + w.w, N, K, w.Kp, sizeof(T));
    if (int rc = p.launch<raw>(st)) return rc;
  }
  GemmArgs a = gemm_args();
  a.m0 = w.pad_k ? ws + w.x : (const char*)x;
  a.n0 = w.pad_k ? ws + w.w : (const char*)wt;
  a.ldm = a.ldn = (long)w.Kp * sizeof(T);
  a.M = (int)M;
  a.N = N;
  a.km = a.kn = w.Kp;
  a.spseg = (int)up_to((long)w.Kp * sizeof(T), 128) / 128;
  a.out = y;
  a.res = res;
  a.vec = N % 8 == 0;
  a.drop = d.thr != 0;
  a.d = d;
  if (M <= skinny_rows<T>(false)) {
    run_skinny<DT, T, false>(st, a);
    HGK_LAUNCH_CHECK();
    return HGK_OK;
  }
  return run_product<DT, T, L_ROW, L_ROW>(st, a, w.fwd, ws + w.slab);
}

template <typename T>
static int linear_bwd(hipStream_t st, const void* x, const void* wt, const void* dy, void* dx, void* dw,
                      long M, int K, int N, const DropArgs& d, char* ws, int dtype, bool f32_wgrad) {
  constexpr int DT = TypeOf<T>::dt;
  constexpr int es = sizeof(T), ks = 128 / es;
  typedef typename TypeOf<T>::raw raw;
  const bool drop = d.thr != 0;
  const LinearWs w = linear_ws(dtype, M, K, N, drop, wanted_code(dx, dw));
  const char *dz = (const char*)dy, *xp = (const char*)x, *wp = (const char*)wt;
  Pads p;
  if (w.rows) {  // nothing to pad
    void* z = drop && dw ? ws + w.dz : nullptr;
    if (int rc = linear_rows_bwd(st, dy, wt, z, dx, M, K, N, d)) return rc;
    if (z) dz = ws + w.dz;
  } else if (w.pad_n) {
    p.add(dy, ws + w.dz, M, N, w.Np, es, drop ? &d : nullptr);
    dz = ws + w.dz;
  } else if (drop) {
    if (int rc = dropout_mask(st, dtype, dy, ws + w.dz, M, N, d)) return rc;
    dz = ws + w.dz;
  }
  if (w.pad_k) {
    if (dw) p.add(x, ws + w.x, M, K, w.Kp, es);
    if (dx) p.add(wt, ws + w.w, N, K, w.Kp, es);
    xp = ws + w.x;
    wp = ws + w.w;
  }
  if (int rc = p.launch<raw>(st)) return rc;
  const float alpha = drop ? d.scale : 1.f;
  if (dx && !w.rows) {
    GemmArgs b = gemm_args();
    b.m0 = dz;
    b.ldm = (long)w.Np * es;
    b.n0 = wp;
    b.ldn = (long)w.Kp * es;
    b.M = (int)M;
    b.N = K;
    b.km = w.Np;
    b.kn = N;
    b.spseg = (N + ks - 1) / ks;
    b.out = dx;
    b.vec = K % 8 == 0;
    b.alpha = alpha;
    if (int rc = run_product<DT, T, L_ROW, L_COL>(st, b, w.dx, ws + w.slab)) return rc;
  }
  if (dw) {
    GemmArgs b = gemm_args();
    b.m0 = dz;
    b.ldm = (long)w.Np * es;
    b.n0 = xp;
    b.ldn = (long)w.Kp * es;
    b.M = N;
    b.N = K;
    b.km = b.kn = (int)M;
    b.spseg = (int)((M + ks - 1) / ks);
    b.out = dw;
    b.vec = K % 8 == 0;
    b.alpha = alpha;
    if (int rc = run_wgrad<DT, T>(st, b, w.dw, ws + w.slab, f32_wgrad)) return rc;
  }
  return HGK_OK;
}

static int zero_words(hipStream_t st, void* p, long words) {
  hipLaunchKernelGGL(zero_kernel, dim3((unsigned)std::min((words + 255) / 256, 1024l)), dim3(256), 0, st,
                     (uint32_t*)p, words);
  HGK_LAUNCH_CHECK();
  return HGK_OK;
}
template <typename T>
__global__ void zero_tail_kernel(T* p, long n0, long n) {
  if (n0 + threadIdx.x < n) p[n0 + threadIdx.x] = T{};
}
// a gradient over no rows at all
template <typename T>
static int zero_out(hipStream_t st, void* p, long n) {
  const long words = n * (long)sizeof(T) / 4;
  if (words)
    if (int rc = zero_words(st, p, words)) return rc;
  hipLaunchKernelGGL((zero_tail_kernel<T>), dim3(1), dim3(64), 0, st, (T*)p, words * 4 / (long)sizeof(T), n);
  HGK_LAUNCH_CHECK();
  return HGK_OK;
}

}  // namespace hgk

using namespace hgk;

extern "C" {

size_t hgk_gated_workspace(int dtype, long M, int C, int F, int backward) {
  dtype &= ~HGK_F32_WGRAD;
  if (M <= 0 || C <= 0 || F <= 0 || (dtype != HGK_F32 && dtype != HGK_BF16)) return 0;
  return (size_t)gated_ws(dtype, M, C, F, backward).total;
}

int hgk_gated_fwd(hgk_stream_t stream, int dtype, const void* x, const void* wg, const void* wu, void* h,
                  long M, int C, int F, int act, void* workspace, size_t ws_bytes) {
  HGK_CHECK_ROWS("gated", M, C, F);
  HGK_CHECK_ARG(act >= 0 && act < HGK_ACT_COUNT, "gated: unknown activation %d", act);
  if (M == 0) return HGK_OK;
  HGK_CHECK_ARG(x && wg && wu && h, "gated: null pointer");
  HGK_CHECK_ARG(al16(x) && al16(wg) && al16(wu) && al16(h) && al16(workspace),
                "gated: pointers must be 16-byte aligned");
  HGK_CHECK_WORKSPACE("gated", workspace, ws_bytes, hgk_gated_workspace(dtype, M, C, F, 0));
  HGK_DISPATCH_DTYPE(dtype, T, return gated_fwd<T>((hipStream_t)stream, x, wg, wu, h, M, C, F, act,
                                                   (char*)workspace, dtype));
}

int hgk_gated_bwd(hgk_stream_t stream, int dtype, const void* x, const void* wg, const void* wu,
                  const void* dh, void* dx, void* dwg, void* dwu, long M, int C, int F, int act,
                  void* workspace, size_t ws_bytes) {
  const bool f32_wgrad = dtype & HGK_F32_WGRAD;
  dtype &= ~HGK_F32_WGRAD;
  HGK_CHECK_ROWS("gated", M, C, F);
  HGK_CHECK_ARG(act >= 0 && act < HGK_ACT_COUNT, "gated: unknown activation %d", act);
  HGK_CHECK_ARG((dwg == nullptr) == (dwu == nullptr), "gated: both weight gradients or neither");
  if (M == 0) {
    if (!dwg) return HGK_OK;
    HGK_DISPATCH_DTYPE(f32_wgrad ? HGK_F32 : dtype, T, {
      if (int rc = zero_out<T>((hipStream_t)stream, dwg, (long)F * C)) return rc;
      return zero_out<T>((hipStream_t)stream, dwu, (long)F * C);
    });
  }
  HGK_CHECK_ARG(x && wg && wu && dh, "gated: null pointer");
  HGK_CHECK_ARG(al16(x) && al16(wg) && al16(wu) && al16(dh) && al16(dx) && al16(dwg) && al16(dwu) &&
                    al16(workspace), "gated: pointers must be 16-byte aligned");
  HGK_CHECK_WORKSPACE("gated", workspace, ws_bytes, hgk_gated_workspace(dtype, M, C, F, wanted_code(dx, dwg)));
  HGK_DISPATCH_DTYPE(dtype, T, return gated_bwd<T>((hipStream_t)stream, x, wg, wu, dh, dx, dwg, dwu, M, C,
                                                   F, act, (char*)workspace, dtype, f32_wgrad));
}

size_t hgk_linear_workspace(int dtype, long M, int K, int N, int dropout, int backward) {
  dtype &= ~HGK_F32_WGRAD;
  if (M <= 0 || K <= 0 || N <= 0 || (dtype != HGK_F32 && dtype != HGK_BF16)) return 0;
  return (size_t)linear_ws(dtype, M, K, N, dropout != 0, backward).total;
}

int hgk_linear_fwd(hgk_stream_t stream, int dtype, const void* x, const void* w, const void* res, void* y,
                   long M, int K, int N, double p, unsigned long long seed, unsigned long long offset,
                   const unsigned long long* step, void* workspace, size_t ws_bytes) {
  HGK_CHECK_ROWS("linear", M, K, N);
  HGK_CHECK_ARG(p >= 0.0 && p <= 1.0, "linear: p = %g is no probability", p);
  if (M == 0) return HGK_OK;
  HGK_CHECK_ARG(x && w && y, "linear: null pointer");
  HGK_CHECK_ARG(al16(x) && al16(w) && al16(res) && al16(y) && al16(workspace),
                "linear: pointers must be 16-byte aligned");
  const DropArgs d = make_drop(p, seed, offset, step);
  HGK_CHECK_WORKSPACE("linear", workspace, ws_bytes, hgk_linear_workspace(dtype, M, K, N, d.thr != 0, 0));
  HGK_DISPATCH_DTYPE(dtype, T, return linear_fwd<T>((hipStream_t)stream, x, w, res, y, M, K, N, d,
                                                    (char*)workspace, dtype));
}

int hgk_linear_bwd(hgk_stream_t stream, int dtype, const void* x, const void* w, const void* dy, void* dx,
                   void* dw, long M, int K, int N, double p, unsigned long long seed,
                   unsigned long long offset, const unsigned long long* step, void* workspace,
                   size_t ws_bytes) {
  const bool f32_wgrad = dtype & HGK_F32_WGRAD;
  dtype &= ~HGK_F32_WGRAD;
  HGK_CHECK_ROWS("linear", M, K, N);
  HGK_CHECK_ARG(p >= 0.0 && p <= 1.0, "linear: p = %g is no probability", p);
  if (M == 0) {
    if (!dw) return HGK_OK;
    HGK_DISPATCH_DTYPE(f32_wgrad ? HGK_F32 : dtype, T, return zero_out<T>((hipStream_t)stream, dw, (long)N * K));
  }
  HGK_CHECK_ARG(x && w && dy, "linear: null pointer");
  HGK_CHECK_ARG(al16(x) && al16(w) && al16(dy) && al16(dx) && al16(dw) && al16(workspace),
                "linear: pointers must be 16-byte aligned");
  const DropArgs d = make_drop(p, seed, offset, step);
  HGK_CHECK_WORKSPACE("linear", workspace, ws_bytes,
                      hgk_linear_workspace(dtype, M, K, N, d.thr != 0, wanted_code(dx, dw)));
  HGK_DISPATCH_DTYPE(dtype, T, return linear_bwd<T>((hipStream_t)stream, x, w, dy, dx, dw, M, K, N, d,
                                                    (char*)workspace, dtype, f32_wgrad));
}
}
