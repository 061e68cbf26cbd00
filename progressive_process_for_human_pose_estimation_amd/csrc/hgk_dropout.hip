// Dropout with the skip added in the same pass, from a counter-based generator (hgk_philox.h): the
// mask is never stored, the backward draws it again.
//   y[r][c] = (kept(r, c) ? x[r][c] * scale : 0) (+ res[r][c])
// One pass: x and res read once, y written once. What is dropped is selected away, not multiplied
// by zero (an infinity or NaN in a dropped place does not reach y).
// y may be x or res: no kernel says that they are apart, and each thread reads an element before it writes it.
#include <algorithm>

#include "hgk_philox.h"

namespace hgk {

struct DropoutArgs {
  const void* x;
  const void* res;
  void* y;
  long rows;
  int C, groups;      // groups = ceil(C / 8)
  long rows_per_mask;
  DropArgs d;
};

// C % 8 == 0, 16-B aligned: a thread owns one 8-channel group of `R` consecutive rows, so that one
// block of random words serves every row of a shared mask row (whole-channel dropout).
template <typename T, int R>
__global__ __launch_bounds__(256) void dropout_vec_kernel(DropoutArgs a) {
  constexpr int V = Vec16<T>::N, NV = 8 / V;
  const long t = (long)blockIdx.x * 256 + threadIdx.x;
  const long r0 = (t / a.groups) * R;
  const int g = (int)(t % a.groups);
  if (r0 >= a.rows) return;
  const uint64_t off = drop_offset(a.d);
  const T* x = (const T*)a.x;
  const T* res = (const T*)a.res;
  T* y = (T*)a.y;
  typename Vec16<T>::type xv[R][NV], rv[R][NV];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const long r = min(r0 + i, a.rows - 1);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      xv[i][j] = load16(x + r * a.C + g * 8 + j * V);
      if (res) rv[i][j] = load16(res + r * a.C + g * 8 + j * V);
    }
  }
  long have = -1;
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const long r = r0 + i;
    if (r >= a.rows) break;
    const long mr = a.rows_per_mask == 1 ? r : r / a.rows_per_mask;
    if (mr != have) {
      m = drop_mask8((uint64_t)mr * a.groups + g, off, a.d.seed, a.d.thr);
      have = mr;
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      float f[V], q[V];
      unpack16<T>(xv[i][j], f);
      if (res) unpack16<T>(rv[i][j], q);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        f[e] = (m >> (j * V + e)) & 1u ? f[e] * a.d.scale : 0.f;
        if (res) f[e] += q[e];
      }
      store16(y + r * a.C + g * 8 + j * V, pack16<T>(f));
    }
  }
}

// Any C: a workgroup owns RB whole rows (a contiguous run of RB * C elements that starts on a 16-B
// border, RB a multiple of 8), puts the mask bytes of its groups into LDS, then walks the run
// element by element in order: coalesced whatever the row length.
static constexpr int kDropLds = 8192;  // mask bytes of a workgroup

template <typename T, bool ALIGNED>
__global__ __launch_bounds__(256) void dropout_flat_kernel(DropoutArgs a, int RB) {
  constexpr int V = ALIGNED ? Vec16<T>::N : 1;
  __shared__ uint8_t mask[kDropLds];
  const long r0 = (long)blockIdx.x * RB;
  const int nr = (int)min((long)RB, a.rows - r0);
  const uint64_t off = drop_offset(a.d);
  const long mr0 = r0 / a.rows_per_mask, mr1 = (r0 + nr - 1) / a.rows_per_mask;
  const int nm = (int)(mr1 - mr0 + 1) * a.groups;
  for (int i = threadIdx.x; i < nm; i += 256)
    mask[i] = (uint8_t)drop_mask8((uint64_t)mr0 * a.groups + i, off, a.d.seed, a.d.thr);
  __syncthreads();
  const T* x = (const T*)a.x + r0 * a.C;
  const T* res = a.res ? (const T*)a.res + r0 * a.C : nullptr;
  T* y = (T*)a.y + r0 * a.C;
  const int n = nr * a.C;  // RB * C <= 2^24 (host)
  auto one = [&](float f, float q, int row, int col) __attribute__((always_inline)) {
    const int mi = a.rows_per_mask == 1 ? row : (int)((r0 + row) / a.rows_per_mask - mr0);
    const bool k = (mask[mi * a.groups + (col >> 3)] >> (col & 7)) & 1;
    f = k ? f * a.d.scale : 0.f;
    return res ? f + q : f;
  };
  for (int i = threadIdx.x * V; i < n; i += 256 * V) {
    int row = i / a.C, col = i - row * a.C;
    if (V > 1 && i + V <= n) {
      float f[8], q[8];
      unpack16<T>(load16(x + i), f);
      if (res) unpack16<T>(load16(res + i), q);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        f[e] = one(f[e], res ? q[e] : 0.f, row, col);
        if (++col == a.C) {
          col = 0;
          ++row;
        }
      }
      store16(y + i, pack16<T>(f));
    } else {
      for (int e = 0; e < V && i + e < n; ++e) {
        y[i + e] = from_f<T>(one(to_f(x[i + e]), res ? to_f(res[i + e]) : 0.f, row, col));
        if (++col == a.C) {
          col = 0;
          ++row;
        }
      }
    }
  }
}

// Runs of 8 rows whose masks are more than kDropLds bytes (C > 8192, off the 16-byte borders): one group of
// one row a thread, element by element
template <typename T>
__global__ __launch_bounds__(256) void dropout_long_kernel(DropoutArgs a) {
  const long t = (long)blockIdx.x * 256 + threadIdx.x;
  const long r = t / a.groups;
  const int g = (int)(t % a.groups);
  if (r >= a.rows) return;
  const uint32_t m = drop_mask8((uint64_t)(r / a.rows_per_mask) * a.groups + g, drop_offset(a.d),
                                a.d.seed, a.d.thr);
  const T* x = (const T*)a.x;
  const T* res = (const T*)a.res;
  T* y = (T*)a.y;
  for (int e = 0; e < 8 && g * 8 + e < a.C; ++e) {
    const long i = r * a.C + g * 8 + e;
    float f = (m >> e) & 1u ? to_f(x[i]) * a.d.scale : 0.f;
    if (res) f += to_f(res[i]);
    y[i] = from_f<T>(f);
  }
}

static inline bool al16(const void* p) { return ((uintptr_t)p & 15) == 0; }

template <typename T>
static int launch_dropout(hipStream_t st, const DropoutArgs& a) {
  const bool al = al16(a.x) && al16(a.res) && al16(a.y);
  HGK_CHECK_ARG(a.rows < (1l << 62) / a.groups, "dropout: too many rows (%ld)", a.rows);
  if (a.C % 8 == 0 && al) {
    if (a.rows_per_mask > 1) {
      const long n = ((a.rows + 3) / 4) * a.groups;
      HGK_CHECK_THREADS("dropout", (n + 255) / 256, 256);
      hipLaunchKernelGGL((dropout_vec_kernel<T, 4>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, a);
    } else {
      const long n = a.rows * a.groups;
      HGK_CHECK_THREADS("dropout", (n + 255) / 256, 256);
      hipLaunchKernelGGL((dropout_vec_kernel<T, 1>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, a);
    }
  } else if (a.groups * 8 <= kDropLds) {
    // RB rows: a multiple of 8, about 8192 elements a workgroup, mask bytes within the LDS
    int RB = 8 * std::max(1, std::min(kDropLds / (8 * a.groups), 8192 / (8 * a.C)));
    const long nb = (a.rows + RB - 1) / RB;
    HGK_CHECK_THREADS("dropout", nb, 256);
    if (al)
      hipLaunchKernelGGL((dropout_flat_kernel<T, true>), dim3((unsigned)nb), dim3(256), 0, st, a, RB);
    else
      hipLaunchKernelGGL((dropout_flat_kernel<T, false>), dim3((unsigned)nb), dim3(256), 0, st, a, RB);
  } else {
    const long n = a.rows * a.groups;
    HGK_CHECK_THREADS("dropout", (n + 255) / 256, 256);
    hipLaunchKernelGGL((dropout_long_kernel<T>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, a);
  }
  HGK_LAUNCH_CHECK();
  return HGK_OK;
}

// dz = kept ? dy : 0, unscaled (the linear's backward, hgk_ffn.hip)
int dropout_mask(hipStream_t st, int dtype, const void* dy, void* dz, long rows, int C, const DropArgs& d) {
  DropoutArgs a;
  a.x = dy;
  a.res = nullptr;
  a.y = dz;
  a.rows = rows;
  a.C = C;
  a.groups = (C + 7) / 8;
  a.rows_per_mask = 1;
  a.d = d;
  a.d.scale = 1.f;
  HGK_DISPATCH_DTYPE(dtype, T, return launch_dropout<T>(st, a));
}

}  // namespace hgk

using namespace hgk;

extern "C" unsigned long long hgk_capture_id(hgk_stream_t stream) {
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  unsigned long long id = 0;
  if (hipStreamGetCaptureInfo((hipStream_t)stream, &status, &id) != hipSuccess) return 0;
  return status == hipStreamCaptureStatusActive ? id : 0;
}

extern "C" int hgk_dropout_add(hgk_stream_t stream, int dtype, const void* x, const void* res, void* y,
                               long rows, int C, long rows_per_mask, double p,
                               unsigned long long seed, unsigned long long offset,
                               const unsigned long long* step) {
  HGK_CHECK_ARG(rows >= 0 && C >= 1 && C <= (1 << 30), "dropout: bad sizes (%ld rows, %d channels)", rows, C);
  HGK_CHECK_ARG(p >= 0.0 && p <= 1.0, "dropout: p = %g is no probability", p);
  HGK_CHECK_ARG(rows_per_mask >= 1, "dropout: rows_per_mask = %ld", rows_per_mask);
  if (rows == 0) return HGK_OK;
  HGK_CHECK_ARG(x && y, "dropout: null pointer");
  DropoutArgs a;
  a.x = x;
  a.res = res;
  a.y = y;
  a.rows = rows;
  a.C = C;
  a.groups = (C + 7) / 8;
  a.rows_per_mask = rows_per_mask;
  a.d = make_drop(p, seed, offset, step);
  HGK_DISPATCH_DTYPE(dtype, T, return launch_dropout<T>((hipStream_t)stream, a));
}
