// Counter-based random words (Philox4x32-10: Salmon, Moraes, Dror, Shaw, "Parallel random numbers:
// as easy as 1, 2, 3", 2011) and the dropout mask made of them.
//
// Element (r, c) of a [rows][C] tensor takes 16-bit word c % 8 of the block at counter
// (gid lo, gid hi, offset lo, offset hi), gid = (r / rows_per_mask) * ceil(C / 8) + c / 8, under
// the key (seed lo, seed hi); word 2 j + b is bits [16 b, 16 b + 16) of output j. It is kept iff
// word >= thr, thr = floor(65536 p + 1/2), and what is kept is scaled by 65536 / (65536 - thr): the
// mean is exact for the probability that is in fact drawn (p to the nearest 2^-16). 16 bits an
// element, not 32: ten rounds are 20 wide multiplies at a quarter of the VALU's rate, and with 4
// elements a block they, not the memory, would bound a bf16 pass. The mask depends on nothing but
// (seed, offset, r, c): any launch shape, the fused epilogue and the backward draw the same one.
#pragma once
#include "hgk_common.h"

namespace hgk {

__device__ __forceinline__ uint4 philox4x32_10(uint4 c, uint32_t k0, uint32_t k1) {
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const uint64_t a = (uint64_t)c.x * 0xD2511F53u, b = (uint64_t)c.z * 0xCD9E8D57u;
    c = make_uint4((uint32_t)(b >> 32) ^ c.y ^ k0, (uint32_t)b, (uint32_t)(a >> 32) ^ c.w ^ k1,
                   (uint32_t)a);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return c;
}

// a launch holds less than 2^32 threads
#define HGK_CHECK_THREADS(what, workgroups, threads) \
  HGK_CHECK_ARG((workgroups) < (1l << 32) / (threads), what ": too many workgroups (%ld of %d threads)", (long)(workgroups), (int)(threads))

struct DropArgs {
  uint32_t thr;  // 0 .. 65536; 0: everything kept
  float scale;   // 65536 / (65536 - thr); 0 at thr = 65536
  uint64_t seed, offset;
  const unsigned long long* step;  // nullable device counter added to `offset`
};

__device__ __forceinline__ uint64_t drop_offset(const DropArgs& d) {
  return d.offset + (d.step ? *d.step : 0ull);
}

// bit e: element e of the 8-channel group is kept
__device__ __forceinline__ uint32_t drop_mask8(uint64_t gid, uint64_t off, uint64_t seed,
                                               uint32_t thr) {
  const uint4 w = philox4x32_10(make_uint4((uint32_t)gid, (uint32_t)(gid >> 32), (uint32_t)off,
                                           (uint32_t)(off >> 32)),
                                (uint32_t)seed, (uint32_t)(seed >> 32));
  const uint32_t v[4] = {w.x, w.y, w.z, w.w};
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    m |= ((v[j] & 0xffffu) >= thr ? 1u : 0u) << (2 * j);
    m |= ((v[j] >> 16) >= thr ? 1u : 0u) << (2 * j + 1);
  }
  return m;
}

// host: the mask's parameters from a probability in [0, 1]
inline DropArgs make_drop(double p, unsigned long long seed, unsigned long long offset,
                          const unsigned long long* step) {
  DropArgs d;
  d.thr = (uint32_t)(p * 65536.0 + 0.5);
  d.scale = d.thr < 65536u ? (float)(65536.0 / (65536.0 - d.thr)) : 0.f;
  d.seed = seed;
  d.offset = offset;
  d.step = step;
  return d;
}

}  // namespace hgk
