// Trees of drafted tokens as the tree kernels read them: parents of up to 64 nodes, and the ancestor set of every node.
#pragma once

#include "common.cuh"

namespace uv {

constexpr int TREE_MAX = 64;

// multiprocessors of the current device, as the rules for grids and parts count them
inline int sm_count() {
  int dev = 0, n = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  return n;
}

// The cache's code of an fp16 or bf16 element: clamp(rint(x / s), -127, 127) with the IEEE quotient and ties to even, s an fp16 value or
// 1e-30, inv within 2^-21 of 1 / s.  Without the division: x and s have at most 11 significant bits, so a quotient between 1/2 and
// 127 that is not halfway between two codes is at least 2^-13 away from it, more than x * inv is off; and halfway is where the
// remainder x - q * s, which one fma gives exactly, is s / 2.
__device__ __forceinline__ float cache_code(float x, float s, float inv) {
  float q = fminf(fmaxf(rintf(x * inv), -127.0f), 127.0f);
  const float rest = fmaf(-q, s, x);
  if (fabsf(rest) * 2.0f == s && ((int)q & 1)) q += rest > 0.f ? 1.0f : -1.0f;
  return fminf(fmaxf(q, -127.0f), 127.0f);
}

// Ancestors of every node, itself included, as a bit mask in shared memory; 0 for a node that is absent (a parent that is neither
// -1 nor an earlier node, or an absent ancestor).  The depth of a present node is popcount(mask) - 1.  Called by one full warp; parents
// are those of one tree.  A node's set is its own bit and its parent's set: the sets double their reach in each of
// log2(64) rounds, since after round r every node knows its 2^r nearest ancestors and the one behind them.
struct TreeSets {
  uint64_t mask[TREE_MAX];
  int up[TREE_MAX];
};
__device__ __forceinline__ void tree_sets(const int32_t* parents, int T, TreeSets& s, int lane) {
  uint64_t m[2];
  int up[2];
  bool bad[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int i = lane + 32 * e;
    const int p = i < T ? parents[i] : -2;
    const bool child = p >= 0 && p < i;
    bad[e] = !child && p != -1;
    up[e] = child ? p : i;
    m[e] = 1ull << i;
  }
#pragma unroll 1
  for (int round = 0; round < 6; ++round) {
#pragma unroll
    for (int e = 0; e < 2; ++e) s.mask[lane + 32 * e] = bad[e] ? 0ull : m[e], s.up[lane + 32 * e] = up[e];
    __syncwarp();
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const uint64_t a = s.mask[up[e]];
      bad[e] = bad[e] || a == 0ull;
      m[e] |= a;
      up[e] = s.up[up[e]];
    }
    __syncwarp();
  }
#pragma unroll
  for (int e = 0; e < 2; ++e) s.mask[lane + 32 * e] = bad[e] ? 0ull : m[e];
  __syncwarp();
}

}  // namespace uv
