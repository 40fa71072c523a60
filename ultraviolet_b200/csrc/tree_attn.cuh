// What the two tree-attention kernels share: parameters, the range of cached positions of a row, the epilogue of a query row.
#pragma once

#include "attn_math.cuh"
#include "common.cuh"
#include "tcgen05.cuh"
#include "tree.cuh"

namespace uv {

struct TreeParams {
  uv_tree_attn_args a;
  int G, M;          // query heads of a kv head; rows of a kv head
  uint32_t g_inv;    // ceil(2^32 / G), 0 for G = 1
  int splits;        // parts of a row's keys
  int cluster;       // the parts form a cluster and merge through distributed shared memory; else through ws
  float scale_log2;
  float *ws_o, *ws_m, *ws_l;
};

// row / G: exact below 2^16 rows (a kv head has at most 1024), where row times what g_inv is too large by stays below 2^32
__device__ __forceinline__ int node_of(const TreeParams& P, int row) { return P.g_inv ? (int)__umulhi((unsigned)row, P.g_inv) : row; }

__device__ __forceinline__ void bulk_copy(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}
__device__ __forceinline__ void mbar_arrive_one(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ float peer_f32(uint32_t local_addr, uint32_t rank) {
  uint32_t remote;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local_addr), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(remote) : "memory");
  return v;
}
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// ---- what every part of a row needs to know: its cache row, the positions that any of its nodes sees
struct RowRange {
  int64_t pos, lo, hi, row;   // cached positions lo .. hi (inclusive, empty when hi < lo), cache row
};
__device__ __forceinline__ RowRange row_range(const uv_tree_attn_args& a, int b) {
  RowRange r;
  r.pos = a.pos[b], r.lo = a.starts[b] > 0 ? a.starts[b] : 0, r.hi = r.pos - 1;
  if (a.window > 0 && r.pos - a.window + 1 > r.lo) r.lo = r.pos - a.window + 1;
  if (a.ring) r.lo = r.pos - a.S > r.lo ? r.pos - a.S : r.lo;
  else r.hi = r.hi < a.S - 1 ? r.hi : a.S - 1;
  r.row = a.row_map ? a.row_map[b] : b;
  if (r.row < 0 || r.row >= a.n_rows) r.row = 0, r.hi = r.lo - 1;
  return r;
}

// ---- 1 / sum of a row's weights.  A present node sees itself at least, so its sum is positive unless its query is not finite or a
//      scale that it sees is no number: then there is no softmax, and NaN says so.
__device__ __forceinline__ float inverse_sum(float sum) { return sum > 0.f ? 1.0f / sum : __int_as_float(0x7fffffff); }
// a part's sum in a merge, weighted: one without a reference has seen no score that is a number, and its sum is 0 or NaN
__device__ __forceinline__ float part_sum(float m, float weight, float sum) { return m == -INFINITY ? sum : weight * sum; }

// ---- epilogue of one query row held by a warp (lane owns dims lane + 32 i), and its store
template <typename QT, int HD>
__device__ __forceinline__ void store_row(const TreeParams& P, float (&z)[(HD + 31) / 32], int b, int kh, int row, bool present,
                                          int lane) {
  constexpr int EPL = (HD + 31) / 32;
  const uv_tree_attn_args& a = P.a;
  const int t = node_of(P, row), h = kh * P.G + row - t * P.G;
  const bool act = HD >= 32 || lane < HD;
#pragma unroll
  for (int i = 0; i < EPL; ++i) z[i] = rnd<QT>(z[i]);
  if (a.xsa_alpha) {
    const QT* v = static_cast<const QT*>(a.v) + (int64_t)b * a.snvb + (int64_t)t * a.snvt + (int64_t)kh * a.snvh;
    float vv[EPL], n2 = 0.f, dot = 0.f;
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      vv[i] = act ? to_f32<QT>(v[lane + 32 * i]) : 0.f;
      n2 += vv[i] * vv[i];
    }
    const float inv = 1.0f / fmaxf(sqrtf(warp_sum(n2)), a.xsa_eps);
#pragma unroll
    for (int i = 0; i < EPL; ++i) vv[i] *= inv, dot += z[i] * vv[i];
    dot = warp_sum(dot);
    const float al = a.xsa_alpha[h];
#pragma unroll
    for (int i = 0; i < EPL; ++i) z[i] = rnd<QT>(z[i] - al * dot * vv[i]);
  }
  const float gate = a.gate_vals ? a.gate_vals[((int64_t)b * a.T + t) * a.H + h] : 1.0f;
  QT* out = static_cast<QT*>(a.out) + (int64_t)b * a.sob + (int64_t)t * a.sot + (int64_t)h * a.soh;
#pragma unroll
  for (int i = 0; i < EPL; ++i)
    if (act) out[lane + 32 * i] = from_f32<QT>(present ? z[i] * gate : 0.f);
}

// tree_attn_tc.cu: many query rows, on the tcgen05 tensor cores
bool tree_tc_wants(const uv_tree_attn_args& a);
size_t tree_tc_workspace(const uv_tree_attn_args& a);
int launch_tree_tc(const TreeParams& P, cudaStream_t st);

}  // namespace uv
