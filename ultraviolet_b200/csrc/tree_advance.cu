// Positions of a tree's nodes, and the end of a step: the accepted path of every tree and its keys and values appended to the
// caches of all layers.
#include "common.cuh"
#include "tree.cuh"

namespace uv {

__global__ void __launch_bounds__(128) tree_positions_kernel(const int32_t* parents, int64_t stride, const int64_t* pos, int B, int T,
                                                             int64_t* out) {
  __shared__ TreeSets sets[4];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, b = blockIdx.x * 4 + warp;
  if (b >= B) return;
  tree_sets(parents + b * stride, T, sets[warp], lane);
  for (int i = lane; i < T; i += 32) {
    const uint64_t m = sets[warp].mask[i];
    out[(int64_t)b * T + i] = pos[b] + (m ? __popcll(m) - 1 : 0);
  }
}

constexpr int ADV_LAYERS = 32;
constexpr int ADV_WARPS = 8;

struct AdvanceParams {
  uv_tree_advance_args a;
  uv_tree_layer layers[ADV_LAYERS];
};

// The walk, by a full warp: lane l learns which node comes l-th (a) and (l + 32)-th (b) on the accepted path; returns how many.
__device__ __forceinline__ int tree_walk(const int32_t* parents, const int64_t* tokens, const int64_t* target, int T, int lane,
                                         int& at_a, int& at_b) {
  int par[2];
  int64_t tok[2], tgt[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int i = lane + 32 * e;
    par[e] = i < T ? parents[i] : -2;
    tok[e] = i < T ? tokens[i] : 0;
    tgt[e] = i < T ? target[i] : 0;
  }
  at_a = at_b = -1;
  auto first = [&](bool lo, bool hi) {
    const unsigned m0 = __ballot_sync(0xffffffffu, lo), m1 = __ballot_sync(0xffffffffu, hi);
    return m0 ? __ffs((int)m0) - 1 : m1 ? 31 + __ffs((int)m1) : -1;
  };
  int cur = first(par[0] == -1, par[1] == -1), n = 0;
  while (cur >= 0 && n < TREE_MAX) {
    if (n < 32) at_a = lane == n ? cur : at_a;
    else at_b = lane == n - 32 ? cur : at_b;
    ++n;
    const int64_t want = __shfl_sync(0xffffffffu, cur < 32 ? tgt[0] : tgt[1], cur & 31);
    cur = first(par[0] == cur && lane > cur && tok[0] == want, par[1] == cur && lane + 32 > cur && tok[1] == want);
  }
  return n;
}

// A block per tree.  Every warp walks the tree for itself (a few ballots), then a group of HD / 8 lanes takes a vector, 8 elements a
// lane: the accepted nodes' keys and values of all layers are far apart in memory and few, so what bounds it is latency: the chain pos,
// parents, tokens -> vectors -> codes, and, with two vectors a group in flight, a round of loads for every 64 vectors of 64 elements.
// Measured on a B200: 3.1 us for one tree of 4 nodes in 10 layers, 11.7 us for 256 trees of 16 nodes, whose paths of nine make 180 vectors
// (three rounds; two blocks on most SMs, a quarter of the issue slots used).  Four blocks to a tree took 12.7 us, a layer to each of 16 warps 12.4 (and 4.8 for the one tree).
template <typename T, int HD>
__global__ void __launch_bounds__(ADV_WARPS * 32) tree_advance_kernel(const __grid_constant__ AdvanceParams P) {
  constexpr int LV = HD / 8, GROUPS = ADV_WARPS * 32 / LV;
  const uv_tree_advance_args& a = P.a;
  const int b = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, group = threadIdx.x / LV, part = threadIdx.x % LV;
  __shared__ int way[TREE_MAX];
  int at[2];
  const int64_t pos = a.pos[b], row = a.row_map ? a.row_map[b] : b;
  const int64_t* target = a.target + (int64_t)b * a.T;
  const int n = tree_walk(a.parents + b * a.parents_stride, a.tokens + (int64_t)b * a.T, target, a.T, lane, at[0], at[1]);
  if (warp == 0) way[lane] = at[0], way[lane + 32] = at[1];
  __syncthreads();                          // the path is there, and every warp has read pos before it moves
  if (warp == 1) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int j = lane + 32 * e;
      if (j >= a.T) continue;
      a.path[(int64_t)b * a.T + j] = at[e];
      a.drawn[(int64_t)b * a.T + j] = at[e] >= 0 ? target[at[e]] : -1;
    }
    if (lane == 0) a.count[b] = n, a.pos_out[b] = pos + n;
  }
  const bool bad_row = row < 0 || row >= a.n_rows;
  const int per = 2 * a.KH, items = n * a.n_layers * per;
  // (whole warps stay in the loop: the groups of a warp share its shuffles)
#pragma unroll 2
  for (int i0 = 0; i0 < items; i0 += GROUPS) {
    const int it = i0 + group;
    const bool live = it < items;
    const int j = live ? it / (per * a.n_layers) : 0, l = live ? it / per % a.n_layers : 0, kv = live ? it % per : 0;
    const int which = kv >= a.KH, kh = which ? kv - a.KH : kv, node = way[j];
    const uv_tree_layer& y = P.layers[l];
    uint4 raw = make_uint4(0u, 0u, 0u, 0u);
    if (live) {
      const T* x = which ? static_cast<const T*>(y.v) + b * a.svb + node * a.svt + kh * a.svh
                         : static_cast<const T*>(y.k) + b * a.skb + node * a.skt + kh * a.skh;
      raw = reinterpret_cast<const uint4*>(x)[part];
    }
    const T* x = reinterpret_cast<const T*>(&raw);
    float amax = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) amax = fmaxf(amax, fabsf(to_f32<T>(x[e])));
#pragma unroll
    for (int o = LV / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    const __half s16 = __float2half_rn(__fdiv_rn(amax, 127.0f));
    const float sf = fmaxf(__half2float(s16), 1e-30f), inv = __frcp_rn(sf);
    uint32_t w[2] = {0u, 0u};
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e / 4] |= (uint32_t)(__float2int_rn(cache_code(to_f32<T>(x[e]), sf, inv)) & 0xff) << (8 * (e & 3));
    int64_t p = pos + j;
    if (y.ring) {
      if (!live || j + y.S < n) continue;
      p = ((p % y.S) + y.S) % y.S;
    }
    if (!live) continue;
    if (p < 0 || p >= y.S || bad_row) {
      if (part == 0 && a.oob_count) atomicAdd(a.oob_count, 1);
      continue;
    }
    const int64_t dst = (row * a.KH + kh) * y.S_alloc + p;
    reinterpret_cast<uint2*>((which ? y.v_cache : y.k_cache) + dst * HD)[part] = make_uint2(w[0], w[1]);
    if (part == 0) (which ? y.v_scale : y.k_scale)[dst] = __half_as_ushort(s16);
  }
}

template <typename T>
static int launch_advance(const AdvanceParams& P, cudaStream_t st) {
  switch (P.a.hd) {
    case 16: tree_advance_kernel<T, 16><<<P.a.B, ADV_WARPS * 32, 0, st>>>(P); break;
    case 32: tree_advance_kernel<T, 32><<<P.a.B, ADV_WARPS * 32, 0, st>>>(P); break;
    case 64: tree_advance_kernel<T, 64><<<P.a.B, ADV_WARPS * 32, 0, st>>>(P); break;
    case 128: tree_advance_kernel<T, 128><<<P.a.B, ADV_WARPS * 32, 0, st>>>(P); break;
    default: return UV_ERR_SHAPE;
  }
  return check_launch();
}

static bool layers_ok(const uv_tree_layer* y, int n, bool nodes) {
  for (int l = 0; l < n; ++l)
    if ((nodes && (!y[l].k || !y[l].v)) || !y[l].k_cache || !y[l].v_cache || !y[l].k_scale || !y[l].v_scale || y[l].S < 1 ||
        (y[l].S_alloc != 0 && y[l].S_alloc < y[l].S))
      return false;
  return true;
}

}  // namespace uv

extern "C" int uv_tree_positions(const int32_t* parents, int64_t parents_stride, const int64_t* pos, int B, int T, int64_t* out,
                                 void* stream) {
  using namespace uv;
  if (B == 0 || T == 0) return UV_OK;
  if (!parents || !pos || !out || B < 0 || T < 0) return UV_ERR_ARG;
  if (T > TREE_MAX) return UV_ERR_SHAPE;
  tree_positions_kernel<<<(B + 3) / 4, 128, 0, static_cast<cudaStream_t>(stream)>>>(parents, parents_stride, pos, B, T, out);
  return check_launch();
}

extern "C" int uv_tree_advance(const uv_tree_advance_args* a, void* stream) {
  using namespace uv;
  if (!a) return UV_ERR_ARG;
  if (a->B == 0) return UV_OK;
  if (!a->parents || !a->tokens || !a->target || !a->pos || !a->path || !a->count || !a->drawn || !a->pos_out || !a->h_layers ||
      a->B < 0 || a->T < 1 || a->KH < 1 || a->n_layers < 1 || a->n_rows < 0)
    return UV_ERR_ARG;
  if (a->dtype != UV_F16 && a->dtype != UV_BF16) return UV_ERR_DTYPE;
  if (a->T > TREE_MAX || a->n_layers > ADV_LAYERS) return UV_ERR_SHAPE;
  if (!layers_ok(a->h_layers, a->n_layers, true)) return UV_ERR_ARG;
  // vectors are read 16 bytes at a time and written 8
  bool aligned = ((a->skb | a->skt | a->skh | a->svb | a->svt | a->svh) & 7) == 0;
  for (int l = 0; l < a->n_layers; ++l) {
    const uv_tree_layer& y = a->h_layers[l];
    aligned = aligned && aligned16(y.k) && aligned16(y.v) &&
              ((reinterpret_cast<uintptr_t>(y.k_cache) | reinterpret_cast<uintptr_t>(y.v_cache)) & 7) == 0;
  }
  if (!aligned) return UV_ERR_ALIGN;
  AdvanceParams P{*a, {}};
  for (int l = 0; l < a->n_layers; ++l) {
    P.layers[l] = a->h_layers[l];
    if (P.layers[l].S_alloc == 0) P.layers[l].S_alloc = P.layers[l].S;
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return a->dtype == UV_F16 ? launch_advance<__half>(P, st) : launch_advance<__nv_bfloat16>(P, st);
}
