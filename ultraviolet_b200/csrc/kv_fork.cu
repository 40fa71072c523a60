// Cached positions of a row copied to other rows, every layer in one launch.
//
// What bounds it is writing the copies, in waves of ten blocks a multiprocessor, and in front of each block's writes the chain pairs -> pos,
// starts -> slots, which is all there is of a few short rows.  A block takes the keys or the values of
// one layer and head for four consecutive pairs; pairs with the same source (a group's, which stand next to each other) are written from one
// read, 16 bytes a thread and four of them in flight, while the last warp copies the scales.
// Measured on a B200: 4.1 us for 7 copies of 48 positions in 10 layers, 41.7 us for 32 prompts of 63 .. 700 tokens to 15 rows each (175 MB
// written: 4.2 TB/s).  8 pairs a block took 43.0 us and 6.2 (fewer blocks), 256 threads 45.7.
#include "common.cuh"

namespace uv {

constexpr int FORK_LAYERS = 32;
constexpr int FORK_THREADS = 128;
constexpr int FORK_PAIRS = 4;

struct ForkParams {
  uv_tree_layer layers[FORK_LAYERS];
  const int64_t *src, *dst;
  int64_t *pos, *starts;
  int* oob;
  int n, KH, hd, n_rows;
};

__global__ void __launch_bounds__(FORK_THREADS, 10) kv_fork_kernel(const __grid_constant__ ForkParams P) {
  __shared__ int64_t from_row[FORK_PAIRS], to_row[FORK_PAIRS];
  __shared__ int to[FORK_PAIRS];                                  // destination rows of the pairs in hand
  const int first = blockIdx.x * FORK_PAIRS, last = min(first + FORK_PAIRS, P.n), part = blockIdx.z & 1, h = blockIdx.z >> 1;
  const uv_tree_layer& y = P.layers[blockIdx.y];
  const bool lead = blockIdx.y == 0 && blockIdx.z == 0;                 // says what was skipped, moves pos and starts
  char* const codes = reinterpret_cast<char*>(part ? y.v_cache : y.k_cache);
  char* const scales = reinterpret_cast<char*>(part ? y.v_scale : y.k_scale);
  const int64_t row = (int64_t)P.KH * y.S_alloc;                  // slots of a cache row
  const bool of_scales = threadIdx.x >= FORK_THREADS - 32;
  const int tid = of_scales ? threadIdx.x - (FORK_THREADS - 32) : threadIdx.x, threads = of_scales ? 32 : FORK_THREADS - 32;
  if (threadIdx.x < FORK_PAIRS && first + (int)threadIdx.x < last)
    from_row[threadIdx.x] = P.src[first + threadIdx.x], to_row[threadIdx.x] = P.dst[first + threadIdx.x];
  __syncthreads();
#pragma unroll 1
  for (int i = first; i < last;) {
    const int64_t s = from_row[i - first];
    const bool ok = s >= 0 && s < P.n_rows;
    const int64_t pos = ok ? P.pos[s] : 0, start = ok ? P.starts[s] : 0;
    int m = 0;
    __syncthreads();
#pragma unroll 1
    for (; i < last && from_row[i - first] == s; ++i) {                      // the pairs from here on that have this source
      const int64_t d = to_row[i - first];
      if (!ok || d < 0 || d >= P.n_rows) {
        if (lead && threadIdx.x == 0 && P.oob) atomicAdd(P.oob, 1);
      } else if (d != s) {
        if (threadIdx.x == 0) {
          to[m] = (int)d;
          if (lead) P.pos[d] = pos, P.starts[d] = start;
        }
        ++m;
      }
    }
    __syncthreads();
    int64_t lo = start > 0 ? start : 0, hi = pos;
    if (y.ring) lo = hi - y.S > lo ? hi - y.S : lo;
    else hi = hi < y.S ? hi : y.S;
    if (m == 0 || hi <= lo) continue;
    // the slots lo .. hi - 1, of a ring in up to two pieces; of each piece the codes, and the scales in three parts: whole groups of 8
    // slots 16 bytes at a time, what stands before and behind them two.  The last warp takes the scales, the others the codes.
    const int64_t a = y.ring ? lo % y.S : lo, n = hi - lo, n1 = y.ring && a + n > y.S ? y.S - a : n;
    const int segments = (n1 < n ? 2 : 1) * (of_scales ? 3 : 1);
#pragma unroll 1
    for (int g = 0; g < segments; ++g) {
      const int piece = of_scales ? g / 3 : g, what = of_scales ? 1 + g % 3 : 0;
      const int64_t at = (int64_t)h * y.S_alloc + (piece ? 0 : a), len = piece ? n - n1 : n1;
      const int64_t head = min(len, -at & 7), body = (len - head) & ~(int64_t)7;
      const int64_t from = what < 2 ? at : what == 2 ? at + head : at + head + body;
      const int64_t slots = what == 0 ? len : what == 1 ? head : what == 2 ? body : len - head - body;
      if (slots == 0) continue;
      char* const base = what ? scales : codes;
      const int64_t unit = what ? 2 : P.hd, bytes = slots * unit, step = row * unit;
      char* const src = base + s * step + from * unit;
      const int64_t off = from * unit;
      const bool wide = ((reinterpret_cast<uintptr_t>(src) | (uintptr_t)bytes) & 15) == 0 && ((reinterpret_cast<uintptr_t>(base + off) | (uintptr_t)step) & 15) == 0;
      if (wide) {
        const int v = (int)(bytes / 16);                          // (a row of a layer holds less than 2^35 bytes)
#pragma unroll 1
        for (int x = tid; x < v; x += 4 * threads) {
          uint4 q[4];
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (x + k * threads < v) q[k] = reinterpret_cast<const uint4*>(src)[x + k * threads];
#pragma unroll 1
          for (int j = 0; j < m; ++j) {
            uint4* d = reinterpret_cast<uint4*>(base + to[j] * step + off);
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (x + k * threads < v) d[x + k * threads] = q[k];
          }
        }
      } else {
#pragma unroll 1
        for (int64_t x = tid; x < bytes / 2; x += threads) {
          const uint16_t q = reinterpret_cast<const uint16_t*>(src)[x];
          for (int j = 0; j < m; ++j) reinterpret_cast<uint16_t*>(base + to[j] * step + off)[x] = q;
        }
      }
    }
  }
}

}  // namespace uv

extern "C" int uv_kv_fork(const uv_tree_layer* h_layers, int n_layers, int KH, int hd, int n_rows, const int64_t* src,
                          const int64_t* dst, int n, int64_t* pos, int64_t* starts, int* oob_count, void* stream) {
  using namespace uv;
  if (n == 0) return UV_OK;
  if (!h_layers || !src || !dst || !pos || !starts || n < 0 || n_layers < 1 || KH < 1 || hd < 1 || n_rows < 0) return UV_ERR_ARG;
  if (n_layers > FORK_LAYERS || KH > 32767 || hd & 1) return UV_ERR_SHAPE;
  ForkParams P{};
  P.src = src, P.dst = dst, P.pos = pos, P.starts = starts, P.oob = oob_count;
  P.n = n, P.KH = KH, P.hd = hd, P.n_rows = n_rows;
  for (int l = 0; l < n_layers; ++l) {
    uv_tree_layer& y = P.layers[l];
    y = h_layers[l];
    if (y.S_alloc == 0) y.S_alloc = y.S;
    if (!y.k_cache || !y.v_cache || !y.k_scale || !y.v_scale || y.S < 1 || y.S_alloc < y.S) return UV_ERR_ARG;
    if ((reinterpret_cast<uintptr_t>(y.k_cache) | reinterpret_cast<uintptr_t>(y.v_cache)) & 1) return UV_ERR_ALIGN;
  }
  kv_fork_kernel<<<dim3((n + FORK_PAIRS - 1) / FORK_PAIRS, n_layers, 2 * KH), FORK_THREADS, 0, static_cast<cudaStream_t>(stream)>>>(P);
  return check_launch();
}
