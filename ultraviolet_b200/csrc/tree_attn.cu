// Attention of a tree of drafted tokens to the int8 cache of its row and to its own ancestors.
//
//   o_i = sum_t softmax_t(scale * q_i . K_t) V_t over the cached positions that node i sees and its ancestors j <= i,
//   K_t = codes * scale (cached), K_j = quantised node key: the numbers the cache will hold.
//
// The query rows of a kv head are the T * G (node, head) pairs, all of which read the same keys.
//
// Arithmetic.  A query row is multiplied by the power of two that puts its largest element just below 2^11 and held in fp16:
// exact for fp16 and bf16 inputs (elements below 2^-35 of the largest one vanish).  Codes are exact in fp16 too, so Q K^T is a sum
// of exact products in fp32; the key's scale and the row's factor multiply the score.  The running reference of a row is the
// largest score + log2(value scale) among the keys that the row sees, so that weight * value scale, which is what is
// rounded to fp16 (once), is at most 2^7 and what fp16 cannot hold is below 2^-24 of the largest contribution, whatever the scales
// of values are and whatever other rows see.  Sums and statistics are fp32.
#include "tree_attn.cuh"

namespace uv {

// ---- nodes' keys and values through the cache's quantiser, into shared memory laid out like a tile of the cache.  Vectors are
//      spread over groups of HD / 8 lanes, 8 elements each; n_warps warps share the work.
template <typename QT, int HD>
__device__ __forceinline__ void quantise_nodes(const uv_tree_attn_args& a, int b, int kh, int warp, int n_warps, int lane, unsigned char* k8,
                                               unsigned char* v8, __half* ks, __half* vs) {
  constexpr int LV = HD / 8, PER = 32 / LV;
  const int n = a.T, sub = lane / LV, part = lane % LV;
  auto load = [&](int i) {
    if (i >= 2 * n) return make_uint4(0u, 0u, 0u, 0u);
    const int j = i >> 1;
    const QT* src = i & 1 ? static_cast<const QT*>(a.v) + (int64_t)b * a.snvb + (int64_t)j * a.snvt + (int64_t)kh * a.snvh
                          : static_cast<const QT*>(a.k) + (int64_t)b * a.snkb + (int64_t)j * a.snkt + (int64_t)kh * a.snkh;
    return *reinterpret_cast<const uint4*>(src + 8 * part);
  };
  uint4 next = load(warp * PER + sub);                             // (the next vectors are under way while these are worked on)
#pragma unroll 1
  for (int i0 = warp * PER; i0 < 2 * n; i0 += n_warps * PER) {
    const int i = i0 + sub, which = i & 1, j = i >> 1;
    float x[8];
    const uint4 raw = next;
    next = load(i + n_warps * PER);
    float amax = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[e] = to_f32<QT>(reinterpret_cast<const QT*>(&raw)[e]);
      amax = fmaxf(amax, fabsf(x[e]));
    }
#pragma unroll
    for (int o = LV / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    const __half s16 = __float2half_rn(__fdiv_rn(amax, 127.0f));
    const float sf = fmaxf(__half2float(s16), 1e-30f), inv = __frcp_rn(sf);
    uint32_t w[2] = {0u, 0u};
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e / 4] |= (uint32_t)(__float2int_rn(cache_code(x[e], sf, inv)) & 0xff) << (8 * (e & 3));
    if (i < 2 * n) {
      *reinterpret_cast<uint2*>((which ? v8 : k8) + j * HD + 8 * part) = make_uint2(w[0], w[1]);
      if (part == 0) (which ? vs : ks)[j] = s16;
    }
  }
}

// ------------------------------------------------------------------------------------------------ few query rows: mma.sync
// One CTA per (batch row, kv head; part of the keys; 16 R query rows).  Cached keys stream in tiles of 128 through a ring of
// shared memory, each of four warps owns 32 keys of a tile and all of the CTA's query rows, with its own running maximum
// and sum; the warps' states, and those of the parts, are merged at the end.  The nodes' own keys are one more tile, of the last part.
// What bounds it: up to a few tiles a CTA, the chain position -> copies and queries -> products -> merge and the fetch of instructions that run
// once (8 us with 16 rows a CTA, 10 with 32); behind that the issue of the softmax and of the codes' conversion, 2 us for 128 keys and 32 rows.
// Four warps with a quarter of the keys each, because a warp then needs no other's scores until the end; 32 rows a CTA, because two row
// blocks share a conversion and four would not leave the registers for two CTAs.  Measured, 8 heads of 64 over one kv head: one row of one node
// 7.2 us over 200 positions, 7 trees of 13 nodes on a ring of 256 13.0, 32 rows of 8 nodes over 2304 19.5
// (0.5 TB/s).
constexpr int TR_TILE = 128, TR_STAGES = 3, TR_WARPS = 4, TR_THREADS = (TR_WARPS + 1) * 32, TR_WKEYS = TR_TILE / TR_WARPS;

template <int HD> struct TreeStage {
  static constexpr int K = 0, V = TR_TILE * HD, KS = 2 * TR_TILE * HD, VS = KS + 2 * TR_TILE, BYTES = KS + 4 * TR_TILE;
};
template <int HD, int R> struct TreeSmem {
  static constexpr int ROWS = 16 * R;
  static constexpr int Q = TR_STAGES * TreeStage<HD>::BYTES;                    // query fragments, fp16
  static constexpr int QF = Q + ROWS * HD * 2;                                  // every row's power of two, undone in its scores
  static constexpr int NODES = QF + ROWS * 4;                                   // the nodes' tile: K, V, two scales
  static constexpr int PART = NODES + 2 * TREE_MAX * HD + 4 * TREE_MAX;         // this part's o, m, l for its cluster
  static constexpr int BYTES = PART + ROWS * (HD + 2) * 4;
};

// Waits for the last copies asked for, after a wait that ran out (out of line: what is not run costs no instruction lines).
__device__ __noinline__ void drain_copies(uint64_t* full, int issued) {
  for (int j = max(0, issued - TR_STAGES); j < issued; ++j)
    tc_mbar_wait(tc_smem_u32(&full[j % TR_STAGES]), (uint32_t)((j / TR_STAGES) & 1));
}

template <typename QT, int HD, int R, bool BULK>
__global__ void __launch_bounds__(TR_THREADS) tree_rows_kernel(const __grid_constant__ TreeParams P) {
  using L = TreeStage<HD>;
  using M = TreeSmem<HD, R>;
  constexpr int ROWS = 16 * R, KSTEPS = HD / 16, NT_S = TR_WKEYS / 8, NT_O = HD / 8, QW = HD / 16;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ __align__(8) uint64_t full[TR_STAGES], empty[TR_STAGES];
  __shared__ TreeSets sets;
  __shared__ int s_dead;
  const uv_tree_attn_args& a = P.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, r = lane >> 2, c = lane & 3;
  const bool producer = warp == TR_WARPS;
  const int b = blockIdx.x / a.KH, kh = blockIdx.x % a.KH, sid = blockIdx.y, row0 = blockIdx.z * ROWS;
  const int rows = min(ROWS, P.M - row0);
  pdl_wait();     // positions, queries, the nodes' keys and values and the caches come from the kernels before this one

  // ---- the part's tiles
  const RowRange rg = row_range(a, b);
  const int64_t lo = rg.lo, hi = rg.hi;
  int64_t t0 = 0;
  int ntile = 0;
  if (hi >= lo) {
    const int64_t t_lo = lo / TR_TILE, t_hi = hi / TR_TILE, per = (t_hi - t_lo + P.splits) / P.splits;
    t0 = t_lo + sid * per;
    const int64_t t1 = t0 + per < t_hi + 1 ? t0 + per : t_hi + 1;
    ntile = t1 > t0 ? (int)(t1 - t0) : 0;
  }
  const bool has_nodes = sid == P.splits - 1;
  const int8_t* kbase = a.k_cache + rg.row * a.skb + kh * a.skh;
  const int8_t* vbase = a.v_cache + rg.row * a.svb + kh * a.svh;
  const __half* ksbase = reinterpret_cast<const __half*>(a.k_scale) + rg.row * a.ssb + kh * a.ssh;
  const __half* vsbase = reinterpret_cast<const __half*>(a.v_scale) + rg.row * a.stb + kh * a.sth;
  if (tid == 0) {
    s_dead = 0;
#pragma unroll
    for (int s = 0; s < TR_STAGES; ++s) {
      tc_mbar_init(tc_smem_u32(&full[s]), 1);
      tc_mbar_init(tc_smem_u32(&empty[s]), TR_WARPS);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();

  // the four linear copies of tile ti into stage s (one thread): whole groups of 8 slots that hold valid positions; a ring's tile that
  // passes slot S - 1 comes in two pieces
  auto issue = [&](int64_t ti, int s) {
    const int64_t T0 = ti * TR_TILE, p0 = (T0 > lo ? T0 : lo) & ~(int64_t)7;
    const int64_t p1 = ((T0 + TR_TILE < hi + 1 ? T0 + TR_TILE : hi + 1) + 7) & ~(int64_t)7;
    const uint32_t n = (uint32_t)(p1 - p0), off = (uint32_t)(p0 - T0), bar = tc_smem_u32(&full[s]);
    const int64_t slot = a.ring ? p0 % a.S : p0;
    const uint32_t st = tc_smem_u32(smem + (size_t)s * L::BYTES);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    tc_mbar_expect_tx(bar, n * (2 * HD + 4));
    const uint32_t n1 = a.ring && slot + n > a.S ? (uint32_t)(a.S - slot) : n;
    auto piece = [&](uint32_t at, int64_t sl, uint32_t cnt) {
      bulk_copy(st + L::K + at * HD, kbase + sl * HD, cnt * HD, bar);
      bulk_copy(st + L::V + at * HD, vbase + sl * HD, cnt * HD, bar);
      bulk_copy(st + L::KS + at * 2, ksbase + sl, cnt * 2, bar);
      bulk_copy(st + L::VS + at * 2, vsbase + sl, cnt * 2, bar);
    };
    piece(off, slot, n1);
    if (n1 < n) piece(off + n1, 0, n - n1);
  };
  // other layouts: 16-byte pieces by all threads, scales through registers
  constexpr int SC = (2 * TR_TILE + TR_THREADS - 1) / TR_THREADS;
  __half sc[SC];
  auto load_pieces = [&](int64_t ti, int s) {
    const int64_t T0 = ti * TR_TILE;
    unsigned char* st = smem + (size_t)s * L::BYTES;
    constexpr int CH = HD / 16;
    for (int i = tid; i < TR_TILE * CH * 2; i += TR_THREADS) {
      const int which = i / (TR_TILE * CH), j = i % (TR_TILE * CH) / CH, ch = i % CH;
      const int64_t t = T0 + j;
      if (t < lo || t > hi) continue;
      const int64_t slot = a.ring ? t % a.S : t;
      const int8_t* src = (which ? vbase + slot * a.svs : kbase + slot * a.sks) + ch * 16;
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(tc_smem_u32(st + (which ? L::V : L::K) + j * HD + ch * 16)), "l"(src)
                   : "memory");
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
#pragma unroll
    for (int n = 0; n < SC; ++n) {
      const int i = tid + n * TR_THREADS, which = i / TR_TILE;
      const int64_t t = T0 + i % TR_TILE;
      sc[n] = __ushort_as_half(0);
      if (i < 2 * TR_TILE && t >= lo && t <= hi) {
        const int64_t slot = a.ring ? t % a.S : t;
        sc[n] = which ? vsbase[slot] : ksbase[slot];
      }
    }
  };

  bool dead = false;
  int issued = ntile;                       // tiles asked for, once the producer is done
  if constexpr (BULK) {
    if (producer && lane == 0)
      for (int j = 0; j < ntile && j < TR_STAGES; ++j) issue(t0 + j, j);
  } else if (ntile > 0) {
    load_pieces(t0, 0);
  }

  // ---- under the copies' latency: ancestor sets, query fragments, the nodes' tile
  if (producer) tree_sets(a.parents + (int64_t)b * a.parents_stride, a.T, sets, lane);
  unsigned char* const nodes = smem + M::NODES;
  __half* const node_ks = reinterpret_cast<__half*>(nodes + 2 * TREE_MAX * HD);
  float* const qf = reinterpret_cast<float*>(smem + M::QF);
  if (!producer) {
    // a group of HD / 8 lanes per row, 8 elements each; row i of a 16-row tile, elements d: the fragment register order of the
    // m16n8k16 A operand with the head dimension permuted so that a lane's four k-columns of a step are four consecutive elements
    constexpr int LV = HD / 8, PER = 32 / LV;
    const int sub = lane / LV, part = lane % LV;
    auto load = [&](int i) {
      if (i >= rows) return make_uint4(0u, 0u, 0u, 0u);
      const int row = row0 + i, t = node_of(P, row);
      return reinterpret_cast<const uint4*>(static_cast<const QT*>(a.q) + (int64_t)b * a.sqb + (int64_t)t * a.sqt +
                                            (int64_t)(kh * P.G + row - t * P.G) * a.sqh)[part];
    };
    uint4 next = load(warp * PER + sub);
#pragma unroll 1
    for (int i0 = warp * PER; i0 < ROWS; i0 += TR_WARPS * PER) {
      const int i = i0 + sub;
      const uint4 raw = next;
      next = load(i + TR_WARPS * PER);
      float x[8], amax = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[e] = to_f32<QT>(reinterpret_cast<const QT*>(&raw)[e]);
        amax = fmaxf(amax, fabsf(x[e]));
      }
#pragma unroll
      for (int o = LV / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
      int ex = ((int)(__float_as_uint(amax) >> 23) & 0xff) - 127;       // amax in [2^ex, 2^(ex + 1))
      ex = amax > 0.f ? max(ex, -100) : 10;                             // (infinite and NaN rows stay what they are)
      const float up = __uint_as_float((uint32_t)(127 + 10 - ex) << 23);
      if (part == 0) qf[i] = __uint_as_float((uint32_t)(127 + ex - 10) << 23);
      const int rm = i >> 4, rr = i & 15;
#pragma unroll
      for (int e2 = 0; e2 < 4; ++e2) {
        const int d = 8 * part + 2 * e2;                 // dims of lane column cc = d / (HD / 4), step j, registers (0 | 1) / (2 | 3)
        const int cc = d / (HD / 4), j = d % (HD / 4) / 4, reg = (rr >> 3) + (d & 2);
        reinterpret_cast<uint32_t*>(smem + M::Q)[((rm * KSTEPS + j) * 32 + (rr & 7) * 4 + cc) * 4 + reg] =
            pack_h2(x[2 * e2] * up, x[2 * e2 + 1] * up);
      }
    }
    if (has_nodes) quantise_nodes<QT, HD>(a, b, kh, warp, TR_WARPS, lane, nodes, nodes + TREE_MAX * HD, node_ks, node_ks + TREE_MAX);
  }
  __syncthreads();

  // ---- every warp's running softmax
  float o_acc[R][NT_O][4], m_run[R][2], l_run[R][2], f[R][2];
  int lo_node[R][2];             // window: how far the row's first position lies behind pos (0: none); see block()
#pragma unroll
  for (int rm = 0; rm < R; ++rm) {
#pragma unroll
    for (int i = 0; i < NT_O; ++i) o_acc[rm][i][0] = o_acc[rm][i][1] = o_acc[rm][i][2] = o_acc[rm][i][3] = 0.f;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int i = 16 * rm + r + 8 * e;
      m_run[rm][e] = -INFINITY, l_run[rm][e] = 0.f, f[rm][e] = qf[i];
      const uint64_t mask = i < rows ? sets.mask[node_of(P, row0 + i)] : 0ull;
      lo_node[rm][e] = a.window > 0 && mask ? __popcll(mask) - a.window : INT32_MIN;     // depth - window + 1
    }
  }
  // positions before pos + deepest are masked for some node
  int deepest = 0;
  if (a.window > 0)
    for (int i = lane; i < a.T; i += 32) deepest = max(deepest, __popcll(sets.mask[i]) - 1);
  deepest = __reduce_max_sync(0xffffffffu, deepest);
  const int64_t lo_all = a.window > 0 && rg.pos + deepest - a.window + 1 > lo ? rg.pos + deepest - a.window + 1 : lo;

  // 32 keys of a warp.  EDGE: lo_rel .. hi_rel are the positions in range, and a node's window may begin inside (base = position of
  // the first key - pos).  NODE: keys are nodes k0 .. k0 + 31 and each row sees its ancestors.
  auto block = [&](const unsigned char* kt, const unsigned char* vt, const __half* kst, const __half* vst, int lo_rel, int hi_rel, int base,
                   auto edge_tag, auto node_tag) {
    constexpr bool EDGE = decltype(edge_tag)::value, NODE = decltype(node_tag)::value;
    float s[R][NT_S][4];
#pragma unroll
    for (int rm = 0; rm < R; ++rm)
#pragma unroll
      for (int t = 0; t < NT_S; ++t) s[rm][t][0] = s[rm][t][1] = s[rm][t][2] = s[rm][t][3] = 0.f;
    uint32_t kw[NT_S][QW];
#pragma unroll
    for (int t = 0; t < NT_S; ++t) {
      const unsigned char* p = kt + (8 * t + r) * HD + c * (HD / 4);
      if constexpr (QW == 1) {
        kw[t][0] = *reinterpret_cast<const uint32_t*>(p);
      } else if constexpr (QW == 2) {
        const uint2 u = *reinterpret_cast<const uint2*>(p);
        kw[t][0] = u.x, kw[t][1] = u.y;
      } else {
#pragma unroll
        for (int j = 0; j < QW / 4; ++j) {
          const uint4 u = *reinterpret_cast<const uint4*>(p + 16 * j);
          kw[t][4 * j] = u.x, kw[t][4 * j + 1] = u.y, kw[t][4 * j + 2] = u.z, kw[t][4 * j + 3] = u.w;
        }
      }
    }
#pragma unroll
    for (int j = 0; j < KSTEPS; ++j) {
      uint4 qa[R];
#pragma unroll
      for (int rm = 0; rm < R; ++rm) qa[rm] = reinterpret_cast<const uint4*>(smem + M::Q)[(rm * KSTEPS + j) * 32 + lane];
#pragma unroll
      for (int t = 0; t < NT_S; ++t) {
        const uint32_t x = kw[t][j] ^ 0x80808080u, b0 = bias_pair(x, 0x4140), b1 = bias_pair(x, 0x4342);
#pragma unroll
        for (int rm = 0; rm < R; ++rm) mma16816(s[rm][t], qa[rm].x, qa[rm].y, qa[rm].z, qa[rm].w, b0, b1);
      }
    }
    float ks[NT_S][2], vs[NT_S][2], lv[NT_S][2];
#pragma unroll
    for (int t = 0; t < NT_S; ++t) {
      const int kk = 8 * t + 2 * c;
      const float2 kf = __half22float2(*reinterpret_cast<const __half2*>(kst + kk));
      const float2 vf = __half22float2(*reinterpret_cast<const __half2*>(vst + kk));
      ks[t][0] = kf.x * P.scale_log2, ks[t][1] = kf.y * P.scale_log2, vs[t][0] = vf.x, vs[t][1] = vf.y;
#pragma unroll
      for (int e = 0; e < 2; ++e)       // floor(log2) of the scale; zero counts as the smallest scale that fp16 has
        lv[t][e] = (float)max((int)((__float_as_uint(vs[t][e]) >> 23) & 0xff) - 127, -24);
    }
    uint32_t pa[R][TR_WKEYS / 16][4];
#pragma unroll
    for (int rm = 0; rm < R; ++rm)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float mx = -INFINITY;
        uint64_t seen = 0;
        if constexpr (NODE) {
          const int i = 16 * rm + r + 8 * h;
          seen = i < rows ? sets.mask[node_of(P, row0 + i)] : 0ull;
        }
#pragma unroll
        for (int t = 0; t < NT_S; ++t)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int kk = 8 * t + 2 * c + e;
            float v = s[rm][t][2 * h + e] * ks[t][e];
            if constexpr (EDGE) v = kk >= lo_rel && kk <= hi_rel && base + kk >= lo_node[rm][h] ? v : -INFINITY;
            if constexpr (NODE) {
              bool on = kk <= hi_rel && (seen >> (base + kk) & 1ull);
              if (on && a.window > 0) on = __popcll(seen) - __popcll(sets.mask[base + kk]) < a.window;
              v = on ? v : -INFINITY;
            }
            s[rm][t][2 * h + e] = v;
            mx = fmaxf(mx, fmaf(v, f[rm][h], lv[t][e]));
          }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        if (__any_sync(0xffffffffu, mx > m_run[rm][h] + RESCALE_GAP)) {
          const float m_new = mx > m_run[rm][h] + RESCALE_GAP ? mx : m_run[rm][h];
          const float alpha = m_new == -INFINITY ? 1.0f : ex2(m_run[rm][h] - m_new);
          l_run[rm][h] *= alpha;
#pragma unroll
          for (int i = 0; i < NT_O; ++i) o_acc[rm][i][2 * h] *= alpha, o_acc[rm][i][2 * h + 1] *= alpha;
          m_run[rm][h] = m_new;
        }
        const float m_use = m_run[rm][h] == -INFINITY ? 0.f : m_run[rm][h];
        float sum = 0.f;
#pragma unroll
        for (int t = 0; t < NT_S; ++t) {
          const float p0 = ex2(fmaf(s[rm][t][2 * h], f[rm][h], -m_use)), p1 = ex2(fmaf(s[rm][t][2 * h + 1], f[rm][h], -m_use));
          sum += p0 + p1;
          float w0 = p0 * vs[t][0], w1 = p1 * vs[t][1];
          if constexpr (EDGE || NODE) w0 = p0 > 0.f ? w0 : 0.f, w1 = p1 > 0.f ? w1 : 0.f;   // (a masked scale may be anything)
          pa[rm][t / 2][2 * (t & 1) + h] = pack_h2(w0, w1);
        }
        l_run[rm][h] += sum;
      }
    // O += P V: lane (r, c) reads HD / 8 bytes at dim r * HD / 8 of keys 2c, 2c + 1, 2c + 8, 2c + 9 of each 16 keys and transposes them
    // into B fragments (n8 tile i <-> dim r * HD / 8 + i)
#pragma unroll
    for (int u = 0; u < TR_WKEYS / 16; ++u) {
      const unsigned char* vrow = vt + (16 * u + 2 * c) * HD + r * (HD / 8);
      constexpr int VW = (NT_O + 3) / 4;
      uint32_t w[4][VW];
      auto ld = [&](const unsigned char* p, uint32_t(&x)[VW]) {
        if constexpr (NT_O == 2) {
          x[0] = *reinterpret_cast<const uint16_t*>(p);
        } else if constexpr (NT_O == 4) {
          x[0] = *reinterpret_cast<const uint32_t*>(p);
        } else if constexpr (NT_O == 8) {
          const uint2 q = *reinterpret_cast<const uint2*>(p);
          x[0] = q.x, x[1] = q.y;
        } else {
#pragma unroll
          for (int j = 0; j < VW / 4; ++j) {
            const uint4 q = *reinterpret_cast<const uint4*>(p + 16 * j);
            x[4 * j] = q.x, x[4 * j + 1] = q.y, x[4 * j + 2] = q.z, x[4 * j + 3] = q.w;
          }
        }
      };
      ld(vrow, w[0]), ld(vrow + HD, w[1]), ld(vrow + 8 * HD, w[2]), ld(vrow + 9 * HD, w[3]);
#pragma unroll
      for (int x = 0; x < VW; ++x)
#pragma unroll
        for (int hw = 0; hw < 2; ++hw) {
          if (4 * x + 2 * hw >= NT_O) break;
          const uint32_t ab = __byte_perm(w[0][x] ^ 0x80808080u, w[1][x] ^ 0x80808080u, hw ? 0x7362 : 0x5140);
          const uint32_t cd = __byte_perm(w[2][x] ^ 0x80808080u, w[3][x] ^ 0x80808080u, hw ? 0x7362 : 0x5140);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int i = 4 * x + 2 * hw + e;
            const uint32_t b0 = bias_pair(ab, e ? 0x4342 : 0x4140), b1 = bias_pair(cd, e ? 0x4342 : 0x4140);
#pragma unroll
            for (int rm = 0; rm < R; ++rm) mma16816(o_acc[rm][i], pa[rm][u][0], pa[rm][u][1], pa[rm][u][2], pa[rm][u][3], b0, b1);
          }
        }
    }
  };
  auto cached = [&](const unsigned char* st, int64_t ti) {
    const int64_t kb = ti * TR_TILE + TR_WKEYS * warp;
    if (kb + TR_WKEYS - 1 < lo || kb > hi) return;
    const unsigned char *kt = st + L::K + TR_WKEYS * warp * HD, *vt = st + L::V + TR_WKEYS * warp * HD;
    const __half *kst = reinterpret_cast<const __half*>(st + L::KS) + TR_WKEYS * warp, *vst = reinterpret_cast<const __half*>(st + L::VS) + TR_WKEYS * warp;
    if (kb < lo_all || kb + TR_WKEYS - 1 > hi) {
      const int64_t a0 = lo - kb, a1 = hi - kb;
      block(kt, vt, kst, vst, a0 < 0 ? 0 : (int)a0, a1 > TR_WKEYS ? TR_WKEYS : (int)a1, (int)(kb - rg.pos), std::true_type{}, std::false_type{});
    } else {
      block(kt, vt, kst, vst, 0, TR_WKEYS, 0, std::false_type{}, std::false_type{});
    }
  };

  // the nodes' tile first: it is there already
  if (has_nodes && !producer) {
    const int k0 = TR_WKEYS * (TR_WARPS - 1 - warp);       // (the last warps: the last tile of a row is often a short one)
    if (k0 < a.T)
      block(nodes + k0 * HD, nodes + (TREE_MAX + k0) * HD, node_ks + k0, node_ks + TREE_MAX + k0, 0, a.T - 1 - k0, k0, std::false_type{},
            std::true_type{});
  }
  if constexpr (BULK) {
    if (producer) {
      if (lane == 0)
        for (int j = TR_STAGES; j < ntile; ++j) {
          const int s = j % TR_STAGES;
          if (!tc_mbar_wait(tc_smem_u32(&empty[s]), (uint32_t)((j / TR_STAGES - 1) & 1))) {
            dead = true, issued = j;
            break;
          }
          issue(t0 + j, s);
        }
    } else {
      for (int it = 0; it < ntile; ++it) {
        const int s = it % TR_STAGES;
        if (!dead) dead = !__all_sync(0xffffffffu, tc_mbar_wait(tc_smem_u32(&full[s]), (uint32_t)((it / TR_STAGES) & 1)));
        if (!dead) cached(smem + (size_t)s * L::BYTES, t0 + it);
        __syncwarp();
        if (lane == 0) mbar_arrive_one(tc_smem_u32(&empty[s]));
      }
    }
    if (dead && lane == 0) {
      if (a.status) atomicOr(a.status, 1);
      s_dead = 1;
    }
  } else {
    for (int it = 0; it < ntile; ++it) {
      unsigned char* st = smem + (size_t)(it & 1) * L::BYTES;
      asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
      for (int n = 0; n < SC; ++n) {
        const int i = tid + n * TR_THREADS;
        if (i < 2 * TR_TILE) reinterpret_cast<__half*>(st + (i / TR_TILE ? L::VS : L::KS))[i % TR_TILE] = sc[n];
      }
      __syncthreads();
      if (it + 1 < ntile) load_pieces(t0 + it + 1, (it + 1) & 1);
      if (!producer) cached(st, t0 + it);
    }
  }
  __syncthreads();

  // ---- merge: the warps' states through shared memory (over the ring: every copy has landed, unless the CTA gave one up: then its
  //      part is reported empty, and the status word says that the output is not to be used)
  const bool lost = s_dead != 0;
  if constexpr (BULK)
    if (lost && producer && lane == 0) drain_copies(full, issued);       // the CTA does not end before its own copies
  float* const mg_o = reinterpret_cast<float*>(smem);
  float* const mg_m = mg_o + TR_WARPS * ROWS * HD;
  float* const mg_l = mg_m + TR_WARPS * ROWS;
  static_assert(TR_WARPS * ROWS * (HD + 2) * 4 <= TR_STAGES * L::BYTES, "the warps' states fit the ring");
  float* const part = reinterpret_cast<float*>(smem + M::PART);
  if (!producer && !lost)
#pragma unroll
    for (int rm = 0; rm < R; ++rm)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float l = l_run[rm][h];
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        const int row = warp * ROWS + 16 * rm + r + 8 * h;
        if (c == 0) mg_m[row] = m_run[rm][h], mg_l[row] = l;
#pragma unroll
        for (int i = 0; i < NT_O; ++i) {
          mg_o[row * HD + 2 * c * (HD / 8) + i] = o_acc[rm][i][2 * h];
          mg_o[row * HD + (2 * c + 1) * (HD / 8) + i] = o_acc[rm][i][2 * h + 1];
        }
      }
  __syncthreads();
  constexpr int EPL = (HD + 31) / 32;
#pragma unroll 2
  for (int row = warp; row < rows; row += TR_WARPS + 1) {
    float mw[TR_WARPS], mx = -INFINITY, lsum = 0.f, z[EPL];
#pragma unroll
    for (int i = 0; i < EPL; ++i) z[i] = 0.f;
    if (!lost) {
#pragma unroll
      for (int w = 0; w < TR_WARPS; ++w) mw[w] = mg_m[w * ROWS + row], mx = fmaxf(mx, mw[w]);
#pragma unroll
      for (int w = 0; w < TR_WARPS; ++w) {
        const float wt = mw[w] == -INFINITY ? 0.f : ex2(mw[w] - mx);          // (what a warp without keys holds is zeros)
        lsum += part_sum(mw[w], wt, mg_l[w * ROWS + row]);
#pragma unroll
        for (int i = 0; i < EPL; ++i)
          if (HD >= 32 || lane < HD) z[i] += wt * mg_o[(w * ROWS + row) * HD + lane + 32 * i];
      }
    }
    if (P.splits == 1) {
      const float inv = inverse_sum(lsum);
#pragma unroll
      for (int i = 0; i < EPL; ++i) z[i] *= inv;
      store_row<QT, HD>(P, z, b, kh, row0 + row, sets.mask[node_of(P, row0 + row)] != 0, lane);
    } else if (P.cluster) {
      if (lane == 0) part[ROWS * HD + row] = mx, part[ROWS * HD + ROWS + row] = lsum;
#pragma unroll
      for (int i = 0; i < EPL; ++i)
        if (HD >= 32 || lane < HD) part[row * HD + lane + 32 * i] = z[i];
    } else {
      const int64_t w = ((int64_t)blockIdx.x * P.splits + sid) * P.M + row0 + row;
      if (lane == 0) P.ws_m[w] = mx, P.ws_l[w] = lsum;
#pragma unroll
      for (int i = 0; i < EPL; ++i)
        if (HD >= 32 || lane < HD) P.ws_o[w * HD + lane + 32 * i] = z[i];
    }
  }
  if (!P.cluster) return;
  cluster_barrier();
  const uint32_t po = tc_smem_u32(part), pm = po + ROWS * HD * 4u, pl = pm + ROWS * 4u;
  for (int row = sid + warp * P.splits; row < rows; row += (TR_WARPS + 1) * P.splits) {
    float m_s = -INFINITY, l_s = 0.f, z[EPL];
    if (lane < P.splits) m_s = peer_f32(pm + row * 4u, lane), l_s = peer_f32(pl + row * 4u, lane);
    const float mx = warp_max(m_s), wt_s = m_s == -INFINITY ? 0.f : ex2(m_s - mx), lsum = warp_sum(part_sum(m_s, wt_s, l_s));
#pragma unroll
    for (int i = 0; i < EPL; ++i) z[i] = 0.f;
#pragma unroll 4
    for (int s = 0; s < P.splits; ++s) {
      const float wt = __shfl_sync(0xffffffffu, wt_s, s);
#pragma unroll
      for (int i = 0; i < EPL; ++i)
        if (HD >= 32 || lane < HD) z[i] += wt * peer_f32(po + (uint32_t)(row * HD + lane + 32 * i) * 4u, s);
    }
    const float inv = inverse_sum(lsum);
#pragma unroll
    for (int i = 0; i < EPL; ++i) z[i] *= inv;
    store_row<QT, HD>(P, z, b, kh, row0 + row, sets.mask[node_of(P, row0 + row)] != 0, lane);
  }
  cluster_barrier();
}

// ------------------------------------------------------------------------------------------------ merge through the workspace
// One warp per query row: log-sum-exp merge of its parts.
template <typename QT, int HD>
__global__ void __launch_bounds__(128) tree_combine_kernel(const __grid_constant__ TreeParams P) {
  constexpr int EPL = (HD + 31) / 32;
  const uv_tree_attn_args& a = P.a;
  const int lane = threadIdx.x & 31, row = blockIdx.y * 4 + (threadIdx.x >> 5);
  const int b = blockIdx.x / a.KH, kh = blockIdx.x % a.KH;
  if (row >= P.M) return;
  // present: the node's way to the root, as tree_sets decides it
  const int32_t* par = a.parents + (int64_t)b * a.parents_stride;
  int up = node_of(P, row);
  while (par[up] >= 0 && par[up] < up) up = par[up];
  const int64_t w0 = (int64_t)blockIdx.x * P.splits * P.M + row;
  float mx = -INFINITY, lsum = 0.f, z[EPL];
  for (int s = lane; s < P.splits; s += 32) mx = fmaxf(mx, P.ws_m[w0 + (int64_t)s * P.M]);
  mx = warp_max(mx);
#pragma unroll
  for (int i = 0; i < EPL; ++i) z[i] = 0.f;
  for (int s = 0; s < P.splits; ++s) {
    const int64_t w = w0 + (int64_t)s * P.M;
    const float m = P.ws_m[w], wt = m == -INFINITY ? 0.f : ex2(m - mx);
    lsum += part_sum(m, wt, P.ws_l[w]);
    if (m == -INFINITY) continue;
#pragma unroll
    for (int i = 0; i < EPL; ++i)
      if (HD >= 32 || lane < HD) z[i] += wt * P.ws_o[w * HD + lane + 32 * i];
  }
  const float inv = inverse_sum(lsum);
#pragma unroll
  for (int i = 0; i < EPL; ++i) z[i] *= inv;
  store_row<QT, HD>(P, z, b, kh, row, par[up] == -1, lane);
}

// ------------------------------------------------------------------------------------------------ host side
// whole groups of 8 slots can be copied linearly, 16-byte aligned on both sides
static bool bulk_ok(const uv_tree_attn_args& a) {
  const int s_alloc = a.S_alloc > a.S ? a.S_alloc : a.S;
  return a.sks == a.hd && a.svs == a.hd && (a.ring ? a.S % 8 == 0 : s_alloc % 8 == 0) && aligned16(a.k_scale) && aligned16(a.v_scale) &&
         ((a.ssb | a.ssh | a.stb | a.sth) & 7) == 0;
}

// Parts of a row's keys: no more CTAs than two to each multiprocessor (three with 16 query rows a CTA or small heads, one with head_dim 128; what
// comes behind them doubles the time), clusters of a power of two; clusters of 8 leave a tenth to a fifth of the places unused, since each stands in
// one group of multiprocessors (head_dim 128: 15 of them run at a time, 21 us, 16 take 42).  What a cluster's exchange costs, some 1 us, is won
// back by fewer tiles a CTA and by rows merged and finished together, from the more tiles on the smaller the heads are.  8 heads to a kv head,
// whole, 2, 4 and 8 parts: head_dim 64, 1 row of 13 nodes over 128 positions 10.1, 11.9, 11.2, 11.1 us; 7 rows of 40 nodes over 256 13.0, 16.3, 14.3;
// 1 row of 4 nodes over 512 15.7, -, 13.6, 11.2 (before the merges were unrolled); 100 rows of 4 nodes over 1024 20.7, 22.1; head_dim 16, 1 row of 4
// nodes over 128 8.2, 10.9, 9.7, 9.3, 60 rows over 512 11.3, 14.0, 12.7; head_dim 128, 7 rows of 40 nodes over 1024 38.5, 33.9.
// More than a cluster of 8 merges pay a second launch and the workspace's traffic, which only rows of hundreds of tiles repay (one row of one
// node over 8192 positions: 17 us with 8 parts, 19 with 32; over 60000: 58 and 29).
static int default_parts(const uv_tree_attn_args& a, int row_tiles, int n_sm) {
  const int64_t ctx = a.window > 0 && a.window < a.S ? a.window : a.S;
  const int tiles = (int)((ctx + TR_TILE - 1) / TR_TILE), size = a.hd > 64 ? 0 : a.hd == 64 ? 1 : 2;
  const int64_t units = (int64_t)a.B * a.KH * row_tiles;
  const bool few = a.T * (a.H / a.KH) <= 16;
  const int64_t places = (size == 0 ? 1 : few || size == 2 ? 3 : 2) * n_sm;
  int64_t s = places / units;
  if (few && s > 2 * tiles) s = 2 * tiles;
  if (s > 8 && tiles < 16 * 8) s = 8;
  if (s > 64) s = 64;
  if (s > 8) return (int)s;
  if (s == 8 && places >= (size == 0 ? 10 : 9) * units && tiles >= 1 << size) return 8;
  if (s >= 4 && tiles >= (size == 0 ? 1 : size == 1 ? 3 : 8)) return 4;
  return s >= 2 && tiles >= (size == 0 ? 8 : 12) ? 2 : 1;
}

struct TreePlan {
  int R, splits;
  bool cluster;
  size_t ws_rows;
};
static TreePlan tree_plan(const uv_tree_attn_args& a) {
  TreePlan p{};
  const int M = a.T * (a.H / a.KH);
  p.R = M > 16 ? 2 : 1;
  p.splits = a.num_splits > 0 ? a.num_splits : default_parts(a, (M + 16 * p.R - 1) / (16 * p.R), sm_count());
  if (p.splits > 1024) p.splits = 1024;
  p.cluster = p.splits > 1 && p.splits <= 8;
  p.ws_rows = p.splits > 1 && !p.cluster ? (size_t)a.B * a.KH * p.splits * M : 0;
  return p;
}

template <typename QT, int HD, int R, bool BULK>
static int launch_rows(const TreeParams& P, cudaStream_t st) {
  auto kern = tree_rows_kernel<QT, HD, R, BULK>;
  constexpr int smem = TreeSmem<HD, R>::BYTES;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) {
    set_last_cuda_error((int)e);
    return UV_ERR_CUDA;
  }
  const dim3 grid((unsigned)(P.a.B * P.a.KH), (unsigned)P.splits, (unsigned)((P.M + 16 * R - 1) / (16 * R)));
  launch_cluster(kern, grid, dim3(TR_THREADS), dim3(1, P.cluster ? (unsigned)P.splits : 1u, 1), smem, st, P);
  int rc = check_launch();
  if (rc != UV_OK || P.splits == 1 || P.cluster) return rc;
  tree_combine_kernel<QT, HD><<<dim3((unsigned)(P.a.B * P.a.KH), (unsigned)((P.M + 3) / 4)), 128, 0, st>>>(P);
  return check_launch();
}

template <typename QT, int HD>
static int launch_tree(const TreeParams& P, int R, cudaStream_t st) {
  const bool bulk = bulk_ok(P.a);
  if (R == 1) return bulk ? launch_rows<QT, HD, 1, true>(P, st) : launch_rows<QT, HD, 1, false>(P, st);
  return bulk ? launch_rows<QT, HD, 2, true>(P, st) : launch_rows<QT, HD, 2, false>(P, st);
}

template <typename QT>
static int launch_tree_hd(const TreeParams& P, int R, cudaStream_t st) {
  switch (P.a.hd) {
    case 16: return launch_tree<QT, 16>(P, R, st);
    case 32: return launch_tree<QT, 32>(P, R, st);
    case 64: return launch_tree<QT, 64>(P, R, st);
    default: return launch_tree<QT, 128>(P, R, st);
  }
}

static int check_tree_args(const uv_tree_attn_args* a) {
  if (!a->q || !a->k || !a->v || !a->parents || !a->k_cache || !a->v_cache || !a->k_scale || !a->v_scale || !a->pos || !a->starts ||
      !a->out)
    return UV_ERR_ARG;
  if (a->B < 0 || a->T < 0 || a->H < 1 || a->KH < 1 || a->S < 1 || a->H % a->KH || a->window < 0 || a->num_splits < 0 || a->n_rows < 0)
    return UV_ERR_ARG;
  if (a->dtype != UV_F16 && a->dtype != UV_BF16) return UV_ERR_DTYPE;
  if (a->T > TREE_MAX || a->H / a->KH > 16) return UV_ERR_SHAPE;
  if (a->hd != 16 && a->hd != 32 && a->hd != 64 && a->hd != 128) return UV_ERR_SHAPE;
  if ((int64_t)a->B * a->KH > INT32_MAX) return UV_ERR_SHAPE;
  // vectors are read in 16-byte pieces
  if (!aligned16(a->q) || !aligned16(a->k) || !aligned16(a->v) || !aligned16(a->k_cache) || !aligned16(a->v_cache) ||
      ((a->sqb | a->sqt | a->sqh | a->snkb | a->snkt | a->snkh | a->snvb | a->snvt | a->snvh) & 7) ||
      ((a->skb | a->skh | a->sks | a->svb | a->svh | a->svs) & 15))
    return UV_ERR_ALIGN;
  return UV_OK;
}

}  // namespace uv

extern "C" size_t uv_tree_attn_workspace_bytes(const uv_tree_attn_args* a) {
  if (!a || a->B < 1 || a->T < 1 || a->T > uv::TREE_MAX || a->KH < 1 || a->H < a->KH || a->S < 1 || a->hd < 1) return 0;
  if (uv::tree_tc_wants(*a)) return uv::tree_tc_workspace(*a);
  return uv::tree_plan(*a).ws_rows * (size_t)(a->hd + 2) * sizeof(float);
}

extern "C" int uv_tree_attn(const uv_tree_attn_args* a, void* stream) {
  using namespace uv;
  if (!a) return UV_ERR_ARG;
  if (a->B == 0 || a->T == 0) return UV_OK;
  const int rc = check_tree_args(a);
  if (rc != UV_OK) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int G = a->H / a->KH;
  const uint32_t g_inv = G > 1 ? (uint32_t)(((1ull << 32) + G - 1) / G) : 0u;
  if (tree_tc_wants(*a)) {
    if (const size_t need = tree_tc_workspace(*a)) {
      if (!a->workspace || a->workspace_bytes < need) return UV_ERR_WORKSPACE;
      if (!aligned16(a->workspace)) return UV_ERR_ALIGN;
    }
    TreeParams P{*a, a->H / a->KH, a->T * (a->H / a->KH), g_inv, 0, 0, a->scale * LOG2E, static_cast<float*>(a->workspace), nullptr, nullptr};
    return launch_tree_tc(P, st);
  }
  const TreePlan plan = tree_plan(*a);
  TreeParams P{*a, a->H / a->KH, a->T * (a->H / a->KH), g_inv, plan.splits, plan.cluster ? 1 : 0, a->scale * LOG2E, nullptr, nullptr, nullptr};
  if (plan.ws_rows) {
    if (!a->workspace || a->workspace_bytes < uv_tree_attn_workspace_bytes(a)) return UV_ERR_WORKSPACE;
    if (!aligned16(a->workspace)) return UV_ERR_ALIGN;
    P.ws_o = static_cast<float*>(a->workspace);
    P.ws_m = P.ws_o + plan.ws_rows * a->hd;
    P.ws_l = P.ws_m + plan.ws_rows;
  }
  return a->dtype == UV_F16 ? launch_tree_hd<__half>(P, plan.R, st) : launch_tree_hd<__nv_bfloat16>(P, plan.R, st);
}
