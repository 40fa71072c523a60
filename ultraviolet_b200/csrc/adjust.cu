// Logits between the head and the sampler: softcap, penalties for tokens of the row's text, biases, and a mask of allowed tokens.
//
//   z = a * sigmoid((x + b) / c);  seen: z = z > 0 ? z / r : z * r;  z -= f n + p [n > 0];  z += bias;  not allowed: -inf
//
// A block owns a run of the vocabulary of one row.  It requests its logits, mask bits and the first round of the row's text together,
// counts the text into a histogram of its run in shared memory, and writes its logits once.  Counting in shared memory needs no pass over
// the text per entry and no scratch in device memory; its price is that every block of a row reads the whole text (a few KB out of L2).
// One thread takes groups of 4 entries: histogram, logits and results move 16 (8) bytes at a time, and a warp's are contiguous (8 entries a
// thread took 38.6 us in place of 26 for 512 rows of 16384: shared-memory conflicts of 8 ways).  Groups without a counted token skip the
// penalties, those without a bias the bias.
// Measured on a B200, L2 warm: 4.3 us for one row of 16384 (latency of the chain lengths -> text -> logits), 10.2 us for 9 trees of 7 nodes
// x 50257 fp16, 25 us for 512 rows of 16384 bf16 with texts of up to 2304 tokens and 32 biases (50 MB moved; the issue slots are 43 %
// busy, the rest is the wait for the text: the same rows with the softcap alone take 11.5 us).
#include "common.cuh"
#include "tree.cuh"

namespace uv {

constexpr uint32_t ADJ_PROMPT = 0x80000000u;   // the token stands in the prompt; the other bits count how often it was drawn

template <typename T> struct alignas(4 * sizeof(T)) Four { T v[4]; };

// TH threads, GR groups of 4 entries each: group g of a thread is entries run + 4 (tid + g TH) .. + 3, so that a warp's loads and stores are
// contiguous.  VEC: groups begin where x and out are aligned to 4 entries; `lead` entries (fewer than 4) stand before the first one and are
// threads 0 .. lead - 1's of the first block.
template <typename TI, typename TO, int TH, int GR, bool VEC, bool BIAS>
__global__ void __launch_bounds__(TH, 6 * 256 / TH) adjust_kernel(const __grid_constant__ uv_adjust_args a) {
  constexpr int RUN = 4 * GR * TH;
  __shared__ __align__(16) uint32_t cnt[RUN + 4];                 // entry of token v: v - run + 4
  __shared__ __align__(16) int which[BIAS ? RUN + 4 : 4];         // 1 + index of the last bias entry of the token
  __shared__ TreeSets sets;
  const int tid = threadIdx.x, r = blockIdx.x, b = a.T == 1 ? r : r / a.T, t = r - b * a.T;
  const TI* x = static_cast<const TI*>(a.x) + b * a.sxb + t * a.sxt;
  TO* out = static_cast<TO*>(a.out) + b * a.sob + t * a.sot;
  const int lead = VEC ? min(a.V, (int)(-(reinterpret_cast<uintptr_t>(x) / sizeof(TI)) & 3)) : 0;
  const int run = lead + blockIdx.y * RUN;
  // ---- requests
  Four<TI> in[GR];
  uint32_t on[GR];
  const uint32_t* bits = reinterpret_cast<const uint32_t*>(a.allowed) + (a.allowed ? b * a.sab + t * a.sat : 0);
#pragma unroll
  for (int g = 0; g < GR; ++g) {
    const int v = run + 4 * (tid + g * TH);
    if (VEC && v + 4 <= a.V) {
      in[g] = *reinterpret_cast<const Four<TI>*>(x + v);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) in[g].v[e] = v + e < a.V ? x[v + e] : from_f32<TI>(0.f);
    }
    on[g] = 0xfu;
    if (a.allowed && v < a.V) {
      const int w = v >> 5, s = v & 31;
      on[g] = bits[w] >> s;
      if (s > 28 && min(v + 4, a.V) > 32 * (w + 1)) on[g] |= bits[w + 1] << (32 - s);
    }
  }
  // (of the text and of the biases what a block reads in its first round, whatever their lengths turn out to be)
  const int32_t* hist = a.history && a.hist_bytes == 4 ? static_cast<const int32_t*>(a.history) + (int64_t)b * a.history_stride : nullptr;
  const bool wide = hist && (reinterpret_cast<uintptr_t>(hist) & 15) == 0;
  int4 text = make_int4(0, 0, 0, 0);
  if (wide && 4 * tid + 3 < a.history_len) text = *reinterpret_cast<const int4*>(hist + 4 * tid);
  int64_t len = a.lengths ? a.lengths[b] : a.history_len;
  int64_t np = a.prompt_lengths ? a.prompt_lengths[b] : 0;
  const int bias_id = BIAS && tid < a.n_bias ? a.bias_ids[b * a.bias_stride + tid] : -1;
  const float rep = a.repetition ? a.repetition[b] : 1.0f, freq = a.frequency ? a.frequency[b] : 0.f, pres = a.presence ? a.presence[b] : 0.f;
  // ---- the row's text
  const bool counted = a.history || a.parents;
  const int lo = blockIdx.y == 0 ? 0 : run, hi = min(a.V, run + RUN);        // tokens that this block counts
  if (counted || BIAS) {
    for (int i = 4 * tid; i < RUN + 4; i += 4 * TH) {
      *reinterpret_cast<uint4*>(&cnt[i]) = make_uint4(0u, 0u, 0u, 0u);
      if (BIAS) *reinterpret_cast<uint4*>(&which[i]) = make_uint4(0u, 0u, 0u, 0u);
    }
    __syncthreads();
  }
  const unsigned span = hi > lo ? (unsigned)(hi - lo) : 0u;       // (the last run may lie behind the vocabulary: `lead` moved it)
  auto narrow = [&](int64_t tok) -> int { return tok < lo || tok >= hi ? -1 : (int)tok; };
  auto count = [&](int tok, bool prompt) {
    if ((unsigned)tok - (unsigned)lo >= span) return;
    uint32_t* c = &cnt[tok - run + 4];
    if (prompt) atomicOr(c, ADJ_PROMPT);
    else atomicAdd(c, 1u);
  };
  if (a.history) {
    len = len < 0 ? 0 : len > a.history_len ? a.history_len : len;
    np = np < 0 ? 0 : np > len ? len : np;
    if (hist) {
      if (wide)
        for (int64_t i = 4 * tid; i + 3 < len; i += 4 * TH) {
          const int4 q = i < 4 * TH ? text : *reinterpret_cast<const int4*>(hist + i);
          const int left = np > i ? (int)min(np - i, (int64_t)4) : 0;   // of them in the prompt
          count(q.x, left > 0), count(q.y, left > 1), count(q.z, left > 2), count(q.w, left > 3);
        }
      // what is left: the last few of an aligned text, or all of it
      for (int64_t i = (wide ? len & ~(int64_t)3 : 0) + tid; i < len; i += TH) count(hist[i], i < np);
    } else {
      const int64_t* h = static_cast<const int64_t*>(a.history) + (int64_t)b * a.history_stride;
      for (int64_t i = tid; i < len; i += TH) count(narrow(h[i]), i < np);
    }
  }
  if (a.parents && tid < 32) {
    tree_sets(a.parents + (int64_t)b * a.parents_stride, a.T, sets, tid);
    const uint64_t way = sets.mask[t];                            // the node and its ancestors; none of an absent one
    for (int i = tid; i < a.T; i += 32)
      if (way >> i & 1ull) count(narrow(a.tokens[(int64_t)b * a.T + i]), false);
  }
  if constexpr (BIAS)
    for (int i = tid; i < a.n_bias; i += TH) {
      const int id = i < TH ? bias_id : a.bias_ids[b * a.bias_stride + i];
      if (id >= lo && id < hi) atomicMax(&which[id - run + 4], i + 1);
    }
  if (counted || BIAS) __syncthreads();
  // ---- the logits
  const float ic = a.softcap ? -1.4426950408889634f / a.cap_c : 0.f, ir = 1.0f / rep;
  // the softcap: e and the reciprocal are each within 2^-21 or so of their values, and 0 comes out where the quotient is below 2^-126
  auto cap = [&](float z) -> float {
    if (!a.softcap) return z;
    float e, q;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"((z + a.cap_b) * ic));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(q) : "f"(1.0f + e));
    return a.cap_a * q;
  };
  // z / r as z * (1 / r): two roundings in place of one
  auto penalty = [&](float z, uint32_t c) -> float {
    if (c) z *= z > 0.f ? ir : rep;
    const uint32_t k = c & ~ADJ_PROMPT;
    return k ? z - (freq * (float)k + pres) : z;
  };
  auto biased = [&](float z, uint32_t w) -> float { return w ? z + a.bias[b * a.bias_stride + w - 1] : z; };
#pragma unroll
  for (int g = 0; g < GR; ++g) {
    const int at = 4 * (tid + g * TH), v = run + at;
    uint4 c = make_uint4(0u, 0u, 0u, 0u), w = c;
    if (counted) c = *reinterpret_cast<const uint4*>(&cnt[at + 4]);
    if constexpr (BIAS) w = *reinterpret_cast<const uint4*>(&which[at + 4]);
    float z[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) z[e] = cap(to_f32<TI>(in[g].v[e]));
    if (c.x | c.y | c.z | c.w) z[0] = penalty(z[0], c.x), z[1] = penalty(z[1], c.y), z[2] = penalty(z[2], c.z), z[3] = penalty(z[3], c.w);
    if constexpr (BIAS)
      if (w.x | w.y | w.z | w.w) z[0] = biased(z[0], w.x), z[1] = biased(z[1], w.y), z[2] = biased(z[2], w.z), z[3] = biased(z[3], w.w);
    Four<TO> res;
#pragma unroll
    for (int e = 0; e < 4; ++e) res.v[e] = from_f32<TO>(on[g] >> e & 1u ? z[e] : -INFINITY);
    if (VEC && v + 4 <= a.V) {
      *reinterpret_cast<Four<TO>*>(out + v) = res;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (v + e < a.V) out[v + e] = res.v[e];
    }
  }
  if (VEC && blockIdx.y == 0 && tid < lead) {
    float z = cap(to_f32<TI>(x[tid]));
    if (counted) z = penalty(z, cnt[4 - lead + tid]);
    if constexpr (BIAS) z = biased(z, which[4 - lead + tid]);
    out[tid] = from_f32<TO>(!a.allowed || bits[0] >> tid & 1u ? z : -INFINITY);
  }
}

template <typename TI, typename TO, int TH, int GR>
static void launch_adjust(const uv_adjust_args& a, bool vec, cudaStream_t st) {
  constexpr int RUN = 4 * GR * TH;
  const dim3 grid(a.B * a.T, (a.V + RUN - 1) / RUN);              // (the entries before the first group only shorten the last run)
  if (vec && a.n_bias) adjust_kernel<TI, TO, TH, GR, true, true><<<grid, TH, 0, st>>>(a);
  else if (vec) adjust_kernel<TI, TO, TH, GR, true, false><<<grid, TH, 0, st>>>(a);
  else if (a.n_bias) adjust_kernel<TI, TO, TH, GR, false, true><<<grid, TH, 0, st>>>(a);
  else adjust_kernel<TI, TO, TH, GR, false, false><<<grid, TH, 0, st>>>(a);
}
// groups of 4 entries are aligned in x and in out at the same places of every row
template <typename TI, typename TO>
static bool groups_meet(const uv_adjust_args& a) {
  const uintptr_t xi = reinterpret_cast<uintptr_t>(a.x), oi = reinterpret_cast<uintptr_t>(a.out);
  return xi % sizeof(TI) == 0 && oi % sizeof(TO) == 0 && ((xi / sizeof(TI) - oi / sizeof(TO)) & 3) == 0 && ((a.sxb - a.sob) & 3) == 0 &&
         ((a.sxt - a.sot) & 3) == 0;
}
template <typename TI, typename TO>
static int adjust_types(const uv_adjust_args& a, cudaStream_t st) {
  const bool vec = groups_meet<TI, TO>(a);
  // runs of 4096 entries where they fill the device twice, so that fewer blocks read the text; 1024 where there are few rows.  One row of
  // 16384: 6.1 us in runs of 4096, 4.3 of 1024; 63 rows of 50257 (819 runs of 4096) 10.5 and 13.3; 512 rows of 16384 26.4 and 33.6
  if ((int64_t)a.B * a.T * ((a.V + 4095) / 4096) >= 2 * sm_count()) launch_adjust<TI, TO, 256, 4>(a, vec, st);
  else launch_adjust<TI, TO, 128, 2>(a, vec, st);
  return check_launch();
}
template <typename TI>
static int adjust_out(const uv_adjust_args& a, cudaStream_t st) {
  switch (a.out_dtype) {
    case UV_F32: return adjust_types<TI, float>(a, st);
    case UV_F16: return adjust_types<TI, __half>(a, st);
    case UV_BF16: return adjust_types<TI, __nv_bfloat16>(a, st);
    default: return UV_ERR_DTYPE;
  }
}

}  // namespace uv

extern "C" int uv_adjust_logits(const uv_adjust_args* a, void* stream) {
  using namespace uv;
  if (!a) return UV_ERR_ARG;
  if (a->B == 0 || a->T == 0 || a->V == 0) return UV_OK;
  if (!a->x || !a->out || a->B < 0 || a->T < 0 || a->V < 0 || a->n_bias < 0 || a->history_len < 0) return UV_ERR_ARG;
  if ((a->parents && !a->tokens) || (a->n_bias && (!a->bias_ids || !a->bias))) return UV_ERR_ARG;
  if (a->history && a->hist_bytes != 4 && a->hist_bytes != 8) return UV_ERR_DTYPE;
  if (a->parents && a->T > TREE_MAX) return UV_ERR_SHAPE;
  if ((int64_t)a->B * a->T > INT32_MAX || a->V > 65535 * 1024) return UV_ERR_SHAPE;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (a->x_dtype) {
    case UV_F32: return adjust_out<float>(*a, st);
    case UV_F16: return adjust_out<__half>(*a, st);
    case UV_BF16: return adjust_out<__nv_bfloat16>(*a, st);
    default: return UV_ERR_DTYPE;
  }
}
