// Attention of a tree of drafted tokens with many query rows, on the tcgen05 tensor cores.
//
// A unit of work is 128 query rows of one (batch row, kv head); its tiles are the tree's own nodes and then the cached keys, 64 a tile.
// (Up to 64 rows stand in both halves of the lanes, of which one takes the tiles of even number and the other those of odd number, each
// with a reference, a sum and an accumulator of its own, joined at the unit's end: 256 rows of 8 nodes of 8 heads over 64 .. 2304 positions
// take 53 us in place of 56.)
// All tiles of a launch form one sequence (rows of any length side by side), which is cut into equal pieces for the CTAs: two
// CTAs per multiprocessor (one for head dimensions over 64), each with its own accumulators, so that one's softmax runs under the other's
// copies and products.
//
//   four converter warps   two for keys, two for values: codes into a ring of shared memory (each thread its own 16-byte pieces, three
//                          tiles ahead), from there as fp16 (exact) into the 128-byte swizzled operand tiles, keys K-major, values
//                          MN-major.  Node keys and values are quantised here, in place.
//   one warp               issues S = Q K^T (128 x 64) and O += P V (128 x head_dim), accumulators in TMEM, two S buffers; Q and P are A
//                          operands in TMEM, so that shared memory feeds one operand only
//   eight softmax warps    16 rows each, S in the fragment layout (a lane has 16 keys of 2 rows, so that it reads a quarter of the tile's
//                          scales), running reference, weights as fp16 back into TMEM over S; O is rescaled only when a reference
//                          grows by more than 2^6
//
// A unit that lies in one piece is finished there; the others leave partial O, reference and sum in the workspace, and a second
// launch merges them.  Arithmetic as in tree_attn.cu, with the reference score + the tile's largest log2(value scale) - 8 on tiles that
// every row sees in full: a weight times its value scale is at most 2^15, and what fp16 cannot hold is below 2^-22 of that.
//
// What bounds it: the issue of instructions, 3880 a warp-tile of 128 rows (0.71 us a tile of a multiprocessor with two CTAs, 87 % of the
// slots), 2590 of 64 rows (0.58 us, 61 %); the softmax's own arithmetic is 1640 of them, conversion some 900, the rest barriers and
// bookkeeping.  Around the tiles 12 us (ranges, queries, the first conversion, the epilogue), with units in pieces 30.  Measured, 8 heads of
// 64 over one kv head: 64 rows of 16 nodes over 8192 positions 72 us (0.99 TB/s, 239 TFLOP/s), 256 rows of 8 nodes over 64 .. 2304 positions
// 53 (the longest row's 37 tiles); 2 x 128 under 4 heads each, 3 rows of 61 nodes over 20001 .. 60007 positions 87 (346 TFLOP/s):
// 244 query rows of a kv head are two units, each of which copies and converts the same keys and values for itself.
//
// What does not run for every tile is kept small (rolled loops, functions out of line): a CTA runs most of it once, and then a
// line of instructions costs its fetch, not its execution.
#include "tree_attn.cuh"

namespace uv {

constexpr int TT_TILE = 64, TT_ROWS = 128;
constexpr int TT_SOFT = 256, TT_CONV = 64, TT_THREADS = TT_SOFT + 2 * TT_CONV + 32;   // softmax 0-7, keys 8-9, values 10-11, MMA warp 12
constexpr int TT_NK = 3, TT_NRAW = 4, TT_NSC = 8;      // operand tiles, raw tiles, tiles of scales
constexpr float TT_LIFT = 8.0f;
constexpr uint32_t TT_O = 2 * TT_TILE;                 // TMEM columns: S 2 x 64, O, Q

__device__ __forceinline__ bool likely(bool x) { return __builtin_expect(x, true); }

// Waits for the phase of that parity.  When one wait of the CTA runs out, all others return at once: the roles run to their ends over
// whatever is in their (own, in-bounds) buffers, and the CTA reports no result.
__device__ __noinline__ void tt_wait_long(uint32_t bar, uint32_t parity, int* dead) {
  unsigned long long begin = 0;
  while (*reinterpret_cast<volatile int*>(dead) == 0) {
    for (int i = 0; i < 1024; ++i)
      if (tc_mbar_try_wait(bar, parity)) return;
    unsigned long long now;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(now));
    if (begin == 0) begin = now;
    else if (now - begin > TC_WAIT_NS) *reinterpret_cast<volatile int*>(dead) = 1;
  }
}
__device__ __forceinline__ void tt_wait(uint64_t& bar, uint32_t parity, int& dead) {
  const uint32_t addr = tc_smem_u32(&bar);
  int tries = 0;
  while (!tc_mbar_try_wait(addr, parity))             // (in place: what wakes here is on the critical path)
    if (!likely(++tries != 4096)) {
      tt_wait_long(addr, parity, &dead);
      break;
    }
}
// the same for a role that runs ahead of the others: its looks leave the issue slots to them
__device__ __forceinline__ void tt_wait_calm(uint64_t& bar, uint32_t parity, int& dead) {
  const uint32_t addr = tc_smem_u32(&bar);
  int tries = 0;
  while (!tc_mbar_try_wait(addr, parity)) {
    __nanosleep(100);
    if (!likely(++tries != 256)) {
      tt_wait_long(addr, parity, &dead);
      break;
    }
  }
}
__device__ __noinline__ int64_t tt_mod(int64_t a, int64_t b) { return a % b; }

template <int HD> struct TcSmem {
  static constexpr int BLK = HD > 64 ? 2 : 1;              // 64-element column blocks of 128 bytes
  static constexpr int CTAS = HD > 64 ? 1 : 2;             // of a multiprocessor
  static constexpr uint32_t COLS = HD > 64 ? 512 : 256, Q = TT_O + (HD > 64 ? 128 : 64);    // TMEM columns, the query operand's
  static constexpr int TILE = BLK * TT_TILE * 128;
  static constexpr int K = 0, V = TT_NK * TILE;            // [NK] tiles each
  static constexpr int SC = V + TT_NK * TILE;              // [NSC] scales: key scale * softmax scale, value scale, fp32
  static constexpr int RAW = SC + TT_NSC * TT_TILE * 8;    // keys, then values: [NRAW] codes and fp16 scales
  static constexpr int RSC = TT_TILE * HD, RBYTES = RSC + 2 * TT_TILE;
  static constexpr int BYTES = RAW + 2 * TT_NRAW * RBYTES;
  // two tiles at a time: the second accumulator's columns behind the first one's; with head_dim 64 the columns are all taken then, and
  // the query operand stands in shared memory
  static constexpr uint32_t O2 = HD > 64 ? 192 : HD == 64 ? 64 : 32;
  static constexpr int QS = (BYTES + 1023) / 1024 * 1024, DUAL_BYTES = HD == 64 ? QS + TT_ROWS * 128 : BYTES;
};

struct Piece {
  int b, kh, rt;
  int n;                   // tiles of the unit: 1 + cached ones; 0: no piece
  int t0, t1, g;           // this piece's; its first one's number in the sequence
  RowRange rg;
  int64_t base;            // position of the first cached tile's first key
};
struct TcRow {
  uint64_t near;           // the ancestors that the row's node sees
  int lo;                  // first cached position it sees, from the unit's first tile on
};
struct TcShared {
  uint64_t kv_full[2][TT_NK], kv_empty[2][TT_NK], p_full[2], s_full[TT_NSC], o_done[2], piece_full, q_full;   // s_full: the products and both scales
  uint64_t drained;                    // every product issued so far, where the CTA gives up
  int lv_max[TT_NSC];                  // floor(log2) of a tile's largest value scale
  uint32_t tmem;
  int dead;
  Piece piece[2];                      // the softmax warps': the warp that issues the products writes them, ahead of time
  TreeSets sets;
  TcRow row[TT_ROWS];                  // by TMEM lane, like f, m, l
  float f[TT_ROWS];                    // the power of two taken out of the query row
  float m[TT_ROWS], l[TT_ROWS], amax[2][TT_ROWS];
  int begin, end, b0, before_b0;       // this CTA's tiles; the batch row that this CTA's pieces begin in, its first tile, and its range
  RowRange rg0;
};

// the sequence of all tiles: batch rows in order, of each its kv heads, of each its blocks of 128 query rows, of each n tiles (the host
// has made sure that they are fewer than 2^31)
struct TcWork {
  int begin, end;          // this CTA's tiles
};
// cached tiles begin at an even position, so that scales can be copied in pairs
__device__ __forceinline__ int64_t tile_base(const RowRange& r) { return r.lo & ~(int64_t)1; }
__device__ __forceinline__ int row_tiles(const RowRange& r) { return 1 + (r.hi >= r.lo ? (int)((r.hi - tile_base(r)) / TT_TILE) + 1 : 0); }

struct PieceWalk {
  const TreeParams& P;
  int RT, b, n;
  int g, end, first;       // next tile; end of the CTA's; first tile of batch row b
  RowRange rg;
  __device__ __forceinline__ PieceWalk(const TreeParams& p, const TcShared& sh, const TcWork& w)
      : P(p), RT((p.M + TT_ROWS - 1) / TT_ROWS), b(sh.b0), n(row_tiles(sh.rg0)), g(w.begin), end(w.end), first(sh.before_b0), rg(sh.rg0) {}
  __device__ __noinline__ bool next(Piece& pc) {
    if (g >= end) return false;
    const int per = n * P.a.KH * RT;
    if (g >= first + per) {
      first += per, ++b;
      rg = row_range(P.a, b), n = row_tiles(rg);
    }
    const unsigned at = (unsigned)(g - first), u = at < (unsigned)n ? 0u : at / (unsigned)n;
    pc.b = b, pc.kh = RT > 1 ? (int)u / RT : (int)u, pc.rt = (int)u - pc.kh * RT, pc.n = n, pc.rg = rg, pc.base = tile_base(rg);
    pc.t0 = (int)(at - u * (unsigned)n);
    pc.t1 = min(n, pc.t0 + (end - g)), pc.g = g;
    g += pc.t1 - pc.t0;
    return true;
  }
};

__device__ __forceinline__ uint64_t tc_desc_mn(uint32_t addr, uint32_t block_bytes) {
  uint64_t d = 0;
  d |= (uint64_t)((addr & 0x3ffffu) >> 4);
  d |= (uint64_t)(block_bytes >> 4) << 16;        // between 64-element blocks of the MN dimension
  d |= (uint64_t)(1024 >> 4) << 32;               // between groups of 8 along K
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;                         // 128-byte swizzle
  return d;
}
__device__ __forceinline__ void tc_mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// row per lane, 8 columns
__device__ __forceinline__ void tc_ld8(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];\n\ttcgen05.wait::ld.sync.aligned;"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr)
               : "memory");
}
// fragment layout, 16 rows: for each group j of 8 columns, lane 4 r + c has columns 8 j + 2 c, + 1 of rows r (registers 4 j, 4 j + 1) and
// r + 8 (4 j + 2, 4 j + 3)
__device__ __forceinline__ void tc_ld_frag64(uint32_t taddr, float2 (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x8.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=f"(r[0].x), "=f"(r[0].y), "=f"(r[1].x), "=f"(r[1].y), "=f"(r[2].x), "=f"(r[2].y), "=f"(r[3].x), "=f"(r[3].y), "=f"(r[4].x),
        "=f"(r[4].y), "=f"(r[5].x), "=f"(r[5].y), "=f"(r[6].x), "=f"(r[6].y), "=f"(r[7].x), "=f"(r[7].y), "=f"(r[8].x), "=f"(r[8].y),
        "=f"(r[9].x), "=f"(r[9].y), "=f"(r[10].x), "=f"(r[10].y), "=f"(r[11].x), "=f"(r[11].y), "=f"(r[12].x), "=f"(r[12].y),
        "=f"(r[13].x), "=f"(r[13].y), "=f"(r[14].x), "=f"(r[14].y), "=f"(r[15].x), "=f"(r[15].y)
      : "r"(taddr)
      : "memory");
}
// 16 columns in the fragment layout
__device__ __forceinline__ void tc_ld_frag16(uint32_t taddr, float (&r)[8]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tc_st_frag16(uint32_t taddr, const float (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.16x256b.x2.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "f"(r[0]), "f"(r[1]), "f"(r[2]),
               "f"(r[3]), "f"(r[4]), "f"(r[5]), "f"(r[6]), "f"(r[7])
               : "memory");
}
// fp16 pairs of the fragment layout, 32 columns of 32 bits: register 2 j is row r, 2 j + 1 row r + 8, column 4 j + c
__device__ __forceinline__ void tc_st_pairs32(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.16x128b.x8.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
// row per lane, 4 columns
__device__ __forceinline__ void tc_st4(uint32_t taddr, const uint32_t (&r)[4]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3])
               : "memory");
}
// address of 16-byte unit `unit` (8 fp16 elements) of row `row` of an operand tile whose column blocks have `rows` rows
__device__ __forceinline__ uint32_t swz(uint32_t base, int rows, int row, int unit) {
  return base + (unit >> 3) * rows * 128 + row * 128 + (((unit & 7) ^ (row & 7)) << 4);
}
__device__ __forceinline__ void sts128(uint32_t addr, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
// two 32-bit operations in one instruction
__device__ __forceinline__ float2 mul2(float2 x, float2 y) {
  float2 r;
  asm("mul.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<uint64_t&>(r))
      : "l"(reinterpret_cast<uint64_t&>(x)), "l"(reinterpret_cast<uint64_t&>(y)));
  return r;
}
__device__ __forceinline__ float2 fma2(float2 x, float2 y, float2 z) {
  float2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<uint64_t&>(r))
      : "l"(reinterpret_cast<uint64_t&>(x)), "l"(reinterpret_cast<uint64_t&>(y)), "l"(reinterpret_cast<uint64_t&>(z)));
  return r;
}
__device__ __forceinline__ float2 add2(float2 x, float2 y) {
  float2 r;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<uint64_t&>(r))
      : "l"(reinterpret_cast<uint64_t&>(x)), "l"(reinterpret_cast<uint64_t&>(y)));
  return r;
}
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}
__device__ __forceinline__ int scale_exponent(float v) { return max((int)((__float_as_uint(v) >> 23) & 0xff) - 127, -24); }
__device__ __forceinline__ void soft_bar() { asm volatile("bar.sync 1, 256;" ::: "memory"); }
__device__ __forceinline__ bool soft_any(bool x) {
  int any;
  asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %1, 0;\n\tbarrier.cta.red.or.aligned.pred q, 1, 256, p;\n\tselp.b32 %0, 1, 0, q;\n\t}" : "=r"(any) : "r"((int)x) : "memory");
  return any != 0;
}
// the query row of a TMEM lane: 16 rows to each warp quadrant first, so that up to 64 rows keep all four schedulers busy
__device__ __forceinline__ int row_of_lane(int l) { return (l >> 4 & 1) * 64 + (l >> 5) * 16 + (l & 15); }
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool on) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}
template <typename QT>
__device__ __forceinline__ float abs_max8(uint4 raw) {
  const QT* x = reinterpret_cast<const QT*>(&raw);
  float m = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) m = fmaxf(m, fabsf(to_f32<QT>(x[e])));
  return m;
}

// ------------------------------------------------------------------------------------------------ converter warps
// 16 codes as fp16 into their two places in an operand tile
__device__ __forceinline__ void store16(uint32_t lo, uint32_t hi, uint4 c) {
  const uint32_t w[4] = {c.x ^ 0x80808080u, c.y ^ 0x80808080u, c.z ^ 0x80808080u, c.w ^ 0x80808080u};
  sts128(lo, bias_pair(w[0], 0x4140), bias_pair(w[0], 0x4342), bias_pair(w[1], 0x4140), bias_pair(w[1], 0x4342));
  sts128(hi, bias_pair(w[2], 0x4140), bias_pair(w[2], 0x4342), bias_pair(w[3], 0x4140), bias_pair(w[3], 0x4342));
}

// The keys (V = 0) or the values (V = 1) of this CTA's tiles, by 64 threads.
template <typename QT, int HD>
__device__ __forceinline__ void convert_tiles(const TreeParams& P, TcShared& sh, const TcWork& w, unsigned char* smem, int V, int tid) {
  using M = TcSmem<HD>;
  constexpr int CH = HD / 16, PIECES = TT_TILE * CH, NC = PIECES / TT_CONV;     // 16-code pieces of a vector, of a tile, of a thread
  static_assert(NC * TT_CONV == PIECES, "");
  const uv_tree_attn_args& a = P.a;
  const int lane = tid & 31;
  const uint32_t tiles = tc_smem_u32(smem) + (V ? M::V : M::K);
  unsigned char* const ring = smem + M::RAW + V * TT_NRAW * M::RBYTES;
  // what is asked for from the cache; vectors of consecutive slots next to each other and scales in pairs on 4-byte boundaries are
  // the quick way
  const int8_t* const codes = V ? a.v_cache : a.k_cache;
  const uint16_t* const scales = V ? a.v_scale : a.k_scale;
  const int64_t cb = V ? a.svb : a.skb, chd = V ? a.svh : a.skh, cs = V ? a.svs : a.sks, sb = V ? a.stb : a.ssb, shd = V ? a.sth : a.ssh;
  const bool quick = cs == HD && (reinterpret_cast<uintptr_t>(scales) & 3) == 0 && ((sb | shd) & 1) == 0 && (!a.ring || (a.S & 1) == 0);
  const float by = V ? 1.0f : P.scale_log2;
  // requests run TT_NRAW - 1 tiles ahead of the conversion
  PieceWalk ahead(P, sh, w), walk(P, sh, w);
  Piece pa, pc;
  const int8_t* kb = nullptr;
  const uint16_t* ks = nullptr;
  int64_t slot = 0;
  int left = 0, ta = 0, ea = 0, t = 0, end = 0;
  uint32_t stage_a = 0, stage = 0, op = 0, phase = 1, at = 0;
  const int total = w.end - w.begin;
  // piece n of this thread: key key0 + n STEP (a multiple of 8, so that the swizzle is the same for all of them)
  constexpr int STEP = TT_CONV / CH;
  const int key0 = (unsigned)tid / CH, ch0 = (unsigned)tid % CH;
  const uint32_t place0 = swz(tiles, TT_TILE, key0, 2 * ch0), place1 = swz(tiles, TT_TILE, key0, 2 * ch0 + 1);
#pragma unroll 1
  for (int i = 1 - TT_NRAW; i < total; ++i) {
    // ---- request
    if (!likely(ta != ea)) {
      if (ahead.next(pa)) {
        ta = pa.t0, ea = pa.t1;
        kb = codes + pa.rg.row * cb + pa.kh * chd, ks = scales + pa.rg.row * sb + pa.kh * shd;
        const int64_t p = pa.base + (int64_t)(ta > 0 ? ta - 1 : 0) * TT_TILE;
        slot = a.ring ? tt_mod(p, a.S) : p;
        left = (int)min((int64_t)INT32_MAX, pa.rg.hi - p + 1);
      } else {
        ta = -1, ea = -2;                                         // nothing is left
      }
    }
    if (ta > 0) {
      unsigned char* const raw = ring + stage_a * M::RBYTES;
      const uint32_t st = tc_smem_u32(raw);
      if (likely(quick && (!a.ring || slot + TT_TILE <= a.S))) {
        const int8_t* src = kb + slot * HD + tid * 16;
        if (likely(left >= TT_TILE)) {
#pragma unroll
          for (int n = 0; n < NC; ++n)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(st + tid * 16 + n * TT_CONV * 16), "l"(src + n * TT_CONV * 16) : "memory");
        } else {
#pragma unroll 1
          for (int n = 0; n < NC; ++n) {
            const bool on = key0 + n * STEP < left;
            copy16(st + (tid + n * TT_CONV) * 16, on ? src + n * TT_CONV * 16 : kb, on);
          }
        }
        if (tid < 32) {
          const int n = min(max(left - 2 * tid, 0), 2) * 2;
          asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(st + M::RSC + tid * 4), "l"(ks + (n ? slot + 2 * tid : 0)), "r"(n)
                       : "memory");
        }
      } else {
        // rings that end inside the tile, other strides and alignments
        auto slot_of = [&](int key) -> int64_t {
          const int64_t x = slot + key;
          return !a.ring || x < a.S ? x : tt_mod(x, a.S);
        };
#pragma unroll 1
        for (int c = tid; c < PIECES; c += TT_CONV) {
          const bool on = c / CH < left;
          copy16(st + c * 16, kb + slot_of(on ? c / CH : 0) * cs + c % CH * 16, on);
        }
        if (tid < 32)
#pragma unroll 1
          for (int e = 2 * tid; e < 2 * tid + 2; ++e) reinterpret_cast<uint16_t*>(raw + M::RSC)[e] = e < left ? ks[slot_of(e)] : (uint16_t)0;
      }
      slot += TT_TILE, left -= TT_TILE;
      if (!likely(!a.ring || slot < a.S)) slot = tt_mod(slot, a.S);
    }
    if (ta >= 0) ++ta;
    asm volatile("cp.async.commit_group;" ::: "memory");
    stage_a = (stage_a + 1) % TT_NRAW;
    if (i < 0) continue;
    // ---- convert
    if (!likely(t != end)) {
      walk.next(pc);
      t = pc.t0, end = pc.t1;
    }
    const uint32_t tile = tiles + op * M::TILE;
    float* const sc = reinterpret_cast<float*>(smem + M::SC) + at * 2 * TT_TILE + V * TT_TILE;
    if (likely(t > 0)) {
      asm volatile("cp.async.wait_group %0;" ::"n"(TT_NRAW - 1) : "memory");
      const unsigned char* raw = ring + stage * M::RBYTES;
      uint4 c[NC];
#pragma unroll
      for (int n = 0; n < NC; ++n) c[n] = reinterpret_cast<const uint4*>(raw)[tid + n * TT_CONV];
      tt_wait_calm(sh.kv_empty[V][op], phase, sh.dead);
      if (tid < 32) {
        const float2 x = __half22float2(reinterpret_cast<const __half2*>(raw + M::RSC)[tid]);
        reinterpret_cast<float2*>(sc)[tid] = make_float2(x.x * by, x.y * by);
        const int e = __reduce_max_sync(0xffffffffu, max(scale_exponent(x.x), scale_exponent(x.y)));
        if (V && tid == 0) sh.lv_max[at] = e;
      }
      const uint32_t shift = op * M::TILE;
#pragma unroll
      for (int n = 0; n < NC; ++n) store16(place0 + shift + n * STEP * 128, place1 + shift + n * STEP * 128, c[n]);
    } else {
      // the tree's own keys or values, in place: as they are, then quantised as the cache would, codes as fp16
      constexpr int LV = HD / 8, PER = TT_CONV / LV;              // lanes of a vector, vectors a pass
      const int sub = tid / LV, part = tid % LV;
      const QT* src = static_cast<const QT*>(V ? a.v : a.k) + (int64_t)pc.b * (V ? a.snvb : a.snkb) + (int64_t)pc.kh * (V ? a.snvh : a.snkh) + 8 * part;
      const int64_t step = V ? a.snvt : a.snkt;
      tt_wait(sh.kv_empty[V][op], phase, sh.dead);
      const int some = (a.T + PER - 1) / PER * PER;               // the passes that hold nodes
#pragma unroll 2
      for (int j = sub; j < some; j += PER) copy16(swz(tile, TT_TILE, j, part), src + (j < a.T ? j * step : 0), j < a.T);
#pragma unroll 2
      for (int j = sub + some; j < TT_TILE; j += PER) {
        sts128(swz(tile, TT_TILE, j, part), 0u, 0u, 0u, 0u);
        if (part == 0) sc[j] = 0.f;
      }
      asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 0;" ::: "memory");
#pragma unroll 2
      for (int j = sub; j < some; j += PER) {
        const uint32_t addr = swz(tile, TT_TILE, j, part);
        uint4 raw;
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(raw.x), "=r"(raw.y), "=r"(raw.z), "=r"(raw.w) : "r"(addr) : "memory");
        float amax = abs_max8<QT>(raw);
#pragma unroll
        for (int o = LV / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        const float s16 = __half2float(__float2half_rn(__fdiv_rn(amax, 127.0f))), sf = fmaxf(s16, 1e-30f), inv = __frcp_rn(sf);
        const QT* x = reinterpret_cast<const QT*>(&raw);
        uint32_t y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = pack_h2(cache_code(to_f32<QT>(x[2 * e]), sf, inv), cache_code(to_f32<QT>(x[2 * e + 1]), sf, inv));
        sts128(addr, y[0], y[1], y[2], y[3]);
        if (part == 0) sc[j] = s16 * by;
      }
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    if (lane == 0) mbar_arrive_one(tc_smem_u32(&sh.s_full[at])), mbar_arrive_one(tc_smem_u32(&sh.kv_full[V][op]));
    ++t;
    stage = (stage + 1) % TT_NRAW, at = (at + 1) % TT_NSC;
    if (++op == TT_NK) op = 0, phase ^= 1;
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

// ------------------------------------------------------------------------------------------------ softmax of a tile that not every row sees in full
// x: the scores of two rows (TMEM lanes row, row + 8) in the fragment layout, -infinity afterwards where a row does not see the key; mx:
// the largest score + log2(value scale) - lift of each among the lane's columns.
__device__ __forceinline__ void mask_scores(const TcShared& sh, float2 (&x)[16], float (&mx)[2], const float2* vf, const float (&fk)[2],
                                            int row, int fc, int p0, int last0) {
  uint32_t on[2][2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const TcRow& rw = sh.row[row + 8 * e];
    uint64_t bits = rw.near;
    if (p0 >= 0) {
      const int first = rw.lo - p0, last = last0 - p0;
      bits = first >= TT_TILE ? 0ull : ~0ull << max(first, 0);
      if (last < TT_TILE - 1) bits &= ~0ull >> (TT_TILE - 1 - last);
    }
    bits >>= 2 * fc;
    on[e][0] = (uint32_t)bits, on[e][1] = (uint32_t)(bits >> 32);
  }
#pragma unroll
  for (int g = 0; g < 8; ++g) {
    const float2 v2 = vf[4 * g];
    const float lx = (float)scale_exponent(v2.x) - TT_LIFT, ly = (float)scale_exponent(v2.y) - TT_LIFT;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float2& y = x[2 * g + e];
      if (!(on[e][g / 4] & (1u << (8 * (g & 3))))) y.x = -INFINITY;
      if (!(on[e][g / 4] & (2u << (8 * (g & 3))))) y.y = -INFINITY;
      mx[e] = fmaxf(mx[e], fmaxf(fmaf(y.x, fk[e], lx), fmaf(y.y, fk[e], ly)));
    }
  }
}

// ------------------------------------------------------------------------------------------------ kernel
template <typename QT, int HD, bool DUAL>
__global__ void __launch_bounds__(TT_THREADS, TcSmem<HD>::CTAS) tree_tc_kernel(const __grid_constant__ TreeParams P, int ctas, int split, int2* meta,
                                                                              float* ws_o, float* ws_ml) {
  using M = TcSmem<HD>;
  constexpr bool Q_SMEM = DUAL && HD == 64;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* const smem = smem_raw + ((1024u - (tc_smem_u32(smem_raw) & 1023u)) & 1023u);
  __shared__ TcShared sh;
  __shared__ int scan[TT_THREADS / 32];
  const uv_tree_attn_args& a = P.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int RT = (P.M + TT_ROWS - 1) / TT_ROWS, units_b = a.KH * RT;

  // ---- the tiles of every batch row; this CTA's share of the sequence and the batch row that it begins in
  auto tiles_of = [&](int b) { return b < a.B ? row_tiles(row_range(a, b)) * units_b : 0; };
  RowRange rg{};
  if (tid < a.B) rg = row_range(a, tid);
  int mine = tid < a.B ? row_tiles(rg) * units_b : 0, sum = mine;
#pragma unroll 1
  for (int b = tid + TT_THREADS; b < a.B; b += TT_THREADS) sum += tiles_of(b);
  if (tid == 0) {
    uint64_t* bar = &sh.kv_full[0][0];
#pragma unroll 1
    for (int i = 0; i < (int)(offsetof(TcShared, lv_max) / 8); ++i) {
      const int at = i * 8;
      int count = 1;                                                                 // a commit of the MMA warp
      if (at < (int)offsetof(TcShared, kv_empty)) count = 2;                          // the converter warps of keys or of values
      else if (at >= (int)offsetof(TcShared, p_full) && at < (int)offsetof(TcShared, s_full)) count = DUAL ? 4 : TT_SOFT / 32;
      else if (at >= (int)offsetof(TcShared, s_full) && at < (int)offsetof(TcShared, o_done)) count = 1 + 4;
      else if (at == (int)offsetof(TcShared, q_full)) count = TT_SOFT / 32;
      tc_mbar_init(tc_smem_u32(bar + i), count);
    }
    sh.dead = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 12) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc_smem_u32(&sh.tmem)), "r"(M::COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  sum = __reduce_add_sync(0xffffffffu, sum);
  if (lane == 0) scan[warp] = sum;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const int total = __reduce_add_sync(0xffffffffu, lane < TT_THREADS / 32 ? scan[lane] : 0);
  // Cut into units, or, with `split`, into equal runs of at least two tiles: the first `extra` CTAs have one more of them.
  const int all = split ? total : a.B * units_b, G = min(ctas, split ? (total + 1) / 2 : all), cta = blockIdx.x, per = all / G, extra = all - per * G;
  const int from = cta < G ? cta * per + min(cta, extra) : 0, upto = cta < G ? from + per + (cta < extra) : 0;
  int base = 0;
#pragma unroll 1
  for (int b0 = 0; b0 < a.B && from < upto; b0 += TT_THREADS) {                      // (the same in every thread)
    const int b = b0 + tid;
    if (b0 && b < a.B) rg = row_range(a, b);
    if (b0) mine = b < a.B ? row_tiles(rg) * units_b : 0;
    int incl = mine;
#pragma unroll 1
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += x;
    }
    __syncthreads();
    if (lane == 31) scan[warp] = incl;
    __syncthreads();
    const int part = lane < TT_THREADS / 32 ? scan[lane] : 0;
    const int first = base + __reduce_add_sync(0xffffffffu, lane < warp ? part : 0) + incl - mine;
    if (b < a.B) {
      // the tiles at which this CTA begins and ends, where they lie in this row
      const int n = row_tiles(rg), at0 = split ? from - first : (from - b * units_b) * n, at1 = split ? upto - 1 - first : (upto - b * units_b) * n - 1;
      if (at0 >= 0 && at0 < mine) sh.b0 = b, sh.before_b0 = first, sh.rg0 = rg, sh.begin = first + at0;
      if (at1 >= 0 && at1 < mine) sh.end = first + at1 + 1;
    }
    base += __reduce_add_sync(0xffffffffu, part);
  }
  __syncthreads();
  TcWork w{0, 0};
  if (from < upto) w.begin = sh.begin, w.end = sh.end;
  pdl_trigger();
  const uint32_t tmem = sh.tmem, t_o = tmem + TT_O;

  if (w.begin >= w.end) {
    // (nothing to do)
  } else if (warp == 12) {
    // ---- products: the warp runs as one, an elected lane issues
    constexpr uint32_t ID = (1u << 4) | ((uint32_t)(TT_ROWS >> 4) << 24);
    constexpr uint32_t ID_S = ID | ((uint32_t)(TT_TILE >> 3) << 17), ID_O = ID | (1u << 16) | ((uint32_t)(HD >> 3) << 17);
    const uint64_t dk = tc_smem_desc(tc_smem_u32(smem + M::K)), dv = tc_desc_mn(tc_smem_u32(smem + M::V), TT_TILE * 128);
    const uint64_t dq = tc_smem_desc(tc_smem_u32(smem + M::QS));
    PieceWalk walk(P, sh, w);
    Piece pc;
    uint32_t pieces = 0, i = 0, kop = 0, kph = 0, vop = 0, vph = 0;
    bool more = walk.next(pc);
    while (true) {
      if (!more) pc.n = 0;
      if (lane == 0) {
        sh.piece[pieces & 1u] = pc;                               // (the softmax warps have got past the piece that stood there: q_full)
        mbar_arrive_one(tc_smem_u32(&sh.piece_full));
      }
      if (!more) break;
      const int n = pc.t1 - pc.t0;
      more = walk.next(pc);                                       // (looked up while the queries come)
      tt_wait(sh.q_full, pieces & 1u, sh.dead);
      ++pieces;
#pragma unroll 1
      for (int j = 0; j <= n; ++j) {
        if (j < n) {
          tt_wait(sh.kv_full[0][kop], kph, sh.dead);
          tc_fence_after();
          const uint64_t d = dk + (uint64_t)(kop * (M::TILE / 16));
          const uint32_t to = tmem + (i & 1u) * TT_TILE;
          if (elect_one()) {
#pragma unroll
            for (int k = 0; k < HD / 16; ++k) {
              if constexpr (Q_SMEM) tc_mma(to, dq + k * 2, d + k * 2, ID_S, (uint32_t)(k > 0));
              else tc_mma_ts(to, tmem + M::Q + k * 8, d + ((k >> 2) * (TT_TILE * 128 / 16) + (k & 3) * 2), ID_S, (uint32_t)(k > 0));
            }
            tc_commit(tc_smem_u32(&sh.s_full[i % TT_NSC]));
            tc_commit(tc_smem_u32(&sh.kv_empty[0][kop]));
          }
          __syncwarp();
          if (++kop == TT_NK) kop = 0, kph ^= 1;
          ++i;
        }
        if (j > 0) {
          const uint32_t pi = i - 1 - (j < n);                    // the tile before
          tt_wait(sh.kv_full[1][vop], vph, sh.dead);
          tt_wait(sh.p_full[pi & 1u], (pi >> 1) & 1u, sh.dead);
          tc_fence_after();
          const uint64_t d = dv + (uint64_t)(vop * (M::TILE / 16));
          const uint32_t from = tmem + (pi & 1u) * TT_TILE;
          if (elect_one()) {
#pragma unroll
            for (int k = 0; k < TT_TILE / 16; ++k)
              tc_mma_ts(t_o + (DUAL ? (pi & 1u) * M::O2 : 0u), from + k * 8, d + k * (2048 / 16), ID_O, (uint32_t)(j > (DUAL ? 2 : 1) || k > 0));
            tc_commit(tc_smem_u32(&sh.kv_empty[1][vop]));
            tc_commit(tc_smem_u32(&sh.o_done[pi & 1u]));
          }
          __syncwarp();
          if (++vop == TT_NK) vop = 0, vph ^= 1;
        }
      }
    }
  } else if (warp >= 8) {
    convert_tiles<QT, HD>(P, sh, w, smem, (warp - 8) >> 1, (tid - TT_SOFT) & (TT_CONV - 1));
  } else {
    // ---- softmax
    auto wait = [&](uint64_t& bar, uint32_t parity) {
      tt_wait(bar, parity, sh.dead);
      __syncwarp();
    };
    const int quad = warp & 3, slab = warp >> 2;                  // TMEM lanes 32 quad + 16 slab .. + 15
    const uint32_t t_quad = (uint32_t)(32 * quad) << 16, t_slab = t_quad + ((uint32_t)(16 * slab) << 16);
    const int fr = lane >> 2, fc = lane & 3, own = 32 * quad + 16 * slab + fr;         // this lane's rows: TMEM lanes own, own + 8
    const int trow = 32 * quad + lane;                            // thread = row: its TMEM lane (two warps share a quadrant's lanes)
    // DUAL: a row has two lanes, 16 apart; the lower ones take the tiles of even number, the upper ones those of odd number
    auto row_at = [](int l) { return DUAL ? row_of_lane(l) & 63 : row_of_lane(l); };
    const uint32_t t_mine = t_o + t_slab + (DUAL ? slab * M::O2 : 0u);
    uint32_t i = 0;
#pragma unroll 1
    for (uint32_t pieces = 0;; ++pieces) {
      // Everybody is done with what the piece before left in shared memory.  Once a wait has run out, all go at once: a piece may not be
      // there then, or may be overwritten, but not before `dead` can be seen.
      wait(sh.piece_full, pieces & 1u);
      const Piece pc = sh.piece[pieces & 1u];
      if (soft_any(*reinterpret_cast<volatile int*>(&sh.dead) != 0) || pc.n == 0) break;
      const int b = pc.b, kh = pc.kh, t0 = pc.t0, n = pc.t1 - pc.t0, row0 = pc.rt * TT_ROWS;
      const int64_t pos = pc.rg.pos;
      const int lo = (int)(pc.rg.lo - pc.base), last0 = (int)min(pc.rg.hi - pc.base, (int64_t)INT32_MAX);   // (positions from the first tile on)
      const int row = row0 + row_at(trow), t = node_of(P, row), h = kh * P.G + row - t * P.G;
      const bool valid = row < P.M;
      // the query row, half of it: times a power of two, fp16, into the A operand (the last products of the piece before have read the
      // old one: their scores have been waited for)
      constexpr int U = HD / 16;                                  // 16-byte units of a half
      uint4 raw[U];
      const uint4* q = reinterpret_cast<const uint4*>(static_cast<const QT*>(a.q) + (int64_t)b * a.sqb + (int64_t)t * a.sqt + (int64_t)h * a.sqh) + slab * U;
      float amax = 0.f;
#pragma unroll
      for (int u = 0; u < U; ++u) raw[u] = valid ? q[u] : make_uint4(0u, 0u, 0u, 0u);
      if (warp == 4) tree_sets(a.parents + (int64_t)b * a.parents_stride, a.T, sh.sets, lane);
#pragma unroll
      for (int u = 0; u < U; ++u) amax = fmaxf(amax, abs_max8<QT>(raw[u]));
      sh.amax[slab][trow] = amax;
      soft_bar();
      amax = fmaxf(amax, sh.amax[slab ^ 1][trow]);
      int ex = ((int)(__float_as_uint(amax) >> 23) & 0xff) - 127;
      ex = amax > 0.f ? max(ex, -100) : 10;
      const float up = __uint_as_float((uint32_t)(127 + 10 - ex) << 23);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const QT* x = reinterpret_cast<const QT*>(&raw[u]);
        uint32_t y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = pack_h2(to_f32<QT>(x[2 * e]) * up, to_f32<QT>(x[2 * e + 1]) * up);
        if constexpr (Q_SMEM) sts128(swz(tc_smem_u32(smem + M::QS), TT_ROWS, trow, slab * U + u), y[0], y[1], y[2], y[3]);
        else tc_st4(tmem + M::Q + t_quad + 4 * (slab * U + u), y);
      }
      if constexpr (Q_SMEM) {
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      } else {
        tc_wait_st();
        tc_fence_before();
      }
      const uint64_t mask = valid ? sh.sets.mask[t] : 0ull;
      uint64_t near = mask;            // the ancestors within the window
      int lo_row = lo, lo_all = lo;
      if (a.window > 0) {
        const int depth = __popcll(mask) - 1;
#pragma unroll 1
        for (uint64_t left = mask; left; left &= left - 1) {
          const int j = __ffsll((long long)left) - 1;
          if (depth - (__popcll(sh.sets.mask[j]) - 1) >= a.window) near &= ~(1ull << j);
        }
        const int64_t first = pos - a.window + 1 - pc.base;       // what a node of depth 0 sees first
        int deepest = max(__popcll(sh.sets.mask[lane]), __popcll(sh.sets.mask[lane + 32])) - 1;
        deepest = __reduce_max_sync(0xffffffffu, deepest);
        if (mask) lo_row = (int)max((int64_t)lo, first + depth);
        lo_all = (int)max((int64_t)lo, first + deepest);
      }
      if ((lane >> 4) == slab) sh.row[trow] = TcRow{near, lo_row}, sh.f[trow] = __uint_as_float((uint32_t)(127 + ex - 10) << 23);
      __syncwarp();
      if (lane == 0) mbar_arrive_one(tc_smem_u32(&sh.q_full));
      const bool busy = row0 + row_at(32 * quad + 16 * slab) < P.M;               // some row of the slab is one
      float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
      const float fk[2] = {sh.f[own], sh.f[own + 8]};
#pragma unroll 1
      for (int j = 0; j < n; ++j, ++i) {
        if (DUAL && (int)(i & 1u) != slab) continue;
        const int at = (int)(i % TT_NSC), p0 = (t0 + j - 1) * TT_TILE;
        const uint32_t ts = tmem + (i & 1u) * TT_TILE + t_slab;
        wait(sh.s_full[at], (i / TT_NSC) & 1u);
        if (busy) {
          tc_fence_after();
          const float2* kf = reinterpret_cast<const float2*>(smem + M::SC) + at * TT_TILE + fc;      // scales of keys 8 g + 2 fc, + 1
          const float2* vf = kf + TT_TILE / 2;
          const bool whole = p0 >= lo_all && p0 + TT_TILE - 1 <= last0 && p0 >= 0;
          float2 x[16];                                          // x[2 g + e]: keys 8 g + 2 fc, + 1 of row e
          float mx[2] = {-INFINITY, -INFINITY};
          tc_ld_frag64(ts, x);
#pragma unroll
          for (int g = 0; g < 8; ++g) {
            const float2 k2 = kf[4 * g];
            x[2 * g] = mul2(x[2 * g], k2), x[2 * g + 1] = mul2(x[2 * g + 1], k2);
          }
          if (likely(whole)) {
#pragma unroll
            for (int g = 0; g < 16; ++g) mx[g & 1] = fmaxf(mx[g & 1], fmaxf(x[g].x, x[g].y));
            const float lift = (float)sh.lv_max[at] - TT_LIFT;
            mx[0] = fmaf(mx[0], fk[0], lift), mx[1] = fmaf(mx[1], fk[1], lift);
          } else {
            mask_scores(sh, x, mx, vf, fk, own, fc, p0, last0);
          }
          bool raise = false;
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 1));
            mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 2));
            raise = raise || mx[e] > m[e] + RESCALE_GAP;
          }
          if (!likely(!__any_sync(0xffffffffu, raise))) {
            float alpha[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float m_new = mx[e] > m[e] + RESCALE_GAP ? mx[e] : m[e];
              alpha[e] = m_new == -INFINITY ? 1.0f : ex2(m[e] - m_new);
              l[e] *= alpha[e], m[e] = m_new;
            }
            if (j > (DUAL ? 1 : 0)) {                             // the products of this lane's tile before
              const uint32_t k = i - (DUAL ? 2 : 1);
              wait(sh.o_done[k & 1u], (k >> 1) & 1u);
              tc_fence_after();
#pragma unroll 1
              for (int c = 0; c < HD; c += 16) {
                float o[8];
                tc_ld_frag16(t_mine + c, o);
#pragma unroll
                for (int e = 0; e < 8; ++e) o[e] *= alpha[(e >> 1) & 1];
                tc_st_frag16(t_mine + c, o);
              }
            }
          }
          uint32_t pk[16];
          float2 f2[2], n2[2], sum[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float neg = m[e] == -INFINITY ? 0.f : -m[e];
            f2[e] = make_float2(fk[e], fk[e]), n2[e] = make_float2(neg, neg), sum[e] = make_float2(0.f, 0.f);
          }
#pragma unroll
          for (int g = 0; g < 8; ++g) {
            const float2 v2 = vf[4 * g];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float2 q = fma2(x[2 * g + e], f2[e], n2[e]);
              q.x = ex2(q.x), q.y = ex2(q.y);
              sum[e] = add2(sum[e], q);
              const float2 y = mul2(q, v2);
              pk[2 * g + e] = pack_h2(y.x, y.y);
            }
          }
          if (!likely(whole)) {                                  // (a masked scale may be anything: 0 * inf)
#pragma unroll
            for (int g = 0; g < 16; ++g)
              pk[g] &= (x[g].x == -INFINITY ? 0u : 0xffffu) | (x[g].y == -INFINITY ? 0u : 0xffff0000u);
          }
          l[0] += sum[0].x + sum[0].y, l[1] += sum[1].x + sum[1].y;
          tc_st_pairs32(ts, pk);
          tc_wait_st();
          tc_fence_before();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive_one(tc_smem_u32(&sh.p_full[i & 1u]));
      }
      wait(sh.o_done[(i - 1) & 1u], ((i - 1) >> 1) & 1u);
      tc_fence_after();
      // ---- back to thread = row; the two warps of a quadrant take half of its columns each
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float x = l[e];
        x += __shfl_xor_sync(0xffffffffu, x, 1);
        x += __shfl_xor_sync(0xffffffffu, x, 2);
        if (fc == 0) sh.m[own + 8 * e] = m[e], sh.l[own + 8 * e] = x;
      }
      soft_bar();
      const bool dead = sh.dead != 0, whole_unit = n == pc.n;
      float row_m = sh.m[trow], row_l = dead ? 0.f : sh.l[trow], share = 1.0f;         // (dead: NaN, and the status word)
      if (DUAL) {                                                 // both lanes of a row get what the two have seen
        const float both = fmaxf(row_m, __shfl_xor_sync(0xffffffffu, row_m, 16));
        share = row_m == -INFINITY ? 0.f : ex2(row_m - both);
        row_l = part_sum(row_m, share, row_l);
        row_l += __shfl_xor_sync(0xffffffffu, row_l, 16);
        row_m = both;
      }
      auto load8 = [&](int c, uint32_t (&o)[8]) {
        tc_ld8(t_o + t_quad + c, o);
        if constexpr (DUAL) {
          uint32_t o2[8];
          tc_ld8(t_o + M::O2 + t_quad + c, o2);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float y = share > 0.f ? __uint_as_float(lane < 16 ? o[e] : o2[e]) * share : 0.f;   // (a lane without tiles: anything)
            o[e] = __float_as_uint(y + __shfl_xor_sync(0xffffffffu, y, 16));
          }
        }
      };
      const bool writes = !DUAL || lane < 16;
      if (split && t0 == 0 && tid == 0) {
        // the CTA that the unit's last tile lies in
        const int g = pc.g + pc.n - 1, cut = extra * (per + 1);
        meta[((int64_t)b * a.KH + kh) * RT + pc.rt] = make_int2(cta, g < cut ? g / (per + 1) : extra + (g - cut) / per);
      }
      const int64_t to = ((int64_t)2 * cta + (t0 == 0 ? 1 : 0)) * TT_ROWS + row_at(trow);
      if (!whole_unit && slab == 0 && writes) ws_ml[2 * to] = dead ? -INFINITY : row_m, ws_ml[2 * to + 1] = row_l;
      if (row0 + row_of_lane(32 * quad) < P.M) {
        const float inv = whole_unit ? inverse_sum(row_l) : 1.0f;
        const uint4* v = reinterpret_cast<const uint4*>(static_cast<const QT*>(a.v) + (int64_t)b * a.snvb + (int64_t)t * a.snvt + (int64_t)kh * a.snvh);
        float xs = 0.f;                            // XSA: z - xs * v
        const bool xsa = whole_unit && a.xsa_alpha != nullptr;
        if (xsa) {
          float n2 = 0.f, dot = 0.f;
#pragma unroll 1
          for (int c = 0; c < HD; c += 8) {
            uint32_t o[8];
            load8(c, o);
            const uint4 vv = valid ? v[c / 8] : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float y = to_f32<QT>(reinterpret_cast<const QT*>(&vv)[e]);
              n2 += y * y, dot += rnd<QT>(__uint_as_float(o[e]) * inv) * y;
            }
          }
          const float nv = 1.0f / fmaxf(sqrtf(n2), a.xsa_eps);
          if (valid) xs = a.xsa_alpha[h] * dot * nv * nv;
        }
        const float gate = a.gate_vals && valid ? a.gate_vals[((int64_t)b * a.T + t) * a.H + h] : 1.0f;
        QT* out = static_cast<QT*>(a.out) + (int64_t)b * a.sob + (int64_t)t * a.sot + (int64_t)h * a.soh;
#pragma unroll 1
        for (int c = slab * (HD / 2); c < (slab + 1) * (HD / 2); c += 8) {
          uint32_t o[8];
          load8(c, o);
          if (!writes) {
            // (the row's other lane does)
          } else if (!whole_unit) {
            uint4* at = reinterpret_cast<uint4*>(ws_o + to * HD + c);
            at[0] = make_uint4(o[0], o[1], o[2], o[3]), at[1] = make_uint4(o[4], o[5], o[6], o[7]);
          } else if (valid) {
            const uint4 vv = xsa ? v[c / 8] : make_uint4(0u, 0u, 0u, 0u);
            uint4 packed;
            QT* y = reinterpret_cast<QT*>(&packed);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              float z = rnd<QT>(__uint_as_float(o[e]) * inv);
              if (xsa) z = rnd<QT>(z - xs * to_f32<QT>(reinterpret_cast<const QT*>(&vv)[e]));
              y[e] = from_f32<QT>(mask ? z * gate : 0.f);
            }
            reinterpret_cast<uint4*>(out + c)[0] = packed;
          }
        }
      }
      tc_fence_before();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (tid == 0 && sh.dead && a.status) atomicOr(a.status, 1);
  if (warp == 12) {
    if (!likely(sh.dead == 0)) {                 // products may be under way: the CTA does not end before them, or this wait
      if (elect_one()) tc_commit(tc_smem_u32(&sh.drained));
      tc_mbar_wait(tc_smem_u32(&sh.drained), 0u);
      __syncwarp();
    }
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(M::COLS) : "memory");
  }
}

// Units that lie in several pieces: a warp per query row merges their partials.
template <typename QT, int HD>
__global__ void __launch_bounds__(256) tree_tc_merge_kernel(const __grid_constant__ TreeParams P, int ctas, const int2* meta, const float* ws_o,
                                                            const float* ws_ml) {
  constexpr int EPL = (HD + 31) / 32;
  const uv_tree_attn_args& a = P.a;
  const int lane = threadIdx.x & 31, RT = (P.M + TT_ROWS - 1) / TT_ROWS;
  const int u = blockIdx.x, rt = u % RT, kh = u / RT % a.KH, b = u / RT / a.KH;
  const int r = blockIdx.y * 8 + (threadIdx.x >> 5), row = rt * TT_ROWS + r;
  pdl_wait();
  const int2 c = meta[u];
  if (c.x < 0 || c.x >= c.y || c.y >= ctas || row >= P.M) return;          // (finished in one piece; or never written, after a wait that ran out)
  const int32_t* par = a.parents + (int64_t)b * a.parents_stride;
  int up = node_of(P, row);
  while (par[up] >= 0 && par[up] < up) up = par[up];
  auto at = [&](int cta) { return ((int64_t)2 * cta + (cta == c.x ? 1 : 0)) * TT_ROWS + r; };
  float mx = -INFINITY;
#pragma unroll 1
  for (int k = c.x + lane; k <= c.y; k += 32) mx = fmaxf(mx, ws_ml[2 * at(k)]);
  mx = warp_max(mx);
  float lsum = 0.f, z[EPL];
#pragma unroll
  for (int i = 0; i < EPL; ++i) z[i] = 0.f;
#pragma unroll 2
  for (int k = c.x; k <= c.y; ++k) {
    const int64_t w = at(k);
    const float m = ws_ml[2 * w], wt = m == -INFINITY ? 0.f : ex2(m - mx);
    lsum += part_sum(m, wt, ws_ml[2 * w + 1]);
    if (m == -INFINITY) continue;
#pragma unroll
    for (int i = 0; i < EPL; ++i)
      if (HD >= 32 || lane < HD) z[i] += wt * ws_o[w * HD + lane + 32 * i];
  }
  const float inv = inverse_sum(lsum);
#pragma unroll
  for (int i = 0; i < EPL; ++i) z[i] *= inv;
  store_row<QT, HD>(P, z, b, kh, row, par[up] == -1, lane);
}

// ------------------------------------------------------------------------------------------------ host side
static int tc_ctas(int hd) { return (hd > 64 ? 1 : 2) * sm_count(); }
static int64_t tc_units(const uv_tree_attn_args& a) {
  return (int64_t)a.B * a.KH * ((a.T * (a.H / a.KH) + TT_ROWS - 1) / TT_ROWS);
}
static int64_t tc_most_tiles(const uv_tree_attn_args& a) {
  const int64_t ctx = a.window > 0 && a.window < a.S ? a.window : a.S;
  return tc_units(a) * (3 + ctx / TT_TILE);
}
// CTAs of a launch: what the device holds at a time, no more than the longest rows could occupy
static int tc_grid(const uv_tree_attn_args& a, bool split) {
  const int64_t most = split ? tc_most_tiles(a) / 2 + 1 : tc_units(a), fit = tc_ctas(a.hd);
  return (int)(most < fit ? most : fit);
}
// Whole units or runs of tiles, by the cache's length (the rows' own are on the device).  Whole: as long as the longest unit takes, 12 us and 1.25 a tile with one CTA on a multiprocessor, 1.45 with
// two; with two tiles at a time 12 us and 0.78, or 17 us and 1.16.  Runs: 30 us -- partials and the merging launch -- and 0.71 us (two tiles
// at a time 0.55; 0.8 for head_dim 128) a tile of a multiprocessor, whatever the rows' lengths are.  (Measured at 64 to 296 rows of 60 to
// 32768 positions; 120 rows of 8 nodes over 2304: whole 41 us, runs 51.)
static bool tc_splits(const uv_tree_attn_args& a) {
  const bool dual = a.T * (a.H / a.KH) <= TT_ROWS / 2;
  const float units = (float)tc_units(a), fit = (float)tc_ctas(a.hd), n_sm = fit / (a.hd > 64 ? 1 : 2);
  const float tiles = (float)((a.window > 0 && a.window < a.S ? a.window : a.S) / TT_TILE + 1);
  const bool pairs = units > n_sm;
  const float run = !dual ? 0.71f : a.hd > 64 ? 0.8f : 0.55f, whole = dual ? (pairs ? 1.16f : 0.78f) : pairs ? 1.45f : 1.25f;
  return 30.0f + units * tiles * run / n_sm < (dual && pairs ? 17.0f : 12.0f) + ceilf(units / fit) * tiles * whole;
}
// Against the mma.sync kernel of tree_attn.cu, which takes 32 rows a CTA (what it needs grows with head_dim, while this kernel's softmax does
// not): either enough rows and more CTAs of that kernel than the device holds one (head_dim 128), two (64) or three to a multiprocessor, or
// more than 32 rows and very many pairs of such a CTA and a key.  This kernel and that one, us, 8 heads to a kv head:
//   head_dim 64   200 x 8 nodes over 256 positions 23, 31; 2304: 58, 70; 8192: 129, 188; 64 x 8: 18, 18; 42, 30; 65, 65; 64 x 16: 19, 17; 47, 42;
//                 77, 112; 600 x 4 (32 rows): over 512 57, 43; 2304: 140, 100
//   head_dim 128  160 x 4 over 100: 25, 29; 2304: 64, 82; 600 x 4: 55, 71; 179, 207; 160 x 2 (16 rows): 25, 20; 62, 58; 64 x 8 over 8192: 81, 122
//   head_dim 32   160 x 12 over 512: 26, 26; 2304: 57, 55; 600 x 12: 58, 67; 152, 160; 600 x 8 (64 rows): 49, 43; 123, 109; 160 x 8 over
//                 16384: 154, 191; 100 x 8: 106, 111
bool tree_tc_wants(const uv_tree_attn_args& a) {
  const int M = a.T * (a.H / a.KH), size = a.hd > 64 ? 0 : a.hd == 64 ? 1 : 2;
  const int64_t rows = (int64_t)a.B * a.KH * ((M + 31) / 32), ctx = a.window > 0 && a.window < a.S ? a.window : a.S;
  const bool many = M > 16 << size && rows > (size + 1) * tc_ctas(128), far = M > 32 && rows * ctx >= 1 << (size == 2 ? 22 : 19 + size);
  return a.num_splits == 0 && (many || far) && tc_most_tiles(a) < INT32_MAX / 2 && (reinterpret_cast<uintptr_t>(a.out) & 15) == 0 &&
         ((a.sob | a.sot | a.soh) & 7) == 0;
}
// [meta: int2 per unit][m, l of 2 partials a CTA][o]
size_t tree_tc_workspace(const uv_tree_attn_args& a) {
  if (!tc_splits(a)) return 0;
  const size_t meta = ((size_t)tc_units(a) * 8 + 255) & ~(size_t)255, rows = (size_t)2 * tc_grid(a, true) * TT_ROWS;
  return meta + rows * 8 + rows * a.hd * 4;
}

template <typename QT, int HD, bool DUAL>
static int launch_tc(const TreeParams& P, cudaStream_t st) {
  auto kern = tree_tc_kernel<QT, HD, DUAL>;
  constexpr int smem = (DUAL ? TcSmem<HD>::DUAL_BYTES : TcSmem<HD>::BYTES) + 1024;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) {
    set_last_cuda_error((int)e);
    return UV_ERR_CUDA;
  }
  const bool split = tc_splits(P.a);
  const int ctas = tc_grid(P.a, split);
  const int64_t units = tc_units(P.a);
  if (units > INT32_MAX) return UV_ERR_SHAPE;
  char* ws = reinterpret_cast<char*>(P.ws_o);
  int2* meta = reinterpret_cast<int2*>(ws);
  float* ml = reinterpret_cast<float*>(ws + (((size_t)units * 8 + 255) & ~(size_t)255));
  float* o = ml + (size_t)4 * ctas * TT_ROWS;
  kern<<<ctas, TT_THREADS, smem, st>>>(P, ctas, split, meta, o, ml);
  const int rc = check_launch();
  if (rc != UV_OK || !split) return rc;
  launch_cluster_pdl(1, tree_tc_merge_kernel<QT, HD>, dim3((unsigned)units, (unsigned)((min(P.M, TT_ROWS) + 7) / 8)), dim3(256), dim3(1, 1, 1), 0,
                     st, P, ctas, meta, o, ml);
  return check_launch();
}
template <typename QT, bool DUAL>
static int launch_tc_hd(const TreeParams& P, cudaStream_t st) {
  switch (P.a.hd) {
    case 16: return launch_tc<QT, 16, DUAL>(P, st);
    case 32: return launch_tc<QT, 32, DUAL>(P, st);
    case 64: return launch_tc<QT, 64, DUAL>(P, st);
    default: return launch_tc<QT, 128, DUAL>(P, st);
  }
}
int launch_tree_tc(const TreeParams& P, cudaStream_t st) {
  if (P.M <= TT_ROWS / 2) return P.a.dtype == UV_F16 ? launch_tc_hd<__half, true>(P, st) : launch_tc_hd<__nv_bfloat16, true>(P, st);
  return P.a.dtype == UV_F16 ? launch_tc_hd<__half, false>(P, st) : launch_tc_hd<__nv_bfloat16, false>(P, st);
}

}  // namespace uv
