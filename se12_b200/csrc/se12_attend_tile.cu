// Attention over the paged cache for many query rows per KV head
// (prompt chunks, drafted tokens of wide groups): tiles of 128 query rows on
// the tensor cores.
//
// The same sums as attend_rows_kernel. A row tile is 128 (query, head) rows of
// one KV head, tokens major; a KV tile is 64 tokens of 256 dimensions or 128
// of 128. S = Q K^T and O += P V are tcgen05.mma with M = 128 and both
// accumulators in tensor memory. Codes have to be FP16 in shared memory for
// that: warps of their own load them (two 16 KB halves in flight per SM, in
// registers), widen them and store them in the 128-byte-swizzled layout, K as
// rows of contraction, V as it lies (a transposed second operand). The
// probabilities go back to tensor memory as P's FP16 operand.
//
//   warps 0-3   softmax: a thread per row
//   warps 4-7   keys, warps 8-11 values: codes to FP16 tiles, two tiles deep
//   warp 12     issues the products: S of tile j + 1 before P V of tile j, so
//               that the tensor pipe works during the softmax
//   warps 13-15 the next pair's queries, while the softmax ends this one
//
// The roles walk the CTA's run on their own and meet at mbarriers only.
// Code that runs once per pair is kept small: it is fetched cold (unrolled by
// four rows, the queries took 20000 cycles a pair, most of it instructions).
//
// The softmax goes over S twice, 64 tokens in registers. First the largest
// product of every 16 tokens, which decides whether the row's references are
// raised (as in attend_rows_kernel; the row's sums in tensor memory are then
// scaled by the row's own thread, after P V of the tile before) and whether
// the tile is usual: block scales within 2^60 of each other, capped logits
// within |x / cap| <= 0.7, or below by so much that they weigh nothing, where
// a polynomial of tanh serves (two special-function calls less per logit). A
// usual tile's second pass takes a handful of instructions per logit; the sum l
// comes from the weights, by a factor per 16 tokens. Other tiles take the slow
// way, eight tokens at a time.
//
// 4-bit pages differ in the loaders, which widen the codes on their lines
// (about 380 instructions of each loading warp per tile instead of 200): 2 x 509
// queries over 5000 to 8191 tokens, 256 dimensions, capped, 259 us instead of 211.
// Their tokens have a power of two each. Where those of 16 tokens are close to each
// other they share one, as a block's scale; tiles with others go the slow way, in
// which every token has its own. With every hundredth token, at random, 2^6 below
// the rest: 345 us (700 queries of 700, 3000 and 9000, 128 dimensions, group 4, no
// cap: 380 us, and 489).
//
// The work list (sequences, KV heads, row tiles, KV tiles) is cut into runs of
// equal cost, one per CTA, and a tile's CTAs are joined as in attend_rows_kernel.
#include "se12_attend.cuh"

#include <cuda_bf16.h>

namespace se12 {

constexpr int kTileAttendRows = 128;  // query rows of a tile
constexpr int kTileSoftmaxWarps = 4;
constexpr int kTileLoaderWarps = 4;   // for keys, and as many for values
constexpr int kTileQueryWarps = 3;
constexpr int kTileAttendThreads = (kTileSoftmaxWarps + 2 * kTileLoaderWarps + 1 + kTileQueryWarps) * 32;
// Registers per thread by role (setmaxnreg), out of the launch's 128 for each
// of the four warp groups.
constexpr int kTileSoftmaxRegs = 208, kTileLoaderRegs = 104, kTileIssuerRegs = 80;
static_assert(kTileSoftmaxRegs + 2 * kTileLoaderRegs + kTileIssuerRegs <= 4 * 128, "more registers than the launch has");
constexpr int kTileKvBytes = 32768;   // an FP16 tile of keys or values
constexpr int kTileMeta = 4;          // tiles whose block scales are kept
// 4 bits: the most that the E of a cell's tokens may differ by for their values to
// stand beside the largest, so that one factor serves the cell. A row that does not
// see the largest, or gives it no weight, loses that many of the 14 powers of two
// that FP16 has below 1 for its weights, and scales and offsets for theirs.
constexpr int kTileSpread = 6;
// What a pair's queries, first loads and output cost, in KV tiles. (Calls
// repeated in a graph, before later checks added a few per cent: 24 sequences
// of 77 to 4093 tokens, 2 to 6 new ones of 8 rows: uncounted 105 us, the SMs
// active 63 % of the time; 2, 3, 4 and 6: 76, 78, 78 and 79 us. 3 sequences of
// 2014 to 8655 tokens, 78 new ones, 256 dimensions: 70 us; 68, 63, 63 and 63.)
constexpr int kTilePairCost = 3;
constexpr int kTileSlotFloats = kTileAttendRows * (256 + 4);

// ------------------------------------------------------------------ tensor memory and tcgen05

__device__ __forceinline__ void tmem_alloc(uint32_t* result, int columns) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(result)), "r"(columns)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}

__device__ __forceinline__ void tmem_free(uint32_t addr, int columns) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(columns) : "memory");
}

__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// The product calls are made by a whole warp, in step, for one elected lane:
// their operands are then warp-uniform registers throughout (issued by one
// thread in a branch of its own, a product took 250 cycles to issue).
__device__ __forceinline__ uint32_t elect_lane() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r;
}

// Arrives on the barrier once every product the lane issued is done.
__device__ __forceinline__ void tc_commit(uint64_t* bar, uint32_t elected) {
  asm volatile(
      "{\n\t.reg .pred e;\n\tsetp.ne.b32 e, %1, 0;\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_addr(bar)),
      "r"(elected)
      : "memory");
}

// Shared-memory operand in 128-byte-swizzled atoms of 8 rows x 128 bytes.
// Low word: address, and for a transposed operand the stride between its
// 128-byte column panels; high word: 1024 bytes between atoms along the rows,
// the descriptor's version and the swizzle.
constexpr uint32_t kOperandHigh = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t operand_low(uint32_t addr, uint32_t panel_bytes) {
  return (addr >> 4) | ((panel_bytes >> 4) << 16);
}

// D = A B (+ D), FP16 operands from shared memory, fp32 accumulator.
__device__ __forceinline__ void tc_mma_ss(uint32_t d, uint32_t a_low, uint32_t b_low, uint32_t idesc, bool add,
                                          uint32_t elected) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t.reg .b64 a, b;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 e, %5, 0;\n\t"
      "mov.b64 a, {%1, %6};\n\tmov.b64 b, {%2, %6};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}" ::"r"(d),
      "r"(a_low), "r"(b_low), "r"(idesc), "r"(static_cast<uint32_t>(add)), "r"(elected), "r"(kOperandHigh)
      : "memory");
}

// The same with A in tensor memory.
__device__ __forceinline__ void tc_mma_ts(uint32_t d, uint32_t a, uint32_t b_low, uint32_t idesc, bool add,
                                          uint32_t elected) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t.reg .b64 b;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 e, %5, 0;\n\t"
      "mov.b64 b, {%2, %6};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b_low), "r"(idesc), "r"(static_cast<uint32_t>(add)), "r"(elected), "r"(kOperandHigh)
      : "memory");
}

// 32 columns of this warp's 32 lanes.
__device__ __forceinline__ void tmem_load_32(uint32_t (&r)[32], uint32_t addr) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]),
        "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]),
        "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr)
      : "memory");
}

__device__ __forceinline__ void tmem_store_32(uint32_t addr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]),
      "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]),
      "r"(r[30]), "r"(r[31])
      : "memory");
}

__device__ __forceinline__ void tmem_store_8(uint32_t addr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(addr), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}

__device__ __forceinline__ void tmem_load_8(uint32_t (&r)[8], uint32_t addr) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(addr)
               : "memory");
}

__device__ __forceinline__ void tmem_store_4(uint32_t addr, const uint32_t (&r)[4]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]),
               "r"(r[3])
               : "memory");
}

// 16 bytes, or zeros where `use` is false (without a branch). A coherent load:
// the kernel may have begun while the one before it, which writes the codes
// and queries, was still running, and .nc asks that nothing writes them meanwhile.
__device__ __forceinline__ uint4 load_or_zero(const uint8_t* p, bool use) {
  uint4 v;
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %5, 0;\n\tmov.b32 %0, 0;\n\tmov.b32 %1, 0;\n\tmov.b32 %2, 0;\n\tmov.b32 %3, 0;\n\t"
      "@p ld.global.v4.u32 {%0, %1, %2, %3}, [%4];\n\t}"
      : "=&r"(v.x), "=&r"(v.y), "=&r"(v.z), "=&r"(v.w)
      : "l"(p), "r"(static_cast<uint32_t>(use))
      : "memory");
  return v;
}

__device__ __forceinline__ uint32_t load_word_or(const uint8_t* p, bool use, uint32_t other) {
  uint32_t v;
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %2, 0;\n\tmov.b32 %0, %3;\n\t@p ld.global.u32 %0, [%1];\n\t}"
               : "=&r"(v)
               : "l"(p), "r"(static_cast<uint32_t>(use)), "r"(other)
               : "memory");
  return v;
}

__device__ __forceinline__ uint32_t load_half_or(const uint8_t* p, bool use, uint32_t other) {
  uint32_t v;
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %2, 0;\n\tmov.b32 %0, %3;\n\t@p ld.global.u16 %0, [%1];\n\t}"
               : "=&r"(v)
               : "l"(p), "r"(static_cast<uint32_t>(use)), "r"(other)
               : "memory");
  return v;
}

// 4 bits: tiles hold the 8 dimensions of a word in the order 0 4 1 5 2 6 3 7, as
// its codes are unpacked. Where dimension d of 8 is, and 8 halves put in that order.
template <int KIND>
__device__ __forceinline__ constexpr int of_eight(int d) {
  return KIND == kKvInt4 ? (d & 3) * 2 + (d >> 2) : d;
}
template <int KIND>
__device__ __forceinline__ uint4 unpacked_order(uint32_t x01, uint32_t x23, uint32_t x45, uint32_t x67) {
  if constexpr (KIND == kKvInt4)
    return make_uint4(prmt(x01, x45, 0x5410u), prmt(x01, x45, 0x7632u), prmt(x23, x67, 0x5410u), prmt(x23, x67, 0x7632u));
  return make_uint4(x01, x23, x45, x67);
}

template <int N>
__device__ __forceinline__ void to_words(uint32_t (&w)[N], int at, const uint4& v) {
  w[at] = v.x, w[at + 1] = v.y, w[at + 2] = v.z, w[at + 3] = v.w;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

__device__ __forceinline__ void tmem_wait_load() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_store() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// FP16 operands, fp32 accumulator, M = 128; B transposed (rows of
// contraction) or not.
__device__ __forceinline__ constexpr uint32_t tc_idesc(int n, bool transposed_b) {
  return (1u << 4) | ((transposed_b ? 1u : 0u) << 16) | (static_cast<uint32_t>(n >> 3) << 17) | ((128u >> 4) << 24);
}

// ------------------------------------------------------------------ work list

struct TileSeq {
  SeqRows s;
  int rows, tiles;
};

__device__ __forceinline__ TileSeq tile_sequence(const AttendArgs& a, int b) {
  TileSeq w;
  w.s = a.t.rows_of(b, list_sizes(a));
  w.rows = w.s.tokens * a.group;
  w.tiles = (w.rows + kTileAttendRows - 1) / kTileAttendRows;
  return w;
}

template <int TT>
__device__ __forceinline__ TileSpan tile_span(const AttendArgs& a, const TileSeq& w, int tile) {
  return tile_span(w.s, tile, kTileAttendRows, list_sizes(a), TT);
}

struct TilePlace {
  int b, head, tile, chunk;
  TileSeq w;
  TileSpan s;
};

// The place of work-list entry g; the next pair after a place.
template <int TT>
__device__ __forceinline__ void tile_start(const AttendArgs& a, const int* before, int g, TilePlace* at) {
  const int heads = a.c.heads;
  int lo = 0, hi = a.t.seqs - 1;  // last b with before[b] * heads <= g
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (static_cast<long long>(before[mid]) * heads <= g) lo = mid;
    else hi = mid - 1;
  }
  at->b = lo;
  at->w = tile_sequence(a, lo);
  const int x = g - before[lo] * heads, each = before[lo + 1] - before[lo];
  at->head = x / each;
  at->tile = 0;
  at->chunk = x - at->head * each;
  at->s = tile_span<TT>(a, at->w, 0);
  while (at->chunk >= at->s.chunks) {
    at->chunk -= at->s.chunks;
    at->s = tile_span<TT>(a, at->w, ++at->tile);
  }
}

template <int TT>
__device__ __forceinline__ void tile_next_pair(const AttendArgs& a, const int* before, TilePlace* at) {  // there is one
  at->chunk = 0;
  if (++at->tile == at->w.tiles) {
    at->tile = 0;
    if (++at->head == a.c.heads) {
      at->head = 0;
      do {
        ++at->b;
      } while (before[at->b + 1] == before[at->b]);
      at->w = tile_sequence(a, at->b);
    }
  }
  at->s = tile_span<TT>(a, at->w, at->tile);
}

// Where the run begins whose first unit is t, when every pair counts `cost`
// units before its KV tiles: the first entry at or past it.
template <int TT>
__device__ __forceinline__ int tile_boundary(const AttendArgs& a, const int* before, const int* pairs, long long t, int cost) {
  const int heads = a.c.heads;
  auto units = [&](int b) { return (before[b] + static_cast<long long>(cost) * pairs[b]) * heads; };
  if (t >= units(a.t.seqs)) return before[a.t.seqs] * heads;
  int lo = 0, hi = a.t.seqs - 1;  // last b with units(b) <= t
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (units(mid) <= t) lo = mid;
    else hi = mid - 1;
  }
  const TileSeq w = tile_sequence(a, lo);
  const int each = before[lo + 1] - before[lo];
  const long long each_units = each + static_cast<long long>(cost) * w.tiles;
  long long x = t - units(lo);
  const int head = static_cast<int>(x / each_units);
  x -= head * each_units;
  int g = before[lo] * heads + head * each;
  for (int tile = 0;; ++tile) {
    const int chunks = tile_span<TT>(a, w, tile).chunks;
    if (x < cost + chunks || tile + 1 == w.tiles) return g + static_cast<int>(max(x - cost, 0ll));
    x -= cost + chunks;
    g += chunks;
  }
}

struct TileSmem {
  // [16 tokens of the tile][scale of keys, log2 of values' scale (4 bits: NaN where each
  // token has its own, in `power`)]
  float meta[kTileMeta][8][2];
  float power[kTileMeta][128];
  int meta_missing[kTileMeta];        // bit g: those tokens' page is not there
  float row_scale[2][kTileAttendRows];  // of this pair and the next
  // Pairs shared with other CTAs (a run's first and last) that this CTA
  // completes: where their parts are and where their rows go.
  struct {
    int cta_first, parts, first_slot, b, head, row0, rows;
  } join[2];
  int joins;
  uint64_t k_full[2], v_full[2], s_full[2], p_full[2], pv_done[2];
  uint64_t q_full[2], q_free, o_free, drained;
  uint64_t meta_full[kTileMeta];
  uint32_t tmem;
  int bounds[2];  // of this CTA's run
  int before[1];  // [seqs + 1] KV tiles of the sequences before, per KV head; then as many counts of row tiles
};

template <int KIND, int DP>
struct TileShape {
  static constexpr int kTokens = kTileKvBytes / 2 / DP;     // of a KV tile: 64 or 128
  static constexpr int kPanels = DP / 64;                   // 128-byte column panels
  static constexpr int kPanelBytes = kTokens * 128;         // of keys or values
  static constexpr int kQueryPanel = kTileAttendRows * 128;
  static constexpr int kGroups = kTokens / 16;
  static constexpr int kColS = 0, kColP = 2 * kTokens, kColO = 3 * kTokens;  // tensor memory columns
  static constexpr size_t kSmem = 1024 + static_cast<size_t>(kPanels) * kQueryPanel + 4 * kTileKvBytes + sizeof(TileSmem);
};

// ------------------------------------------------------------------ softmax of a tile

// What a row keeps over its tiles.
struct RowSoftmax {
  float m, l, mp;  // reference and sum of 2^(logit - m); reference of the weights
};

struct TileLogits {
  uint32_t from, to;        // S and P of this tile in tensor memory, this warp's lanes
  const float (*meta)[2];   // per 16 tokens: scale of keys, log2 of values' scale
  const float* power;       // per token, where that is NaN (4 bits)
  float row_scale;          // logits per product (capped: logits / cap)
  float cap2;               // cap * log2(e)
  int low, high;            // this row sees the tile's tokens low .. high
};

// The largest product of each 16 of the 64 tokens in s.
template <bool MASK>
__device__ __forceinline__ void group_maxima(float* t, const uint32_t (&s)[2][32], int k0, int low, int high) {
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    float v[16];
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      v[k] = __uint_as_float(s[q >> 1][(q & 1) * 16 + k]);
      if (MASK && (k0 + q * 16 + k < low || k0 + q * 16 + k > high)) v[k] = kNegInf;
    }
    float top = max3(v[0], v[1], v[2]);
#pragma unroll
    for (int k = 3; k < 15; k += 2) top = max3(top, v[k], v[k + 1]);
    t[q] = fmaxf(top, v[15]);
  }
}

__device__ __forceinline__ unsigned long long twice(float x) { return pair_of(x, x); }

// cap tanh(u) in units of log 2, and `add`: u times a polynomial of u^2 of
// degree 4 (Chebyshev fit of tanh(u) / u on |u| <= 0.7, off by 1.9e-7), two at a time.
__device__ __forceinline__ unsigned long long capped_pair(unsigned long long u, float cap2, unsigned long long add) {
  const unsigned long long c0 = twice(0.999999706f * cap2), c1 = twice(-0.33330266f * cap2), c2 = twice(0.132816473f * cap2),
                           c3 = twice(-0.0508535559f * cap2), c4 = twice(0.0137912829f * cap2);
  const unsigned long long t = mul_pair(u, u);
  return fma_pair(fma_pair(fma_pair(fma_pair(fma_pair(c4, t, c3), t, c2), t, c1), t, c0), u, add);
}

// Weights of the 64 tokens in s into P, and their sum, two tokens at a time.
template <bool CAP, bool MASK>
__device__ __forceinline__ void group_weights(RowSoftmax& r, const TileLogits& z, const uint32_t (&s)[2][32], int k0) {
#pragma unroll
  for (int c = 0; c < 2; ++c) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t p[8];
      const int q = (k0 >> 4) + c * 2 + h;
      const float shift = z.meta[q][1] - r.mp;
      const unsigned long long f = twice(z.row_scale * z.meta[q][0]), shift2 = twice(shift);
      unsigned long long sum = 0;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int i = h * 16 + 2 * k;
        const unsigned long long v = pair_of(__uint_as_float(s[c][i]), __uint_as_float(s[c][i + 1]));
        const unsigned long long x = CAP ? capped_pair(mul_pair(v, f), z.cap2, shift2) : fma_pair(v, f, shift2);
        float w0, w1;
        unpair(x, w0, w1);
        w0 = ex2(w0);
        w1 = ex2(w1);
        if (MASK) {
          const int at = k0 + c * 32 + i;
          if (at < z.low || at > z.high) w0 = 0.f;
          if (at + 1 < z.low || at + 1 > z.high) w1 = 0.f;
        }
        sum = add_pair(sum, pair_of(w0, w1));
        p[k] = half2_bits(__floats2half2_rn(w0, w1));
      }
      float sum0, sum1;
      unpair(sum, sum0, sum1);
      // 2^(logit - m) = w 2^(mp - lv - m); where the row sees none of the 16, lv may be anything
      if (!MASK || sum0 + sum1 != 0.f) r.l = fmaf(sum0 + sum1, ex2(-shift - r.m), r.l);
      tmem_store_8(z.to + k0 / 2 + c * 16 + h * 8, p);
    }
  }
}

__device__ __forceinline__ void load_64(uint32_t (&s)[2][32], uint32_t from) {
  tmem_load_32(s[0], from);
  tmem_load_32(s[1], from + 32);
  tmem_wait_load();
}

// Whether the row sees a logit below -0.7 of its cap. (Seldom asked: small.)
template <int TT>
__device__ __forceinline__ bool reaches_below(const TileLogits& z) {
  bool below = false;
#pragma unroll 1
  for (int k0 = 0; k0 < TT; k0 += 8) {
    uint32_t s[8];
    tmem_load_8(s, z.from + k0);
    tmem_wait_load();
    const float f = z.row_scale * z.meta[k0 >> 4][0];
#pragma unroll
    for (int k = 0; k < 8; ++k) below |= k0 + k >= z.low && k0 + k <= z.high && __uint_as_float(s[k]) * f < -0.7f;
  }
  return below;
}

// A tile's weights, if it is usual. `scale_sums(f)` multiplies the row's sums
// so far by f. False (for the whole warp): take the slow way.
template <int TT, bool CAP, bool MASK, typename ScaleSums>
__device__ __forceinline__ bool usual_tile(RowSoftmax& r, const TileLogits& z, ScaleSums&& scale_sums) {
  constexpr int kHalves = TT / 64, kGroups = TT / 16;
  uint32_t s[2][32];
  float t[kGroups];
  bool unusual = false;
  float top = r.mp, top_lv = 0.f;
#pragma unroll
  for (int h = 0; h < kHalves; ++h) {
    load_64(s, z.from + h * 64);
    group_maxima<MASK>(t + h * 4, s, h * 64, z.low, z.high);
#pragma unroll
    for (int q = h * 4; q < h * 4 + 4; q += 2) {
      // the groups' largest logits, capped as the weights will be (the cap
      // bends them by up to 0.1 of it: more than a weight has room for)
      float u[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float f = z.row_scale * z.meta[q + e][0];
        u[e] = t[q + e] * f;
        unusual |= !(f > 0.f) || (CAP && !(MASK && t[q + e] == kNegInf) && !(fabsf(u[e]) <= 0.7f));
      }
      if (CAP) unpair(capped_pair(pair_of(u[0], u[1]), z.cap2, twice(0.f)), u[0], u[1]);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float lv = z.meta[q + e][1];
        const float v = MASK && t[q + e] == kNegInf ? kNegInf : u[e] + lv;
        if (v > top) {
          top = v;
          top_lv = lv;
        }
      }
    }
  }
  if (__any_sync(0xFFFFFFFFu, !unusual && top - r.mp > kAttendRaise)) {
    const bool raise = !unusual && top - r.mp > kAttendRaise;
    const float mp = raise ? top : r.mp, m = mp - top_lv;
    if (raise && m - r.m > kAttendRaiseSum) {
      r.l *= ex2(r.m - m);
      r.m = m;
    }
    scale_sums(ex2(r.mp - mp));
    r.mp = mp;
  }
  // Below u = -0.7 the polynomial falls faster than tanh. That changes nothing
  // where a logit there, at most cap tanh(-0.7), weighs below 2^-36 of both
  // references (a cap of 50 with a largest logit of -5 or more); elsewhere the
  // tile is usual only if it has no such logit. Looked for at the end, where no
  // registers are held (here it cost 4 % of a prompt chunk).
  const float reach = 0.6043f * z.cap2 - 36.f;
  bool deep = CAP && !(reach + r.m >= 0.f);
#pragma unroll
  for (int q = 0; q < kGroups; ++q) {
    const float above = r.mp - z.meta[q][1];
    unusual |= !(fabsf(above - r.m) <= 60.f) && !(MASK && t[q] == kNegInf && r.m == kAttendStart);
    deep |= CAP && !(reach + above >= 0.f);
  }
  if (__any_sync(0xFFFFFFFFu, unusual)) return false;
  const float l_before = r.l;
#pragma unroll
  for (int h = kHalves - 1; h >= 0; --h) {  // the last 64 are still in registers
    if (h < kHalves - 1) load_64(s, z.from + h * 64);
    group_weights<CAP, MASK>(r, z, s, h * 64);
  }
  if (CAP && __any_sync(0xFFFFFFFFu, deep) && __any_sync(0xFFFFFFFFu, reaches_below<TT>(z))) {
    r.l = l_before;
    tmem_wait_store();  // the weights are written again
    return false;
  }
  return true;
}

// Any tile, eight tokens at a time. `missing`: bit q set where the 16 tokens'
// page is not there; masked and missing tokens weigh nothing.
template <int KIND, int TT, typename ScaleSums>
__device__ __forceinline__ void any_tile(RowSoftmax& r, const TileLogits& z, int missing, ScaleSums&& scale_sums) {
  auto logits = [&](float (&y)[8], int k0) {
    uint32_t s[8];
    tmem_load_8(s, z.from + k0);
    tmem_wait_load();
    const float f = z.row_scale * z.meta[k0 >> 4][0];
    const bool there = !((missing >> (k0 >> 4)) & 1);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      float v = __uint_as_float(s[k]) * f;
      if (z.cap2 != 0.f) v = capped_by(v, z.cap2);
      y[k] = k0 + k < z.low || k0 + k > z.high || !there ? kNegInf : v;
    }
  };
  auto value_scales = [&](float (&lv)[8], int k0) {
    const float of_all = z.meta[k0 >> 4][1];
    const bool own = KIND == kKvInt4 && of_all != of_all;
#pragma unroll
    for (int k = 0; k < 8; ++k) lv[k] = own ? z.power[k0 + k] : of_all;
  };
  float top = r.m, top_v = r.mp;
#pragma unroll 1
  for (int k0 = 0; k0 < TT; k0 += 8) {
    float y[8], lv[8];
    logits(y, k0);
    value_scales(lv, k0);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      top = fmaxf(top, y[k]);
      if (y[k] != kNegInf) top_v = fmaxf(top_v, y[k] + lv[k]);
    }
  }
  r.l *= ex2(r.m - top);
  r.m = top;
  scale_sums(ex2(r.mp - top_v));
  r.mp = top_v;
#pragma unroll 1
  for (int k0 = 0; k0 < TT; k0 += 8) {
    float y[8], lv[8];
    logits(y, k0);
    value_scales(lv, k0);
    uint32_t p[4];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      r.l += ex2(y[k] - r.m);
      y[k] = y[k] == kNegInf ? 0.f : ex2(y[k] + (lv[k] - r.mp));
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) p[k] = half2_bits(__floats2half2_rn(y[2 * k], y[2 * k + 1]));
    tmem_store_4(z.to + k0 / 2, p);
  }
}

// Eight BF16 values of an output row, from dimension d.
__device__ __forceinline__ void store_8(uint16_t* out, int d, int dim, int vec, const uint32_t (&w)[4]) {
  if (d >= dim) return;
  if (vec) {
    *reinterpret_cast<uint4*>(out + d) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      out[d + 2 * e] = static_cast<uint16_t>(w[e]);
      out[d + 2 * e + 1] = static_cast<uint16_t>(w[e] >> 16);
    }
  }
}

// ------------------------------------------------------------------ kernel

// NARROW: 64 dimensions (of 4-bit codes; 8-bit ones take any number in their stride).
template <int KIND, int DP, bool NARROW>
__global__ void __launch_bounds__(kTileAttendThreads, 1) attend_tile_kernel(const AttendArgs a) {
  using Shape = TileShape<KIND, DP>;
  constexpr int TT = Shape::kTokens, PANELS = Shape::kPanels, GROUPS = Shape::kGroups;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* q_tile = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  unsigned char* k_tiles = q_tile + PANELS * Shape::kQueryPanel;
  unsigned char* v_tiles = k_tiles + 2 * kTileKvBytes;
  TileSmem& sm = *reinterpret_cast<TileSmem*>(v_tiles + 2 * kTileKvBytes);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  constexpr int kIssuer = kTileSoftmaxWarps + 2 * kTileLoaderWarps;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sm.k_full[i], kTileLoaderWarps);
      mbar_init(&sm.v_full[i], kTileLoaderWarps);
      mbar_init(&sm.s_full[i], 1);
      mbar_init(&sm.p_full[i], kTileSoftmaxWarps);
      mbar_init(&sm.pv_done[i], 1);
    }
    for (int i = 0; i < kTileMeta; ++i) mbar_init(&sm.meta_full[i], KIND == kKvInt4 ? kTileLoaderWarps : 1);
    mbar_init(&sm.q_free, 1);
    mbar_init(&sm.q_full[0], kTileQueryWarps);
    mbar_init(&sm.q_full[1], kTileQueryWarps);
    sm.joins = 0;
    mbar_init(&sm.o_free, kTileSoftmaxWarps);
    mbar_init(&sm.drained, 1);
    fence_barrier_init();
  }
  if (warp == kIssuer) tmem_alloc(&sm.tmem, 512);
  grid_launch_dependents();
  grid_dependency_wait();

  // ---- the work list
  const int heads = a.c.heads;
  int* pairs = sm.before + a.t.seqs + 1;
  const int limit = static_cast<int>(kWorkLimit / heads);
  for (int b = threadIdx.x; b < a.t.seqs; b += kTileAttendThreads) {
    const TileSeq w = tile_sequence(a, b);
    check_length(a, b);
    int n = 0;
    for (int t = 0; t < w.tiles; ++t) n = add_work(n, tile_span<TT>(a, w, t).chunks, limit);
    sm.before[b + 1] = n;
    pairs[b + 1] = w.tiles;
  }
  if (threadIdx.x == 0) sm.before[0] = pairs[0] = 0;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp < 2) sum_up_to(warp == 0 ? sm.before : pairs, a.t.seqs, limit, lane);
  __syncthreads();
  constexpr uint32_t tmem = 0;  // all 512 columns are this CTA's: they begin at 0
  const int total = sm.before[a.t.seqs] * heads;
  // Runs are equal in units, a pair's beginning counting as `cost` KV tiles
  // (fewer when a run is short: they would leave CTAs without work).
  const int cost = min(kTilePairCost, total / (4 * static_cast<int>(gridDim.x)));
  const long long units = total + static_cast<long long>(cost) * pairs[a.t.seqs] * heads;
  const long long per = (units + gridDim.x - 1) / gridDim.x;
  const bool fits = sm.before[a.t.seqs] < limit;
  if (!fits && threadIdx.x == 0) raise_status(kStatusBadArgument);
  if (lane == 0 && warp < 2)
    sm.bounds[warp] = fits ? tile_boundary<TT>(a, sm.before, pairs, (blockIdx.x + warp) * per, cost) : 0;
  __syncthreads();
  const int g0 = sm.bounds[0], g1 = sm.bounds[1];

  // ---- each role walks the CTA's run pair by pair
  TilePlace at;
  // Once a wait has run out (status raised) a role waits no more: the results
  // are void, but every thread still meets the barriers and returns.
  bool dead = false;
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    if (!dead) dead = !mbar_wait(bar, parity);
  };

  if (g0 >= g1) {
    // nothing to do
  } else if (warp >= kIssuer) {
    // ---- products
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kTileIssuerRegs));
    if (warp == kIssuer) {
      tile_start<TT>(a, sm.before, g0, &at);
      const uint32_t elected = elect_lane();
      const uint32_t q_low = operand_low(smem_addr(q_tile), 16), k_low = operand_low(smem_addr(k_tiles), 16),
                     v_low = operand_low(smem_addr(v_tiles), Shape::kPanelBytes);
      // (what the compiler cannot see to be uniform passes through a reduction)
      auto wait_warp = [&](uint64_t* bar, uint32_t parity) {
        wait(bar, parity);
        dead = __any_sync(0xFFFFFFFFu, dead);
      };
      auto scores = [&](uint32_t j, bool last) {  // S of tile j (of the ring)
        wait_warp(&sm.k_full[j & 1], (j >> 1) & 1);
        if (dead) return;
        tc_fence_after();
        const uint32_t k_at = k_low + (j & 1) * (kTileKvBytes >> 4), s_at = Shape::kColS + (j & 1) * TT;
#pragma unroll
        for (int k = 0; k < DP / 16; ++k)
          tc_mma_ss(s_at, q_low + (((k >> 2) * Shape::kQueryPanel + (k & 3) * 32) >> 4),
                    k_at + (((k >> 2) * Shape::kPanelBytes + (k & 3) * 32) >> 4), tc_idesc(TT, false), k > 0, elected);
        tc_commit(&sm.s_full[j & 1], elected);
        if (last) tc_commit(&sm.q_free, elected);
      };
      uint32_t done = 0, pair = 0;  // KV tiles and pairs before: the rings' phases
      for (int g = g0; g < g1; ++pair) {
        const uint32_t run = __reduce_max_sync(0xFFFFFFFFu, static_cast<unsigned>(min(at.s.chunks - at.chunk, g1 - g)));
        wait_warp(&sm.q_full[pair & 1], (pair >> 1) & 1);
        scores(done, run == 1);
        for (uint32_t i = 0; i < run && !dead; ++i) {
          const uint32_t j = done + i;
          if (i + 1 < run) scores(j + 1, i + 2 == run);
          wait_warp(&sm.v_full[j & 1], (j >> 1) & 1);
          wait_warp(&sm.p_full[j & 1], (j >> 1) & 1);
          if (i == 0 && pair > 0) wait_warp(&sm.o_free, (pair - 1) & 1);
          if (dead) break;
          tc_fence_after();
          const uint32_t v_at = v_low + (j & 1) * (kTileKvBytes >> 4), p_at = Shape::kColP + (j & 1) * (TT / 2);
#pragma unroll
          for (int k = 0; k < TT / 16; ++k)
            tc_mma_ts(Shape::kColO, p_at + k * 8, v_at + ((k * 2048) >> 4), tc_idesc(DP, true), i > 0 || k > 0, elected);
          tc_commit(&sm.pv_done[j & 1], elected);
        }
        if (dead) break;
        done += run;
        g += run;
        if (g < g1) tile_next_pair<TT>(a, sm.before, &at);
      }
      if (dead) {  // products may still be reading the tiles and tensor memory
        tc_commit(&sm.drained, elected);
        mbar_wait(&sm.drained, 0);
      }
    }
    __syncwarp();
    if (warp > kIssuer) {
      // ---- queries as FP16 times 2^-e (and the scale's sign), eight threads per row
      constexpr int kVectors = DP / 64, kRowsAtOnce = kTileQueryWarps * 4;
      const int tid = threadIdx.x - (kIssuer + 1) * 32, part = tid & 7;
      tile_start<TT>(a, sm.before, g0, &at);
      int pair = 0;
      for (int g = g0; g < g1; ++pair) {
        const int run = min(at.s.chunks - at.chunk, g1 - g);
        // the pair before has been multiplied
        if (pair > 0) wait(&sm.q_free, (pair - 1) & 1);
        const int token0 = a.t.begin_of(at.b, list_sizes(a));
        const int rows_left = at.w.rows - at.tile * kTileAttendRows;
        auto load_row = [&](uint4 (&r)[kVectors], int q_row) {
          const int all = at.tile * kTileAttendRows + q_row;
          const bool live = q_row < rows_left && q_row < kTileAttendRows;
          const int i = live ? all / a.group : 0;
          const uint16_t* src = a.q + (token0 + i) * a.q_ts + (at.head * a.group + (live ? all - i * a.group : 0)) * a.q_hs;
#pragma unroll
          for (int j = 0; j < kVectors; ++j) {
            const int d = (j * 8 + part) * 8;
            const bool use = live && d < a.c.dim;
            if (a.q_vec) {
              r[j] = load_or_zero(reinterpret_cast<const uint8_t*>(src + d), use);
            } else {
              uint32_t w[4];
#pragma unroll
              for (int k = 0; k < 4; ++k)
                w[k] = use ? src[d + 2 * k] | (static_cast<uint32_t>(src[d + 2 * k + 1]) << 16) : 0;
              r[j] = make_uint4(w[0], w[1], w[2], w[3]);
            }
          }
        };
        uint4 next[kVectors];
        load_row(next, tid >> 3);
#pragma unroll 1
        for (int q_row = tid >> 3; q_row - (tid >> 3) < kTileAttendRows; q_row += kRowsAtOnce) {
          uint4 raw[kVectors];
#pragma unroll
          for (int j = 0; j < kVectors; ++j) raw[j] = next[j];
          load_row(next, q_row + kRowsAtOnce);
          unsigned big = 0;
#pragma unroll
          for (int j = 0; j < kVectors; ++j)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const uint32_t w = word_of(raw[j], k);
              big = max(big, max((w << 16) & 0x7FFFFFFFu, w & 0x7FFF0000u));
            }
#pragma unroll
          for (int d = 1; d < 8; d <<= 1) big = max(big, __shfl_xor_sync(0xFFFFFFFFu, big, d));
          int e = static_cast<int>(big >> 23) - 127;
          e = big == 0 ? 0 : max(min(e, 120), -120);
          const float down = copysignf(__uint_as_float(static_cast<unsigned>(127 - e) << 23), a.scale);
          auto halves = [&](uint32_t w) {
            return half2_bits(__floats2half2_rn(__uint_as_float(w << 16) * down, __uint_as_float(w & 0xFFFF0000u) * down));
          };
          if (q_row < kTileAttendRows) {
#pragma unroll
            for (int j = 0; j < kVectors; ++j)
              *reinterpret_cast<uint4*>(q_tile + j * Shape::kQueryPanel + q_row * 128 + ((part ^ (q_row & 7)) << 4)) =
                  unpacked_order<KIND>(halves(raw[j].x), halves(raw[j].y), halves(raw[j].z), halves(raw[j].w));
            if (part == 0)
              sm.row_scale[pair & 1][q_row] = __uint_as_float(static_cast<unsigned>(127 + e) << 23) * fabsf(a.scale);
          }
        }
        fence_proxy_async_shared();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.q_full[pair & 1]);
        g += run;
        if (g < g1) tile_next_pair<TT>(a, sm.before, &at);
      }
    }
  } else if (warp >= kTileSoftmaxWarps) {
    // ---- codes to FP16 tiles
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kTileLoaderRegs));
    const bool keys = warp < kTileSoftmaxWarps + kTileLoaderWarps;
    const int tid = threadIdx.x - (kTileSoftmaxWarps + (keys ? 0 : kTileLoaderWarps)) * 32;  // 0 .. 127
    const uint8_t* codes = keys ? a.c.k_codes : a.c.v_codes;
    unsigned char* tiles = keys ? k_tiles : v_tiles;
    constexpr int kHalf = 4;  // 16-byte vectors per thread and half tile
    constexpr bool kFour = KIND == kKvInt4;
    // A warp's vector: 8 tokens x 64 bytes. The 8 lanes of a shared-memory
    // phase hold one column of 8 tokens: all banks, in the swizzled layout.
    constexpr int kStep = Shape::kTokens / 8;  // tokens between a thread's vectors: 8 or 16
    const int w4 = tid >> 5;
    const int panel = w4 % PANELS, sub = kFour ? 0 : (w4 / PANELS) * 8 + (lane & 7);  // panel of 64 dimensions, token of a vector
    const int column = panel * 64 + (lane >> 3) * 16;
    const int dim = a.c.dim;
    const bool wanted = kFour || column < dim;
    const uint8_t* source = codes + column;
    const int place = panel * Shape::kPanelBytes + sub * 128;
    const int place0 = place + ((((lane >> 3) * 2) ^ (lane & 7)) << 4), place1 = place + ((((lane >> 3) * 2 + 1) ^ (lane & 7)) << 4);

    // Lane g < GROUPS keeps, for the tile to load, the row (of all the
    // cache's rows of `dim` codes) where its 16 tokens begin, -1 if none; its
    // page for the tile after that is on its way too.
    tile_start<TT>(a, sm.before, g0, &at);
    int walk_t0 = at.s.low + at.chunk * TT, walk_left = min(at.s.chunks - at.chunk, g1 - g0), walk_g = g0 + walk_left;
    int walk_head = at.head, walk_end = span_end(at.w.s, at.s.pos_max), walk_from = visible_from(at.s.pos_min, a.window);
    const int32_t* walk_table = a.t.table + at.b * a.t.table_stride;
    int page_next = 0;
    auto fetch_pages = [&]() {
      const int t = walk_t0 + lane * 16;
      page_next = -2;  // none due: past the last row's position, or below the first row's window
      if (lane < GROUPS && t < walk_end && t + 16 > walk_from)
        page_next = (t >> a.c.page_shift) < a.t.max_pages ? walk_table[t >> a.c.page_shift] : -1;
    };
    bool missing = false;  // a page that is due is not there
    int rows_at = -1, limit = 0;  // limit: of a vector's first token, for this lane's token to count
    float ks = 0.f, vs = 0.f;  // this lane's block scales of that tile (first warp of the keys)
    auto take_tile = [&]() {   // the fetched pages become the tile to load; fetch the next one's
      rows_at = -1;
      missing = page_next != -2 && (page_next < 0 || page_next >= a.c.pages);
      if (missing)
        raise_status(kStatusBadArgument);
      else if (page_next != -2)
        rows_at = (page_next * heads + walk_head) * a.c.page_size + ((walk_t0 + lane * 16) & (a.c.page_size - 1));
      limit = wanted ? walk_end - walk_t0 - sub : 0;
      walk_t0 += TT;
      if (--walk_left == 0) {
        if (walk_g >= g1) return;
        tile_next_pair<TT>(a, sm.before, &at);  // (a pair cut at the run's end is its last)
        walk_t0 = at.s.low;
        walk_left = min(at.s.chunks, g1 - walk_g);
        walk_g += walk_left;
        walk_head = at.head;
        walk_end = span_end(at.w.s, at.s.pos_max);
        walk_from = visible_from(at.s.pos_min, a.window);
        walk_table = a.t.table + at.b * a.t.table_stride;
      }
      fetch_pages();
    };
    auto load = [&](uint4 (&r)[kHalf], int first) {
      int row[kHalf];
#pragma unroll
      for (int v = 0; v < kHalf; ++v) row[v] = __shfl_sync(0xFFFFFFFFu, rows_at, ((first + v) * kStep) >> 4);
#pragma unroll
      for (int v = 0; v < kHalf; ++v) {
        const int in_group = ((first + v) * kStep & 15) + sub;
        const bool use = row[v] >= 0 && (first + v) * kStep < limit;
        r[v] = load_or_zero(source + static_cast<long long>(row[v] + in_group) * dim, use);
      }
    };
    auto store = [&](const uint4 (&r)[kHalf], int first, unsigned char* tile) {
#pragma unroll
      for (int v = 0; v < kHalf; ++v) {
        uint4 h;
        widen<KIND>(r[v].x, h.x, h.y);
        widen<KIND>(r[v].y, h.z, h.w);
        *reinterpret_cast<uint4*>(tile + place0 + (first + v) * kStep * 128) = h;
        widen<KIND>(r[v].z, h.x, h.y);
        widen<KIND>(r[v].w, h.z, h.w);
        *reinterpret_cast<uint4*>(tile + place1 + (first + v) * kStep * 128) = h;
      }
    };
    fetch_pages();
    take_tile();
    const int tiles_all = g1 - g0;
    if constexpr (kFour) {
      // ---- 4 bits. A warp has two cells of 16 tokens of a tile (256 dimensions:
      // half of each row's codes), four vectors of 8 tokens x 64 bytes of codes.
      // Keys become FP16 values; values become FP16 times 2^-X, X the largest E of
      // the cell's tokens that count, which takes the place of a block's scale; where
      // a token's E is more than kTileSpread below it, FP16 times 2^-E of their own,
      // and the tile goes the slow way. (A token of zeros may have any E.) The 8
      // of a word stay in the order their codes are unpacked in (of_eight). A
      // token whose E is no number has NaN for a key and zero for a value: the
      // rows that see it are NaN, as their weights are.
      constexpr int groups = DP == 256 ? 4 : NARROW ? 1 : 2;
      const int part = DP == 256 ? (w4 & 1) * 4 + (lane >> 3) : lane >> 3;  // 16 bytes of a row's codes
      const bool mine = !NARROW || part < 2;
      constexpr int row_codes = 32 * groups, key_lines = 4 * groups, cell_bytes = 64 * groups + 32;
      constexpr int kWords = DP == 256 ? 8 : 4;  // of a vector's lines (keys: the first half of them)
      const uint8_t* lines_of = static_cast<const uint8_t*>(keys ? a.c.k_scales : a.c.v_scales);
      const uint8_t* cells = static_cast<const uint8_t*>(a.c.v_scales);
      auto cell_of = [&](int v) { return DP == 256 ? (v >> 1) * 2 + (w4 >> 1) : (v >> 1) * 4 + w4; };
      // Where word w of a vector goes: the 64 dimensions of a panel, 8 per column.
      auto place_of = [&](int v, int w) {
        const int to_panel = DP == 256 ? w : NARROW ? part >> 1 : w & 1;
        const int to_column = DP == 256 ? part : NARROW ? (part & 1) * 4 + w : 2 * part + (w >> 1);
        const int token = cell_of(v) * 16 + (v & 1) * 8 + (lane & 7);
        return to_panel * Shape::kPanelBytes + token * 128 + ((to_column ^ (lane & 7)) << 4);
      };
      struct Vector {
        uint4 codes;
        uint32_t lines[kWords];  // keys: (scale, offset) of each group; values: scales, then offsets, of two tokens each
        uint32_t power;          // E
      };
      Vector r[4];
      auto load_cell = [&](int i) {  // the i-th of the warp's: vectors 2 i and 2 i + 1
        const int row = __shfl_sync(0xFFFFFFFFu, rows_at, cell_of(2 * i));
        const int token = lane & 7, left = row >= 0 ? limit - cell_of(2 * i) * 16 - token : 0;
        const uint8_t* code = codes + static_cast<long long>(row + token) * row_codes + part * 16;
        const uint8_t* cell = cells + static_cast<long long>(row >> 4) * cell_bytes;
        const uint8_t* line = keys ? lines_of + static_cast<long long>(row + token) * key_lines : cell + (token >> 1) * (8 * groups);
        const uint8_t* power = cell + 64 * groups + 2 * token;
        const int line_step = keys ? 8 * key_lines : 32 * groups;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          Vector& x = r[2 * i + h];
          const bool use = left > 8 * h, wanted_lines = use && mine;
          x.codes = load_or_zero(code + h * (8 * row_codes), wanted_lines);
          if constexpr (DP == 256) {
            to_words(x.lines, 0, load_or_zero(line + h * line_step, wanted_lines));
            if (!keys) to_words(x.lines, kWords - 4, load_or_zero(line + h * line_step + 16, wanted_lines));
          } else if constexpr (NARROW) {
            x.lines[0] = x.lines[1] = load_word_or(line + h * line_step, wanted_lines, 0u);
            x.lines[2] = x.lines[3] = load_word_or(line + h * line_step + 4, wanted_lines && !keys, 0u);
          } else if (keys) {
            x.lines[0] = load_word_or(line + h * line_step, wanted_lines, 0u);
            x.lines[1] = load_word_or(line + h * line_step + 4, wanted_lines, 0u);
          } else {
            to_words(x.lines, 0, load_or_zero(line + h * line_step, wanted_lines));
          }
          x.power = load_half_or(power + 16 * h, use, 0xFC00u);  // (-inf: a token that does not count)
        }
      };
      auto power_of = [&](int v) { return __half2float(__ushort_as_half(static_cast<unsigned short>(r[v].power))); };
      // Whether a token of the warp's cells (in `far`, a bit per vector, its own lanes)
      // has a line that is not zeros: bits of the cells. (Seldom asked: small.)
      auto cells_with_lines = [&](unsigned far) {
        unsigned found = 0;
#pragma unroll 1
        for (int v = 0; v < 4; ++v) {
          const int row = __shfl_sync(0xFFFFFFFFu, rows_at, cell_of(v & 2));
          const uint8_t* pair = cells + static_cast<long long>(row >> 4) * cell_bytes + ((lane & 7) >> 1) * (8 * groups) + (v & 1) * (32 * groups);
          uint32_t any = 0;
#pragma unroll 1
          for (int w = lane >> 3; w < 2 * groups; w += 4) any |= load_word_or(pair + 4 * w, (far >> v) & 1, 0u);
          if (__any_sync(0xFFFFFFFFu, (any & ((lane & 1) ? 0x7FFF0000u : 0x7FFFu)) != 0)) found |= 1u << (v >> 1);
        }
        return found;
      };
      // A vector's codes on their lines, to the tile. `cell_power`: X, or NaN.
      auto store4 = [&](int v, unsigned char* tile, float cell_power) {
        const float e = power_of(v);
        const bool number = e == e;
        const float to_cell = cell_power == cell_power ? ex2(e - cell_power) : 1.f;
        const uint32_t down = half2_bits(__half2half2(__float2half_rn(number ? to_cell : 0.f)));
        const uint32_t side = (lane & 1) ? 0x3232u : 0x1010u;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const int g = DP == 256 ? w : w & 1;
          uint32_t scale, offset;
          if (keys) {
            scale = prmt(r[v].lines[g], 0u, 0x1010u);
            offset = prmt(r[v].lines[g], 0u, 0x3232u);
            if (!number) scale = offset = 0x7FFF7FFFu;
          } else {
            const __half2 d = *reinterpret_cast<const __half2*>(&down);
            const uint32_t s = prmt(r[v].lines[g], 0u, side), o = prmt(r[v].lines[kWords / 2 + g], 0u, side);
            scale = half2_bits(__hmul2(*reinterpret_cast<const __half2*>(&s), d));
            offset = half2_bits(__hmul2(*reinterpret_cast<const __half2*>(&o), d));
          }
          const uint32_t x = word_of(r[v].codes, w), y = x >> 8;
          // u + 1024 and u + 64 in FP16, codes 0 and 4, 1 and 5, 2 and 6, 3 and 7
          uint32_t h[4] = {(x & 0x000F000Fu) | 0x64006400u, (x & 0x00F000F0u) | 0x54005400u, (y & 0x000F000Fu) | 0x64006400u,
                           (y & 0x00F000F0u) | 0x54005400u};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            asm("sub.f16x2 %0, %0, %1;" : "+r"(h[k]) : "r"(k & 1 ? 0x54805480u : 0x64086408u));
            asm("fma.rn.f16x2 %0, %0, %1, %2;" : "+r"(h[k]) : "r"(scale), "r"(offset));
          }
          *reinterpret_cast<uint4*>(tile + place_of(v, w)) = make_uint4(h[0], h[1], h[2], h[3]);
        }
      };
      load_cell(0);
      load_cell(1);
#pragma unroll 1
      for (int j = 0; j < tiles_all; ++j) {
        const int stage = j & 1;
        unsigned char* tile = tiles + stage * kTileKvBytes;
        float cell_power[2];  // of the warp's cells: X (0 where no token counts), or NaN
        unsigned far = 0;     // this lane's tokens that are too far below X
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float x = fmaxf(power_of(2 * i), power_of(2 * i + 1));  // (NaN is left out)
#pragma unroll
          for (int d = 1; d < 8; d <<= 1) x = fmaxf(x, __shfl_xor_sync(0xFFFFFFFFu, x, d));
          cell_power[i] = fabsf(x) <= 64.f ? x : 0.f;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float below = cell_power[i] - power_of(2 * i + h);
            if (below > kTileSpread && below < 1000.f) far |= 1u << (2 * i + h);  // (not -inf: no token)
          }
        }
        if (__any_sync(0xFFFFFFFFu, far != 0)) {
          far = cells_with_lines(far);
#pragma unroll
          for (int i = 0; i < 2; ++i)
            if ((far >> i) & 1) cell_power[i] = __uint_as_float(0x7FC00000u);
        }
        // the tile two before has been read by its products
        if (j >= 2) wait(keys ? &sm.s_full[stage] : &sm.pv_done[stage], ((j >> 1) + 1) & 1);
        const bool more = j + 1 < tiles_all;
        const unsigned missing_groups = __ballot_sync(0xFFFFFFFFu, missing);
        if (keys) {
          const int slot = j % kTileMeta;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int cell = cell_of(2 * i);
            if (lane == 0) {
              sm.meta[slot][cell][0] = 1.f;
              sm.meta[slot][cell][1] = cell_power[i];
            }
            if (cell_power[i] != cell_power[i] && lane < 8) {
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const float e = power_of(2 * i + h);
                sm.power[slot][cell * 16 + h * 8 + lane] = fabsf(e) <= 64.f ? e : 0.f;
              }
            }
          }
          if (tid == 0) sm.meta_missing[slot] = static_cast<int>(missing_groups);
          __syncwarp();
          if (lane == 0) mbar_arrive(&sm.meta_full[slot]);
        }
        if (more) take_tile();
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          store4(2 * i, tile, cell_power[i]);
          store4(2 * i + 1, tile, cell_power[i]);
          if (more) load_cell(i);
        }
        fence_proxy_async_shared();
        __syncwarp();
        if (lane == 0) mbar_arrive(keys ? &sm.k_full[stage] : &sm.v_full[stage]);
      }
    } else {
    // Two halves per tile, each loaded a tile ahead: 32 KB per SM on the way.
    uint4 ra[kHalf], rb[kHalf];
    load(ra, 0);
    load(rb, kHalf);
#pragma unroll 1
    for (int j = 0; j < tiles_all; ++j) {
      const int stage = j & 1;
      unsigned char* tile = tiles + stage * kTileKvBytes;
      if (keys && tid < 32) {
        ks = rows_at >= 0 ? static_cast<const float*>(a.c.k_scales)[rows_at >> a.c.page_shift] : 1.f;
        vs = rows_at >= 0 ? static_cast<const float*>(a.c.v_scales)[rows_at >> a.c.page_shift] : 1.f;
      }
      // the tile two before has been read by its products
      if (j >= 2) wait(keys ? &sm.s_full[stage] : &sm.pv_done[stage], ((j >> 1) + 1) & 1);
      const bool more = j + 1 < tiles_all;
      const unsigned missing_groups = __ballot_sync(0xFFFFFFFFu, missing);
      if (more) take_tile();
      store(ra, 0, tile);
      if (more) load(ra, 0);
      store(rb, kHalf, tile);
      if (more) load(rb, kHalf);
      fence_proxy_async_shared();
      if (keys && tid < 32) {
        const int slot = j % kTileMeta;
        if (lane < GROUPS) {
          sm.meta[slot][lane][0] = ks;
          sm.meta[slot][lane][1] = lg2(vs);
        }
        if (lane == 0) sm.meta_missing[slot] = static_cast<int>(missing_groups);
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.meta_full[slot]);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(keys ? &sm.k_full[stage] : &sm.v_full[stage]);
    }
    }
  } else {
    // ---- softmax: row 32 warp + lane
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kTileSoftmaxRegs));
    constexpr int kSoftmaxThreads = kTileSoftmaxWarps * 32;
    const int row = threadIdx.x;
    const uint32_t lanes = static_cast<uint32_t>(warp * 32) << 16;
    const bool capped_logits = a.softcap != 0.f;
    const float cap2 = a.softcap * kLog2e;
    tile_start<TT>(a, sm.before, g0, &at);
    int done = 0, pair = 0;  // KV tiles of the pairs before: the rings' phases
    for (int g = g0; g < g1;) {
      const int run = min(at.s.chunks - at.chunk, g1 - g);
      const int rows = min(kTileAttendRows, at.w.rows - at.tile * kTileAttendRows);
      const int t_first = at.s.low + at.chunk * TT;
      const int last = at.w.s.length - 1;  // the last token there is: rows past the page table see up to it
      const int pos_min = min(at.s.pos_min, last), pos_max = at.s.pos_max;
      const bool active = warp * 32 < rows;  // rows past the tile's are left out, warp by warp
      wait(&sm.q_full[pair & 1], (pair >> 1) & 1);
      const float row_scale = sm.row_scale[pair & 1][row] * (capped_logits ? 1.f / a.softcap : kLog2e);
      const int pos = at.w.s.first + min(at.tile * kTileAttendRows + row, at.w.rows - 1) / a.group;
      RowSoftmax r{kAttendStart, 0.f, kAttendStart};
#pragma unroll 1
      for (int i = 0; i < run; ++i) {
        const int j = done + i, slot = j % kTileMeta;
        const int t0 = t_first + i * TT;
        wait(&sm.meta_full[slot], (j / kTileMeta) & 1);
        // S of this tile is there; the products run in order, so P V of the
        // tile two before, which was issued earlier, has read its P
        wait(&sm.s_full[j & 1], (j >> 1) & 1);
        tc_fence_after();
        if (active) {
          TileLogits z;
          z.from = tmem + lanes + Shape::kColS + (j & 1) * TT;
          z.to = tmem + lanes + Shape::kColP + (j & 1) * (TT / 2);
          z.meta = sm.meta[slot];
          z.power = sm.power[slot];
          z.row_scale = row_scale;
          z.cap2 = cap2;
          z.low = a.window ? pos - t0 - (a.window - 1) : 0;
          z.high = min(pos, last) - t0;
          const int missing = sm.meta_missing[slot];
          auto scale_sums = [&](float f) {
            if (i == 0 || !__any_sync(0xFFFFFFFFu, f != 1.f)) return;
            wait(&sm.pv_done[(j - 1) & 1], ((j - 1) >> 1) & 1);
            tc_fence_after();
#pragma unroll 1
            for (int q = 0; q < DP / 32; ++q) {
              const uint32_t addr = tmem + lanes + Shape::kColO + q * 32;
              uint32_t o[32];
              tmem_load_32(o, addr);
              tmem_wait_load();
#pragma unroll
              for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
              tmem_store_32(addr, o);
            }
            tmem_wait_store();  // (the slow way may scale them again)
          };
          const bool masked = t0 + TT - 1 > pos_min || (a.window && pos_max - t0 >= a.window);
          bool finished = false;
          if (missing == 0) {
            if (capped_logits)
              finished = masked ? usual_tile<TT, true, true>(r, z, scale_sums) : usual_tile<TT, true, false>(r, z, scale_sums);
            else
              finished = masked ? usual_tile<TT, false, true>(r, z, scale_sums) : usual_tile<TT, false, false>(r, z, scale_sums);
          }
          if (!finished) any_tile<KIND, TT>(r, z, missing, scale_sums);
          tmem_wait_store();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.p_full[j & 1]);
      }
      // ---- the row's sums
      const int pair_start = g - at.chunk, pair_end = pair_start + at.s.chunks;
      const long long cost_before = static_cast<long long>(cost) * (pairs[at.b] * heads + at.head * at.w.tiles + at.tile);
      const int cta_first = static_cast<int>((pair_start + cost_before + cost) / per),
                cta_last = static_cast<int>((pair_end - 1 + cost_before + cost) / per);
      const bool whole = cta_first == cta_last;
      float* part_out = a.partials + (static_cast<size_t>(blockIdx.x) * 2 + (pair_start > g0 ? 1 : 0)) * kTileSlotFloats;
      const int token0 = a.t.begin_of(at.b, list_sizes(a));
      const int row0 = at.tile * kTileAttendRows;
      wait(&sm.pv_done[(done + run - 1) & 1], ((done + run - 1) >> 1) & 1);
      tc_fence_after();
      if (active) {
        const float f = whole ? (r.l == 0.f ? 0.f : ex2(r.mp - r.m) / r.l) : 1.f;
        if (!whole) {  // statistics after the sums, all with the rows side by side
          part_out[256 * kTileAttendRows + row] = r.m;
          part_out[257 * kTileAttendRows + row] = r.l;
          part_out[258 * kTileAttendRows + row] = r.mp;
        }
        const int all = row0 + row, i_tok = all / a.group;
        uint16_t* out = a.out + (token0 + i_tok) * a.o_ts + (at.head * a.group + all - i_tok * a.group) * a.o_hs;
#pragma unroll 1
        for (int q = 0; q < DP / 32; ++q) {
          const int d0 = q * 32;
          uint32_t o[32];
          tmem_load_32(o, tmem + lanes + Shape::kColO + d0);
          tmem_wait_load();
          if (!whole) {
#pragma unroll
            for (int k = 0; k < 32; ++k) part_out[(d0 + k) * kTileAttendRows + row] = __uint_as_float(o[k]);
          } else if (row < rows) {
#pragma unroll
            for (int k = 0; k < 32; k += 8) {
              uint32_t w[4];
#pragma unroll
              for (int e = 0; e < 4; ++e)
                w[e] = __bfloat16_as_ushort(__float2bfloat16_rn(__uint_as_float(o[k + of_eight<KIND>(2 * e)]) * f)) |
                       (static_cast<uint32_t>(__bfloat16_as_ushort(
                            __float2bfloat16_rn(__uint_as_float(o[k + of_eight<KIND>(2 * e + 1)]) * f)))
                        << 16);
              store_8(out, d0 + k, a.c.dim, a.o_vec, w);
            }
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.o_free);
      if (!whole) {
        // the last of the tile's CTAs to arrive joins them, once its run is done
        __threadfence();
        named_barrier(1, kSoftmaxThreads);
        if (threadIdx.x == 0 && atomic_add_acq_rel_gpu(a.counters + cta_first, 1) == cta_last - cta_first) {
          a.counters[cta_first] = 0;
          auto& join = sm.join[sm.joins++];
          join.cta_first = cta_first;
          join.parts = cta_last - cta_first + 1;
          join.first_slot = pair_start + cost_before > cta_first * per ? 1 : 0;
          join.b = at.b;
          join.head = at.head;
          join.row0 = row0;
          join.rows = rows;
        }
      }
      done += run;
      g += run;
      ++pair;
      if (g < g1) tile_next_pair<TT>(a, sm.before, &at);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kIssuer) tmem_free(sm.tmem, 512);

  // ---- join: a thread per row and quarter of the dimensions, parts in order
  const int joins = sm.joins;
  for (int n = 0; n < joins; ++n) {
    __threadfence();
    const auto join = sm.join[n];
    const int row = threadIdx.x & (kTileAttendRows - 1);
    const float* rest = a.partials + static_cast<size_t>(join.cta_first) * 2 * kTileSlotFloats + row;
    auto part_of = [&](int i) { return rest + static_cast<size_t>(i == 0 ? join.first_slot : 2 * i) * kTileSlotFloats; };
    float m = kAttendStart, mp = kAttendStart, sum = 0.f;
    for (int i = 0; i < join.parts; ++i) {
      m = fmaxf(m, __ldcg(part_of(i) + 256 * kTileAttendRows));
      mp = fmaxf(mp, __ldcg(part_of(i) + 258 * kTileAttendRows));
    }
    for (int i = 0; i < join.parts; ++i)
      sum += __ldcg(part_of(i) + 257 * kTileAttendRows) * ex2(__ldcg(part_of(i) + 256 * kTileAttendRows) - m);
    const float f = sum == 0.f ? 0.f : ex2(mp - m) / sum;
    const int token0 = a.t.begin_of(join.b, list_sizes(a));
    const int all = join.row0 + row, i_tok = all / a.group;
    uint16_t* out = a.out + (token0 + i_tok) * a.o_ts + (join.head * a.group + all - i_tok * a.group) * a.o_hs;
    static_assert(kTileAttendThreads == 4 * kTileAttendRows, "a quarter of the dimensions per thread");
#pragma unroll 1
    for (int d0 = (threadIdx.x / kTileAttendRows) * (DP / 4); d0 < (threadIdx.x / kTileAttendRows + 1) * (DP / 4); d0 += 16) {
      float v[16];
#pragma unroll
      for (int k = 0; k < 16; ++k) v[k] = 0.f;
#pragma unroll 1
      for (int i = 0; i < join.parts; ++i) {
        const float* part = part_of(i);
        const float w = ex2(__ldcg(part + 258 * kTileAttendRows) - mp);
#pragma unroll
        for (int k = 0; k < 16; ++k) v[k] = fmaf(__ldcg(part + (d0 + k) * kTileAttendRows), w, v[k]);
      }
      if (row < join.rows) {
#pragma unroll
        for (int k = 0; k < 16; k += 8) {
          uint32_t w[4];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            w[e] = __bfloat16_as_ushort(__float2bfloat16_rn(v[k + of_eight<KIND>(2 * e)] * f)) |
                   (static_cast<uint32_t>(__bfloat16_as_ushort(__float2bfloat16_rn(v[k + of_eight<KIND>(2 * e + 1)] * f))) << 16);
          store_8(out, d0 + k, a.c.dim, a.o_vec, w);
        }
      }
    }
  }
}

// ------------------------------------------------------------------ launch

size_t kv_attend_tile_partial_bytes(int sm_count) { return static_cast<size_t>(sm_count) * 2 * kTileSlotFloats * 4; }

template <int KIND, int DP, bool NARROW = false>
cudaError_t launch_attend_tile_as(const AttendArgs& a, int sm_count, cudaStream_t stream) {
  const size_t smem = TileShape<KIND, DP>::kSmem + (2 * a.t.seqs + 1) * sizeof(int);
  return launch_overlapped(attend_tile_kernel<KIND, DP, NARROW>, dim3(sm_count), kTileAttendThreads, smem, stream, a);
}

cudaError_t launch_attend_tile(const AttendArgs& a, int sm_count, cudaStream_t stream) {
  if (a.c.kind == kKvInt4)
    return a.c.dim == 64    ? launch_attend_tile_as<kKvInt4, 128, true>(a, sm_count, stream)
           : a.c.dim == 128 ? launch_attend_tile_as<kKvInt4, 128>(a, sm_count, stream)
                            : launch_attend_tile_as<kKvInt4, 256>(a, sm_count, stream);
  if (a.c.kind == kKvInt8)
    return a.c.dim <= 128 ? launch_attend_tile_as<kKvInt8, 128>(a, sm_count, stream)
                          : launch_attend_tile_as<kKvInt8, 256>(a, sm_count, stream);
  return a.c.dim <= 128 ? launch_attend_tile_as<kKvE4m3, 128>(a, sm_count, stream)
                        : launch_attend_tile_as<kKvE4m3, 256>(a, sm_count, stream);
}

}  // namespace se12
