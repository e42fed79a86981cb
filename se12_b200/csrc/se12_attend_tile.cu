// Attention over the paged 8-bit cache for many query rows per KV head
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
//   warps 0-7   softmax: a thread per row, two warps per 32 rows, one for each
//               half of the tile's tokens
//   warps 8-11  keys, warps 12-15 values: codes to FP16 tiles, two tiles deep
//   warp 16     one thread issues the products: S of tile j + 1 before P V of
//               tile j, so that the tensor pipe works during the softmax
//               (17-19 only complete its warp group)
//
// The roles walk the CTA's run on their own and meet at mbarriers only; the
// register file is split by role (setmaxnreg).
//
// As in attend_rows_kernel a row's references are raised only when a value
// passes them by 2^8; then the row's sums in tensor memory are scaled by the
// row's own threads, after P V of the tile before. The two warps of a row
// agree by one barrier with a vote per tile. The sum l is taken from the weights,
// a factor per 16 tokens, unless scales differ by more than 2^80.
// A row's capped logits take a polynomial of tanh for |x / cap| < 0.7 (two
// special-function calls less per logit; the unit has 16 a clock, and the
// softmax is what bounds the kernel).
//
// The work list (sequences, KV heads, row tiles, KV tiles) is cut into equal
// runs, one per CTA, and a tile's CTAs are joined as in attend_rows_kernel.
#include "se12_device.cuh"
#include "se12_serve.h"

#include <cuda_fp16.h>

namespace se12 {

constexpr int kTileAttendRows = 128;  // query rows of a tile
constexpr int kTileSoftmaxWarps = 8;
constexpr int kTileLoaderWarps = 4;   // for keys, and as many for values
constexpr int kTileAttendThreads = (kTileSoftmaxWarps + 2 * kTileLoaderWarps + 4) * 32;
// Registers per thread: 96 at launch (20 warps); 2 x 128 + 2 x 88 + 40 per
// thread of the five warp groups stays below 5 x 96.
constexpr int kTileSoftmaxRegs = 128, kTileLoaderRegs = 88, kTileIssuerRegs = 40;
static_assert(2 * kTileSoftmaxRegs + 2 * kTileLoaderRegs + kTileIssuerRegs <= 5 * 96, "more registers than the launch has");
constexpr int kTileKvBytes = 32768;   // an FP16 tile of keys or values
constexpr int kTileMeta = 4;          // tiles whose block scales are kept
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

// Arrives on the barrier once every product this thread issued is done.
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar)) : "memory");
}

// D = A B (+ D), FP16 operands from shared memory, fp32 accumulator.
__device__ __forceinline__ void tc_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(static_cast<uint32_t>(add))
      : "memory");
}

// The same with A in tensor memory.
__device__ __forceinline__ void tc_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(static_cast<uint32_t>(add))
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

__device__ __forceinline__ void tmem_store_16(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

__device__ __forceinline__ void tmem_wait_load() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_store() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Shared-memory operand in 128-byte-swizzled atoms of 8 rows x 128 bytes:
// stride between atoms along the rows (1024 bytes here) and, for a
// transposed operand, between 128-byte column panels.
__device__ __forceinline__ uint64_t tc_operand(uint32_t addr, uint32_t panel_bytes) {
  return static_cast<uint64_t>((addr >> 4) & 0x3FFF) | (static_cast<uint64_t>((panel_bytes >> 4) & 0x3FFF) << 16) |
         (static_cast<uint64_t>(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

// FP16 operands, fp32 accumulator, M = 128; B transposed (rows of
// contraction) or not.
__device__ __forceinline__ constexpr uint32_t tc_idesc(int n, bool transposed_b) {
  return (1u << 4) | ((transposed_b ? 1u : 0u) << 16) | (static_cast<uint32_t>(n >> 3) << 17) | ((128u >> 4) << 24);
}

// A barrier of `threads` threads that returns the OR of their predicates.
__device__ __forceinline__ bool vote_barrier(int id, int threads, bool x) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 q, %3, 0;\n\t"
      "barrier.cta.red.or.pred p, %1, %2, q;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r)
      : "r"(id), "r"(threads), "r"(static_cast<uint32_t>(x))
      : "memory");
  return r != 0;
}

// ------------------------------------------------------------------ work list

// A row tile's part of the work list.
struct TileSpan {
  int low;      // first token, a multiple of the KV tile
  int chunks;   // KV tiles (at least one: its CTA writes the rows)
  int pos_min, pos_max;
};

struct TileSeq {
  int tokens, first, length;
  int rows, tiles;
};

__device__ __forceinline__ TileSeq tile_sequence(const AttendArgs& a, int b) {
  TileSeq w;
  const int q0 = a.t.query_start ? max(a.t.query_start[b], 0) : b;
  const int q1 = a.t.query_start ? min(a.t.query_start[b + 1], a.t.tokens) : b + 1;
  w.tokens = max(q1 - q0, 0);
  w.length = max(a.t.lens[b], 0);
  w.first = w.length - w.tokens;
  w.rows = w.tokens * a.group;
  w.tiles = (w.rows + kTileAttendRows - 1) / kTileAttendRows;
  return w;
}

template <int TT>
__device__ __forceinline__ TileSpan tile_span(const AttendArgs& a, const TileSeq& w, int tile) {
  TileSpan s;
  s.pos_min = w.first + tile * kTileAttendRows / a.group;
  s.pos_max = w.first + min(tile * kTileAttendRows + kTileAttendRows - 1, w.rows - 1) / a.group;
  const int visible = a.window ? max(s.pos_min - a.window + 1, 0) : 0;
  s.low = visible / TT * TT;
  s.chunks = max((s.pos_max + 1 - s.low + TT - 1) / TT, 1);
  return s;
}

struct TilePlace {
  int b, head, tile, chunk;
  TileSeq w;
  TileSpan s;
};

struct TileSmem {
  float meta[kTileMeta][8][2];        // [16 tokens of the tile][scale of keys, log2 of values' scale]
  int meta_ok[kTileMeta];             // bit g: those tokens' page is good
  float row_scale[kTileAttendRows];
  float exchange[2][kTileAttendRows][2];
  float out_scale[kTileAttendRows];
  float merged_ref[kTileAttendRows];
  uint64_t k_full[2], v_full[2], s_full[2], p_full[2], pv_done[2];
  uint64_t q_full, o_free;
  uint64_t meta_full[kTileMeta];
  uint32_t tmem;
  int last;
  int before[1];  // [seqs + 1] KV tiles of the sequences before, per KV head
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

// ------------------------------------------------------------------ kernel

template <int KIND, int DP>
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
    for (int i = 0; i < kTileMeta; ++i) mbar_init(&sm.meta_full[i], 1);
    mbar_init(&sm.q_full, kTileSoftmaxWarps);
    mbar_init(&sm.o_free, kTileSoftmaxWarps);
    fence_barrier_init();
  }
  if (warp == kIssuer) tmem_alloc(&sm.tmem, 512);
  grid_launch_dependents();
  grid_dependency_wait();

  // ---- the work list
  const int heads = a.c.heads;
  for (int b = threadIdx.x; b < a.t.seqs; b += kTileAttendThreads) {
    const TileSeq w = tile_sequence(a, b);
    int n = 0;
    for (int t = 0; t < w.tiles; ++t) n += tile_span<TT>(a, w, t).chunks;
    sm.before[b + 1] = n;
  }
  if (threadIdx.x == 0) sm.before[0] = 0;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 0) {
    int carry = 0;
    for (int i = 1; i <= a.t.seqs; i += 32) {
      int v = i + lane <= a.t.seqs ? sm.before[i + lane] : 0;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int u = __shfl_up_sync(0xFFFFFFFFu, v, d);
        if (lane >= d) v += u;
      }
      v += carry;
      if (i + lane <= a.t.seqs) sm.before[i + lane] = v;
      carry = __shfl_sync(0xFFFFFFFFu, v, 31);
    }
  }
  __syncthreads();
  const uint32_t tmem = sm.tmem;
  const int total = sm.before[a.t.seqs] * heads;
  const int per = (total + static_cast<int>(gridDim.x) - 1) / static_cast<int>(gridDim.x);
  const int g0 = static_cast<int>(min(static_cast<long long>(blockIdx.x) * per, static_cast<long long>(total)));
  const int g1 = min(g0 + per, total);

  // ---- each role walks the CTA's run pair by pair
  TilePlace at{};
  auto start = [&]() {
    int lo = 0, hi = a.t.seqs - 1;  // last b with before[b] * heads <= g0
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (static_cast<long long>(sm.before[mid]) * heads <= g0) lo = mid;
      else hi = mid - 1;
    }
    at.b = lo;
    at.w = tile_sequence(a, lo);
    const int x = g0 - sm.before[lo] * heads, each = sm.before[lo + 1] - sm.before[lo];
    at.head = x / each;
    at.tile = 0;
    at.chunk = x - at.head * each;
    at.s = tile_span<TT>(a, at.w, 0);
    while (at.chunk >= at.s.chunks) {
      at.chunk -= at.s.chunks;
      at.s = tile_span<TT>(a, at.w, ++at.tile);
    }
  };
  auto next_pair = [&]() {  // there is one
    at.chunk = 0;
    if (++at.tile == at.w.tiles) {
      at.tile = 0;
      if (++at.head == heads) {
        at.head = 0;
        do {
          ++at.b;
        } while (sm.before[at.b + 1] == sm.before[at.b]);
        at.w = tile_sequence(a, at.b);
      }
    }
    at.s = tile_span<TT>(a, at.w, at.tile);
  };
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
    if (warp == kIssuer && lane == 0) {
      start();
      const uint32_t q_addr = smem_addr(q_tile), k_base = smem_addr(k_tiles), v_base = smem_addr(v_tiles);
      auto scores = [&](int j) {  // S of tile j (of the ring)
        const uint32_t k_addr = k_base + (j & 1) * kTileKvBytes;
        wait(&sm.k_full[j & 1], (j >> 1) & 1);
        if (dead) return;
        tc_fence_after();
#pragma unroll
        for (int k = 0; k < DP / 16; ++k)
          tc_mma_ss(tmem + Shape::kColS + (j & 1) * TT, tc_operand(q_addr + (k >> 2) * Shape::kQueryPanel + (k & 3) * 32, 16),
                    tc_operand(k_addr + (k >> 2) * Shape::kPanelBytes + (k & 3) * 32, 16), tc_idesc(TT, false), k > 0);
        tc_commit(&sm.s_full[j & 1]);
      };
      int done = 0, pair = 0;  // KV tiles and pairs before: the rings' phases
      for (int g = g0; g < g1; ++pair) {
        const int run = min(at.s.chunks - at.chunk, g1 - g);
        wait(&sm.q_full, pair & 1);
        scores(done);
        for (int i = 0; i < run && !dead; ++i) {
          const int j = done + i;
          if (i + 1 < run) scores(j + 1);
          wait(&sm.v_full[j & 1], (j >> 1) & 1);
          wait(&sm.p_full[j & 1], (j >> 1) & 1);
          if (i == 0 && pair > 0) wait(&sm.o_free, (pair - 1) & 1);
          if (dead) break;
          tc_fence_after();
          const uint32_t v_addr = v_base + (j & 1) * kTileKvBytes;
#pragma unroll
          for (int k = 0; k < TT / 16; ++k)
            tc_mma_ts(tmem + Shape::kColO, tmem + Shape::kColP + (j & 1) * (TT / 2) + k * 8,
                      tc_operand(v_addr + k * 2048, Shape::kPanelBytes), tc_idesc(DP, true), i > 0 || k > 0);
          tc_commit(&sm.pv_done[j & 1]);
        }
        if (dead) break;
        done += run;
        g += run;
        if (g < g1) next_pair();
      }
    }
    __syncwarp();
  } else if (warp >= kTileSoftmaxWarps) {
    // ---- codes to FP16 tiles
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kTileLoaderRegs));
    const bool keys = warp < kTileSoftmaxWarps + kTileLoaderWarps;
    const int tid = threadIdx.x - (kTileSoftmaxWarps + (keys ? 0 : kTileLoaderWarps)) * 32;  // 0 .. 127
    const uint8_t* codes = keys ? a.c.k_codes : a.c.v_codes;
    unsigned char* tiles = keys ? k_tiles : v_tiles;
    constexpr int kHalf = 4;                   // 16-byte vectors per thread and half tile
    constexpr int kPerToken = DP / 16;         // vectors per token
    constexpr int kStep = 128 / kPerToken;     // tokens per round: 8 or 16
    const int ch = tid % kPerToken, sub = tid / kPerToken;
    // The halves of all tiles in order, two on the way while a third is
    // widened: `ahead` is the place of the next one to load.
    start();
    int load_g = g0, load_run = min(at.s.chunks - at.chunk, g1 - g0), load_i = 0, load_half = 0;
    int pages = -1;  // of this lane's (lane < GROUPS) 16 tokens of the tile to load
    auto find_pages = [&]() {
      pages = -1;
      const int t0 = at.s.low + (at.chunk + load_i) * TT + lane * 16;
      if (lane < GROUPS && t0 <= at.s.pos_max) {
        const int column = t0 >> a.c.page_shift;
        pages = column < a.t.max_pages ? a.t.table[at.b * a.t.table_stride + column] : -1;
        if (pages < 0 || pages >= a.c.pages) {
          raise_status(kStatusBadArgument);
          pages = -1;
        }
      }
    };
    float ks = 0.f, vs = 0.f;  // this lane's block scales of the tile loaded last (first warp of the keys)
    unsigned ok = 0;
    auto load = [&](uint4 (&r)[kHalf]) {
      if (load_g >= g1) return;
      const int t0 = at.s.low + (at.chunk + load_i) * TT;
#pragma unroll
      for (int v = 0; v < kHalf; ++v) {
        const int token = (load_half * kHalf + v) * kStep + sub;
        const int page = __shfl_sync(0xFFFFFFFFu, pages, token >> 4);
        r[v] = make_uint4(0, 0, 0, 0);
        if (page >= 0 && t0 + token <= at.s.pos_max && ch * 16 < a.c.dim) {
          const long long row =
              (static_cast<long long>(page) * heads + at.head) * a.c.page_size + ((t0 + token) & (a.c.page_size - 1));
          r[v] = __ldg(reinterpret_cast<const uint4*>(codes + row * a.c.dim + ch * 16));
        }
      }
      load_half ^= 1;
      if (load_half) {  // a new tile begins
        if (keys && tid < 32) {
          const long long block = static_cast<long long>(pages) * heads + at.head;
          ks = pages >= 0 ? a.c.k_scales[block] : 0.f;
          vs = pages >= 0 ? a.c.v_scales[block] : 1.f;
          ok = __ballot_sync(0xFFFFFFFFu, pages >= 0);
        }
        return;
      }
      if (++load_i == load_run) {
        load_g += load_run;
        load_i = 0;
        if (load_g >= g1) return;
        if (at.chunk + load_run == at.s.chunks) next_pair();
        else at.chunk += load_run;
        load_run = min(at.s.chunks - at.chunk, g1 - load_g);
      }
      find_pages();
    };
    auto store = [&](const uint4 (&r)[kHalf], int half, unsigned char* tile) {
#pragma unroll
      for (int v = 0; v < kHalf; ++v) {
        const int token = (half * kHalf + v) * kStep + sub;
        uint4 h0, h1;
        widen<KIND>(r[v].x, h0.x, h0.y);
        widen<KIND>(r[v].y, h0.z, h0.w);
        widen<KIND>(r[v].z, h1.x, h1.y);
        widen<KIND>(r[v].w, h1.z, h1.w);
        // neighbouring panels' lanes write their two vectors in opposite
        // order, so that a quarter-warp covers all banks
        const bool flip = (ch >> 2) & 1;
        unsigned char* row = tile + (ch >> 2) * Shape::kPanelBytes + token * 128;
        const int c16 = (ch & 3) * 2;
        *reinterpret_cast<uint4*>(row + (((c16 + flip) ^ (token & 7)) << 4)) = flip ? h1 : h0;
        *reinterpret_cast<uint4*>(row + (((c16 + !flip) ^ (token & 7)) << 4)) = flip ? h0 : h1;
      }
    };
    uint4 r0[kHalf], r1[kHalf], r2[kHalf];
    find_pages();
    load(r0);
    load(r1);
    const int halves = 2 * (g1 - g0);
    auto step = [&](int n, uint4 (&cur)[kHalf], uint4 (&later)[kHalf]) {
      if (n >= halves) return;
      const int j = n >> 1, half = n & 1, stage = j & 1;  // ring tile
      if (half == 0) {
        // the tile two before has been read by its products
        if (j >= 2) wait(keys ? &sm.s_full[stage] : &sm.pv_done[stage], ((j >> 1) + 1) & 1);
        if (keys && tid < 32) {  // loaded with this tile's first half; the next tile's are loaded below
          const int slot = j % kTileMeta;
          if (lane < GROUPS) {
            sm.meta[slot][lane][0] = ks;
            sm.meta[slot][lane][1] = lg2(vs);
          }
          if (lane == 0) sm.meta_ok[slot] = static_cast<int>(ok);
          __syncwarp();
          if (lane == 0) mbar_arrive(&sm.meta_full[slot]);
        }
      }
      load(later);
      store(cur, half, tiles + stage * kTileKvBytes);
      if (half == 1) {
        fence_proxy_async_shared();
        __syncwarp();
        if (lane == 0) mbar_arrive(keys ? &sm.k_full[stage] : &sm.v_full[stage]);
      }
    };
    for (int n = 0; n < halves; n += 3) {
      step(n, r0, r2);
      step(n + 1, r1, r0);
      step(n + 2, r2, r1);
    }
  } else {
    // ---- softmax: row 32 (warp % 4) + lane, tokens half * TT / 2 ..
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kTileSoftmaxRegs));
    constexpr int HC = TT / 2, HG = HC / 16;
    constexpr int kSoftmaxThreads = kTileSoftmaxWarps * 32;
    const int quarter = warp & 3, half = warp >> 2;
    const int row = quarter * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
    const bool capped_logits = a.softcap != 0.f;
    const float cap2 = a.softcap * kLog2e;
    auto wait_all = [&](uint64_t* bar, uint32_t parity) {  // one answer for the warp
      wait(bar, parity);
      dead = __any_sync(0xFFFFFFFFu, dead);
    };
    // A pair's queries as FP16 times 2^-e, two threads per row.
    auto load_queries = [&]() {
      const int q_row = threadIdx.x >> 1, part = threadIdx.x & 1;
      const int token0 = a.t.query_start ? a.t.query_start[at.b] : at.b;
      const int all = at.tile * kTileAttendRows + q_row;
      const bool live = all < at.w.rows;
      const int i = live ? all / a.group : 0;
      const uint16_t* src = a.q + (token0 + i) * a.q_ts + (at.head * a.group + (live ? all - i * a.group : 0)) * a.q_hs;
      auto vector = [&](int c) {  // 16-byte chunk c of the row
        uint4 v = make_uint4(0, 0, 0, 0);
        if (live && c * 8 < a.c.dim) {
          if (a.q_vec) {
            v = *reinterpret_cast<const uint4*>(src + c * 8);
          } else {
            const uint16_t* s = src + c * 8;
            v = make_uint4(s[0] | (static_cast<uint32_t>(s[1]) << 16), s[2] | (static_cast<uint32_t>(s[3]) << 16),
                           s[4] | (static_cast<uint32_t>(s[5]) << 16), s[6] | (static_cast<uint32_t>(s[7]) << 16));
          }
        }
        return v;
      };
      unsigned big = 0;
#pragma unroll 4
      for (int j = 0; j < DP / 16; ++j) {
        const uint4 v = vector(j * 2 + part);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t w = word_of(v, k);
          big = max(big, max((w << 16) & 0x7FFFFFFFu, w & 0x7FFF0000u));
        }
      }
      big = max(big, __shfl_xor_sync(0xFFFFFFFFu, big, 1));
      int e = static_cast<int>(big >> 23) - 127;
      e = max(min(e, 120), -120);
      const float down = __uint_as_float(static_cast<unsigned>(127 - e) << 23);
      auto halves = [&](uint32_t w) {
        return half2_bits(__floats2half2_rn(__uint_as_float(w << 16) * down, __uint_as_float(w & 0xFFFF0000u) * down));
      };
#pragma unroll 4
      for (int j = 0; j < DP / 16; ++j) {  // (from the cache again: fewer registers)
        const int c = j * 2 + part;
        const uint4 v = vector(c);
        *reinterpret_cast<uint4*>(q_tile + (c >> 3) * Shape::kQueryPanel + q_row * 128 + (((c & 7) ^ (q_row & 7)) << 4)) =
            make_uint4(halves(v.x), halves(v.y), halves(v.z), halves(v.w));
      }
      if (part == 0) sm.row_scale[q_row] = __uint_as_float(static_cast<unsigned>(127 + e) << 23) * a.scale;
      fence_proxy_async_shared();
      named_barrier(5, kSoftmaxThreads);
      if (lane == 0) mbar_arrive(&sm.q_full);
    };
    start();
    load_queries();
    int done = 0;  // KV tiles of the pairs before: the rings' phases
    for (int g = g0; g < g1;) {
      const int run = min(at.s.chunks - at.chunk, g1 - g);
      const int rows = min(kTileAttendRows, at.w.rows - at.tile * kTileAttendRows);
      const int t_first = at.s.low + at.chunk * TT;
      const int pos_min = at.s.pos_min, pos_max = at.s.pos_max;
      const bool active = quarter * 32 < rows;  // rows past the tile's are left out, warp by warp
      const float row_scale = sm.row_scale[row] * (capped_logits ? 1.f / a.softcap : kLog2e);
      const int pos = at.w.first + min(at.tile * kTileAttendRows + row, at.w.rows - 1) / a.group;
      float m = kAttendStart, l = 0.f, mp = kAttendStart;
      for (int i = 0; i < run; ++i) {
        const int j = done + i, slot = j % kTileMeta;
        const int t0 = t_first + i * TT + half * HC;
        wait_all(&sm.meta_full[slot], (j / kTileMeta) & 1);
        wait_all(&sm.s_full[j & 1], (j >> 1) & 1);
        tc_fence_after();
        if (active) {
          float x[HC];
#pragma unroll
          for (int q = 0; q < HC / 32; ++q) {
            uint32_t s[32];
            tmem_load_32(s, tmem + lanes + Shape::kColS + (j & 1) * TT + half * HC + q * 32);
            tmem_wait_load();
#pragma unroll
            for (int k = 0; k < 32; ++k) x[q * 32 + k] = __uint_as_float(s[k]);
          }
          float lv[HG];
#pragma unroll
          for (int q = 0; q < HG; ++q) {
            const float f = row_scale * sm.meta[slot][half * HG + q][0];
            lv[q] = sm.meta[slot][half * HG + q][1];
#pragma unroll
            for (int k = 0; k < 16; ++k) x[q * 16 + k] *= f;
          }
          if (capped_logits) {
            // cap tanh(u), u = x / cap: u times a polynomial of u^2 of degree
            // 4 (Chebyshev fit of tanh(u) / u on |u| <= 0.7, off by 1.9e-7)
            float wide = 0.f;
#pragma unroll
            for (int k = 0; k < HC; ++k) wide = fmaxf(wide, fabsf(x[k]));
            if (!__any_sync(0xFFFFFFFFu, wide > 0.7f)) {
#pragma unroll
              for (int k = 0; k < HC; ++k) {
                const float u = x[k], t = u * u;
                float y = fmaf(0.0137912829f, t, -0.0508535559f);
                y = fmaf(y, t, 0.132816473f);
                y = fmaf(y, t, -0.33330266f);
                y = fmaf(y, t, 0.999999706f);
                x[k] = y * (u * cap2);
              }
            } else {
#pragma unroll
              for (int k = 0; k < HC; ++k)
                x[k] = cap2 - __fdividef(2.f * cap2, ex2(x[k] * (2.f * kLog2e)) + 1.f);
            }
          }
          const int ok = sm.meta_ok[slot] >> (half * HG);
          const bool masked = t0 + HC - 1 > pos_min || (a.window && pos_max - t0 >= a.window) ||
                              (ok & ((1 << HG) - 1)) != (1 << HG) - 1;
          if (masked) {
#pragma unroll
            for (int k = 0; k < HC; ++k) {
              const int t = t0 + k;
              if (t > pos || (a.window && pos - t >= a.window) || !((ok >> (k >> 4)) & 1)) x[k] = kNegInf;
            }
          }
          float top = kNegInf, top_v = kNegInf;
#pragma unroll
          for (int q = 0; q < HG; ++q) {
            float t = x[q * 16];
#pragma unroll
            for (int k = 1; k < 16; ++k) t = fmaxf(t, x[q * 16 + k]);
            top = fmaxf(top, t);
            top_v = fmaxf(top_v, t + lv[q]);
          }
          if (top - m > kAttendRaiseSum) {  // this half's own reference
            l *= ex2(m - top);
            m = top;
          }
          if (vote_barrier(1 + quarter, 64, top_v - mp > kAttendRaise)) {
            sm.exchange[half][row][0] = top_v;
            named_barrier(1 + quarter, 64);
            const float tv = fmaxf(mp, fmaxf(top_v, sm.exchange[half ^ 1][row][0]));
            const float f = ex2(mp - tv);
            mp = tv;
            if (i > 0) {  // the sums so far, half of the columns each
              wait_all(&sm.pv_done[(j - 1) & 1], ((j - 1) >> 1) & 1);
              tc_fence_after();
#pragma unroll
              for (int q = 0; q < DP / 64; ++q) {
                const uint32_t addr = tmem + lanes + Shape::kColO + half * (DP / 2) + q * 32;
                uint32_t o[32];
                tmem_load_32(o, addr);
                tmem_wait_load();
#pragma unroll
                for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
                tmem_store_32(addr, o);
              }
              tmem_wait_store();
            }
            named_barrier(1 + quarter, 64);  // the exchange has been read
          }
          // weights, and the sum from them: 2^(x - m) = w 2^(mp - lv - m)
          float up[HG];
          bool far = false;
#pragma unroll
          for (int q = 0; q < HG; ++q) {
            up[q] = mp - lv[q] - m;
            far |= !(up[q] <= 80.f);
          }
          uint32_t p[HC / 2];
          if (!__any_sync(0xFFFFFFFFu, far)) {
#pragma unroll
            for (int q = 0; q < HG; ++q) {
              const float shift = lv[q] - mp;
              float sum = 0.f;
#pragma unroll
              for (int k = 0; k < 8; ++k) {
                const float w0 = ex2(x[q * 16 + 2 * k] + shift), w1 = ex2(x[q * 16 + 2 * k + 1] + shift);
                sum += w0 + w1;
                p[q * 8 + k] = half2_bits(__floats2half2_rn(w0, w1));
              }
              l = fmaf(sum, ex2(up[q]), l);
            }
          } else {
#pragma unroll
            for (int q = 0; q < HG; ++q) {
              const float shift = lv[q] - mp;
#pragma unroll
              for (int k = 0; k < 8; ++k) {
                const float x0 = x[q * 16 + 2 * k], x1 = x[q * 16 + 2 * k + 1];
                l += ex2(x0 - m) + ex2(x1 - m);
                // a masked token weighs nothing, whatever its block's scale holds
                const float w0 = x0 == kNegInf ? 0.f : ex2(x0 + shift), w1 = x1 == kNegInf ? 0.f : ex2(x1 + shift);
                p[q * 8 + k] = half2_bits(__floats2half2_rn(w0, w1));
              }
            }
          }
          // P of the tile two before has been read
          if (j >= 2) wait_all(&sm.pv_done[j & 1], ((j >> 1) + 1) & 1);
          const uint32_t to = tmem + lanes + Shape::kColP + (j & 1) * (TT / 2) + half * (HC / 2);
#pragma unroll
          for (int q = 0; q < HC / 32; ++q) tmem_store_16(to + q * 16, p + q * 16);
          tmem_wait_store();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.p_full[j & 1]);
      }
      // ---- the pair's end: the next pair's queries first (this one's products
      // with them are done), then the row's sums
      const int pair_start = g - at.chunk, pair_end = pair_start + at.s.chunks;
      const int cta_first = pair_start / per, cta_last = (pair_end - 1) / per;
      const bool whole = cta_first == cta_last;
      float* part_out = a.partials + (static_cast<size_t>(blockIdx.x) * 2 + (pair_start > g0 ? 1 : 0)) * kTileSlotFloats;
      const int token0 = a.t.query_start ? a.t.query_start[at.b] : at.b;
      const int row0 = at.tile * kTileAttendRows, head = at.head;
      const bool more = g + run < g1;
      named_barrier(5, kSoftmaxThreads);  // every warp has read row_scale and seen the last scores
      if (more) {
        next_pair();
        load_queries();
      }
      wait_all(&sm.pv_done[(done + run - 1) & 1], ((done + run - 1) >> 1) & 1);
      tc_fence_after();
      if (active) {
        sm.exchange[half][row][0] = m;
        sm.exchange[half][row][1] = l;
        named_barrier(1 + quarter, 64);
        const float m2 = sm.exchange[half ^ 1][row][0], l2 = sm.exchange[half ^ 1][row][1];
        const float mm = fmaxf(m, m2);
        const float sum = half ? l2 * ex2(m2 - mm) + l * ex2(m - mm) : l * ex2(m - mm) + l2 * ex2(m2 - mm);
        const float f = whole ? (sum == 0.f ? 0.f : ex2(mp - mm) / sum) : 1.f;
        if (!whole && half == 0 && row < rows) {
          float* st = part_out + kTileAttendRows * 256 + row * 4;
          st[0] = mm;
          st[1] = sum;
          st[2] = mp;
        }
        const int all = row0 + row, i_tok = all / a.group;
        uint16_t* out = a.out + (token0 + i_tok) * a.o_ts + (head * a.group + all - i_tok * a.group) * a.o_hs;
#pragma unroll
        for (int q = 0; q < DP / 64; ++q) {
          const int d0 = half * (DP / 2) + q * 32;
          uint32_t o[32];
          tmem_load_32(o, tmem + lanes + Shape::kColO + d0);
          tmem_wait_load();
          if (row < rows && d0 < a.c.dim) {
            if (whole) {
#pragma unroll
              for (int k = 0; k < 32; k += 8) {
                uint32_t w[4];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  w[e] = __bfloat16_as_ushort(__float2bfloat16_rn(__uint_as_float(o[k + 2 * e]) * f)) |
                         (static_cast<uint32_t>(__bfloat16_as_ushort(__float2bfloat16_rn(__uint_as_float(o[k + 2 * e + 1]) * f))) << 16);
                if (d0 + k < a.c.dim) {
                  if (a.o_vec) {
                    *reinterpret_cast<uint4*>(out + d0 + k) = make_uint4(w[0], w[1], w[2], w[3]);
                  } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                      out[d0 + k + 2 * e] = static_cast<uint16_t>(w[e]);
                      out[d0 + k + 2 * e + 1] = static_cast<uint16_t>(w[e] >> 16);
                    }
                  }
                }
              }
            } else {
              float4* dst = reinterpret_cast<float4*>(part_out + row * 256 + d0);
#pragma unroll
              for (int k = 0; k < 8; ++k)
                dst[k] = make_float4(__uint_as_float(o[4 * k]), __uint_as_float(o[4 * k + 1]), __uint_as_float(o[4 * k + 2]),
                                     __uint_as_float(o[4 * k + 3]));
            }
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.o_free);
      if (!whole) {
        // ---- join the CTAs of the tile: the last to arrive adds all in order
        __threadfence();
        named_barrier(5, kSoftmaxThreads);
        if (threadIdx.x == 0) {
          const int arrived = atomic_add_acq_rel_gpu(a.counters + cta_first, 1);
          sm.last = arrived == cta_last - cta_first;
          if (sm.last) a.counters[cta_first] = 0;
        }
        named_barrier(5, kSoftmaxThreads);
        if (sm.last) {
          __threadfence();
          const int parts = cta_last - cta_first + 1;
          const float* rest = a.partials + static_cast<size_t>(cta_first) * 2 * kTileSlotFloats;
          const float* first = rest + (pair_start > cta_first * per ? kTileSlotFloats : 0);
          auto part_of = [&](int i) { return i == 0 ? first : rest + static_cast<size_t>(i) * 2 * kTileSlotFloats; };
          if (threadIdx.x < rows) {
            float mm = kAttendStart, mmp = kAttendStart;
            for (int i = 0; i < parts; ++i) {
              const float* st = part_of(i) + kTileAttendRows * 256 + threadIdx.x * 4;
              mm = fmaxf(mm, __ldcg(st));
              mmp = fmaxf(mmp, __ldcg(st + 2));
            }
            float sum = 0.f;
            for (int i = 0; i < parts; ++i) {
              const float* st = part_of(i) + kTileAttendRows * 256 + threadIdx.x * 4;
              sum += __ldcg(st + 1) * ex2(__ldcg(st) - mm);
            }
            sm.merged_ref[threadIdx.x] = mmp;
            sm.out_scale[threadIdx.x] = sum == 0.f ? 0.f : ex2(mmp - mm) / sum;
          }
          named_barrier(5, kSoftmaxThreads);
          const int vectors = a.c.dim / 4;
          for (int i = threadIdx.x; i < rows * vectors; i += kSoftmaxThreads) {
            const int r = i / vectors, d = (i - r * vectors) * 4;
            const float ref = sm.merged_ref[r], f = sm.out_scale[r];
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
            for (int n = 0; n < parts; ++n) {
              const float* pt = part_of(n);
              const float4 u = __ldcg(reinterpret_cast<const float4*>(pt + r * 256 + d));
              const float w = ex2(__ldcg(pt + kTileAttendRows * 256 + r * 4 + 2) - ref);
              v.x += u.x * w, v.y += u.y * w, v.z += u.z * w, v.w += u.w * w;
            }
            const int all = row0 + r, i_tok = all / a.group;
            uint16_t* out = a.out + (token0 + i_tok) * a.o_ts + (head * a.group + all - i_tok * a.group) * a.o_hs + d;
            out[0] = __bfloat16_as_ushort(__float2bfloat16_rn(v.x * f));
            out[1] = __bfloat16_as_ushort(__float2bfloat16_rn(v.y * f));
            out[2] = __bfloat16_as_ushort(__float2bfloat16_rn(v.z * f));
            out[3] = __bfloat16_as_ushort(__float2bfloat16_rn(v.w * f));
          }
          named_barrier(5, kSoftmaxThreads);  // sm.last and the references are free
        }
      }
      done += run;
      g += run;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kIssuer) tmem_free(tmem, 512);
}

// ------------------------------------------------------------------ launch

size_t kv_attend_tile_partial_bytes(int sm_count) { return static_cast<size_t>(sm_count) * 2 * kTileSlotFloats * 4; }

template <int KIND, int DP>
cudaError_t launch_attend_tile_as(const AttendArgs& a, int sm_count, cudaStream_t stream) {
  const size_t smem = TileShape<KIND, DP>::kSmem + a.t.seqs * sizeof(int);
  return launch_overlapped(attend_tile_kernel<KIND, DP>, dim3(sm_count), kTileAttendThreads, smem, stream, a);
}

cudaError_t launch_attend_tile(const AttendArgs& a, int sm_count, cudaStream_t stream) {
  if (a.c.kind == kKvInt8)
    return a.c.dim <= 128 ? launch_attend_tile_as<kKvInt8, 128>(a, sm_count, stream)
                          : launch_attend_tile_as<kKvInt8, 256>(a, sm_count, stream);
  return a.c.dim <= 128 ? launch_attend_tile_as<kKvE4m3, 128>(a, sm_count, stream)
                        : launch_attend_tile_as<kKvE4m3, 256>(a, sm_count, stream);
}

}  // namespace se12
