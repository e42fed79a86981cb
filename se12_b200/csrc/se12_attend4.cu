// Attention over the paged 4-bit cache for few query rows per KV head (next
// tokens, drafted tokens): split over the tokens, joined in the same launch.
//
//   s_ij = sum_g ks_jg sum_{d in g} q_id (u_jd - 8) + ko_jg sum_{d in g} q_id
//   o_id = sum_j p_ij (vs_jg (u_jd - 8) + vo_jg),  p_ij = 2^(s_ij + E_j) / sum_j 2^s_ij
//
// for groups g of 64 dimensions, u the codes, ks, ko, vs, vo scales and
// offsets. A code never becomes a value: its four bits, shifted and masked, are
// the FP16 subnormal u 2^-22 (or u 2^-18, four bits higher, met by a query's or a
// sum's factor of 1/16), which mma.sync multiplies exactly. So 8 keys take six
// instructions and 8 values seven; subtracting the zero point from each pair of
// them would take four more. Zero points are put right afterwards: keys' with
// the sums of the query's groups, values' by the products of one more instruction
// per group, whose second operand is the same rounded weights that the codes were
// multiplied by (a difference of roundings would not cancel where weights are
// equal).
//
// A group's products are scaled in fp32 (keys) or through its weights
// p vs in FP16 (values; the scales are relative to 2^E, so that both factors
// have FP16's full precision whatever the values' size).
//
// Work list, warps' parts of a run, joins: as attend_rows_kernel, see there. A
// warp's chunks come by asynchronous copies of 16 bytes per lane, three chunks
// (of 2048 codes of keys and of values) deep: a whole chunk takes ten copies, where
// boxes copied by one lane each are a loop over the lanes (206 us for the first case
// below, 190 with copies by all).
//
// 64 sequences of 1000 to 16384 tokens, 64 query and 8 KV heads of 128: 166 us,
// 3.9 TB/s (copies alone 114; with the keys' products 131); one of 131071, 32 and
// 16 heads of 128, capped: 81 us, 3.8 TB/s. What bounds it is the issue of 305
// instructions per 16 tokens and head at 2.1 of 4 a cycle with 12 warps per SM. 16
// warps of 128 registers work out again what they cannot hold (351 instructions,
// 174 us); a warp that copies for four others does not keep up (183 us).
#include "se12_attend.cuh"

#include <cuda_bf16.h>
#include <type_traits>

namespace se12 {

constexpr int kRows4Warps = 4;
constexpr int kRows4Threads = kRows4Warps * 32;
constexpr int kRows4SlotRows = 16;
constexpr int kRows4SlotFloats = kRows4SlotRows * (256 + 4);  // sums, then (mp, l) per row
constexpr int kRows4MaxCtas = 3;       // per SM
// What a pair's queries, joins and output cost, in chunks. (4, 8, 12, 16 and 24: 24
// sequences with drafted tokens 87, 77, 68, 68 and 71 us; 16 with a window 53, 48,
// 46, 45 and 45; equal lengths do not care.)
constexpr int kRows4PairCost = 16;
constexpr float kRows4WideCap = 128.f;  // as kAttendWideCap

template <int DIM>
struct Rows4Shape {
  static constexpr int kGroups = DIM / 64;
  static constexpr int kSubs = 256 / DIM;                     // 16 tokens each, of a chunk
  static constexpr int kStages = 3;
  static constexpr int kChunk = 16 * kSubs;
  static constexpr int kBox = 8 * DIM;                        // codes of 16 tokens
  static constexpr int kCodes = 2 * kSubs * kBox;             // of a stage: keys, then values
  static constexpr int kKeyLines = 64 * kGroups;              // scales of 16 tokens
  static constexpr int kValueLines = 64 * kGroups + 32;
  static constexpr int kLines = kSubs * (kKeyLines + kValueLines);
  static constexpr int kStage = kCodes + kLines;              // (a multiple of 16)
};

template <int DIM>
struct Rows4Smem {
  using Shape = Rows4Shape<DIM>;
  alignas(128) unsigned char pipes[kRows4Warps][Shape::kStages][Shape::kStage];
  union {
    uint4 queries[2 * DIM / 32 * 32];     // FP16 fragments: [n-tile][group][word][lane]
    float deposit[2048];                  // the warps' sums while they are joined
  };
  float query_sums[2 * DIM / 64][8];       // 2^-22 sum of a group's, [n-tile][group][row]
  float row_scale[kRows4SlotRows];
  float stat[kRows4Warps][kRows4SlotRows][2];  // mp, l of each warp
  float factor[kRows4Warps][kRows4SlotRows];
  float out_scale[kRows4SlotRows];
  int last;
  int most;
  int before[1];  // [seqs + 1] units of the sequences before (per KV head)
};

// A value that stays in its register: the compiler would rather work out again
// for every chunk what it knows from the lane (40 of 350 instructions per 16
// tokens).
__device__ __forceinline__ void keep(uint32_t& x) { asm volatile("" : "+r"(x)); }

__device__ __forceinline__ uint2 lds64(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
  return v;
}

__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr));
  return v;
}

__device__ __forceinline__ float lds_half(uint32_t addr) {
  uint16_t v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(addr));
  return __half2float(__ushort_as_half(v));
}

// N consecutive words.
template <int N>
__device__ __forceinline__ void lds_words(uint32_t (&w)[N], uint32_t addr) {
  if constexpr (N == 1) {
    w[0] = lds32(addr);
  } else if constexpr (N == 2) {
    const uint2 v = lds64(addr);
    w[0] = v.x, w[1] = v.y;
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const uint4 v = lds128(addr + 4 * i);
      w[i] = v.x, w[i + 1] = v.y, w[i + 2] = v.z, w[i + 3] = v.w;
    }
  }
}

// The first product of a sum.
__device__ __forceinline__ void mma_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

__device__ __forceinline__ uint32_t mul_halves(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

__device__ __forceinline__ float2 halves_of(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }

// Where codes lie in each half of a word to be FP16 subnormals, u 2^-22 and u
// 2^-18: the first and second of a half's four shifted up by two bits, the third
// and fourth down by six. (A product is cut 24 bits or so below the largest one of
// its sum as if a subnormal began at 2^-14: two bits more are worth a shift.)
constexpr uint32_t kLowCodes = 0x003C003Cu, kHighCodes = 0x03C003C0u;

// 16 bytes, asynchronously; the second only where `use`.
__device__ __forceinline__ void copy_16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_16_if(bool use, uint32_t dst, const void* src) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %2, 0;\n\t@p cp.async.cg.shared.global [%0], [%1], 16;\n\t}" ::"r"(dst), "l"(src),
      "r"(static_cast<uint32_t>(use))
      : "memory");
}

// Where in a box of 16 tokens' codes a sixteenth of token `token`'s row lies:
// rows of 64 and 128 bytes are swizzled, so that a warp's reads meet all banks.
template <int DIM>
__device__ __forceinline__ uint32_t row_part(int token, int sixteenth) {
  if (DIM == 256) return token * 128 + ((sixteenth ^ (token & 7)) << 4);
  if (DIM == 128) return token * 64 + ((sixteenth ^ ((token >> 1) & 3)) << 4);
  return token * 32 + (sixteenth << 4);
}

// Four dimensions, from d on, of row `row` of a sequence's (token, head) rows.
__device__ __forceinline__ void store_four(const AttendArgs& a, int token0, int head, int row, int d, const float4& v, float f) {
  const int i = row / a.group;
  uint16_t* out = a.out + (token0 + i) * a.o_ts + (head * a.group + row - i * a.group) * a.o_hs + d;
  auto bits = [&](float x) { return static_cast<uint32_t>(__bfloat16_as_ushort(__float2bfloat16_rn(x * f))); };
  if (a.o_vec) {
    *reinterpret_cast<uint2*>(out) = make_uint2(bits(v.x) | (bits(v.y) << 16), bits(v.z) | (bits(v.w) << 16));
  } else {
    out[0] = static_cast<uint16_t>(bits(v.x));
    out[1] = static_cast<uint16_t>(bits(v.y));
    out[2] = static_cast<uint16_t>(bits(v.z));
    out[3] = static_cast<uint16_t>(bits(v.w));
  }
}

// ONE: pages are as long as a chunk or longer (a chunk lies in one page).
template <int DIM, int NT, int CTAS, bool ONE>
__global__ void __launch_bounds__(kRows4Threads, CTAS)
    attend4_rows_kernel(const AttendArgs a) {
  using Shape = Rows4Shape<DIM>;
  // A place in the work list, which counts units: a pair's (KV head x row tile) are
  // kRows4PairCost for its beginning and end, from `start` on, and one per chunk. The
  // pair's chunks in this CTA's run end before `stop`.
  struct Spot {
    int b, head, tile, chunk, stop;
    int start;
    SeqWork w;
  };
  constexpr int G = Shape::kGroups, SUBS = Shape::kSubs, CHUNK = Shape::kChunk, STAGES = Shape::kStages, ROWS = 8 * NT;
  constexpr int Z = (G + 1) / 2;
  extern __shared__ unsigned char smem_raw[];
  Rows4Smem<DIM>& sm = *reinterpret_cast<Rows4Smem<DIM>*>((reinterpret_cast<uintptr_t>(smem_raw) + 127) & ~uintptr_t(127));
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int r = lane >> 2, c = lane & 3;

  grid_launch_dependents();
  grid_dependency_wait();

  // ---- the work list
  const int heads = a.c.heads;
  if (threadIdx.x == 0) sm.before[0] = sm.most = 0;
  __syncthreads();
  const int limit = static_cast<int>(kWorkLimit / heads);
  int most = 0;
  for (int b = threadIdx.x; b < a.t.seqs; b += kRows4Threads) {
    const SeqWork w = sequence_work<CHUNK, ROWS>(a, b);
    check_length(a, b);
    sm.before[b + 1] = times_work(w.chunks + kRows4PairCost, w.tiles, limit);
    most = max(most, w.chunks);
  }
  atomicMax(&sm.most, most);
  __syncthreads();
  if (warp == 0) sum_up_to(sm.before, a.t.seqs, limit, lane);
  __syncthreads();
  if (sm.before[a.t.seqs] == limit) {
    if (threadIdx.x == 0) raise_status(kStatusBadArgument);
    return;
  }
  const int total = sm.before[a.t.seqs] * heads;
  // short pairs are not cut below a chunk per warp
  const int per = max(min(kRows4Warps, sm.most), (total + static_cast<int>(gridDim.x) - 1) / static_cast<int>(gridDim.x));
  const int u0 = static_cast<int>(min(static_cast<long long>(blockIdx.x) * per, static_cast<long long>(total)));
  const int u1 = min(u0 + per, total);
  if (u0 >= u1) return;

  // The first chunk at or past a unit of the list.
  auto locate = [&](int u) {
    int lo = 0, hi = a.t.seqs - 1;  // last b with before[b] * heads <= u
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (static_cast<long long>(sm.before[mid]) * heads <= u) lo = mid;
      else hi = mid - 1;
    }
    Spot p;
    p.b = lo;
    p.w = sequence_work<CHUNK, ROWS>(a, lo);
    const int x = u - sm.before[lo] * heads, each = p.w.chunks + kRows4PairCost;
    const int pair = x / each, at = x - pair * each;
    p.head = pair / p.w.tiles;
    p.tile = pair - p.head * p.w.tiles;
    p.start = u - at;
    p.chunk = max(at - kRows4PairCost, 0);
    p.stop = min(p.w.chunks, u1 - p.start - kRows4PairCost);
    return p;
  };
  // To the place `by` chunks on; false where that is past this CTA's run.
  auto advance = [&](Spot& p, int by) {
    p.chunk += by;
    if (p.chunk < p.stop) return true;
#pragma unroll 1
    while (p.chunk >= p.w.chunks) {
      p.chunk -= p.w.chunks;
      p.start += p.w.chunks + kRows4PairCost;
      if (p.start + kRows4PairCost >= u1) return false;
      if (++p.tile == p.w.tiles) {
        p.tile = 0;
        if (++p.head == heads) {
          p.head = 0;
          do {
            ++p.b;
          } while (sm.before[p.b + 1] == sm.before[p.b]);
          // (chunks left over continue in the next sequence)
          p.w = sequence_work<CHUNK, ROWS>(a, p.b);
        }
      }
    }
    p.stop = min(p.w.chunks, u1 - p.start - kRows4PairCost);
    return p.chunk < p.stop;
  };

  // ---- this warp's pipeline: every fourth chunk of the run. A lane copies the
  // same 16 bytes of every box; a chunk is one group of its copies.
  const uint32_t pipe = smem_addr(sm.pipes[warp]);
  Spot next = locate(u0);
  bool more = advance(next, warp);  // `next` is a chunk of the run
  // ONE: a chunk is one piece, whose row every lane has; otherwise 16 tokens are,
  // and lane `sub` has theirs.
  constexpr int kPiece = ONE ? CHUNK : 16;
  int next_row = -1;  // of the next chunk to issue: where a piece of it begins, -1: not to be read
  auto fetch_rows = [&]() {
    const int t0 = next.w.low + next.chunk * CHUNK + (ONE ? 0 : lane * 16);
    const bool due = (ONE || lane < SUBS) && t0 < next.w.s.length && t0 + kPiece > visible_from(next.w.s.first, a.window);
    unsigned page = 0;  // (a sequence's length is one that its table row has pages for)
    if (due) page = a.t.table[next.b * a.t.table_stride + (t0 >> a.c.page_shift)];
    const bool there = due && page < static_cast<unsigned>(a.c.pages);
    next_row = there ? (static_cast<int>(page) * heads + next.head) * a.c.page_size + (t0 & (a.c.page_size - 1)) : -1;
    if (due && !there) raise_status(kStatusBadArgument);
  };
  constexpr int kCopies = Shape::kBox / 512;  // of 512 bytes, of a box
  uint32_t copy_to[kCopies];
#pragma unroll
  for (int i = 0; i < kCopies; ++i) {
    const int vector = i * 32 + lane;
    copy_to[i] = pipe + row_part<DIM>(vector / (DIM / 32), vector % (DIM / 32));
    keep(copy_to[i]);
  }
  uint32_t line_to = pipe + Shape::kCodes + lane * 16;
  keep(line_to);
  // N boxes of codes and their lines, from `row` on, to the stage's `sub`-th
  auto copy_boxes = [&](auto n, int row, int sub, uint32_t stage_at) {
    constexpr int N = decltype(n)::value;
    const long long from = static_cast<long long>(row) * (DIM / 2) + lane * 16;
    const uint8_t* keys = a.c.k_codes + from;
    const uint8_t* values = a.c.v_codes + from;
#pragma unroll
    for (int b = 0; b < N; ++b)
#pragma unroll
      for (int i = 0; i < kCopies; ++i) {
        copy_16(copy_to[i] + stage_at + (sub + b) * Shape::kBox, keys + b * Shape::kBox + i * 512);
        copy_16(copy_to[i] + stage_at + (SUBS + sub + b) * Shape::kBox, values + b * Shape::kBox + i * 512);
      }
    copy_16_if(lane < N * Shape::kKeyLines / 16, line_to + stage_at + sub * Shape::kKeyLines,
               static_cast<const char*>(a.c.k_scales) + static_cast<long long>(row) * (4 * G) + lane * 16);
    copy_16_if(lane < N * Shape::kValueLines / 16, line_to + stage_at + SUBS * Shape::kKeyLines + sub * Shape::kValueLines,
               static_cast<const char*>(a.c.v_scales) + static_cast<long long>(row >> 4) * Shape::kValueLines + lane * 16);
  };
  constexpr uint32_t kAll = (1u << SUBS) - 1;
  uint32_t usable = 0;    // bits of the chunks on the way, the oldest lowest
  uint32_t fill = 0;      // stage of the next chunk to issue, in bytes
  auto issue = [&]() {    // the chunk at `next`, if there is one, then move on
    uint32_t bits = 0;
    if (more) {
      if constexpr (ONE) {
        if (next_row >= 0) {
          copy_boxes(std::integral_constant<int, SUBS>{}, next_row, 0, fill);
          bits = kAll;
        }
      } else {
#pragma unroll
        for (int sub = 0; sub < SUBS; ++sub) {
          const int row = __shfl_sync(0xFFFFFFFFu, next_row, sub);
          if (row < 0) continue;
          copy_boxes(std::integral_constant<int, 1>{}, row, sub, fill);
          bits |= 1u << sub;
        }
      }
      more = advance(next, kRows4Warps);
      if (more) fetch_rows();
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    usable = (usable >> SUBS) | (bits << (SUBS * (STAGES - 2)));
    fill = fill == (STAGES - 1) * Shape::kStage ? 0 : fill + Shape::kStage;
  };
  if (more) fetch_rows();
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) issue();

  const bool capped = a.softcap != 0.f, wide = a.softcap > kRows4WideCap;
  const float cap2 = a.softcap * kLog2e;
  // Where this lane's parts of a stage lie.
  uint32_t key_at[DIM / 128 + (DIM < 128)], value_at[2];
#pragma unroll
  for (int i = 0; i < DIM / 128; ++i) key_at[i] = pipe + row_part<DIM>(r, c * (DIM / 128) + i);
  if (DIM == 64) key_at[0] = pipe + r * 32 + c * 8;
#pragma unroll
  for (int i = 0; i < DIM / 128 + (DIM < 128); ++i) keep(key_at[i]);
  // The tokens 2 c and 2 c + 1 in the order that meets all banks.
  const bool swapped = DIM == 256 ? false : DIM == 128 ? c & 1 : c >> 1;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int token = 2 * c + (i ^ static_cast<int>(swapped));
    value_at[i] = pipe + SUBS * Shape::kBox +
                  (DIM == 256 ? row_part<DIM>(token, r) : DIM == 128 ? row_part<DIM>(token, r >> 1) + (r & 1) * 8 : token * 32 + r * 4);
    keep(value_at[i]);
  }
  uint32_t low_pair = swapped ? 0x1054u : 0x5410u, high_pair = swapped ? 0x3276u : 0x7632u;
  keep(low_pair);
  keep(high_pair);
  uint32_t key_line_at = pipe + Shape::kCodes + r * (4 * G), value_line_at = pipe + Shape::kCodes + SUBS * Shape::kKeyLines + c * (8 * G),
           power_at = pipe + Shape::kCodes + SUBS * Shape::kKeyLines + 64 * G + 2 * r;
  keep(key_line_at);
  keep(value_line_at);
  keep(power_at);
  uint32_t queries_at = smem_addr(sm.queries) + lane * 16, sums_at = smem_addr(sm.query_sums) + c * 8;
  keep(queries_at);
  keep(sums_at);
  uint32_t minus8[G > 1 ? 2 : 1][4];  // a first operand of -8 in the upper rows, and one in the lower (kept as they are)
#pragma unroll
  for (int i = 0; i < (G > 1 ? 2 : 1); ++i)
#pragma unroll
    for (int k = 0; k < 4; ++k)
      asm volatile("mov.b32 %0, %1;" : "=r"(minus8[i][k]) : "r"((k & 1) == i ? 0xC800C800u : 0u));
  uint32_t stage = 0;  // in bytes

  // ---- the pairs of this CTA's run
  Spot at = locate(u0);
  int done = 0;  // chunks of the run before this pair
  for (bool here = advance(at, 0); here;) {
    const int run = at.stop - at.chunk;  // chunks of this pair here
    const int head = at.head, tile = at.tile;
    const int token0 = a.t.begin_of(at.b, list_sizes(a));
    const int rows_all = at.w.s.tokens * a.group;

    // Queries as the second operand's fragments: lane (r, c) of an n-tile has, of
    // row r, the words 2 c and 2 c + 1 of each group, its halves paired as the
    // masks pair the codes. Every second one of a word's pairs is a sixteenth.
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      // (a warp takes every fourth group of the n-tiles)
      if (G < kRows4Warps && (warp < n * G % kRows4Warps || warp >= n * G % kRows4Warps + G)) continue;
      const int row = tile * ROWS + n * 8 + r;
      uint4 raw[G][2];
      unsigned big = 0;
      const bool live = row < rows_all;
      const int i = live ? row / a.group : 0;
      const uint16_t* src = a.q + (token0 + i) * a.q_ts + (head * a.group + (live ? row - i * a.group : 0)) * a.q_hs;
#pragma unroll
      for (int g = 0; g < G; ++g)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int d = g * 64 + c * 16 + j * 8;
          uint4 v = make_uint4(0, 0, 0, 0);
          if (live) {
            if (a.q_vec) {
              v = *reinterpret_cast<const uint4*>(src + d);
            } else {
              const uint16_t* s = src + d;
              v = make_uint4(s[0] | (static_cast<uint32_t>(s[1]) << 16), s[2] | (static_cast<uint32_t>(s[3]) << 16),
                             s[4] | (static_cast<uint32_t>(s[5]) << 16), s[6] | (static_cast<uint32_t>(s[7]) << 16));
            }
          }
          raw[g][j] = v;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t w = word_of(v, k);
            big = max(big, max((w << 16) & 0x7FFFFFFFu, w & 0x7FFF0000u));
          }
        }
      big = max(big, __shfl_xor_sync(0xFFFFFFFFu, big, 1));
      big = max(big, __shfl_xor_sync(0xFFFFFFFFu, big, 2));
      // the row times 2^(14 - e), largest in [2^14, 2^15): FP16 holds all but
      // elements below 2^-24 of it without loss (a sixteenth: 2^-20). Zero rows,
      // infinities and rows from 2^118 on: e clamped.
      int e = static_cast<int>(big >> 23) - 127;
      e = max(min(e, 117), -100);
      const float down = __uint_as_float(static_cast<unsigned>(127 + 14 - e) << 23);
#pragma unroll
      for (int g = 0; g < G; ++g) {
        if (((n * G + g) & (kRows4Warps - 1)) != warp) continue;
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float x[8];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t w = word_of(raw[g][j], k);
            x[2 * k] = __uint_as_float(w << 16) * down;
            x[2 * k + 1] = __uint_as_float(w & 0xFFFF0000u) * down;
          }
          uint32_t f[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float part = k & 1 ? 0.0625f : 1.f;
            const __half2 h = __floats2half2_rn(x[k] * part, x[k + 4] * part);
            const float2 back = __half22float2(h);
            sum += (back.x + back.y) * (k & 1 ? 16.f : 1.f);
            f[k] = half2_bits(h);
          }
          sm.queries[((n * G + g) * 2 + j) * 32 + lane] = make_uint4(f[0], f[1], f[2], f[3]);
        }
        sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 1);
        sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 2);
        if (c == 0) sm.query_sums[n * G + g][r] = sum * 0x1p-22f;
      }
      if (c == 0) sm.row_scale[n * 8 + r] = __uint_as_float(static_cast<unsigned>(127 + e + 8) << 23) * a.scale;
    }
    __syncthreads();
    float row_scale[NT][2];  // of rows 2c, 2c + 1
    int row_pos[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int row = n * 8 + 2 * c + k;
        row_scale[n][k] = sm.row_scale[row] * (capped ? 2.f * kLog2e / a.softcap : kLog2e);
        row_pos[n][k] = at.w.s.first + min(tile * ROWS + row, rows_all - 1) / a.group;
      }
    const int pos_min = at.w.s.first + min(tile * ROWS, rows_all - 1) / a.group;
    const int pos_max = at.w.s.first + min(tile * ROWS + ROWS - 1, rows_all - 1) / a.group;

    float l[NT][2], mp[NT][2];
    float acc[G][4][NT][4];  // sums of codes: rows 2 j and 2 j + 1 of the lane's word of a group
    float zero[NT][Z][4];    // what zero points and offsets add: rows 0 .. 7 of group 2 z, 8 .. 15 of 2 z + 1
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        mp[n][k] = kAttendStart;
        l[n][k] = 0.f;
      }
#pragma unroll
      for (int z = 0; z < Z; ++z)
#pragma unroll
        for (int k = 0; k < 4; ++k) zero[n][z][k] = 0.f;
#pragma unroll
      for (int g = 0; g < G; ++g)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int k = 0; k < 4; ++k) acc[g][j][n][k] = 0.f;
    }

    // this warp's first chunk of the pair
    int mine = (warp - done) & (kRows4Warps - 1);
    for (; mine < run; mine += kRows4Warps) {
      asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
      __syncwarp();  // every lane's copies are there, and every lane has read the stage filled next
      const uint32_t there = usable & kAll;
      issue();
      const int t0 = at.w.low + (at.chunk + mine) * CHUNK;
      float power[SUBS][2];   // E of tokens r, r + 8
      float p[SUBS][NT][4];   // logits in units of log 2, with E, then weights
      // S^T: 16 tokens x 8 rows at a time, group by group
      uint32_t x[SUBS][2][2 * G];  // of tokens r and r + 8: words 2 c of all groups, then 2 c + 1's
      uint32_t line[SUBS][2][G];   // (scale, offset) of tokens r and r + 8
#pragma unroll
      for (int sub = 0; sub < SUBS; ++sub)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t keys = stage + sub * Shape::kBox + h * (4 * DIM);
          if constexpr (DIM == 64) {
            lds_words<2>(x[sub][h], keys + key_at[0]);
          } else {
#pragma unroll
            for (int i = 0; i < DIM / 128; ++i) {
              const uint4 v = lds128(keys + key_at[i]);
              x[sub][h][4 * i] = v.x, x[sub][h][4 * i + 1] = v.y, x[sub][h][4 * i + 2] = v.z, x[sub][h][4 * i + 3] = v.w;
            }
          }
          lds_words<G>(line[sub][h], key_line_at + stage + sub * Shape::kKeyLines + h * (32 * G));
          power[sub][h] = lds_half(power_at + stage + sub * Shape::kValueLines + 16 * h);
#pragma unroll
          for (int n = 0; n < NT; ++n) p[sub][n][2 * h] = p[sub][n][2 * h + 1] = 0.f;
        }
#pragma unroll
      for (int g = 0; g < G; ++g) {
        float d[SUBS][NT][4];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          uint4 q[NT];
#pragma unroll
          for (int n = 0; n < NT; ++n) q[n] = lds128(queries_at + ((n * G + g) * 2 + j) * 512);
#pragma unroll
          for (int sub = 0; sub < SUBS; ++sub) {
            const uint32_t w0 = x[sub][0][j * G + g] << 2, w1 = x[sub][1][j * G + g] << 2;
            const uint32_t v0 = x[sub][0][j * G + g] >> 6, v1 = x[sub][1][j * G + g] >> 6;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              if (j == 0)
                mma_first(d[sub][n], w0 & kLowCodes, w1 & kLowCodes, w0 & kHighCodes, w1 & kHighCodes, q[n].x, q[n].y);
              else
                mma_f16_16816(d[sub][n], w0 & kLowCodes, w1 & kLowCodes, w0 & kHighCodes, w1 & kHighCodes, q[n].x, q[n].y);
              mma_f16_16816(d[sub][n], v0 & kLowCodes, v1 & kLowCodes, v0 & kHighCodes, v1 & kHighCodes, q[n].z, q[n].w);
            }
          }
        }
        float2 sums[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const uint2 v = lds64(sums_at + (n * G + g) * 32);
          sums[n] = make_float2(__uint_as_float(v.x), __uint_as_float(v.y));
        }
#pragma unroll
        for (int sub = 0; sub < SUBS; ++sub)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float2 l2 = halves_of(line[sub][h][g]);
            const float low = fmaf(-8.f, l2.x, l2.y);  // what code 0 stands for
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              p[sub][n][2 * h] = fmaf(d[sub][n][2 * h], l2.x, fmaf(low, sums[n].x, p[sub][n][2 * h]));
              p[sub][n][2 * h + 1] = fmaf(d[sub][n][2 * h + 1], l2.x, fmaf(low, sums[n].y, p[sub][n][2 * h + 1]));
            }
          }
      }
      auto each_logit = [&](auto&& f) {
#pragma unroll
        for (int sub = 0; sub < SUBS; ++sub)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int k = 0; k < 4; ++k) p[sub][n][k] = f(p[sub][n][k], row_scale[n][k & 1], power[sub][k >> 1]);
      };
      if (!capped)
        each_logit([&](float x, float scale, float e) { return fmaf(x, scale, e); });
      else if (!wide)
        // cap * tanh(x / cap) = cap - 2 cap / (exp(2 x / cap) + 1); the factor
        // 2 log2(e) / cap is in row_scale. The difference is off by some 2^-23 of
        // the cap: above kRows4WideCap not taken.
        each_logit([&](float x, float scale, float e) { return cap2 - __fdividef(2.f * cap2, ex2(x * scale) + 1.f) + e; });
      else
        each_logit([&](float x, float scale, float e) { return capped_by(x * scale * (0.5f / kLog2e), cap2) + e; });
      const bool masked = there != kAll || t0 + CHUNK - 1 > pos_min || (a.window && pos_max - t0 >= a.window);
      if (masked) {
#pragma unroll
        for (int sub = 0; sub < SUBS; ++sub)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int j = t0 + sub * 16 + r + (k >> 1) * 8, pos = row_pos[n][k & 1];
              if (j > pos || (a.window && pos - j >= a.window) || !((there >> sub) & 1)) p[sub][n][k] = kNegInf;
            }
        // E that is no number has made the weights NaN of the rows that see the
        // token; it does not reach the others (neither does what lies where no token is)
#pragma unroll
        for (int sub = 0; sub < SUBS; ++sub)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            if (!(fabsf(power[sub][h]) <= 64.f)) power[sub][h] = 0.f;
      }
      // raise the references where a weight passes them
      bool passes = false;
      float top[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          top[n][k] = kNegInf;
#pragma unroll
          for (int sub = 0; sub < SUBS; ++sub) top[n][k] = fmaxf(top[n][k], fmaxf(p[sub][n][k], p[sub][n][k + 2]));
          passes |= top[n][k] - mp[n][k] > kAttendRaise;
        }
      if (__any_sync(0xFFFFFFFFu, passes)) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            float t = top[n][k];
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) t = fmaxf(t, __shfl_xor_sync(0xFFFFFFFFu, t, d));
            t = fmaxf(t, mp[n][k]);
            const float f = ex2(mp[n][k] - t);
            mp[n][k] = t;
            l[n][k] *= f;
#pragma unroll
            for (int z = 0; z < Z; ++z) {
              zero[n][z][k] *= f;
              zero[n][z][k + 2] *= f;
            }
#pragma unroll
            for (int g = 0; g < G; ++g)
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                acc[g][j][n][k] *= f;
                acc[g][j][n][k + 2] *= f;
              }
          }
      }
#pragma unroll
      for (int sub = 0; sub < SUBS; ++sub) {
        uint32_t pf[NT][2];
        const float back[2] = {ex2(-power[sub][0]), ex2(-power[sub][1])};
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            p[sub][n][k] = ex2(p[sub][n][k] - mp[n][k & 1]);
            l[n][k & 1] = fmaf(p[sub][n][k], back[k >> 1], l[n][k & 1]);
          }
          pf[n][0] = transpose_8x8(half2_bits(__floats2half2_rn(p[sub][n][0], p[sub][n][1])));
          pf[n][1] = transpose_8x8(half2_bits(__floats2half2_rn(p[sub][n][2], p[sub][n][3])));
        }
        // O^T += V^T P^T: lane (r, c) has word r of each group, of the tokens
        // 2 c, 2 c + 1, 2 c + 8, 2 c + 9
        const uint32_t values = stage + sub * Shape::kBox, lines = value_line_at + stage + sub * Shape::kValueLines;
        uint32_t y[2][2][G];  // [tokens, + 8][first, second to be read][group]
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 2; ++i) lds_words<G>(y[h][i], values + value_at[i] + h * (4 * DIM));
        uint32_t scale[2][G], offset[2][G];  // of two tokens each
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          lds_words<G>(scale[h], lines + h * (32 * G));
          lds_words<G>(offset[h], lines + h * (32 * G) + 4 * G);
        }
        if (masked) {  // lines past the sequence, or of a page that is not there, may be anything
          const int left = (there >> sub) & 1 ? at.w.s.length - (t0 + sub * 16) : 0;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int t = 2 * c + 8 * h;
            const uint32_t keep = (t < left ? 0xFFFFu : 0u) | (t + 1 < left ? 0xFFFF0000u : 0u);
#pragma unroll
            for (int g = 0; g < G; ++g) scale[h][g] &= keep, offset[h][g] &= keep;
          }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int z = 0; z < Z; ++z)
            mma_f16_16816(zero[n][z], offset[0][2 * z], offset[0][2 * z + (G > 1)], offset[1][2 * z], offset[1][2 * z + (G > 1)],
                          pf[n][0], pf[n][1]);
#pragma unroll
        for (int g = 0; g < G; ++g) {
          uint32_t w[NT][2];
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            w[n][0] = mul_halves(pf[n][0], scale[0][g]);
            w[n][1] = mul_halves(pf[n][1], scale[1][g]);
            mma_f16_16816(zero[n][g >> 1], minus8[g & 1][0], minus8[g & 1][1], minus8[g & 1][2], minus8[g & 1][3], w[n][0], w[n][1]);
          }
#pragma unroll
          for (int hi = 0; hi < 2; ++hi) {
            const uint32_t pair = hi ? high_pair : low_pair;
            const uint32_t x0 = prmt(y[0][0][g], y[0][1][g], pair), x1 = prmt(y[1][0][g], y[1][1][g], pair);
            const uint32_t y0 = x0 << 2, y1 = x1 << 2, z0 = x0 >> 6, z1 = x1 >> 6;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              mma_f16_16816(acc[g][2 * hi][n], y0 & kLowCodes, y0 & kHighCodes, y1 & kLowCodes, y1 & kHighCodes, w[n][0], w[n][1]);
              mma_f16_16816(acc[g][2 * hi + 1][n], z0 & kLowCodes, z0 & kHighCodes, z1 & kLowCodes, z1 & kHighCodes, w[n][0], w[n][1]);
            }
          }
        }
      }
      stage = stage == (STAGES - 1) * Shape::kStage ? 0 : stage + Shape::kStage;
    }

    // ---- join the warps
    const int rows = min(ROWS, rows_all - tile * ROWS);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float v = l[n][k];
        v += __shfl_xor_sync(0xFFFFFFFFu, v, 4);
        v += __shfl_xor_sync(0xFFFFFFFFu, v, 8);
        v += __shfl_xor_sync(0xFFFFFFFFu, v, 16);
        if (r == 0) {
          float* st = sm.stat[warp][n * 8 + 2 * c + k];
          st[0] = mp[n][k];
          st[1] = v;
        }
      }
    __syncthreads();
    const int first_unit = at.start + kRows4PairCost;  // of the pair's chunks
    const int cta_first = first_unit / per, cta_last = (first_unit + at.w.chunks - 1) / per;
    const bool whole = cta_first == cta_last;
    const int slot = at.start > u0 ? 1 : 0;
    float* part = a.partials + (static_cast<size_t>(blockIdx.x) * 2 + slot) * kRows4SlotFloats;
    if (threadIdx.x < rows) {
      const int row = threadIdx.x;
      float mm = kAttendStart;
      for (int w = 0; w < kRows4Warps; ++w) mm = fmaxf(mm, sm.stat[w][row][0]);
      float sum = 0.f;
      for (int w = 0; w < kRows4Warps; ++w) {
        const float f = ex2(sm.stat[w][row][0] - mm);
        sum += sm.stat[w][row][1] * f;
        sm.factor[w][row] = f;
      }
      if (whole) {
        sm.out_scale[row] = sum == 0.f ? 0.f : 1.f / sum;
      } else {
        float* st = part + kRows4SlotRows * 256 + row * 4;
        st[0] = mm;
        st[1] = sum;
      }
    }
    __syncthreads();
    // A pass joins 8 rows of one group, or fewer rows of more groups.
    const int per_pass = min(G, rows <= 2 ? 4 : rows <= 4 ? 2 : 1);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int rows_n = min(8, rows - n * 8);
      if (rows_n <= 0) break;
      for (int g0 = 0; g0 < G; g0 += per_pass) {
#pragma unroll
        for (int g = 0; g < G; ++g) {
          if (g < g0 || g >= g0 + per_pass) continue;
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int row = 2 * c + k;
            if (row < rows_n) {
              const float f = sm.factor[warp][n * 8 + row], z = zero[n][g >> 1][2 * (g & 1) + k] * f;
              float* to = &sm.deposit[((warp * rows_n + row) * per_pass + g - g0) * 64 + r * 8];
#pragma unroll
              for (int hi = 0; hi < 2; ++hi)
                *reinterpret_cast<float4*>(to + 4 * hi) = make_float4(
                    fmaf(acc[g][2 * hi][n][k], f * 0x1p22f, z), fmaf(acc[g][2 * hi][n][k + 2], f * 0x1p18f, z),
                    fmaf(acc[g][2 * hi + 1][n][k], f * 0x1p22f, z), fmaf(acc[g][2 * hi + 1][n][k + 2], f * 0x1p18f, z));
            }
          }
        }
        __syncthreads();
        const int width = per_pass * 64;
        for (int i = threadIdx.x; i < rows_n * width / 4; i += kRows4Threads) {
          const int row = i / (width / 4), d = (i - row * (width / 4)) * 4;
          float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int w = 0; w < kRows4Warps; ++w) {
            const float4 u = *reinterpret_cast<const float4*>(&sm.deposit[(w * rows_n + row) * width + d]);
            v.x += u.x, v.y += u.y, v.z += u.z, v.w += u.w;
          }
          if (whole) {
            store_four(a, token0, head, tile * ROWS + n * 8 + row, g0 * 64 + d, v, sm.out_scale[n * 8 + row]);
          } else {
            *reinterpret_cast<float4*>(part + (n * 8 + row) * 256 + g0 * 64 + d) = v;
          }
        }
        __syncthreads();
      }
    }
    if (!whole) {
      // ---- join the CTAs of the pair: the last to arrive adds all in order
      __threadfence();
      __syncthreads();
      if (threadIdx.x == 0) {
        const int arrived = atomic_add_acq_rel_gpu(a.counters + cta_first, 1);
        sm.last = arrived == cta_last - cta_first;
        if (sm.last) a.counters[cta_first] = 0;
      }
      __syncthreads();
      if (sm.last) {
        __threadfence();
        const int parts = cta_last - cta_first + 1;
        const float* first = a.partials + (static_cast<size_t>(cta_first) * 2 + (at.start > cta_first * per ? 1 : 0)) * kRows4SlotFloats;
        const float* rest = a.partials + static_cast<size_t>(cta_first) * 2 * kRows4SlotFloats;  // + 2 slots per CTA
        auto part_of = [&](int i) { return i == 0 ? first : rest + static_cast<size_t>(i) * 2 * kRows4SlotFloats; };
        if (threadIdx.x < rows) {
          float mm = kAttendStart;
          for (int i = 0; i < parts; ++i) mm = fmaxf(mm, __ldcg(part_of(i) + kRows4SlotRows * 256 + threadIdx.x * 4));
          float sum = 0.f;
          for (int i = 0; i < parts; ++i) {
            const float* st = part_of(i) + kRows4SlotRows * 256 + threadIdx.x * 4;
            sum += __ldcg(st + 1) * ex2(__ldcg(st) - mm);
          }
          sm.factor[0][threadIdx.x] = mm;
          sm.out_scale[threadIdx.x] = sum == 0.f ? 0.f : 1.f / sum;
        }
        __syncthreads();
        constexpr int kVectors = DIM / 4;
        for (int i = threadIdx.x; i < rows * kVectors; i += kRows4Threads) {
          const int row = i / kVectors, d = (i - row * kVectors) * 4;
          const float mm = sm.factor[0][row];
          float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
          for (int j = 0; j < parts; ++j) {
            const float* pt = part_of(j);
            const float4 u = __ldcg(reinterpret_cast<const float4*>(pt + row * 256 + d));
            const float w = ex2(__ldcg(pt + kRows4SlotRows * 256 + row * 4) - mm);
            v.x += u.x * w, v.y += u.y * w, v.z += u.z * w, v.w += u.w * w;
          }
          store_four(a, token0, head, tile * ROWS + row, d, v, sm.out_scale[row]);
        }
      }
      __syncthreads();
    }
    done += run;
    here = advance(at, run);
  }
}

// ------------------------------------------------------------------ launch

// This file's kernel reads and widens the codes again for every 16 query rows of a
// sequence, attend_tile_kernel for every 128, at a cost that hardly depends on how
// many of them there are. us by this kernel and by that one, 8 KV heads (small
// ones: 2), sequences of 77 to 4093, 1000, 100 to 3000, 2000 to 8000 tokens:
//   128 dimensions  24 seqs      1       64       4
//     32 rows       62, 102   17, 31  116, 205  36, 52
//     48            85, 104   18, 32  166, 206  43, 53
//     64           108, 105   23, 32  209, 207  49, 53
//   256 dimensions, capped
//     32           160, 166   42, 55  298, 317  70, 79
//     48           231, 172   35, 55  444, 328  87, 81
//   64 dimensions, capped
//     64            36, 58    16, 35   55, 86   25, 56
//    128            54, 59    16, 36   91, 89   30, 55
//    192            70, 81    16, 35  123, 143  35, 56
bool kv_attend4_takes_tiles(int max_query, int group, int dim) {
  return static_cast<long long>(max_query) * group > (dim == 64 ? 128 : dim == 128 ? 48 : 32);
}

size_t kv_attend4_partial_bytes(int sm_count, bool tile) {
  if (tile) return kv_attend_tile_partial_bytes(sm_count);
  return static_cast<size_t>(sm_count) * kRows4MaxCtas * 2 * kRows4SlotFloats * 4;
}

template <int DIM, int NT, int CTAS>
cudaError_t launch_attend4_rows(const AttendArgs& a, int sm_count, cudaStream_t stream) {
  using Shape = Rows4Shape<DIM>;
  static_assert(CTAS <= kRows4MaxCtas, "workspace slots");
  const size_t smem = 128 + sizeof(Rows4Smem<DIM>) + a.t.seqs * sizeof(int);
  const auto kernel = Shape::kSubs == 1 || a.c.page_size >= Shape::kChunk
                          ? attend4_rows_kernel<DIM, NT, CTAS, true>
                          : attend4_rows_kernel<DIM, NT, CTAS, Shape::kSubs == 1>;
  return launch_overlapped(kernel, dim3(sm_count * CTAS), kRows4Threads, smem, stream, a);
}

cudaError_t launch_attend4(const AttendArgs& a, int max_query, int sm_count, cudaStream_t stream) {
  if (kv_attend4_takes_tiles(max_query, a.group, a.c.dim)) return launch_attend_tile(a, sm_count, stream);
  const bool one = static_cast<long long>(max_query) * a.group <= 8;  // query rows per KV head in one n-tile
  switch (a.c.dim) {
    case 64: return one ? launch_attend4_rows<64, 1, 3>(a, sm_count, stream) : launch_attend4_rows<64, 2, 3>(a, sm_count, stream);
    case 128: return one ? launch_attend4_rows<128, 1, 3>(a, sm_count, stream) : launch_attend4_rows<128, 2, 2>(a, sm_count, stream);
    default: return one ? launch_attend4_rows<256, 1, 3>(a, sm_count, stream) : launch_attend4_rows<256, 2, 2>(a, sm_count, stream);
  }
}

}  // namespace se12
