// Attention over the paged 4-bit cache for few query rows per KV head (next
// tokens, drafted tokens): split over the tokens, joined in the same launch.
//
//   s_ij = sum_g ks_jg sum_{d in g} q_id (u_jd - 8) + ko_jg sum_{d in g} q_id
//   o_id = sum_j p_ij (vs_jg (u_jd - 8) + vo_jg),  p_ij = 2^(s_ij + E_j) / sum_j 2^s_ij
//
// for groups g of 64 dimensions, u the codes, ks, ko, vs, vo scales and
// offsets. A code never becomes a value: its four bits, masked where they lie,
// are the FP16 subnormal u 2^-24 (or 16 u 2^-24, four bits higher, met by a
// query's or a sum's factor of 1/16), which mma.sync multiplies exactly. So 8
// keys take six instructions and 8 values seven, where widening to signed
// numbers takes nine more, at a rate of codes at which issue slots are what runs
// out. Zero points are put right afterwards: keys' with the sums of the query's
// groups, values' by the products of one more instruction per group, whose
// second operand is the same rounded weights that the codes were multiplied by
// (a difference of roundings would not cancel where weights are equal).
//
// A group's products are scaled in fp32 (keys) or through its weights
// p vs in FP16 (values; the scales are relative to 2^E, so that both factors
// have FP16's full precision whatever the values' size).
//
// Work list, warps' pipelines, joins: as attend_rows_kernel, see there.
#include "se12_attend.cuh"

#include <cuda_bf16.h>

namespace se12 {

constexpr int kRows4Warps = 4;
constexpr int kRows4Threads = kRows4Warps * 32;
constexpr int kRows4SlotRows = 16;
constexpr int kRows4SlotFloats = kRows4SlotRows * (256 + 4);  // sums, then (mp, l) per row
constexpr int kRows4MaxCtas = 3;       // per SM
constexpr int kRows4PairCost = 8;      // what a pair's queries, joins and output cost, in chunks
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
  float query_sums[2][DIM / 64][8];       // 2^-22 sum of a group's, [n-tile][group][row]
  float row_scale[kRows4SlotRows];
  float stat[kRows4Warps][kRows4SlotRows][2];  // mp, l of each warp
  float factor[kRows4Warps][kRows4SlotRows];
  float out_scale[kRows4SlotRows];
  int last;
  int most;
  int before[1];  // [seqs + 1] units of the sequences before (per KV head)
};

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

// 16 bytes, asynchronously.
__device__ __forceinline__ void copy_16(uint32_t dst, const void* src, uint64_t policy) {
  asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "l"(policy) : "memory");
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

template <int DIM, int NT, int CTAS>
__global__ void __launch_bounds__(kRows4Threads, CTAS)
    attend4_rows_kernel(const AttendArgs a) {
  using Shape = Rows4Shape<DIM>;
  // A place in the list, with its pair's KV head and row tile.
  struct Spot : Place<kRows4PairCost> {
    int head, tile;
  };
  constexpr int G = Shape::kGroups, SUBS = Shape::kSubs, CHUNK = Shape::kChunk, STAGES = Shape::kStages, ROWS = 8 * NT;
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
    p.pair = x / each;
    p.head = p.pair / p.w.tiles;
    p.tile = p.pair - p.head * p.w.tiles;
    const int at = x - p.pair * each;
    p.start = u - at;
    p.chunk = max(at - kRows4PairCost, 0);
    return p;
  };
  // To the place `by` chunks on; false where that is past this CTA's run.
  auto advance = [&](Spot& p, int by) {
    p.chunk += by;
    while (p.chunk >= p.w.chunks) {
      p.chunk -= p.w.chunks;
      p.start += p.w.chunks + kRows4PairCost;
      if (p.start + kRows4PairCost >= u1) return false;
      if (++p.tile < p.w.tiles) continue;
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
    return p.unit() < u1;
  };

  // ---- this warp's pipeline: every fourth chunk of the run. A lane copies the
  // same 16 bytes of every box; a chunk is one group of its copies.
  const uint32_t pipe = smem_addr(sm.pipes[warp]);
  const uint64_t policy = policy_evict_first();
  Spot next = locate(u0);
  bool more = advance(next, warp);  // `next` is a chunk of the run
  int next_row = -1;  // of the next chunk to issue: where 16 tokens of it begin (lane `sub`'s), -1: not to be read
  auto fetch_rows = [&]() {
    next_row = -1;
    const int t0 = next.w.low + next.chunk * CHUNK + lane * 16;
    if (lane < SUBS && t0 < next.w.s.length && t0 + 16 > visible_from(next.w.s.first, a.window)) {
      const int i = t0 >> a.c.page_shift;
      const int page = i < a.t.max_pages ? a.t.table[next.b * a.t.table_stride + i] : -1;
      if (page >= 0 && page < a.c.pages)
        next_row = (page * heads + next.head) * a.c.page_size + (t0 & (a.c.page_size - 1));
      else
        raise_status(kStatusBadArgument);
    }
  };
  constexpr int kCopies = Shape::kBox / 512 > 0 ? Shape::kBox / 512 : 1;  // of 512 bytes, of a box
  uint32_t copy_to[kCopies];
#pragma unroll
  for (int i = 0; i < kCopies; ++i) {
    const int vector = i * 32 + lane;
    copy_to[i] = row_part<DIM>(vector / (DIM / 32), vector % (DIM / 32));
  }
  uint32_t usable = 0;  // bits of the chunks on the way, the oldest lowest
  int fill = 0;         // stage of the next chunk to issue
  auto issue = [&]() {  // the chunk at `next`, if there is one, then move on
    uint32_t bits = 0;
    if (more) {
      const uint32_t to = pipe + fill * Shape::kStage;
#pragma unroll
      for (int sub = 0; sub < SUBS; ++sub) {
        const int row = __shfl_sync(0xFFFFFFFFu, next_row, sub);
        if (row < 0) continue;
        bits |= 1u << sub;
        const long long from = static_cast<long long>(row) * (DIM / 2) + lane * 16;
#pragma unroll
        for (int i = 0; i < kCopies; ++i) {
          copy_16(to + sub * Shape::kBox + copy_to[i], a.c.k_codes + from + i * 512, policy);
          copy_16(to + (SUBS + sub) * Shape::kBox + copy_to[i], a.c.v_codes + from + i * 512, policy);
        }
        if (lane < Shape::kKeyLines / 16)
          copy_16(to + Shape::kCodes + sub * Shape::kKeyLines + lane * 16,
                  static_cast<const char*>(a.c.k_scales) + static_cast<long long>(row) * (4 * G) + lane * 16, policy);
        if (lane < Shape::kValueLines / 16)
          copy_16(to + Shape::kCodes + SUBS * Shape::kKeyLines + sub * Shape::kValueLines + lane * 16,
                  static_cast<const char*>(a.c.v_scales) + static_cast<long long>(row >> 4) * Shape::kValueLines + lane * 16, policy);
      }
      more = advance(next, kRows4Warps);
      if (more) fetch_rows();
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    usable = (usable >> SUBS) | (bits << (SUBS * (STAGES - 2)));
    fill = fill + 1 == STAGES ? 0 : fill + 1;
  };
  if (more) fetch_rows();
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) issue();

  const bool capped = a.softcap != 0.f, wide = a.softcap > kRows4WideCap;
  // where this lane's parts of a sub lie
  uint32_t key_at[DIM / 128 + (DIM < 128)], value_at[2];
#pragma unroll
  for (int i = 0; i < DIM / 128; ++i) key_at[i] = row_part<DIM>(r, c * (DIM / 128) + i);
  if (DIM == 64) key_at[0] = r * 32 + c * 8;
  // The tokens 2 c and 2 c + 1 in the order that meets all banks.
  const bool swapped = DIM == 256 ? false : DIM == 128 ? c & 1 : c >> 1;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int token = 2 * c + (i ^ static_cast<int>(swapped));
    value_at[i] = DIM == 256 ? row_part<DIM>(token, r) : DIM == 128 ? row_part<DIM>(token, r >> 1) + (r & 1) * 8 : token * 32 + r * 4;
  }
  const uint32_t low_pair = swapped ? 0x1054u : 0x5410u, high_pair = swapped ? 0x3276u : 0x7632u;
  int stage = 0;

  // ---- the pairs of this CTA's run
  Spot at = locate(u0);
  int done = 0;  // chunks of the run before this pair
  for (bool here = advance(at, 0); here;) {
    const int run = min(at.w.chunks - at.chunk, u1 - at.unit());  // chunks of this pair here
    const int head = at.head, tile = at.tile;
    const int token0 = a.t.begin_of(at.b, list_sizes(a));
    const int rows_all = at.w.s.tokens * a.group;

    // Queries as the second operand's fragments: lane (r, c) of an n-tile has, of
    // row r, the words 2 c and 2 c + 1 of each group, its halves paired as the
    // masks pair the codes. Every second one of a word's pairs is a sixteenth.
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      if ((n & (kRows4Warps - 1)) != warp) continue;
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
        if (c == 0) sm.query_sums[n][g][r] = sum * 0x1p-22f;
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
    float zero[NT][4];       // row g < G: what the zero points and offsets of group g add
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        mp[n][k] = kAttendStart;
        l[n][k] = 0.f;
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) zero[n][k] = 0.f;
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
      const uint32_t base = pipe + stage * Shape::kStage;
      const uint32_t key_lines = base + Shape::kCodes, value_lines = key_lines + SUBS * Shape::kKeyLines;
      const uint32_t there = usable;
      issue();
      const int t0 = at.w.low + (at.chunk + mine) * CHUNK;
      bool use[SUBS];
      float power[SUBS][2];   // E of tokens r, r + 8
      float p[SUBS][NT][4];   // logits in units of log 2, with E, then weights
#pragma unroll
      for (int sub = 0; sub < SUBS; ++sub) {
        use[sub] = (there >> sub) & 1;
        power[sub][0] = power[sub][1] = 0.f;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int k = 0; k < 4; ++k) p[sub][n][k] = kNegInf;
        if (!use[sub]) continue;
        // S^T: 16 tokens x 8 rows, group by group
        const uint32_t keys = base + sub * Shape::kBox;
        uint32_t x[2][2 * G];  // of tokens r and r + 8: words 2 c of all groups, then 2 c + 1's
        if constexpr (DIM == 64) {
#pragma unroll
          for (int h = 0; h < 2; ++h) lds_words<2>(x[h], keys + key_at[0] + h * 256);
        } else {
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < DIM / 128; ++i) {
              const uint4 v = lds128(keys + key_at[i] + h * (4 * DIM));
              x[h][4 * i] = v.x, x[h][4 * i + 1] = v.y, x[h][4 * i + 2] = v.z, x[h][4 * i + 3] = v.w;
            }
        }
        uint32_t line[2][G];  // (scale, offset) of tokens r and r + 8
#pragma unroll
        for (int h = 0; h < 2; ++h) lds_words<G>(line[h], key_lines + sub * Shape::kKeyLines + (r + 8 * h) * (4 * G));
        float s[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int k = 0; k < 4; ++k) s[n][k] = 0.f;
#pragma unroll
        for (int g = 0; g < G; ++g) {
          float d[NT][4];
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int k = 0; k < 4; ++k) d[n][k] = 0.f;
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const uint32_t w0 = x[0][j * G + g] << 2, w1 = x[1][j * G + g] << 2, v0 = x[0][j * G + g] >> 6, v1 = x[1][j * G + g] >> 6;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              const uint4 q = sm.queries[((n * G + g) * 2 + j) * 32 + lane];
              mma_f16_16816(d[n], w0 & kLowCodes, w1 & kLowCodes, w0 & kHighCodes, w1 & kHighCodes, q.x, q.y);
              mma_f16_16816(d[n], v0 & kLowCodes, v1 & kLowCodes, v0 & kHighCodes, v1 & kHighCodes, q.z, q.w);
            }
          }
          const float2 line0 = halves_of(line[0][g]), line1 = halves_of(line[1][g]);
          const float low0 = fmaf(-8.f, line0.x, line0.y), low1 = fmaf(-8.f, line1.x, line1.y);  // what code 0 stands for
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const float2 qs = *reinterpret_cast<const float2*>(&sm.query_sums[n][g][2 * c]);
            s[n][0] = fmaf(d[n][0], line0.x, fmaf(low0, qs.x, s[n][0]));
            s[n][1] = fmaf(d[n][1], line0.x, fmaf(low0, qs.y, s[n][1]));
            s[n][2] = fmaf(d[n][2], line1.x, fmaf(low1, qs.x, s[n][2]));
            s[n][3] = fmaf(d[n][3], line1.x, fmaf(low1, qs.y, s[n][3]));
          }
        }
        const uint32_t exponents = value_lines + sub * Shape::kValueLines + 64 * G;
        power[sub][0] = lds_half(exponents + 2 * r);
        power[sub][1] = lds_half(exponents + 2 * r + 16);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if (!capped) {
              p[sub][n][k] = fmaf(s[n][k], row_scale[n][k & 1], power[sub][k >> 1]);
              continue;
            }
            // cap * tanh(x / cap) = cap - 2 cap / (exp(2 x / cap) + 1); the
            // factor 2 log2(e) / cap is in row_scale. The difference is off by
            // some 2^-23 of the cap: above kRows4WideCap not taken.
            float y = s[n][k] * row_scale[n][k & 1];
            if (wide)
              y = capped_by(y * (0.5f / kLog2e), a.softcap * kLog2e);
            else
              y = a.softcap * kLog2e - __fdividef(2.f * kLog2e * a.softcap, ex2(y) + 1.f);
            p[sub][n][k] = y + power[sub][k >> 1];
          }
      }
      const bool masked = t0 + CHUNK - 1 > pos_min || (a.window && pos_max - t0 >= a.window);
      if (masked) {
#pragma unroll
        for (int sub = 0; sub < SUBS; ++sub)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int j = t0 + sub * 16 + r + (k >> 1) * 8, pos = row_pos[n][k & 1];
              if (j > pos || (a.window && pos - j >= a.window)) p[sub][n][k] = kNegInf;
            }
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
            zero[n][k] *= f;
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
        if (!use[sub]) continue;
        uint32_t pf[NT][2];
        const float back[2] = {ex2(-power[sub][0]), ex2(-power[sub][1])};
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const bool hidden = masked && p[sub][n][k] == kNegInf;  // weighs nothing, whatever E is
            const float w = ex2(p[sub][n][k] - mp[n][k & 1]);
            p[sub][n][k] = hidden ? 0.f : w;
            l[n][k & 1] += hidden ? 0.f : w * back[k >> 1];
          }
          pf[n][0] = transpose_8x8(half2_bits(__floats2half2_rn(p[sub][n][0], p[sub][n][1])));
          pf[n][1] = transpose_8x8(half2_bits(__floats2half2_rn(p[sub][n][2], p[sub][n][3])));
        }
        // O^T += V^T P^T: lane (r, c) has word r of each group, of the tokens
        // 2 c, 2 c + 1, 2 c + 8, 2 c + 9
        const uint32_t values = base + (SUBS + sub) * Shape::kBox, lines = value_lines + sub * Shape::kValueLines;
        uint32_t x[2][2][G];  // [tokens, + 8][first, second to be read][group]
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 2; ++i) lds_words<G>(x[h][i], values + value_at[i] + h * (4 * DIM));
        uint32_t scale[2][G], offset[2];  // of two tokens each; offsets: row min(r, G - 1)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          lds_words<G>(scale[h], lines + (c + 4 * h) * (8 * G));
          offset[h] = lds32(lines + (c + 4 * h) * (8 * G) + 4 * G + 4 * min(r, G - 1));
        }
        const int left = at.w.s.length - (t0 + sub * 16);
        if (left < 16) {  // lines past the sequence may be anything
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int t = 2 * c + 8 * h;
            const uint32_t keep = (t < left ? 0xFFFFu : 0u) | (t + 1 < left ? 0xFFFF0000u : 0u);
            offset[h] &= keep;
#pragma unroll
            for (int g = 0; g < G; ++g) scale[h][g] &= keep;
          }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) mma_f16_16816(zero[n], offset[0], 0u, offset[1], 0u, pf[n][0], pf[n][1]);
#pragma unroll
        for (int g = 0; g < G; ++g) {
          uint32_t w[NT][2];
          const uint32_t minus8 = r == g ? 0xC800C800u : 0u;
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            w[n][0] = mul_halves(pf[n][0], scale[0][g]);
            w[n][1] = mul_halves(pf[n][1], scale[1][g]);
            mma_f16_16816(zero[n], minus8, 0u, minus8, 0u, w[n][0], w[n][1]);
          }
#pragma unroll
          for (int hi = 0; hi < 2; ++hi) {
            const uint32_t pair = hi ? high_pair : low_pair;
            const uint32_t x0 = prmt(x[0][0][g], x[0][1][g], pair), x1 = prmt(x[1][0][g], x[1][1][g], pair);
            const uint32_t y0 = x0 << 2, y1 = x1 << 2, z0 = x0 >> 6, z1 = x1 >> 6;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              mma_f16_16816(acc[g][2 * hi][n], y0 & kLowCodes, y0 & kHighCodes, y1 & kLowCodes, y1 & kHighCodes, w[n][0], w[n][1]);
              mma_f16_16816(acc[g][2 * hi + 1][n], z0 & kLowCodes, z0 & kHighCodes, z1 & kLowCodes, z1 & kHighCodes, w[n][0], w[n][1]);
            }
          }
        }
      }
      stage = stage + 1 == STAGES ? 0 : stage + 1;
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
          const float z0 = __shfl_sync(0xFFFFFFFFu, zero[n][0], g * 4 + c), z1 = __shfl_sync(0xFFFFFFFFu, zero[n][1], g * 4 + c);
          if (g < g0 || g >= g0 + per_pass) continue;
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int row = 2 * c + k;
            if (row < rows_n) {
              const float f = sm.factor[warp][n * 8 + row], z = (k ? z1 : z0) * f;
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

size_t kv_attend4_partial_bytes(int sm_count) {
  return static_cast<size_t>(sm_count) * kRows4MaxCtas * 2 * kRows4SlotFloats * 4;
}

template <int DIM, int NT, int CTAS>
cudaError_t launch_attend4_rows(const AttendArgs& a, int sm_count, cudaStream_t stream) {
  static_assert(CTAS <= kRows4MaxCtas, "workspace slots");
  const size_t smem = 128 + sizeof(Rows4Smem<DIM>) + a.t.seqs * sizeof(int);
  return launch_overlapped(attend4_rows_kernel<DIM, NT, CTAS>, dim3(sm_count * CTAS), kRows4Threads, smem, stream, a);
}

cudaError_t launch_attend4(const AttendArgs& a, int max_query, int sm_count, cudaStream_t stream) {
  const bool one = static_cast<long long>(max_query) * a.group <= 8;  // query rows per KV head in one n-tile
  switch (a.c.dim) {
    case 64: return one ? launch_attend4_rows<64, 1, 3>(a, sm_count, stream) : launch_attend4_rows<64, 2, 3>(a, sm_count, stream);
    case 128: return one ? launch_attend4_rows<128, 1, 3>(a, sm_count, stream) : launch_attend4_rows<128, 2, 3>(a, sm_count, stream);
    default: return one ? launch_attend4_rows<256, 1, 3>(a, sm_count, stream) : launch_attend4_rows<256, 2, 2>(a, sm_count, stream);
  }
}

}  // namespace se12
