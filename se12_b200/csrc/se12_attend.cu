// Attention over the paged 8-bit cache for few query rows per KV head (next
// tokens, drafted tokens): split over the tokens, joined in the same launch.
//
//   s_ij = scale * ks_j * (q_i . kc_j)          kc, vc: codes; ks, vs: scales
//   o_i  = sum_j exp(s_ij) vs_j vc_j / sum_j exp(s_ij)
//
// The codes never become values: a code is exact in FP16, the scales
// multiply the logits and the probabilities, and q enters as FP16 times a
// power of two per row (a BF16 row fits without loss but for elements below
// 2^-16 of its largest).
//
// Work is the list of all (sequence, KV head, row tile, chunk of tokens), a
// chunk being 8 KB of keys and values, cut into runs of equal cost, one per
// CTA; the list comes from the lengths in device memory, so that the launch
// does not depend on them (a captured graph follows the lengths) and a ragged
// batch is balanced. A CTA's 4 warps take its chunks in turn, each with
// a TMA pipeline of its own (no CTA-wide barrier inside a pair's chunks) and
// its own references and sums; a pair's warps are joined in shared memory,
// its CTAs through global memory by the CTA that finishes last, in CTA order.
// Small CTAs, 2 or 3 per SM: 8 or 12 warps hide each other's latencies (131071
// tokens of 16 KV heads of 128, capped, calls repeated in a graph: 109 us, 4.9
// TB/s; 8 warps in one CTA per SM took a third longer), and short sequences'
// pairs run side by side.
//
// Layout of the products (mma.sync m16n8k16, tokens or dimensions as M,
// query rows as N = 8): with a group of up to 8 query rows per KV head the
// tensor pipe needs half of what rows-as-M would, and every lane reads whole
// 16-byte vectors of codes: S^T = K Q^T takes the contraction in the order
// the bytes lie in, O^T = V^T P^T interleaves two tokens' bytes with one
// byte permute per pair. P^T is S^T's accumulator transposed by movmatrix.
// The floor is HBM's; what bounds the kernel is the issue of its instructions
// and their latencies (2.2 of 4 a cycle with 12 warps per SM, DRAM 58 % busy,
// the tensor pipe 16 %). tcgen05 would need the codes widened into shared
// memory first and pads the rows to 64 or more.
//
// Two references instead of one running maximum: m for the sum l of 2^(s - m),
// and mp for the weights 2^(s + log2 vs - mp) that multiply the codes, so that
// the FP16 weights keep their precision whatever the blocks' scales are. Both
// are raised only when a value passes them by more than fits (2^8 of FP16's
// 2^16; 2^30 of fp32's 2^127), which a vote per chunk decides: the usual chunk
// pays neither the reduction over the lanes nor the scaling of the sums.
#include "se12_attend.cuh"

#include <cuda_bf16.h>

namespace se12 {

constexpr int kAttendWarps = 4;
constexpr int kAttendThreads = kAttendWarps * 32;
constexpr int kAttendStages = 2;
constexpr int kAttendBox = 2048;         // 16 tokens x 128 bytes
constexpr int kAttendStageBytes = 8192;  // keys and values of a chunk
constexpr int kAttendDeposit = 8192;     // joining the warps' sums
constexpr int kAttendSlotRows = 16;
constexpr int kAttendSlotFloats = kAttendSlotRows * (256 + 4);  // sums, then (m, l, mp) per row
constexpr int kAttendMaxCtas = 3;        // per SM
// What a pair's queries, joins and output cost, in chunks. (Calls repeated in a
// graph; calls among others take more, 64 sequences 210 us. 64 of 1000
// to 16384 tokens, 8 KV heads of 128, e4m3: uncounted 196 us; 4, 8 and 16: 188,
// 183 and 185. 16 of 301 to 8191, window 4096, 8 heads of 256: 57 us; 52, 51 and
// 50. 7 of 86 to 702 tokens: 24 us; 17, 16 and 16. Equal lengths gain little.)
constexpr int kAttendPairCost = 8;
constexpr float kAttendWideCap = 128.f;  // a logit off by 2^-15 there, an eighth of a weight's FP16 rounding

__device__ __forceinline__ void cp_async_4(void* dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_addr(dst)), "l"(src) : "memory");
}

template <int KIND, int DP, int NT>
struct AttendShape {
  static constexpr int kBoxes = DP / 128;                           // boxes per 16 tokens
  static constexpr int kChunk = kAttendStageBytes / 2 / DP;         // tokens per chunk: 16 or 32
  static constexpr int kSubs = kChunk / 16;
  static constexpr int kRows = 8 * NT;
};

// After the pipelines (1024-byte aligned).
struct AttendSmem {
  union {
    uint4 queries[512];                   // FP16 fragments: [n-tile][box][4 pairs of words][lane]
    float deposit[kAttendDeposit / 4];    // the warps' sums while they are joined
  };
  float row_scale[kAttendSlotRows];       // 2^e * scale of each query row
  float stat[kAttendWarps][kAttendSlotRows][3];   // m, l, mp of each warp
  float factor[kAttendWarps][kAttendSlotRows];
  float out_scale[kAttendSlotRows];
  float scales[kAttendWarps][kAttendStages][2][2];  // [sub][keys, values]
  int usable[kAttendWarps][kAttendStages][2];
  uint64_t full[kAttendWarps][kAttendStages];
  int last;
  int most;                               // chunks of the longest pair
  int before[1];  // [seqs + 1] units of the sequences before (per KV head)
};

// A place in the work list: chunk `chunk` of pair `pair` (KV head x row
// tile) of sequence b. The list counts units: a pair's are kAttendPairCost for
// its beginning and end, from `start` on, and one per chunk.
struct Place {
  int b, pair, chunk;
  int start;
  SeqWork w;
  __device__ __forceinline__ int unit() const { return start + kAttendPairCost + chunk; }
};

template <int KIND, int DP, int NT, int CTAS>
__global__ void __launch_bounds__(kAttendThreads, CTAS)
    attend_rows_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                       const AttendArgs a) {
  using Shape = AttendShape<KIND, DP, NT>;
  constexpr int HB = Shape::kBoxes, CHUNK = Shape::kChunk, SUBS = Shape::kSubs, ROWS = Shape::kRows;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* pipes = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  AttendSmem& sm = *reinterpret_cast<AttendSmem*>(pipes + kAttendWarps * kAttendStages * kAttendStageBytes);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int r = lane >> 2, c = lane & 3;

  if (lane == 0) {
    for (int s = 0; s < kAttendStages; ++s) mbar_init(&sm.full[warp][s], 1);
    fence_barrier_init();
    if (warp == 0) {
      prefetch_tmap(&kmap);
      prefetch_tmap(&vmap);
    }
  }
  grid_launch_dependents();
  grid_dependency_wait();

  // ---- the work list
  const int heads = a.c.heads;
  if (threadIdx.x == 0) sm.before[0] = sm.most = 0;
  __syncthreads();
  const int limit = static_cast<int>(kWorkLimit / heads);
  int most = 0;
  for (int b = threadIdx.x; b < a.t.seqs; b += kAttendThreads) {
    const SeqWork w = sequence_work<CHUNK, ROWS>(a, b);
    check_length(a, b);
    sm.before[b + 1] = times_work(w.chunks + kAttendPairCost, w.tiles, limit);
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
  const int per = max(min(kAttendWarps, sm.most), (total + static_cast<int>(gridDim.x) - 1) / static_cast<int>(gridDim.x));
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
    Place p;
    p.b = lo;
    p.w = sequence_work<CHUNK, ROWS>(a, lo);
    const int x = u - sm.before[lo] * heads, each = p.w.chunks + kAttendPairCost;
    p.pair = x / each;
    const int at = x - p.pair * each;
    p.start = u - at;
    p.chunk = max(at - kAttendPairCost, 0);
    return p;
  };
  // To the place `by` chunks on; false where that is past this CTA's run.
  auto advance = [&](Place& p, int by) {
    p.chunk += by;
    while (p.chunk >= p.w.chunks) {
      p.chunk -= p.w.chunks;
      p.start += p.w.chunks + kAttendPairCost;
      if (p.start + kAttendPairCost >= u1) return false;
      if (++p.pair == p.w.tiles * heads) {
        p.pair = 0;
        do {
          ++p.b;
        } while (sm.before[p.b + 1] == sm.before[p.b]);
        // (chunks left over continue in the next sequence)
        p.w = sequence_work<CHUNK, ROWS>(a, p.b);
      }
    }
    return p.unit() < u1;
  };

  // ---- this warp's pipeline: every fourth chunk of the run
  unsigned char* pipe = pipes + warp * (kAttendStages * kAttendStageBytes);
  const uint32_t pipe_addr = smem_addr(pipe);
  const uint64_t policy = policy_evict_first();
  Place next = locate(u0);
  bool more = advance(next, warp);  // `next` is a chunk of the run
  int next_page = -1;  // this lane's (lane < SUBS) page for the next chunk to issue
  auto fetch_page = [&]() {
    next_page = -1;
    if (lane < SUBS) {
      const int t0 = next.w.low + next.chunk * CHUNK + lane * 16;
      if (t0 < next.w.s.length && t0 + 16 > visible_from(next.w.s.first, a.window)) {
        const int i = t0 >> a.c.page_shift;
        next_page = i < a.t.max_pages ? a.t.table[next.b * a.t.table_stride + i] : -1;
        if (next_page < 0 || next_page >= a.c.pages) {
          raise_status(kStatusBadArgument);
          next_page = -1;
        }
      }
    }
  };
  auto issue = [&](int stage) {  // the chunk at `next`, then move on
    uint64_t* bar = &sm.full[warp][stage];
    const bool use = next_page >= 0;
    const int head = next.pair / next.w.tiles;
    const long long block = static_cast<long long>(next_page) * heads + head;
    if (lane < SUBS) {
      sm.usable[warp][stage][lane] = use;
      if (use) {
        cp_async_4(&sm.scales[warp][stage][lane][0], static_cast<const float*>(a.c.k_scales) + block);
        cp_async_4(&sm.scales[warp][stage][lane][1], static_cast<const float*>(a.c.v_scales) + block);
        cp_async_mbar_arrive(bar);
      }
    }
    const int boxes = __popc(__ballot_sync(0xFFFFFFFFu, use)) * 2 * HB;
    if (lane == 0) mbar_arrive_expect_tx(bar, boxes * kAttendBox);
    __syncwarp();
    if (use) {
      const int t0 = next.w.low + next.chunk * CHUNK + lane * 16;
      const int row = static_cast<int>(block * a.c.page_size + (t0 & (a.c.page_size - 1)));
      unsigned char* dst = pipe + stage * kAttendStageBytes + lane * HB * kAttendBox;
#pragma unroll
      for (int hb = 0; hb < HB; ++hb) {
        tma_load_2d(dst + hb * kAttendBox, &kmap, hb * 128, row, bar, policy);
        tma_load_2d(dst + kAttendStageBytes / 2 + hb * kAttendBox, &vmap, hb * 128, row, bar, policy);
      }
    }
    more = advance(next, kAttendWarps);
    if (more) fetch_page();
  };
  if (more) fetch_page();
#pragma unroll
  for (int s = 0; s < kAttendStages; ++s)
    if (more) issue(s);

  const bool wide = a.softcap > kAttendWideCap;
  int stage = 0;
  uint32_t phase = 0;
  bool dead = false;  // a wait ran out: skip the rest (status raised)

  // ---- the pairs of this CTA's run
  Place at = locate(u0);
  int done = 0;  // chunks of the run before this pair
  for (bool here = advance(at, 0); here;) {
    const int run = min(at.w.chunks - at.chunk, u1 - at.unit());  // chunks of this pair here
    const int head = at.pair / at.w.tiles, tile = at.pair % at.w.tiles;
    const int token0 = a.t.begin_of(at.b, list_sizes(a));
    const int rows_all = at.w.s.tokens * a.group;

    // queries as the second operand's fragments: lane (r, c) of an n-tile
    // needs, of row r, the dimensions 128 hb + 32 c .. + 31 in byte order. A
    // warp prepares every fourth n-tile.
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      if ((n & (kAttendWarps - 1)) != warp) continue;
      const int row = tile * ROWS + n * 8 + r;
      uint4 raw[HB][4];
      unsigned big = 0;
      const bool live = row < rows_all;
      const int i = live ? row / a.group : 0;
      const uint16_t* src = a.q + (token0 + i) * a.q_ts + (head * a.group + (live ? row - i * a.group : 0)) * a.q_hs;
#pragma unroll
      for (int hb = 0; hb < HB; ++hb)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int d = hb * 128 + c * 32 + j * 8;
          uint4 v = make_uint4(0, 0, 0, 0);
          if (live && d < a.c.dim) {  // dim is a multiple of 16
            if (a.q_vec) {
              v = *reinterpret_cast<const uint4*>(src + d);
            } else {
              const uint16_t* s = src + d;
              v = make_uint4(s[0] | (static_cast<uint32_t>(s[1]) << 16), s[2] | (static_cast<uint32_t>(s[3]) << 16),
                             s[4] | (static_cast<uint32_t>(s[5]) << 16), s[6] | (static_cast<uint32_t>(s[7]) << 16));
            }
          }
          raw[hb][j] = v;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t w = word_of(v, k);
            big = max(big, max((w << 16) & 0x7FFFFFFFu, w & 0x7FFF0000u));
          }
        }
      big = max(big, __shfl_xor_sync(0xFFFFFFFFu, big, 1));
      big = max(big, __shfl_xor_sync(0xFFFFFFFFu, big, 2));
      // the row times 2^-e, largest in [1, 2) (zero rows and infinities: e clamped)
      int e = static_cast<int>(big >> 23) - 127;
      e = max(min(e, 120), -120);
      const float down = __uint_as_float(static_cast<unsigned>(127 - e) << 23);
      auto halves = [&](uint32_t w) {
        return half2_bits(__floats2half2_rn(__uint_as_float(w << 16) * down, __uint_as_float(w & 0xFFFF0000u) * down));
      };
#pragma unroll
      for (int hb = 0; hb < HB; ++hb)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          sm.queries[((n * HB + hb) * 4 + j) * 32 + lane] =
              make_uint4(halves(raw[hb][j].x), halves(raw[hb][j].y), halves(raw[hb][j].z), halves(raw[hb][j].w));
      if (c == 0) sm.row_scale[n * 8 + r] = __uint_as_float(static_cast<unsigned>(127 + e) << 23) * a.scale;
    }
    __syncthreads();
    float row_scale[NT][2];  // of rows 2c, 2c + 1
    int row_pos[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int row = n * 8 + 2 * c + k;
        row_scale[n][k] = sm.row_scale[row] * (a.softcap != 0.f ? 2.f * kLog2e / a.softcap : kLog2e);
        row_pos[n][k] = at.w.s.first + min(tile * ROWS + row, rows_all - 1) / a.group;
      }
    const int pos_min = at.w.s.first + min(tile * ROWS, rows_all - 1) / a.group;
    const int pos_max = at.w.s.first + min(tile * ROWS + ROWS - 1, rows_all - 1) / a.group;

    float m[NT][2], l[NT][2], mp[NT][2];
    float acc[HB][4][2][NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        m[n][k] = mp[n][k] = kAttendStart;
        l[n][k] = 0.f;
      }
#pragma unroll
    for (int hb = 0; hb < HB; ++hb)
#pragma unroll
      for (int w = 0; w < 4; ++w)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int k = 0; k < 4; ++k) acc[hb][w][h][n][k] = 0.f;

    // this warp's first chunk of the pair
    int mine = (warp - done) & (kAttendWarps - 1);
    for (; mine < run; mine += kAttendWarps) {
      if (!dead) dead = !__all_sync(0xFFFFFFFFu, mbar_wait(&sm.full[warp][stage], phase));
      if (dead) break;
      const uint32_t base = pipe_addr + stage * kAttendStageBytes;
      const int t0 = at.w.low + (at.chunk + mine) * CHUNK;
      bool use[SUBS];
      float lv[SUBS];
      float p[SUBS][NT][4];  // logits in units of log 2, then weights
#pragma unroll
      for (int sub = 0; sub < SUBS; ++sub) {
        use[sub] = sm.usable[warp][stage][sub];
        lv[sub] = 0.f;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int k = 0; k < 4; ++k) p[sub][n][k] = kNegInf;
        if (!use[sub]) continue;
        // S^T: 16 tokens x 8 rows
        float s[NT][2][4];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int k = 0; k < 4; ++k) s[n][h][k] = 0.f;
        const uint32_t kbase = base + sub * HB * kAttendBox + r * 128;
#pragma unroll
        for (int hb = 0; hb < HB; ++hb)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t off = kbase + hb * kAttendBox + (((2 * c + i) ^ r) << 4);
            const uint4 x = lds128(off), y = lds128(off + 1024);
            uint4 qf[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int j = 0; j < 2; ++j) qf[n][j] = sm.queries[((n * HB + hb) * 4 + 2 * i + j) * 32 + lane];
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              uint32_t a0, a1, a2, a3;
              widen<KIND>(word_of(x, w), a0, a2);
              widen<KIND>(word_of(y, w), a1, a3);
#pragma unroll
              for (int n = 0; n < NT; ++n)
                mma_f16_16816(s[n][w & 1], a0, a1, a2, a3, word_of(qf[n][w >> 1], 2 * (w & 1)),
                              word_of(qf[n][w >> 1], 2 * (w & 1) + 1));
            }
          }
        const float ks = sm.scales[warp][stage][sub][0];
        lv[sub] = lg2(sm.scales[warp][stage][sub][1]);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            float x = (s[n][0][k] + s[n][1][k]) * (row_scale[n][k & 1] * ks);
            // cap * tanh(x / cap) = cap - 2 cap / (exp(2 x / cap) + 1); the
            // factor 2 log2(e) / cap is in row_scale. The difference is off by
            // some 2^-23 of the cap: above kAttendWideCap not taken.
            if (a.softcap != 0.f && !wide) x = a.softcap * kLog2e - __fdividef(2.f * kLog2e * a.softcap, ex2(x) + 1.f);
            p[sub][n][k] = x;
          }
        if (wide) {
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int k = 0; k < 4; ++k) p[sub][n][k] = capped_by(p[sub][n][k] * (0.5f / kLog2e), a.softcap * kLog2e);
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
      // raise the references where a value passes them
      bool passes = false;
      float top[NT][2], top_v[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          top[n][k] = top_v[n][k] = kNegInf;
#pragma unroll
          for (int sub = 0; sub < SUBS; ++sub) {
            const float t = fmaxf(p[sub][n][k], p[sub][n][k + 2]);
            top[n][k] = fmaxf(top[n][k], t);
            top_v[n][k] = fmaxf(top_v[n][k], t + lv[sub]);
          }
          passes |= top[n][k] - m[n][k] > kAttendRaiseSum || top_v[n][k] - mp[n][k] > kAttendRaise;
        }
      if (__any_sync(0xFFFFFFFFu, passes)) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            float t = top[n][k], tv = top_v[n][k];
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) {
              t = fmaxf(t, __shfl_xor_sync(0xFFFFFFFFu, t, d));
              tv = fmaxf(tv, __shfl_xor_sync(0xFFFFFFFFu, tv, d));
            }
            t = fmaxf(t, m[n][k]);
            tv = fmaxf(tv, mp[n][k]);
            l[n][k] *= ex2(m[n][k] - t);
            const float f = ex2(mp[n][k] - tv);
            m[n][k] = t;
            mp[n][k] = tv;
#pragma unroll
            for (int hb = 0; hb < HB; ++hb)
#pragma unroll
              for (int w = 0; w < 4; ++w)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                  acc[hb][w][h][n][k] *= f;
                  acc[hb][w][h][n][k + 2] *= f;
                }
          }
      }
#pragma unroll
      for (int sub = 0; sub < SUBS; ++sub) {
        if (!use[sub]) continue;
        uint32_t pf[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float x = p[sub][n][k];
            l[n][k & 1] += ex2(x - m[n][k & 1]);
            p[sub][n][k] = ex2(x + (lv[sub] - mp[n][k & 1]));
            // a masked token weighs nothing, whatever its block's scale holds
            if (masked && x == kNegInf) p[sub][n][k] = 0.f;
          }
          pf[n][0] = transpose_8x8(half2_bits(__floats2half2_rn(p[sub][n][0], p[sub][n][1])));
          pf[n][1] = transpose_8x8(half2_bits(__floats2half2_rn(p[sub][n][2], p[sub][n][3])));
        }
        // O^T += V^T P^T: lane (r, c) reads dimensions 128 hb + 16 r .. + 15
        // of tokens 2c, 2c + 1, 2c + 8, 2c + 9
        const uint32_t vbase = base + kAttendStageBytes / 2 + sub * HB * kAttendBox + 2 * c * 128;
        const int ts = t0 + sub * 16;
        const bool clip = ts + 16 > at.w.s.length;  // codes past the sequence may be anything
#pragma unroll
        for (int hb = 0; hb < HB; ++hb) {
          uint4 v[4];
#pragma unroll
          for (int i = 0; i < 4; ++i)
            v[i] = lds128(vbase + hb * kAttendBox + (i & 1) * 128 + (i >> 1) * 1024 + ((r ^ (2 * c + (i & 1))) << 4));
          if (clip) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (ts + 2 * c + (i & 1) + (i >> 1) * 8 >= at.w.s.length) v[i] = make_uint4(0, 0, 0, 0);
          }
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const uint32_t x0 = word_of(v[0], w), x1 = word_of(v[1], w), y0 = word_of(v[2], w), y1 = word_of(v[3], w);
            uint32_t a0, a1, a2, a3;
            widen<KIND>(prmt(x0, x1, 0x5140u), a0, a1);
            widen<KIND>(prmt(y0, y1, 0x5140u), a2, a3);
#pragma unroll
            for (int n = 0; n < NT; ++n) mma_f16_16816(acc[hb][w][0][n], a0, a1, a2, a3, pf[n][0], pf[n][1]);
            widen<KIND>(prmt(x0, x1, 0x7362u), a0, a1);
            widen<KIND>(prmt(y0, y1, 0x7362u), a2, a3);
#pragma unroll
            for (int n = 0; n < NT; ++n) mma_f16_16816(acc[hb][w][1][n], a0, a1, a2, a3, pf[n][0], pf[n][1]);
          }
        }
      }
      __syncwarp();  // every lane has read the stage
      if (more) issue(stage);
      if (++stage == kAttendStages) {
        stage = 0;
        phase ^= 1;
      }
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
          st[0] = m[n][k];
          st[1] = v;
          st[2] = mp[n][k];
        }
      }
    __syncthreads();
    const int first_unit = at.start + kAttendPairCost;  // of the pair's chunks
    const int cta_first = first_unit / per, cta_last = (first_unit + at.w.chunks - 1) / per;
    const bool whole = cta_first == cta_last;
    const int slot = at.start > u0 ? 1 : 0;
    float* part = a.partials + (static_cast<size_t>(blockIdx.x) * 2 + slot) * kAttendSlotFloats;
    if (threadIdx.x < rows) {
      const int row = threadIdx.x;
      float mm = kAttendStart, mmp = kAttendStart;
      for (int w = 0; w < kAttendWarps; ++w) {
        mm = fmaxf(mm, sm.stat[w][row][0]);
        mmp = fmaxf(mmp, sm.stat[w][row][2]);
      }
      float sum = 0.f;
      for (int w = 0; w < kAttendWarps; ++w) {
        sum += sm.stat[w][row][1] * ex2(sm.stat[w][row][0] - mm);
        sm.factor[w][row] = ex2(sm.stat[w][row][2] - mmp);
      }
      if (whole) {
        sm.out_scale[row] = sum == 0.f ? 0.f : ex2(mmp - mm) / sum;
      } else {
        float* st = part + kAttendSlotRows * 256 + row * 4;
        st[0] = mm;
        st[1] = sum;
        st[2] = mmp;
      }
    }
    __syncthreads();
    // words (of 4 dimensions per lane: 32 in all) joined at a time
    const int words = max(1, min(HB * 4, kAttendDeposit / (kAttendWarps * 32 * 4) / rows));
    for (int w0 = 0; w0 < HB * 4; w0 += words) {
      const int nw = min(words, HB * 4 - w0);
#pragma unroll
      for (int hb = 0; hb < HB; ++hb)
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const int word = hb * 4 + w - w0;
          if (word >= 0 && word < nw) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                const int row = n * 8 + 2 * c + k;
                if (row < rows) {
                  const float f = sm.factor[warp][row];
                  float4 v = make_float4(acc[hb][w][0][n][k] * f, acc[hb][w][0][n][k + 2] * f, acc[hb][w][1][n][k] * f,
                                         acc[hb][w][1][n][k + 2] * f);
                  *reinterpret_cast<float4*>(&sm.deposit[((warp * rows + row) * nw + word) * 32 + r * 4]) = v;
                }
              }
          }
        }
      __syncthreads();
      const int count = rows * nw * 8;  // vectors of 4 dimensions
      for (int i = threadIdx.x; i < count; i += kAttendThreads) {
        const int row = i / (nw * 8), word = i / 8 % nw, rr = i & 7;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kAttendWarps; ++w) {
          const float4 u = *reinterpret_cast<const float4*>(&sm.deposit[((w * rows + row) * nw + word) * 32 + rr * 4]);
          v.x += u.x, v.y += u.y, v.z += u.z, v.w += u.w;
        }
        const int wd = w0 + word;
        const int d = (wd >> 2) * 128 + rr * 16 + (wd & 3) * 4;
        if (whole) {
          if (d < a.c.dim) {
            const float f = sm.out_scale[row];
            const int all = tile * ROWS + row, i_tok = all / a.group;
            uint16_t* out = a.out + (token0 + i_tok) * a.o_ts + (head * a.group + all - i_tok * a.group) * a.o_hs + d;
            out[0] = __bfloat16_as_ushort(__float2bfloat16_rn(v.x * f));
            out[1] = __bfloat16_as_ushort(__float2bfloat16_rn(v.y * f));
            out[2] = __bfloat16_as_ushort(__float2bfloat16_rn(v.z * f));
            out[3] = __bfloat16_as_ushort(__float2bfloat16_rn(v.w * f));
          }
        } else {
          *reinterpret_cast<float4*>(part + row * 256 + d) = v;
        }
      }
      __syncthreads();
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
        const float* first = a.partials + (static_cast<size_t>(cta_first) * 2 + (at.start > cta_first * per ? 1 : 0)) * kAttendSlotFloats;
        const float* rest = a.partials + static_cast<size_t>(cta_first) * 2 * kAttendSlotFloats;  // + 2 slots per CTA
        auto part_of = [&](int i) { return i == 0 ? first : rest + static_cast<size_t>(i) * 2 * kAttendSlotFloats; };
        if (threadIdx.x < rows) {
          float mm = kAttendStart, mmp = kAttendStart;
          for (int i = 0; i < parts; ++i) {
            const float* st = part_of(i) + kAttendSlotRows * 256 + threadIdx.x * 4;
            mm = fmaxf(mm, __ldcg(st));
            mmp = fmaxf(mmp, __ldcg(st + 2));
          }
          float sum = 0.f;
          for (int i = 0; i < parts; ++i) {
            const float* st = part_of(i) + kAttendSlotRows * 256 + threadIdx.x * 4;
            sum += __ldcg(st + 1) * ex2(__ldcg(st) - mm);
          }
          sm.factor[0][threadIdx.x] = mmp;
          sm.out_scale[threadIdx.x] = sum == 0.f ? 0.f : ex2(mmp - mm) / sum;
        }
        __syncthreads();
        const int vectors = a.c.dim / 4;
        for (int i = threadIdx.x; i < rows * vectors; i += kAttendThreads) {
          const int row = i / vectors, d = (i - row * vectors) * 4;
          const float mpr = sm.factor[0][row], f = sm.out_scale[row];
          float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
          for (int j = 0; j < parts; ++j) {
            const float* pt = part_of(j);
            const float4 u = __ldcg(reinterpret_cast<const float4*>(pt + row * 256 + d));
            const float w = ex2(__ldcg(pt + kAttendSlotRows * 256 + row * 4 + 2) - mpr);
            v.x += u.x * w, v.y += u.y * w, v.z += u.z * w, v.w += u.w * w;
          }
          const int all = tile * ROWS + row, i_tok = all / a.group;
          uint16_t* out = a.out + (token0 + i_tok) * a.o_ts + (head * a.group + all - i_tok * a.group) * a.o_hs + d;
          out[0] = __bfloat16_as_ushort(__float2bfloat16_rn(v.x * f));
          out[1] = __bfloat16_as_ushort(__float2bfloat16_rn(v.y * f));
          out[2] = __bfloat16_as_ushort(__float2bfloat16_rn(v.z * f));
          out[3] = __bfloat16_as_ushort(__float2bfloat16_rn(v.w * f));
        }
      }
      __syncthreads();
    }
    done += run;
    here = advance(at, run);
  }
  if (dead) {  // copies may still be on their way into this warp's stages
    for (int i = 0; i < kAttendStages; ++i) mbar_wait(&sm.full[warp][i], i >= stage ? phase : phase ^ 1);
  }
}

// ------------------------------------------------------------------ launch

// This file's kernel reads the codes again for every 16 query rows of a
// sequence, attend_tile_kernel for every 128, at a cost that hardly depends on
// how many of them there are. This kernel and that one, 8 KV heads of 128, 32
// rows per KV head (e4m3; int8 with capped logits): one sequence of 1000 tokens
// 18 and 25 us (18 and 28), 24 of 2040 70 and 72 (78 and 93), 24 of 77 to 4093
// 72 and 75 (79 and 94), 64 of 100 to 8000 256 and 277 (292 and 334); at worst 16
// of 1000 to 2000 48 and 47. At 48 rows 24 of 2040 took 96 and 78 us (106 and
// 100). Heads of 256 (int8, capped), 24 of 2040: 135 and 121 at 24 rows.
// The batch's largest sequence decides for all: 63 sequences with one new token
// (2000 to 16000 tokens, 8 rows) and one with 512 (6000 tokens) take 765 us in
// one call and 189 and 223 in two; batches like that are better split.
bool kv_attend_takes_tiles(int max_query, int group, int dim) {
  return static_cast<long long>(max_query) * group > (dim <= 128 ? 32 : 16);
}

size_t kv_attend_partial_bytes(int sm_count, bool tile) {
  if (tile) return kv_attend_tile_partial_bytes(sm_count);
  return static_cast<size_t>(sm_count) * kAttendMaxCtas * 2 * kAttendSlotFloats * 4;
}

template <int KIND, int DP, int NT, int CTAS>
cudaError_t launch_attend_rows(const CUtensorMap& kmap, const CUtensorMap& vmap, const AttendArgs& a, int sm_count,
                               cudaStream_t stream) {
  static_assert(CTAS <= kAttendMaxCtas, "workspace slots");
  const size_t smem = 1024 + kAttendWarps * kAttendStages * kAttendStageBytes + sizeof(AttendSmem) + a.t.seqs * sizeof(int);
  return launch_overlapped(attend_rows_kernel<KIND, DP, NT, CTAS>, dim3(sm_count * CTAS), kAttendThreads, smem, stream, kmap,
                           vmap, a);
}

template <int KIND>
cudaError_t launch_attend_kind(const CUtensorMap& kmap, const CUtensorMap& vmap, const AttendArgs& a, int max_query,
                               int sm_count, cudaStream_t stream) {
  const bool one = static_cast<long long>(max_query) * a.group <= 8;  // query rows per KV head in one n-tile
  if (a.c.dim <= 128)
    return one ? launch_attend_rows<KIND, 128, 1, 3>(kmap, vmap, a, sm_count, stream)
               : launch_attend_rows<KIND, 128, 2, 3>(kmap, vmap, a, sm_count, stream);
  return one ? launch_attend_rows<KIND, 256, 1, 3>(kmap, vmap, a, sm_count, stream)
             : launch_attend_rows<KIND, 256, 2, 2>(kmap, vmap, a, sm_count, stream);
}

cudaError_t launch_kv_attend(const CUtensorMap& kmap, const CUtensorMap& vmap, const AttendArgs& a, int max_query,
                             int sm_count, cudaStream_t stream) {
  if (a.c.kind == kKvInt4) return launch_attend4(a, max_query, sm_count, stream);
  if (kv_attend_takes_tiles(max_query, a.group, a.c.dim)) return launch_attend_tile(a, sm_count, stream);
  return a.c.kind == kKvInt8 ? launch_attend_kind<kKvInt8>(kmap, vmap, a, max_query, sm_count, stream)
                             : launch_attend_kind<kKvE4m3>(kmap, vmap, a, max_query, sm_count, stream);
}

}  // namespace se12
