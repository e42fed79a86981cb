// Log probabilities of given tokens, entropy and the top alternatives of
// rows of logits (the LM head's output), in one pass over them.
//
//   z = x, or cap * tanh(x / cap); lse = M + log S, S = sum exp(z - M)
//   logprob = z[token] - lse,  entropy = log S - (sum exp(z - M) (z - M)) / S
//   top: the k largest x, ties to the lowest index (the cap keeps the order)
//
// The pass keeps, per thread, the running maximum with S and the weighted
// sum below it, and the largest value the thread has met. The top list is found
// afterwards: the k-th largest of the 256 threads' own largest is no larger
// than the k-th value, so that only the threads whose largest reaches it, k of
// them but for equal values, hold anything of the list; their values are read
// again from L2, a warp per thread, and the few that reach the bound are sorted
// (32 at a time over a warp's lanes, the warps' lists then merged). Rows with
// too many equal values for that (nearly all tokens banned) go through memory
// once more. 1023 x 128256 BF16 logits, top 20, against a list kept during the
// pass with the candidates pushed into a buffer: 117 us and 137 us, rows in
// ascending order 126 us and 2604 us; but all rows with ten tokens or none left
// 245 us and 201 us (16 rows of 256000 34 us and 30 us).
//
// Rows come in batches of 8 KB (4 KB when there are few) by bulk copies, four
// batches ahead, whatever row they belong to: with three CTAs per SM 96 KB are
// on the way. (Three CTAs of 256 threads, 80 registers: at two of 512 and 64
// the spilled registers of the inner loop cost four times the loop.) The warps
// of a CTA meet at a row's end only. The batches of all rows are cut into
// equal runs, one per CTA, and a row's CTAs are joined by the last to finish,
// in CTA order. Streaming alone takes 85 us of the 117, twice what HBM needs
// for the bytes. Neither fills its pipes: 2.1 of 4 instructions a cycle, special
// functions 32 %, DRAM 36 %; the warps wait for memory (2.4 warps per issue) and,
// at the rows' ends, for each other (1.6). Rows that are not on 16 bytes come by
// scalar loads (1023 x 50257 BF16, top 20: 103 us, the bytes alone 16).
#include "se12_device.cuh"
#include "se12_serve.h"

#include <algorithm>

#include <cuda_bf16.h>

namespace se12 {

constexpr int kLogprobThreads = 256;
constexpr int kLogprobCtas = 3;  // per SM
constexpr int kLogprobWarps = kLogprobThreads / 32;
constexpr int kLogprobStages = 4;
constexpr int kLogprobTop = 32;
constexpr int kLogprobBuffer = 2048;  // candidates
constexpr int kLogprobHolders = 128;  // threads whose values are looked through for them
// -inf and masks of the type's lowest value become this: its exponential is
// zero and its product with log2(e) still finite.
constexpr float kLogprobFloor = -2.0e38f;
// Where every running maximum starts: far enough above the floor that floor
// values add nothing to a sum, below every logit that counts.
constexpr float kLogprobStart = -1.0e38f;

// Whether a maximum (in units of log 2) is one the sums below it can be told
// from. Elsewhere the row's largest value itself decides: with infinities the
// row is NaN; with finite values that large (masks of the type's lowest value
// alone, forced tokens near its largest) any two that differ do so by more than
// 2^100, so that the sum is the number of values equal to the largest.
__device__ __forceinline__ bool usual_maximum(float max) { return max > kLogprobStart && max < 1e38f; }

// A CTA's part of a row, for the CTA that joins them.
struct LogprobPart {
  float max, sum, weighted;  // of z * log2(e): max; sum 2^(z - max); sum 2^(z - max) (z - max)
  float largest;             // value of the part, where the maximum is not a usual one (0 otherwise)
  unsigned long long list[kLogprobTop];  // sorted, largest first
};

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Order of the top list: larger value first (NaN above all, -0 as 0), then
// the lower index. 0: no entry.
__device__ __forceinline__ unsigned long long list_key(float x, int index) {
  unsigned u = __float_as_uint(x + 0.f);
  u = x != x ? 0xFFFFFFFFu : (u & 0x80000000u) ? ~u : u | 0x80000000u;
  return (static_cast<unsigned long long>(u) << 32) | static_cast<unsigned>(~index);
}

__device__ __forceinline__ float key_value(unsigned long long key) {
  const unsigned u = static_cast<unsigned>(key >> 32);
  if (u == 0xFFFFFFFFu || u == 0) return __uint_as_float(0x7FC00000u);
  return __uint_as_float((u & 0x80000000u) ? u & 0x7FFFFFFFu : ~u);
}

__device__ __forceinline__ int key_index(unsigned long long key) { return static_cast<int>(~static_cast<unsigned>(key)); }

// One compare-exchange step of a descending bitonic network over the lanes.
template <typename K>
__device__ __forceinline__ K exchange(K v, int lane, int distance, bool descending) {
  const K o = __shfl_xor_sync(0xFFFFFFFFu, v, distance);
  const bool keep_large = ((lane & distance) == 0) == descending;
  return keep_large ? (v > o ? v : o) : (v < o ? v : o);
}

template <typename K>
__device__ __forceinline__ K sort_lanes(K v, int lane) {  // lane 0 the largest
#pragma unroll
  for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
    for (int d = size >> 1; d > 0; d >>= 1) v = exchange(v, lane, d, (lane & size) == 0);
  return v;
}

// The 32 largest of two sorted lists, sorted.
template <typename K>
__device__ __forceinline__ K merge_lanes(K a, K b, int lane) {
  const K o = __shfl_sync(0xFFFFFFFFu, b, 31 - lane);
  K v = a > o ? a : o;
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v = exchange(v, lane, d, true);
  return v;
}

struct LogprobSmem {
  unsigned long long buffer[kLogprobBuffer];
  unsigned long long lists[kLogprobWarps][32];
  unsigned long long list[32];
  float stat[kLogprobWarps][4];
  float maxima[kLogprobWarps][32];
  float bound;
  int holders[kLogprobThreads];  // threads that hold something of the list
  int held;
  int count;
  int last;
  int equal;      // 1: the row's sum is the number of values equal to `extreme`
  float extreme;
  uint64_t full[kLogprobStages], empty[kLogprobStages];
};

// The largest 32 of every warp's sorted list (`v` of this warp), in all
// lanes of warp 0. All threads call it.
template <typename K>
__device__ __forceinline__ K merge_warps(K v, K (*lists)[32], int warp, int lane) {
  lists[warp][lane] = v;
#pragma unroll
  for (int n = kLogprobWarps / 2; n > 0; n >>= 1) {
    __syncthreads();
    if (warp < n) {
      v = merge_lanes(v, lists[warp + n][lane], lane);
      if (n > 1) lists[warp][lane] = v;
    }
  }
  return v;
}

// Sorts the buffer's `count` candidates and the kept list into the list.
__device__ __forceinline__ void rebuild_list(LogprobSmem& sm, int count, int warp, int lane) {
  unsigned long long v = warp == 0 ? sm.list[lane] : 0ull;
  for (int i = warp * 32; i < count; i += kLogprobThreads) {
    const unsigned long long x = i + lane < count ? sm.buffer[i + lane] : 0ull;
    v = merge_lanes(v, sort_lanes(x, lane), lane);
  }
  v = merge_warps(v, sm.lists, warp, lane);
  if (warp == 0) {
    sm.list[lane] = v;
    if (lane == 0) sm.count = 0;
  }
  __syncthreads();
}

// The capped logit; -inf stays. The sums, their reference and the logits that
// are reported all take this value, so that the largest one's term is 1.
__device__ __forceinline__ float capped(float x, float cap, float inverse) {
  return x == kNegInf ? kNegInf : capped_by(__fmul_rn(x, inverse), cap);
}

template <bool BF16>
__device__ __forceinline__ float load_logit(const void* row, long long i) {
  if constexpr (BF16) return __uint_as_float(static_cast<uint32_t>(static_cast<const uint16_t*>(row)[i]) << 16);
  return static_cast<const float*>(row)[i];
}

__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// Values of a 16-byte vector.
template <bool BF16>
__device__ __forceinline__ void unpack(float* x, const uint4& v) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint32_t w = word_of(v, k);
    if constexpr (BF16) {
      x[2 * k] = __uint_as_float(w << 16);
      x[2 * k + 1] = __uint_as_float(w & 0xFFFF0000u);
    } else {
      x[k] = __uint_as_float(w);
    }
  }
}

// The list of a row's values [begin, end), from memory, whatever they are: a
// buffer of them at a time, the next one on its way. The warps meet once a
// buffer, and sort only when it holds something.
template <bool BF16>
__device__ __noinline__ void list_all(LogprobSmem& sm, const void* row, int begin, int end, int top, bool vec, int warp, int lane) {
  constexpr int kPer = BF16 ? 8 : 4, kVecs = kLogprobBuffer / (kLogprobThreads * kPer);
  const int tid = static_cast<int>(threadIdx.x);
  auto at = [&](int base, int n) { return base + (n * kLogprobThreads + tid) * kPer; };  // first value of vector n
  uint4 next[kVecs];
  auto fetch = [&](int base) {
#pragma unroll
    for (int n = 0; n < kVecs; ++n)
      if (vec && at(base, n) + kPer <= end)
        next[n] = __ldcg(reinterpret_cast<const uint4*>(static_cast<const char*>(row) + static_cast<long long>(at(base, n)) * (BF16 ? 2 : 4)));
  };
  fetch(begin);
  __syncthreads();  // (the list is there, the counter zero)
  unsigned long long kth = sm.list[top - 1];
  for (int base = begin; base < end; base += kLogprobBuffer) {
    float x[kVecs * kPer];
#pragma unroll
    for (int n = 0; n < kVecs; ++n) {
      if (vec && at(base, n) + kPer <= end) {
        unpack<BF16>(x + n * kPer, next[n]);
      } else {
#pragma unroll
        for (int j = 0; j < kPer; ++j) x[n * kPer + j] = at(base, n) + j < end ? load_logit<BF16>(row, at(base, n) + j) : 0.f;
      }
    }
    fetch(base + kLogprobBuffer);
    bool found = false;
#pragma unroll
    for (int k = 0; k < kVecs * kPer; ++k) {
      const int i = at(base, k / kPer) + k % kPer;
      const unsigned long long key = list_key(x[k], i);
      if (i < end && key > kth) {
        sm.buffer[atomicAdd(&sm.count, 1)] = key;
        found = true;
      }
    }
    if (__syncthreads_or(found)) {
      rebuild_list(sm, sm.count, warp, lane);
      kth = sm.list[top - 1];
    }
  }
}

__device__ __forceinline__ void join_sums(float& max, float& sum, float& weighted, float m2, float s2, float w2) {
  // with d = m_old - m_new <= 0: sum 2^d, weighted 2^d + sum 2^d d (d no
  // less than -1000, where 2^d is zero, so that the product stays finite)
  const float m = max_nan(max, m2);
  const float d1 = max_nan(max - m, -1000.f), d2 = max_nan(m2 - m, -1000.f);
  const float f1 = ex2(d1), f2 = ex2(d2);
  weighted = (weighted + sum * d1) * f1 + (w2 + s2 * d2) * f2;
  sum = sum * f1 + s2 * f2;
  max = m;
}

// VECS: 16-byte vectors a thread takes of a batch.
template <bool BF16, bool CAP, int VECS>
__global__ void __launch_bounds__(kLogprobThreads, kLogprobCtas) token_logprobs_kernel(const LogprobArgs a) {
  constexpr int kPer = BF16 ? 8 : 4;                 // values per vector
  constexpr int kValues = kPer * VECS;               // per thread and batch
  constexpr int kBatch = kLogprobThreads * kValues;
  constexpr int kBatchBytes = kLogprobThreads * 16 * VECS;
  constexpr int kSize = BF16 ? 2 : 4;
  extern __shared__ __align__(128) unsigned char smem_raw[];
  LogprobSmem& sm = *reinterpret_cast<LogprobSmem*>(smem_raw + kLogprobStages * kBatchBytes);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kLogprobStages; ++i) {
      mbar_init(&sm.full[i], 1);
      mbar_init(&sm.empty[i], kLogprobWarps);
    }
    fence_barrier_init();
  }
  grid_launch_dependents();
  grid_dependency_wait();
  __syncthreads();

  const int units = a.rows * a.chunks_per_row;  // (the host sees to it that they fit)
  const int u0 = blockIdx.x * a.units_per_cta, u1 = min(u0 + a.units_per_cta, units), batches = u1 - u0;
  const float inverse = CAP ? 1.f / a.softcap : 0.f;
  const uint64_t policy = policy_evict_first();
  // batch n of this CTA's run on its way into its stage: whole vectors only
  int copy_row = u0 / a.chunks_per_row, copy_chunk = u0 - copy_row * a.chunks_per_row;
  int dead = 0;  // a wait ran out (status raised); in thread 0: after so many copies, its last
  auto copy = [&](int n) {  // in order, by thread 0
    if (n >= batches || dead) return;
    const int stage = n % kLogprobStages;
    if (n >= kLogprobStages && !mbar_wait(&sm.empty[stage], (n / kLogprobStages + 1) & 1)) {
      dead = n;
      return;
    }
    const int base = copy_chunk * kBatch;
    const int bytes = min(kBatch, a.vocab - base) * kSize / 16 * 16;
    mbar_arrive_expect_tx(&sm.full[stage], bytes);
    if (bytes)
      bulk_load(smem_raw + stage * kBatchBytes, static_cast<const char*>(a.logits) + (copy_row * a.ld + base) * kSize, bytes,
                &sm.full[stage], policy);
    if (++copy_chunk == a.chunks_per_row) {
      copy_chunk = 0;
      ++copy_row;
    }
  };
  if (a.vec && threadIdx.x == 0)
    for (int n = 0; n < kLogprobStages; ++n) copy(n);
  int batch = 0;  // of the run

  for (int u = u0; u < u1;) {
    const int row_id = u / a.chunks_per_row;
    const int row_u0 = row_id * a.chunks_per_row, row_u1 = row_u0 + a.chunks_per_row;
    const int stop = min(row_u1, u1);
    const void* row = static_cast<const char*>(a.logits) + row_id * a.ld * kSize;
    const int first = u - row_u0, chunks = stop - u;
    // the given token's logit, on its way while the row streams
    long long token = -1;
    float token_logit = 0.f;
    if (threadIdx.x == 0) {
      token = a.tokens[row_id];
      if (token >= 0 && token < a.vocab) token_logit = load_logit<BF16>(row, token);
    }

    float max = kLogprobStart, sum = 0.f, weighted = 0.f;
    float largest = kNegInf;  // of this thread's values; NaN counts as +inf
#pragma unroll 1
    for (int c = 0; c < chunks; ++c, ++batch) {
      const int base = (first + c) * kBatch;
      const int left = a.vocab - base;  // values from here to the row's end
      const int stage_id = batch % kLogprobStages;
      const unsigned char* stage = smem_raw + stage_id * kBatchBytes;
      const int whole = a.vec ? (left < kBatch ? left * kSize / 16 * kPer : kBatch) : 0;  // values the copy brings
      // place of this thread's value j in the batch; the batch's value i
      auto index_of = [](int j) { return (j / kPer * kLogprobThreads + static_cast<int>(threadIdx.x)) * kPer + j % kPer; };
      auto value_of = [&](int i) {
        return i < whole ? load_logit<BF16>(stage, i) : load_logit<BF16>(row, static_cast<long long>(base) + i);
      };
      float x[kValues];
      if (a.vec) {
        if (!dead && !mbar_wait(&sm.full[stage_id], (batch / kLogprobStages) & 1))
          dead = int_min(int_max(batch - 1, 0) + kLogprobStages, batches);
#pragma unroll
        for (int j = 0; j < VECS; ++j)
          unpack<BF16>(x + j * kPer, *reinterpret_cast<const uint4*>(stage + (j * kLogprobThreads + threadIdx.x) * 16));
      }
      if (whole < kBatch) {
        // past the copy: one by one; past the row: -inf, never a candidate
#pragma unroll
        for (int j = 0; j < kValues; ++j) {
          const int i = index_of(j);
          if (i >= left) x[j] = kNegInf;
          else if (i >= whole) x[j] = value_of(i);
        }
      }
      float top = max_nan(x[0], x[1]);
#pragma unroll
      for (int j = 2; j < kValues; j += 2) top = max3_nan(top, x[j], x[j + 1]);

      largest = fmaxf(largest, top != top ? INFINITY : top);
      if (a.vec) {
        __syncwarp();  // every lane has read its values
        if (lane == 0) mbar_arrive(&sm.empty[stage_id]);
        if (threadIdx.x == 0 && batch > 0) copy(batch - 1 + kLogprobStages);
      }

      // sums relative to the running maximum, in units of log 2 (z log2(e)
      // - max is one rounding everywhere: the maximum's own cancels)
      float high = top;
      if constexpr (CAP) {
        // |x / cap| below 0.7 but for banned tokens, usually: the polynomial
        // alone, two values at a time. The lowest value that is not -inf: as
        // unsigned numbers, negative ones are the larger the lower they are, and
        // an exponent step more turns -inf into 0.
        constexpr unsigned kStep = 0x00800000u;
        const float range = 0.6999f * a.softcap;
        unsigned low = 0;
#pragma unroll
        for (int j = 0; j < kValues; ++j) low = umax(low, __float_as_uint(x[j]) + kStep);
        if (__all_sync(0xFFFFFFFFu, top <= range && low <= __float_as_uint(-range) + kStep)) {
#pragma unroll
          for (int j = 0; j < kValues; j += 2)
            unpair(capped_pair_near(mul_pair(pair_of(x[j], x[j + 1]), pair_of(inverse, inverse)), a.softcap), x[j], x[j + 1]);
          high = fmaxf(x[0], x[1]);
#pragma unroll
          for (int j = 2; j < kValues; j += 2) high = max3_nan(high, x[j], x[j + 1]);
        } else {
          high = kNegInf;
#pragma unroll
          for (int j = 0; j < kValues; ++j) {
            x[j] = capped(x[j], a.softcap, inverse);
            high = max_nan(high, x[j]);
          }
        }
      }
      high = max_nan(high, kLogprobFloor) * kLog2e;
      if (!(high <= max)) {
        const float d = max_nan(max - high, -1000.f), f = ex2(d);
        weighted = (weighted + sum * d) * f;
        sum *= f;
        max = high;
      }
      unsigned long long s = 0, w = 0;  // pairs of zeros
      const unsigned long long scale = pair_of(kLog2e, kLog2e), shift = pair_of(-max, -max);
#pragma unroll
      for (int j = 0; j < kValues; j += 2) {
        const unsigned long long d =
            fma_pair(pair_of(max_nan(x[j], kLogprobFloor), max_nan(x[j + 1], kLogprobFloor)), scale, shift);
        float d0, d1;
        unpair(d, d0, d1);
        const unsigned long long e = pair_of(ex2(d0), ex2(d1));
        s = add_pair(s, e);
        w = fma_pair(e, d, w);
      }
      float lo, hi;
      unpair(s, lo, hi);
      sum += lo + hi;
      unpair(w, lo, hi);
      weighted += lo + hi;
    }

    // ---- join the threads, then the CTAs of the row
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
      const float m2 = __shfl_xor_sync(0xFFFFFFFFu, max, d), s2 = __shfl_xor_sync(0xFFFFFFFFu, sum, d),
                  w2 = __shfl_xor_sync(0xFFFFFFFFu, weighted, d);
      join_sums(max, sum, weighted, m2, s2, w2);
    }
    float extreme = 0.f;  // the largest value, where the maximum is not a usual one
    if (!usual_maximum(max)) {
      extreme = largest;
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) extreme = fmaxf(extreme, __shfl_xor_sync(0xFFFFFFFFu, extreme, d));
    }
    if (lane == 0) {
      sm.stat[warp][0] = max;
      sm.stat[warp][1] = sum;
      sm.stat[warp][2] = weighted;
      sm.stat[warp][3] = extreme;
    }
    if (a.top) {
      // ---- the segment's list
      float v = sort_lanes(largest, lane);
      v = merge_warps(v, sm.maxima, warp, lane);
      if (threadIdx.x < 32) sm.list[threadIdx.x] = 0ull;
      if (threadIdx.x == a.top - 1) sm.bound = v;
      if (threadIdx.x == 0) sm.count = sm.held = 0;
      __syncthreads();
      const float bound = sm.bound;
      const int begin = first * kBatch, end = min(a.vocab, (first + chunks) * kBatch);
      if (bound > kNegInf) {
        if (largest >= bound) sm.holders[atomicAdd(&sm.held, 1)] = threadIdx.x;
        __syncthreads();
        const int held = sm.held <= kLogprobHolders ? sm.held : 0;  // more: equal values, nearly everywhere
        for (int n = warp; n < held; n += kLogprobWarps) {
          const int of = sm.holders[n];
          for (int k = lane; k < chunks * VECS; k += 32) {
            const int i0 = begin + (k * kLogprobThreads + of) * kPer;  // (vectors of a thread: every 256th)
            float y[kPer];
            if (a.vec && i0 + kPer <= end) {
              unpack<BF16>(y, __ldcg(reinterpret_cast<const uint4*>(static_cast<const char*>(row) + static_cast<long long>(i0) * kSize)));
            } else {
#pragma unroll
              for (int j = 0; j < kPer; ++j) y[j] = i0 + j < end ? load_logit<BF16>(row, i0 + j) : kNegInf;
            }
#pragma unroll
            for (int j = 0; j < kPer; ++j)
              if (!(y[j] < bound)) {
                const int at = atomicAdd(&sm.count, 1);
                if (at < kLogprobBuffer) sm.buffer[at] = list_key(y[j], i0 + j);
              }
          }
        }
        __syncthreads();
      }
      const int count = sm.count;
      if (count && count <= kLogprobBuffer) {
        rebuild_list(sm, count, warp, lane);
      } else {
        __syncthreads();
        if (threadIdx.x == 0) sm.count = 0;
        list_all<BF16>(sm, row, begin, end, a.top, a.vec, warp, lane);
      }
    }
    __syncthreads();
    if (warp == 0) {
      max = sm.stat[lane & (kLogprobWarps - 1)][0];
      sum = lane < kLogprobWarps ? sm.stat[lane & (kLogprobWarps - 1)][1] : 0.f;
      weighted = lane < kLogprobWarps ? sm.stat[lane & (kLogprobWarps - 1)][2] : 0.f;
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) {
        const float m2 = __shfl_xor_sync(0xFFFFFFFFu, max, d), s2 = __shfl_xor_sync(0xFFFFFFFFu, sum, d),
                    w2 = __shfl_xor_sync(0xFFFFFFFFu, weighted, d);
        join_sums(max, sum, weighted, m2, s2, w2);
      }
      extreme = 0.f;
      if (!usual_maximum(max)) {
        extreme = kNegInf;
        for (int i = 0; i < kLogprobWarps; ++i) extreme = fmaxf(extreme, sm.stat[i][3]);
      }
    }
    const int cta_first = row_u0 / a.units_per_cta, cta_last = (row_u1 - 1) / a.units_per_cta;
    unsigned long long mine = warp == 0 ? sm.list[lane] : 0ull;
    bool finish = true;
    if (cta_first != cta_last) {
      LogprobPart* parts = reinterpret_cast<LogprobPart*>(a.partials);
      LogprobPart* part = parts + blockIdx.x * 2 + (row_u0 > u0 ? 1 : 0);
      if (warp == 0) {
        part->list[lane] = mine;
        if (lane == 0) part->max = max, part->sum = sum, part->weighted = weighted, part->largest = extreme;
        __threadfence();
        __syncwarp();
        if (lane == 0) {
          const int arrived = atomic_add_acq_rel_gpu(a.counters + cta_first, 1);
          sm.last = arrived == cta_last - cta_first;
          if (sm.last) a.counters[cta_first] = 0;
        }
      }
      __syncthreads();
      finish = sm.last;
      if (finish) {
        __threadfence();
        // a warp takes every eighth part, then the warps' results are merged
        const LogprobPart* first_part = parts + cta_first * 2 + (row_u0 > cta_first * a.units_per_cta ? 1 : 0);
        const int count = cta_last - cta_first + 1;
        unsigned long long v = 0ull;
        float pm = kLogprobStart, ps = 0.f, pw = 0.f;
        constexpr int kAhead = 4;  // parts whose lists are on the way together
        for (int i0 = warp; i0 < count; i0 += kAhead * kLogprobWarps) {
          unsigned long long list[kAhead];
          float3 stat[kAhead];
#pragma unroll
          for (int k = 0; k < kAhead; ++k) {
            const int i = i0 + k * kLogprobWarps;
            const LogprobPart* p = i == 0 ? first_part : parts + (cta_first + min(i, count - 1)) * 2;
            list[k] = a.top && i < count ? __ldcg(&p->list[lane]) : 0ull;
            stat[k] = i < count ? make_float3(__ldcg(&p->max), __ldcg(&p->sum), __ldcg(&p->weighted))
                                : make_float3(kLogprobStart, 0.f, 0.f);
          }
#pragma unroll
          for (int k = 0; k < kAhead; ++k) {
            join_sums(pm, ps, pw, stat[k].x, stat[k].y, stat[k].z);
            if (a.top && i0 + k * kLogprobWarps < count) v = merge_lanes(v, list[k], lane);
          }
        }
        if (lane == 0) {
          sm.stat[warp][0] = pm;
          sm.stat[warp][1] = ps;
          sm.stat[warp][2] = pw;
        }
        mine = merge_warps(v, sm.lists, warp, lane);
        __syncthreads();
        if (warp == 0) {
          max = sm.stat[0][0], sum = sm.stat[0][1], weighted = sm.stat[0][2];
          for (int i = 1; i < kLogprobWarps; ++i) join_sums(max, sum, weighted, sm.stat[i][0], sm.stat[i][1], sm.stat[i][2]);
          if (!usual_maximum(max)) {
            extreme = kNegInf;
            for (int i = 0; i < count; ++i) extreme = fmaxf(extreme, __ldcg(&(i == 0 ? first_part : parts + (cta_first + i) * 2)->largest));
          }
        }
      }
    }
    if (finish && warp == 0) {
      bool equal = false;
      if (!usual_maximum(max)) {
        equal = !CAP && fabsf(extreme) < INFINITY;
        if (!equal) sum = __uint_as_float(0x7FC00000u);
      }
      if (lane == 0) sm.equal = equal, sm.extreme = extreme, sm.count = 0;
      // lse = (max + log2 sum) ln 2; differences to the maximum first, so
      // that large logits lose nothing
      constexpr float kLn2 = 0.6931471805599453f;
      const float log_sum = logf(sum);
      // (a probability is at most 1: what rounding leaves above that goes)
      auto at_most_zero = [](float v) { return v > 0.f ? 0.f : v; };
      auto log_prob = [&](float x) {
        const float z = CAP ? capped(x, a.softcap, inverse) : x;
        if (sum != sum) return sum;
        if (z < kLogprobStart) return z - (max * kLn2 + log_sum);  // would leave fp32's range in units of log 2
        return at_most_zero(fmaf(z, kLog2e, -max) * kLn2 - log_sum);
      };
      if (lane == 0) {
        float lp = __uint_as_float(0x7FC00000u);
        if (token >= a.vocab) raise_status(kStatusBadArgument);
        else if (token >= 0) lp = log_prob(token_logit);
        a.logprob[row_id] = lp;
        a.entropy[row_id] = 0.f - at_most_zero((weighted / sum) * kLn2 - log_sum);
      }
      if (lane < a.top) {
        a.top_ids[static_cast<long long>(row_id) * a.top + lane] = key_index(mine);
        a.top_logprobs[static_cast<long long>(row_id) * a.top + lane] = log_prob(key_value(mine));
      }
    }
    __syncthreads();
    if (!CAP && finish && sm.equal) {
      // ---- the values equal to the largest, counted by all threads
      const float value = sm.extreme;
      int count = 0;
      const int whole = a.vec ? a.vocab / kPer : 0;  // vectors
#pragma unroll 4
      for (int i = threadIdx.x; i < whole; i += kLogprobThreads) {
        float x[kPer];
        unpack<BF16>(x, __ldcg(static_cast<const uint4*>(row) + i));
#pragma unroll
        for (int j = 0; j < kPer; ++j) count += x[j] == value;
      }
      for (long long i = static_cast<long long>(whole) * kPer + threadIdx.x; i < a.vocab; i += kLogprobThreads)
        count += load_logit<BF16>(row, i) == value;
      count = __reduce_add_sync(0xFFFFFFFFu, count);
      if (lane == 0) atomicAdd(&sm.count, count);
      __syncthreads();
      if (warp == 0) {
        const float log_count = logf(static_cast<float>(sm.count));
        if (lane == 0) {
          if (token >= 0 && token < a.vocab) a.logprob[row_id] = (token_logit - value) - log_count;
          a.entropy[row_id] = log_count;
        }
        if (lane < a.top) {
          const long long at = static_cast<long long>(row_id) * a.top + lane;
          a.top_logprobs[at] = (load_logit<BF16>(row, a.top_ids[at]) - value) - log_count;
        }
      }
      __syncthreads();
    }
    u = stop;
  }
  if (dead && threadIdx.x == 0) {  // copies may still be on their way into the stages
    for (int n = int_max(dead - kLogprobStages, 0); n < dead; ++n) mbar_wait(&sm.full[n % kLogprobStages], (n / kLogprobStages) & 1);
  }
}

// ------------------------------------------------------------------ launch

size_t logprob_partial_bytes(int sm_count) { return static_cast<size_t>(sm_count) * kLogprobCtas * 2 * sizeof(LogprobPart); }

template <bool BF16, int VECS>
cudaError_t launch_logprobs_as(LogprobArgs a, int sm_count, cudaStream_t stream) {
  const int batch = kLogprobThreads * VECS * (BF16 ? 8 : 4);
  a.chunks_per_row = (a.vocab + batch - 1) / batch;
  const long long units = static_cast<long long>(a.rows) * a.chunks_per_row;
  if (units > INT32_MAX - kLogprobCtas * sm_count) return cudaErrorInvalidValue;  // 2^31 batches: more than a GPU's memory of rows
  // at most 64 CTAs to a row: joining more takes longer than they save (one
  // row of 256000 fp32 logits: 19.4 us with 250 CTAs, 15.1 with 63)
  const long long ctas =
      std::min({units, static_cast<long long>(kLogprobCtas) * sm_count, static_cast<long long>(a.rows) * 64});
  a.units_per_cta = static_cast<int>((units + ctas - 1) / ctas);
  const unsigned grid = static_cast<unsigned>((units + a.units_per_cta - 1) / a.units_per_cta);
  const size_t smem = kLogprobStages * kLogprobThreads * 16 * VECS + sizeof(LogprobSmem);
  return launch_overlapped(a.softcap != 0.f ? token_logprobs_kernel<BF16, true, VECS> : token_logprobs_kernel<BF16, false, VECS>,
                           dim3(grid), kLogprobThreads, smem, stream, a);
}

// Two vectors per thread where that leaves every CTA several batches: half
// the barriers per value; one where the rows are few: more CTAs to each row.
cudaError_t launch_token_logprobs(bool bf16, LogprobArgs a, int sm_count, cudaStream_t stream) {
  const long long bytes = static_cast<long long>(a.rows) * a.vocab * (bf16 ? 2 : 4);
  const bool two = bytes >= 12ll * sm_count * kLogprobThreads * 32;
  if (bf16) return two ? launch_logprobs_as<true, 2>(a, sm_count, stream) : launch_logprobs_as<true, 1>(a, sm_count, stream);
  return two ? launch_logprobs_as<false, 2>(a, sm_count, stream) : launch_logprobs_as<false, 1>(a, sm_count, stream);
}

}  // namespace se12
