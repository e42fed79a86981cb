// Log probabilities of given tokens, entropy and the top alternatives of
// rows of logits (the LM head's output), in one pass over them.
//
//   z = x, or cap * tanh(x / cap); lse = M + log S, S = sum exp(z - M)
//   logprob = z[token] - lse,  entropy = log S - (sum exp(z - M) (z - M)) / S
//   top: the k largest x, ties to the lowest index (the cap keeps the order)
//
// The pass keeps, per thread, the running maximum with S and the weighted
// sum below it, and per CTA a buffer of candidates for the top list: values
// above the list's k-th, pushed by whichever thread meets them. The list is
// rebuilt (each warp sorts 32 candidates at a time and merges them into its
// own 32, then the warps' lists are merged) only when the buffer fills up,
// after the first batch and at the end; before the first batch is pushed,
// the k-th largest of the threads' own maxima already bounds the list from
// below. Work units of whole batches are cut into equal runs, one per CTA,
// and a row's CTAs are joined by the last to finish, in CTA order. The bound
// is HBM for plain logits, the special-function unit (three calls a value)
// for capped ones.
#include "se12_device.cuh"
#include "se12_serve.h"

#include <algorithm>

#include <cuda_bf16.h>

namespace se12 {

constexpr int kLogprobThreads = 512;
constexpr int kLogprobWarps = kLogprobThreads / 32;
constexpr int kLogprobValues = 16;                               // per thread and batch
constexpr int kLogprobBatch = kLogprobThreads * kLogprobValues;  // values of a batch
constexpr int kLogprobTop = 32;
constexpr int kLogprobSpare = 1024;                              // candidates kept before the list is rebuilt
constexpr int kLogprobBuffer = kLogprobSpare + kLogprobBatch;
// -inf and masks of the type's lowest value become this: its exponential is
// zero and its product with log2(e) still finite.
constexpr float kLogprobFloor = -2.0e38f;
// Where every running maximum starts: far enough above the floor that floor
// values add nothing to a sum, below every logit that counts. A row that
// ends there is summed again in 64 bits.
constexpr float kLogprobStart = -1.0e38f;

// A CTA's part of a row, for the CTA that joins them.
struct LogprobPart {
  float max, sum, weighted, pad;  // of z * log2(e): max; sum 2^(z - max); sum 2^(z - max) (z - max)
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
  if (u == 0xFFFFFFFFu) return __uint_as_float(0x7FC00000u);
  return __uint_as_float((u & 0x80000000u) ? u & 0x7FFFFFFFu : ~u);
}

__device__ __forceinline__ int key_index(unsigned long long key) { return static_cast<int>(~static_cast<unsigned>(key)); }

__device__ __forceinline__ unsigned long long larger(unsigned long long a, unsigned long long b) { return a > b ? a : b; }
__device__ __forceinline__ unsigned long long smaller(unsigned long long a, unsigned long long b) { return a < b ? a : b; }

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
  float maxima[kLogprobWarps][32];
  float stat[kLogprobWarps][3];
  unsigned long long list[32];
  float joined[3];
  int count;
  int last;
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

// cap * tanh(x / cap) = cap - 2 cap / (exp(2 x / cap) + 1); -inf stays.
__device__ __forceinline__ float capped(float x, float cap) {
  const float e = ex2(x * (2.f * kLog2e / cap));
  const float z = cap - __fdividef(2.f * cap, e + 1.f);
  return x == kNegInf ? kNegInf : z;
}

template <bool BF16>
__device__ __forceinline__ float load_logit(const void* row, long long i) {
  if constexpr (BF16) return __uint_as_float(static_cast<uint32_t>(static_cast<const uint16_t*>(row)[i]) << 16);
  return static_cast<const float*>(row)[i];
}

// This thread's kLogprobValues values of the batch at `base`: vector j of
// thread t holds values base + (j * threads + t) * per vector ... Values at
// or past `end` are -inf and never candidates.
template <bool BF16>
__device__ __forceinline__ void load_batch(float (&x)[kLogprobValues], const void* row, long long base, long long end,
                                           bool vec) {
  constexpr int kPer = BF16 ? 8 : 4;
#pragma unroll
  for (int j = 0; j < kLogprobValues / kPer; ++j) {
    const long long i = base + (j * kLogprobThreads + threadIdx.x) * kPer;
    if (vec && i + kPer <= end) {
      const uint4 v = __ldcs(reinterpret_cast<const uint4*>(static_cast<const char*>(row) + i * (BF16 ? 2 : 4)));
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if constexpr (BF16) {
          x[j * 8 + 2 * k] = __uint_as_float(w[k] << 16);
          x[j * 8 + 2 * k + 1] = __uint_as_float(w[k] & 0xFFFF0000u);
        } else {
          x[j * 4 + k] = __uint_as_float(w[k]);
        }
      }
    } else {
#pragma unroll
      for (int k = 0; k < kPer; ++k) x[j * kPer + k] = i + k < end ? load_logit<BF16>(row, i + k) : kNegInf;
    }
  }
}

template <bool BF16>
__device__ __forceinline__ int batch_index(int value) {
  constexpr int kPer = BF16 ? 8 : 4;
  return ((value / kPer) * kLogprobThreads + static_cast<int>(threadIdx.x)) * kPer + value % kPer;
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

template <bool BF16, bool CAP>
__global__ void __launch_bounds__(kLogprobThreads, 2) token_logprobs_kernel(const LogprobArgs a) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  LogprobSmem& sm = *reinterpret_cast<LogprobSmem*>(smem_raw);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  grid_launch_dependents();
  grid_dependency_wait();

  const long long units = static_cast<long long>(a.rows) * a.chunks_per_row;
  const long long u0 = blockIdx.x * a.units_per_cta, u1 = min(u0 + a.units_per_cta, units);
  for (long long u = u0; u < u1;) {
    const int row_id = static_cast<int>(u / a.chunks_per_row);
    const long long row_u0 = static_cast<long long>(row_id) * a.chunks_per_row, row_u1 = row_u0 + a.chunks_per_row;
    const long long stop = min(row_u1, u1);
    const void* row = static_cast<const char*>(a.logits) + row_id * a.ld * (BF16 ? 2 : 4);
    const long long begin = (u - row_u0) * a.chunk;
    const long long end = min(static_cast<long long>(a.vocab), (stop - row_u0) * a.chunk);

    float max = kLogprobStart, sum = 0.f, weighted = 0.f;
    float bound = kNegInf;  // candidates: values not below it (first batch) or above it
    if (threadIdx.x < 32) sm.list[threadIdx.x] = 0ull;
    if (threadIdx.x == 0) sm.count = 0;
    __syncthreads();
    bool strict = false;
    for (long long base = begin; base < end; base += kLogprobBatch) {
      float x[kLogprobValues];
      load_batch<BF16>(x, row, base, end, a.vec);
      float top = x[0];
#pragma unroll
      for (int j = 1; j < kLogprobValues; ++j) top = max_nan(top, x[j]);
      if (a.top) {
        if (!strict) {
          // the k-th largest of the threads' maxima
          float v = sort_lanes(top != top ? INFINITY : top, lane);
          v = merge_warps(v, sm.maxima, warp, lane);
          if (warp == 0 && lane == a.top - 1) sm.joined[0] = v;
          __syncthreads();
          bound = sm.joined[0];
        }
        bool full = false;
        if (strict ? !(top <= bound) : !(top < bound)) {
#pragma unroll
          for (int j = 0; j < kLogprobValues; ++j) {
            const long long i = base + batch_index<BF16>(j);
            if ((strict ? !(x[j] <= bound) : !(x[j] < bound)) && i < end) {
              const int at = atomicAdd(&sm.count, 1);
              sm.buffer[at] = list_key(x[j], static_cast<int>(i));
              full |= at >= kLogprobSpare;
            }
          }
        }
        // (the first batch may hold fewer than k values: -inf stays inclusive)
        if (__syncthreads_or(full || !strict)) {
          rebuild_list(sm, sm.count, warp, lane);
          const unsigned long long kth = sm.list[a.top - 1];
          strict = kth != 0ull;
          bound = strict ? key_value(kth) : kNegInf;
          if (bound != bound) bound = INFINITY;  // a list of NaN takes no more
        }
      }
      // sums relative to the running maximum, in units of log 2 (z log2(e)
      // - max is one rounding everywhere: the maximum's own cancels)
      float high = kLogprobFloor;
#pragma unroll
      for (int j = 0; j < kLogprobValues; ++j) {
        x[j] = max_nan(CAP ? capped(x[j], a.softcap) : x[j], kLogprobFloor);
        high = max_nan(high, x[j]);
      }
      high *= kLog2e;
      if (!(high <= max)) {
        const float d = max_nan(max - high, -1000.f), f = ex2(d);
        weighted = (weighted + sum * d) * f;
        sum *= f;
        max = high;
      }
      float s = 0.f, w = 0.f;
#pragma unroll
      for (int j = 0; j < kLogprobValues; ++j) {
        const float d = fmaf(x[j], kLog2e, -max), e = ex2(d);
        s += e;
        w = fmaf(e, d, w);
      }
      sum += s;
      weighted += w;
    }

    // ---- join the threads, then the CTAs of the row
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
      const float m2 = __shfl_xor_sync(0xFFFFFFFFu, max, d), s2 = __shfl_xor_sync(0xFFFFFFFFu, sum, d),
                  w2 = __shfl_xor_sync(0xFFFFFFFFu, weighted, d);
      join_sums(max, sum, weighted, m2, s2, w2);
    }
    if (lane == 0) {
      sm.stat[warp][0] = max;
      sm.stat[warp][1] = sum;
      sm.stat[warp][2] = weighted;
    }
    if (a.top) {
      __syncthreads();
      if (sm.count) rebuild_list(sm, sm.count, warp, lane);
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
    }
    const long long cta_first = row_u0 / a.units_per_cta, cta_last = (row_u1 - 1) / a.units_per_cta;
    unsigned long long mine = warp == 0 ? sm.list[lane] : 0ull;
    bool finish = true;
    if (cta_first != cta_last) {
      LogprobPart* parts = reinterpret_cast<LogprobPart*>(a.partials);
      LogprobPart* part = parts + blockIdx.x * 2 + (row_u0 > u0 ? 1 : 0);
      if (warp == 0) {
        part->list[lane] = mine;
        if (lane == 0) part->max = max, part->sum = sum, part->weighted = weighted;
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
        // a warp takes every 16th part, then the warps' results are merged
        const LogprobPart* first = parts + cta_first * 2 + (row_u0 > cta_first * a.units_per_cta ? 1 : 0);
        const int count = static_cast<int>(cta_last - cta_first) + 1;
        unsigned long long v = 0ull;
        float pm = kLogprobStart, ps = 0.f, pw = 0.f;
        for (int i = warp; i < count; i += kLogprobWarps) {
          const LogprobPart* p = i == 0 ? first : parts + (cta_first + i) * 2;
          join_sums(pm, ps, pw, __ldcg(&p->max), __ldcg(&p->sum), __ldcg(&p->weighted));
          if (a.top) v = merge_lanes(v, __ldcg(&p->list[lane]), lane);
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
        }
      }
    }
    if (finish && warp == 0) {
      // a row with nothing above the start, values past fp32's range in units
      // of log 2, infinities or NaN: again in 64 bits from its true maximum
      float low_max = kNegInf;
      const bool again = !(max > kLogprobStart && max < 1e38f);
      if (again) {
        double s = 0.0, w = 0.0;
        for (long long i = lane; i < a.vocab; i += 32) {
          const float x = load_logit<BF16>(row, i);
          low_max = fmaxf(low_max, CAP ? capped(x, a.softcap) : x);
        }
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) low_max = fmaxf(low_max, __shfl_xor_sync(0xFFFFFFFFu, low_max, d));
        for (long long i = lane; i < a.vocab; i += 32) {
          const float x = load_logit<BF16>(row, i);
          const double below = static_cast<double>(CAP ? capped(x, a.softcap) : x) - low_max;  // -inf - -inf: NaN, as it must be
          const double e = exp(below);
          s += e;
          if (e > 0.0) w += e * below;
          else if (e != e) w = e;
        }
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) {
          s += __shfl_xor_sync(0xFFFFFFFFu, s, d);
          w += __shfl_xor_sync(0xFFFFFFFFu, w, d);
        }
        sum = static_cast<float>(s);
        weighted = static_cast<float>(w * 1.4426950408889634);
      }
      // lse = (max + log2 sum) ln 2; differences to the maximum first, so
      // that large logits lose nothing
      constexpr float kLn2 = 0.6931471805599453f;
      const float log_sum = logf(sum);
      auto log_prob = [&](float x) {
        const float z = CAP ? capped(x, a.softcap) : x;
        if (sum != sum) return sum;
        if (again) return (z - low_max) - log_sum;
        if (z < kLogprobStart) return z - (max * kLn2 + log_sum);  // would leave fp32's range in units of log 2
        return fmaf(z, kLog2e, -max) * kLn2 - log_sum;
      };
      if (lane == 0) {
        const long long t = a.tokens[row_id];
        float lp = __uint_as_float(0x7FC00000u);
        if (t >= a.vocab) raise_status(kStatusBadArgument);
        else if (t >= 0) lp = log_prob(load_logit<BF16>(row, t));
        a.logprob[row_id] = lp;
        a.entropy[row_id] = log_sum - (weighted / sum) * kLn2;
      }
      if (lane < a.top) {
        a.top_ids[static_cast<long long>(row_id) * a.top + lane] = key_index(mine);
        a.top_logprobs[static_cast<long long>(row_id) * a.top + lane] = log_prob(key_value(mine));
      }
    }
    __syncthreads();
    u = stop;
  }
}

// ------------------------------------------------------------------ launch

// Two CTAs per SM at most (their candidate buffers fill the shared memory).
size_t logprob_partial_bytes(int sm_count) { return static_cast<size_t>(sm_count) * 2 * 2 * sizeof(LogprobPart); }

cudaError_t launch_token_logprobs(bool bf16, LogprobArgs a, int sm_count, cudaStream_t stream) {
  // units of one batch, or of less when the rows alone do not fill the GPU
  a.chunk = kLogprobBatch;
  a.chunks_per_row = (a.vocab + a.chunk - 1) / a.chunk;
  const long long units = static_cast<long long>(a.rows) * a.chunks_per_row;
  const long long ctas = std::min<long long>(units, 2ll * sm_count);
  a.units_per_cta = (units + ctas - 1) / ctas;
  const unsigned grid = static_cast<unsigned>((units + a.units_per_cta - 1) / a.units_per_cta);
  const size_t smem = sizeof(LogprobSmem);
  const bool cap = a.softcap != 0.f;
  if (bf16)
    return launch_overlapped(cap ? token_logprobs_kernel<true, true> : token_logprobs_kernel<true, false>, dim3(grid),
                             kLogprobThreads, smem, stream, a);
  return launch_overlapped(cap ? token_logprobs_kernel<false, true> : token_logprobs_kernel<false, false>, dim3(grid),
                           kLogprobThreads, smem, stream, a);
}

}  // namespace se12
