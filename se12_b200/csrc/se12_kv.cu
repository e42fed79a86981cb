// The paged 8-bit key/value cache: appending new tokens, with the position
// rotation applied on the way, and reading pages back.
//
// A block (one page of one KV head, keys and values separately) holds codes
// c and one scale s = 2^e; a value is c * s. e is the smallest integer >=
// kMinScaleExponent with amax <= qmax * 2^e over the block's tokens (qmax 127
// for int8, 448 for e4m3). Powers of two cost int8 up to one of its seven
// bits, and buy two things: when a later token raises the block's scale, the
// older codes shrink by an exact power of two and are rounded once more (for
// e4m3 that only touches subnormals), so that the rounding errors of
// repeated growth form a geometric series below one step; and code * scale
// is exact in BF16 and in every product with a query, whatever order the
// kernels apply the scale in.
//
// Both kernels are bound by memory: the new tokens are read once from HBM
// (the second pass of a prompt block hits L2) and the codes written once.
#include "se12_device.cuh"
#include "se12_serve.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

namespace se12 {

constexpr int kMinScaleExponent = -100;
constexpr unsigned kInfBits = 0x7F800000u;
constexpr unsigned kNanBits = 0x7FC00000u;

// Bits of the least admissible scale for a block whose largest magnitude has
// the fp32 bits `amax`; NaN where that is not finite.
template <int KIND>
__device__ __forceinline__ float fit_scale(unsigned amax) {
  if (amax >= kInfBits) return __uint_as_float(kNanBits);
  // qmax = 1.984375 * 2^6 (127) or 1.75 * 2^8 (448)
  constexpr int q_exponent = KIND == kKvInt8 ? 6 : 8;
  constexpr unsigned q_mantissa = KIND == kKvInt8 ? 0x7E0000u : 0x600000u;
  int e = static_cast<int>(amax >> 23) - 127 - q_exponent + ((amax & 0x7FFFFFu) > q_mantissa ? 1 : 0);
  if (e < kMinScaleExponent) e = kMinScaleExponent;
  return __uint_as_float(static_cast<unsigned>(e + 127) << 23);
}

// Scaled value to code, rounded to nearest, ties to even. |x| <= qmax.
template <int KIND>
__device__ __forceinline__ uint32_t to_code(float x) {
  if constexpr (KIND == kKvInt8) return static_cast<uint32_t>(__float2int_rn(x)) & 0xFFu;
  return __nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3);
}

template <int KIND>
__device__ __forceinline__ float code_value(uint32_t c) {
  if constexpr (KIND == kKvInt8) return static_cast<float>(static_cast<int8_t>(c));
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(c), __NV_E4M3)));
}

__device__ __forceinline__ float load_value(const float* p) { return *p; }
__device__ __forceinline__ float load_value(const __nv_bfloat16* p) { return __bfloat162float(*p); }

// VP consecutive elements (VP > 1: the address is a multiple of their size).
template <int VP>
__device__ __forceinline__ void load_vector(float (&x)[VP], const float* p) {
  if constexpr (VP == 4) {
    const float4 v = *reinterpret_cast<const float4*>(p);
    x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
  } else if constexpr (VP == 2) {
    const float2 v = *reinterpret_cast<const float2*>(p);
    x[0] = v.x, x[1] = v.y;
  } else {
    x[0] = *p;
  }
}

template <int VP>
__device__ __forceinline__ void load_vector(float (&x)[VP], const __nv_bfloat16* p) {
  if constexpr (VP == 4) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    x[0] = __uint_as_float(v.x << 16), x[1] = __uint_as_float(v.x & 0xFFFF0000u);
    x[2] = __uint_as_float(v.y << 16), x[3] = __uint_as_float(v.y & 0xFFFF0000u);
  } else if constexpr (VP == 2) {
    const uint32_t v = *reinterpret_cast<const uint32_t*>(p);
    x[0] = __uint_as_float(v << 16), x[1] = __uint_as_float(v & 0xFFFF0000u);
  } else {
    x[0] = load_value(p);
  }
}

// A row of `dim` values as dim / 2 pairs (a, b): the pairs the rotation turns
// together first, then neighbours. A lane takes VP consecutive pairs at a
// time, so that both members stay in one lane.
struct PairMap {
  int pairs;   // dim / 2
  int turned;  // pairs below this are rotated
  int split;   // pairs below this have members p and p + half, the others 2p and 2p + 1
  int half;

  __device__ __forceinline__ void at(int p, int& a, int& b) const {
    if (p < split) {
      a = p;
      b = p + half;
    } else {
      a = 2 * p;
      b = 2 * p + 1;
    }
  }
};

// (a, b) turned by the angle whose cosine and sine are c and s; each product
// and each sum is rounded by itself, as elementary tensor operations do.
__device__ __forceinline__ void turn(float& a, float& b, float c, float s) {
  const float x = __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s));
  b = __fadd_rn(__fmul_rn(b, c), __fmul_rn(a, s));
  a = x;
}

// Calls f(a index, b index, values a, values b) for this lane's pairs of one row.
template <int VP, typename T, typename F>
__device__ __forceinline__ void for_row(const T* row, const PairMap& map, const float* cos, const float* sin, int lane,
                                        F&& f) {
  for (int p = lane * VP; p < map.pairs; p += 32 * VP) {
    float a[VP], b[VP];
    int ia, ib;
    map.at(p, ia, ib);
    load_vector<VP>(a, row + ia);
    load_vector<VP>(b, row + ib);
    if (p < map.turned) {
      float c[VP], s[VP];
      load_vector<VP>(c, cos + p);
      load_vector<VP>(s, sin + p);
#pragma unroll
      for (int j = 0; j < VP; ++j) turn(a[j], b[j], c[j], s[j]);
    }
    f(ia, ib, a, b);
  }
}

// A row in registers, for vector lanes (one step covers the row): what
// lane `lane` has of its first and second halves.
template <int VP>
struct RowPart {
  float a[VP], b[VP];

  template <typename T>
  __device__ __forceinline__ void load(const T* row, int lane) {
    load_vector<VP>(a, row + lane * VP);
    load_vector<VP>(b, row + 32 * VP + lane * VP);
  }

  __device__ __forceinline__ void rotate(const float (&c)[VP], const float (&s)[VP]) {
#pragma unroll
    for (int j = 0; j < VP; ++j) turn(a[j], b[j], c[j], s[j]);
  }
};

template <int VP>
__device__ __forceinline__ unsigned magnitude_bits(const float (&x)[VP], unsigned m) {
#pragma unroll
  for (int j = 0; j < VP; ++j) m = max(m, __float_as_uint(x[j]) & 0x7FFFFFFFu);
  return m;
}

template <int KIND, int VP>
__device__ __forceinline__ void store_codes(uint8_t* p, const float (&x)[VP], float inv) {
  uint32_t w = 0;
#pragma unroll
  for (int j = 0; j < VP; ++j) w |= to_code<KIND>(x[j] * inv) << (8 * j);
  if constexpr (VP == 4)
    *reinterpret_cast<uint32_t*>(p) = w;
  else if constexpr (VP == 2)
    *reinterpret_cast<uint16_t*>(p) = static_cast<uint16_t>(w);
  else
    *p = static_cast<uint8_t>(w);
}

template <int VP>
__device__ __forceinline__ void store_bf16(uint16_t* p, const float (&x)[VP]) {
  uint16_t h[VP];
#pragma unroll
  for (int j = 0; j < VP; ++j) h[j] = __bfloat16_as_ushort(__float2bfloat16_rn(x[j]));
  if constexpr (VP == 4)
    *reinterpret_cast<uint2*>(p) = make_uint2(h[0] | (static_cast<uint32_t>(h[1]) << 16), h[2] | (static_cast<uint32_t>(h[3]) << 16));
  else if constexpr (VP == 2)
    *reinterpret_cast<uint32_t*>(p) = h[0] | (static_cast<uint32_t>(h[1]) << 16);
  else
    *p = h[0];
}

// Rounds `bytes` codes (a multiple of 16) again after the scale grew by 1 / ratio.
template <int KIND>
__device__ __forceinline__ void shrink_codes(uint8_t* codes, int bytes, float ratio, int thread, int threads) {
  for (int i = thread * 16; i < bytes; i += threads * 16) {
    uint4 v = *reinterpret_cast<const uint4*>(codes + i);
    uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t r = 0;
#pragma unroll
      for (int b = 0; b < 4; ++b) r |= to_code<KIND>(code_value<KIND>((w[j] >> (8 * b)) & 0xFFu) * ratio) << (8 * b);
      w[j] = r;
    }
    *reinterpret_cast<uint4*>(codes + i) = v;
  }
}

// Page of position `pos` of sequence b, or -1 (and the status word raised)
// where the table has none for it.
__device__ __forceinline__ int page_of(const TokenBatch& t, const KvView& c, int b, int pos) {
  const int i = pos >> c.page_shift;
  if (i < t.max_pages) {
    const int page = t.table[b * t.table_stride + i];
    if (page >= 0 && page < c.pages) return page;
  }
  raise_status(kStatusBadArgument);
  return -1;
}

// Scale of a block with older tokens at scale `before` (`older`) once tokens
// with largest magnitude `amax` have joined it; `ratio` = what the older codes
// shrink by.
template <int KIND>
__device__ __forceinline__ float joined_scale(float before, bool older, unsigned amax, float& ratio) {
  const float need = fit_scale<KIND>(amax);
  ratio = 1.f;
  if (!older) return need;
  if (!(before >= need)) {  // grows, or one of the two is not finite
    if (before < need) {
      ratio = before * __frcp_rn(need);
      return need;
    }
    return __uint_as_float(kNanBits);
  }
  return before;
}

// How a row of queries or keys (turned) or values (not) splits into pairs.
// Vector lanes (vp > 1) serve rows that are turned in halves, whole or not
// at all, and split both kinds in halves.
__device__ __forceinline__ PairMap pair_map(const AppendArgs& a, bool turned, int vp) {
  PairMap m;
  m.pairs = a.c.dim / 2;
  m.turned = turned && a.cos ? a.rotary / 2 : 0;
  m.split = vp > 1 ? m.pairs : a.interleaved ? 0 : m.turned;
  m.half = vp > 1 ? m.pairs : m.turned;
  return m;
}

// One query row (token t, head h), rotated, as BF16. `pos` < 0: an inactive
// row, written as zeros.
template <typename T, int VP>
__device__ __forceinline__ void rotate_query(const AppendArgs& a, int token, int head, int pos, int lane) {
  uint16_t* out = a.q_out + token * a.o_ts + head * a.o_hs;
  const bool bad = a.cos && pos >= a.rope_rows;
  if (pos < 0 || bad) {
    if (bad) raise_status(kStatusBadArgument);
    for (int i = lane; i < a.c.dim; i += 32) out[i] = 0;
    return;
  }
  const T* row = static_cast<const T*>(a.q) + token * a.q_ts + head * a.q_hs;
  PairMap map = pair_map(a, true, VP);
  for_row<VP>(row, map, a.cos + pos * a.rope_stride, a.sin + pos * a.rope_stride, lane,
              [&](int ia, int ib, const float(&x)[VP], const float(&y)[VP]) {
                store_bf16<VP>(out + ia, x);
                store_bf16<VP>(out + ib, y);
              });
}

// One token per sequence: a warp per (sequence, KV head, keys or values) and
// one per (sequence, query head).
template <typename T, int KIND, int VP>
__global__ void __launch_bounds__(128) kv_append_step_kernel(const AppendArgs a) {
  grid_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int per_seq = 2 * a.c.heads + (a.q ? a.q_heads : 0);
  const long long item = static_cast<long long>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  const int b = static_cast<int>(item / per_seq);
  const int what = static_cast<int>(item % per_seq);
  grid_dependency_wait();
  if (b >= a.t.seqs) return;
  const int pos = max(a.t.lens[b], 0) - 1;
  if (what >= 2 * a.c.heads) {
    rotate_query<T, VP>(a, b, what - 2 * a.c.heads, pos, lane);
    return;
  }
  if (pos < 0) return;
  const bool keys = what < a.c.heads;
  const int head = keys ? what : what - a.c.heads;
  if (a.cos && pos >= a.rope_rows) {  // neither half of the token is stored
    raise_status(kStatusBadArgument);
    return;
  }
  const T* row = static_cast<const T*>(keys ? a.k : a.v) + b * (keys ? a.k_ts : a.v_ts) + head * (keys ? a.k_hs : a.v_hs);
  const PairMap map = pair_map(a, keys, VP);
  const float* cos = a.cos + pos * a.rope_stride;
  const float* sin = a.sin + pos * a.rope_stride;
  const int page = page_of(a.t, a.c, b, pos);
  if (page < 0) return;
  const int slot = pos & (a.c.page_size - 1);
  const long long block = static_cast<long long>(page) * a.c.heads + head;
  uint8_t* codes = (keys ? a.c.k_codes : a.c.v_codes) + block * a.c.page_size * a.c.dim;
  float* scale = (keys ? a.c.k_scales : a.c.v_scales) + block;
  const float before = *scale;
  unsigned amax = 0;
  for_row<VP>(row, map, cos, sin, lane, [&](int, int, const float(&x)[VP], const float(&y)[VP]) {
    amax = magnitude_bits<VP>(y, magnitude_bits<VP>(x, amax));
  });
  amax = __reduce_max_sync(0xFFFFFFFFu, amax);
  float ratio;
  const float now = joined_scale<KIND>(before, slot > 0, amax, ratio);
  const bool finite = now == now;
  if (ratio != 1.f) shrink_codes<KIND>(codes, slot * a.c.dim, ratio, lane, 32);
  const float inv = finite ? __frcp_rn(now) : 0.f;  // exact for the powers of two stored here
  uint8_t* to = codes + slot * a.c.dim;
  for_row<VP>(row, map, cos, sin, lane, [&](int ia, int ib, const float(&x)[VP], const float(&y)[VP]) {
    if (finite) {
      store_codes<KIND, VP>(to + ia, x, inv);
      store_codes<KIND, VP>(to + ib, y, inv);
    } else {
#pragma unroll
      for (int j = 0; j < VP; ++j) to[ia + j] = to[ib + j] = 0;
    }
  });
  __syncwarp();
  if (lane == 0) *scale = now;
}

// The sequence token t belongs to: the number of sequences 1 .. seqs - 1
// that start at or before it, counted 32 at a time by one warp.
__device__ __forceinline__ int sequence_of(const TokenBatch& t, int token, int lane) {
  if (!t.query_start) return token;
  int n = 0;
  for (int i = 1; i < t.seqs; i += 32) {
    const int b = i + lane;
    n += __popc(__ballot_sync(0xFFFFFFFFu, b < t.seqs && t.query_start[b] <= token));
  }
  return n;
}

// New tokens of one page (rows 0 .. count - 1 at src, slots slot ..) joined to
// it by a CTA of 8 warps, for the heads head .. head + heads - 1 one after the
// other: the next head's rows are on their way while this one's scale is found.
template <typename T, int KIND, int VP>
__device__ __forceinline__ void append_page(const AppendArgs& a, bool keys, const T* src, long long ts, long long hs, int head,
                                            int heads, int pos, int slot, int count, int page, unsigned (*s_amax)[8]) {
  constexpr int kHeld = 4;  // rows a warp keeps in registers from one pass to the next
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, dim = a.c.dim;
  const PairMap map = pair_map(a, keys, VP);
  const bool turned = keys && a.cos;
  const bool held = VP > 1 && count <= 8 * kHeld;
  RowPart<VP> row[kHeld];
  auto rotate = [&](RowPart<VP>& r, int i) {
    if (turned) {
      float c[VP], s[VP];
      load_vector<VP>(c, a.cos + (pos + i) * a.rope_stride + lane * VP);
      load_vector<VP>(s, a.sin + (pos + i) * a.rope_stride + lane * VP);
      r.rotate(c, s);
    }
  };
  auto load = [&](int h, int i0) {
#pragma unroll
    for (int k = 0; k < kHeld; ++k)
      if (i0 + 8 * k < count) row[k].load(src + h * hs + (i0 + 8 * k) * ts, lane);
  };
  if (VP > 1 && held) load(head, warp);
  for (int n = 0; n < heads; ++n) {
    const int h = head + n;
    const T* rows = src + h * hs;
    const long long block = static_cast<long long>(page) * a.c.heads + h;
    float* scale = (keys ? a.c.k_scales : a.c.v_scales) + block;
    uint8_t* codes = (keys ? a.c.k_codes : a.c.v_codes) + block * a.c.page_size * dim;
    const float before = slot > 0 ? *scale : 0.f;
    unsigned amax = 0;
    if constexpr (VP > 1) {
      for (int i0 = warp; i0 < count; i0 += 8 * kHeld) {
        if (!held) load(h, i0);
#pragma unroll
        for (int k = 0; k < kHeld; ++k)
          if (i0 + 8 * k < count) {
            rotate(row[k], i0 + 8 * k);
            amax = magnitude_bits<VP>(row[k].b, magnitude_bits<VP>(row[k].a, amax));
          }
      }
    } else {
      for (int i = warp; i < count; i += 8)
        for_row<VP>(rows + i * ts, map, a.cos + (pos + i) * a.rope_stride, a.sin + (pos + i) * a.rope_stride, lane,
                    [&](int, int, const float(&x)[VP], const float(&y)[VP]) {
                      amax = magnitude_bits<VP>(y, magnitude_bits<VP>(x, amax));
                    });
    }
    amax = __reduce_max_sync(0xFFFFFFFFu, amax);
    if (lane == 0) s_amax[n & 1][warp] = amax;
    __syncthreads();  // the maxima are there, and every thread has read the old scale
    amax = s_amax[n & 1][lane & 7];
    amax = __reduce_max_sync(0xFFFFFFFFu, amax);
    float ratio;
    const float now = joined_scale<KIND>(before, slot > 0, amax, ratio);
    const bool finite = now == now;
    if (ratio != 1.f) shrink_codes<KIND>(codes, slot * dim, ratio, threadIdx.x, 256);
    const float inv = finite ? __frcp_rn(now) : 0.f;  // exact for the powers of two stored here
    auto put = [&](uint8_t* to, const float(&x)[VP]) {
      if (finite) {
        store_codes<KIND, VP>(to, x, inv);
      } else {
#pragma unroll
        for (int j = 0; j < VP; ++j) to[j] = 0;
      }
    };
    uint8_t* to = codes + slot * dim;
    if constexpr (VP > 1) {
      for (int i0 = warp; i0 < count; i0 += 8 * kHeld) {
        if (!held) {
          load(h, i0);
#pragma unroll
          for (int k = 0; k < kHeld; ++k)
            if (i0 + 8 * k < count) rotate(row[k], i0 + 8 * k);
        }
#pragma unroll
        for (int k = 0; k < kHeld; ++k)
          if (i0 + 8 * k < count) {
            put(to + (i0 + 8 * k) * dim + lane * VP, row[k].a);
            put(to + (i0 + 8 * k) * dim + 32 * VP + lane * VP, row[k].b);
          }
      }
      if (held && n + 1 < heads) load(h + 1, warp);
    } else {
      for (int i = warp; i < count; i += 8)
        for_row<VP>(rows + i * ts, map, a.cos + (pos + i) * a.rope_stride, a.sin + (pos + i) * a.rope_stride, lane,
                    [&](int ia, int ib, const float(&x)[VP], const float(&y)[VP]) {
                      put(to + i * dim + ia, x);
                      put(to + i * dim + ib, y);
                    });
    }
    if (threadIdx.x == 0) *scale = now;
  }
  __syncthreads();  // the maxima are free
}

// One token's queries, a warp: the angle's cosines and sines are loaded once
// for all heads.
template <typename T, int VP>
__device__ __forceinline__ void rotate_queries(const AppendArgs& a, int token, int pos, int lane) {
  if (VP == 1 || pos < 0 || (a.cos && pos >= a.rope_rows)) {
    for (int h = 0; h < a.q_heads; ++h) rotate_query<T, VP>(a, token, h, pos, lane);
    return;
  }
  float c[VP], s[VP];
  if (a.cos) {
    load_vector<VP>(c, a.cos + pos * a.rope_stride + lane * VP);
    load_vector<VP>(s, a.sin + pos * a.rope_stride + lane * VP);
  }
  const T* src = static_cast<const T*>(a.q) + token * a.q_ts;
  uint16_t* out = a.q_out + token * a.o_ts;
  constexpr int kHeads = 4;  // on their way together
  for (int h0 = 0; h0 < a.q_heads; h0 += kHeads) {
    RowPart<VP> row[kHeads];
#pragma unroll
    for (int k = 0; k < kHeads; ++k)
      if (h0 + k < a.q_heads) row[k].load(src + (h0 + k) * a.q_hs, lane);
#pragma unroll
    for (int k = 0; k < kHeads; ++k)
      if (h0 + k < a.q_heads) {
        if (a.cos) row[k].rotate(c, s);
        store_bf16<VP>(out + (h0 + k) * a.o_hs + lane * VP, row[k].a);
        store_bf16<VP>(out + (h0 + k) * a.o_hs + 32 * VP + lane * VP, row[k].b);
      }
  }
}

// Any number of tokens per sequence. All blockIdx.y but the last, each for
// `heads_each` heads of the keys or of the values: a CTA looks through `span`
// consecutive tokens for the first new token of a block (of its sequence, or
// of a page) and stores that block's new tokens, four rows per warp on their
// way at a time; up to 32 stay in registers while the scale is found, more are
// read again from L2. The last blockIdx.y rotates the queries, a warp per
// token.
template <typename T, int KIND, int VP>
__global__ void __launch_bounds__(256, 3) kv_append_prompt_kernel(const AppendArgs a, const int span, const int heads_each) {
  __shared__ unsigned s_amax[2][8];
  grid_launch_dependents();
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int groups = (a.c.heads + heads_each - 1) / heads_each, what = blockIdx.y;
  const int first = blockIdx.x * span, end = min(first + span, a.t.tokens);
  const ListSizes sizes{a.t.tokens, a.t.max_pages << a.c.page_shift, 1, 0};
  if (what == 2 * groups) {
    for (int t = first + warp; t < end; t += 8) {
      const int b = sequence_of(a.t, t, lane);
      const SeqRows s = a.t.rows_of(b, sizes);
      const int row = t - a.t.begin_of(b, sizes);
      rotate_queries<T, VP>(a, t, row >= 0 && row < s.tokens ? s.first + row : -1, lane);
    }
    return;
  }
  int b = sequence_of(a.t, first, lane);
  const bool keys = what < groups;
  const int head = (keys ? what : what - groups) * heads_each;
  const T* src = static_cast<const T*>(keys ? a.k : a.v);
  const long long ts = keys ? a.k_ts : a.v_ts;
  for (int t = first; t < end; ++t) {
    while (b + 1 < a.t.seqs && a.t.query_start[b + 1] <= t) ++b;
    const SeqRows s = a.t.rows_of(b, sizes);
    const int start = a.t.begin_of(b, sizes), stop = start + s.tokens;
    const int pos = s.first + (t - start);
    if (t < start || t >= stop || pos < 0) continue;  // not a sequence's token, or an inactive one
    const int slot = pos & (a.c.page_size - 1);
    if (t != start && slot != 0) {  // a token inside a block: on to the next block
      t += min(min(a.c.page_size - slot, stop - t), end - t) - 1;
      continue;
    }
    const int page = page_of(a.t, a.c, b, pos);
    if (page < 0) continue;
    int count = min(a.c.page_size - slot, stop - t);
    if (a.cos && pos + count > a.rope_rows) {  // tokens past the rotation table: neither half is stored
      raise_status(kStatusBadArgument);
      count = a.rope_rows - pos;
      if (count <= 0) continue;
    }
    append_page<T, KIND, VP>(a, keys, src + t * ts, ts, keys ? a.k_hs : a.v_hs, head, min(heads_each, a.c.heads - head), pos,
                             slot, count, page, s_amax);
  }
}

// Pages read back as BF16 (exact: a code has at most 8 significant bits), a
// CTA per block (page of a head), keys and values by blockIdx.y.
template <int KIND>
__global__ void __launch_bounds__(256) kv_decode_kernel(const KvView c, const int32_t* pages, int count, uint16_t* k_out,
                                                        uint16_t* v_out) {
  grid_launch_dependents();
  grid_dependency_wait();
  const int block_codes = c.page_size * c.dim;  // a multiple of 256
  const uint8_t* codes = blockIdx.y ? c.v_codes : c.k_codes;
  const float* scales = blockIdx.y ? c.v_scales : c.k_scales;
  uint16_t* outs = blockIdx.y ? v_out : k_out;
  const long long blocks = static_cast<long long>(count) * c.heads;
  for (long long n = blockIdx.x; n < blocks; n += gridDim.x) {
    const int nth = static_cast<int>(n / c.heads), head = static_cast<int>(n - static_cast<long long>(nth) * c.heads);
    const int page = pages ? pages[nth] : nth;
    uint16_t* out = outs + n * block_codes;
    if (page < 0 || page >= c.pages) {
      raise_status(kStatusBadArgument);
      for (int i = threadIdx.x * 8; i < block_codes; i += 2048) *reinterpret_cast<uint4*>(out + i) = make_uint4(0, 0, 0, 0);
      continue;
    }
    const long long block = static_cast<long long>(page) * c.heads + head;
    const uint8_t* in = codes + block * block_codes;
    const float s = scales[block];
#pragma unroll 4
    for (int i = threadIdx.x * 8; i < block_codes; i += 2048) {
      const uint2 v = *reinterpret_cast<const uint2*>(in + i);
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t pair = (j < 2 ? v.x : v.y) >> (16 * (j & 1));
        const float lo = code_value<KIND>(pair & 0xFFu) * s, hi = code_value<KIND>((pair >> 8) & 0xFFu) * s;
        w[j] = __bfloat16_as_ushort(__float2bfloat16_rn(lo)) |
               (static_cast<uint32_t>(__bfloat16_as_ushort(__float2bfloat16_rn(hi))) << 16);
      }
      *reinterpret_cast<uint4*>(out + i) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}

// ------------------------------------------------------------------ launches

template <typename T, int KIND, int VP>
cudaError_t launch_append_as(const AppendArgs& a, cudaStream_t stream) {
  if (!a.t.query_start) {
    const long long warps = static_cast<long long>(a.t.seqs) * (2 * a.c.heads + (a.q ? a.q_heads : 0));
    return launch_overlapped(kv_append_step_kernel<T, KIND, VP>, dim3(static_cast<unsigned>((warps + 3) / 4)), 128, 0,
                             stream, a);
  }
  // Few tokens: one per CTA, so that short sequences' blocks run side by side;
  // more: 16, among them one CTA's queries. A CTA takes four heads of short
  // pages, which it finds once for them, one of long ones, two where there are
  // many. us for one, two and four heads per CTA, BF16 with the queries: pages
  // of 32, 16 query and 8 KV heads of 256, 500 tokens 11, 12, 13; 2100 tokens 26,
  // 24, 17; 16000 tokens 141, 122, 111. Pages of 128, 2100 tokens 26, 45, 84;
  // 8000 (992 blocks) 81, 75, 104. Pages of 256, 8000 tokens (496 blocks) 94,
  // 113, 184; 16000 (992) 164, 161, 222. 32 tokens per CTA instead of 16: pages
  // of 128, 64 query heads of 128, 2100 tokens 41 -> 62; 16000 170 -> 183 (four heads).
  const int span = a.t.tokens <= 256 ? 1 : 16;
  const long long blocks = static_cast<long long>(a.t.tokens) / a.c.page_size * 2 * a.c.heads;
  const int heads_each = a.t.tokens <= 256 ? 1 : a.c.page_size <= 32 ? 4 : blocks >= 900 ? 2 : 1;
  const dim3 grid((a.t.tokens + span - 1) / span, 2 * ((a.c.heads + heads_each - 1) / heads_each) + (a.q ? 1 : 0));
  return launch_overlapped(kv_append_prompt_kernel<T, KIND, VP>, grid, 256, 0, stream, a, span, heads_each);
}

template <typename T, int KIND>
cudaError_t launch_append_kind(const AppendArgs& a, cudaStream_t stream) {
  // vector lanes: whole rows turned in halves (or not at all), 32 * VP pairs
  // a step, and every row and table address a multiple of VP elements
  const int vp = a.c.dim % 256 == 0 ? 4 : a.c.dim % 128 == 0 ? 2 : 1;
  bool vec = vp > 1 && (!a.cos || (!a.interleaved && a.rotary == a.c.dim && a.rope_stride % vp == 0 &&
                                   reinterpret_cast<uintptr_t>(a.cos) % (vp * 4) == 0 &&
                                   reinterpret_cast<uintptr_t>(a.sin) % (vp * 4) == 0));
  const void* ptr[3] = {a.k, a.v, a.q};
  const long long stride[6] = {a.k_ts, a.k_hs, a.v_ts, a.v_hs, a.q_ts, a.q_hs};
  for (int i = 0; i < 3; ++i)
    if (ptr[i] && (reinterpret_cast<uintptr_t>(ptr[i]) % (vp * sizeof(T)) || stride[2 * i] % vp || stride[2 * i + 1] % vp))
      vec = false;
  if (a.q && (reinterpret_cast<uintptr_t>(a.q_out) % (vp * 2) || a.o_ts % vp || a.o_hs % vp)) vec = false;
  if (!vec) return launch_append_as<T, KIND, 1>(a, stream);
  return vp == 4 ? launch_append_as<T, KIND, 4>(a, stream) : launch_append_as<T, KIND, 2>(a, stream);
}

cudaError_t launch_kv_append(bool bf16, const AppendArgs& a, cudaStream_t stream) {
  if (bf16)
    return a.c.kind == kKvInt8 ? launch_append_kind<__nv_bfloat16, kKvInt8>(a, stream)
                               : launch_append_kind<__nv_bfloat16, kKvE4m3>(a, stream);
  return a.c.kind == kKvInt8 ? launch_append_kind<float, kKvInt8>(a, stream) : launch_append_kind<float, kKvE4m3>(a, stream);
}

cudaError_t launch_kv_decode(const KvView& c, const int32_t* pages, int count, uint16_t* k_out, uint16_t* v_out,
                             cudaStream_t stream) {
  const long long blocks = static_cast<long long>(count) * c.heads;
  const dim3 grid(static_cast<unsigned>(blocks < (1 << 20) ? blocks : (1 << 20)), 2);
  return launch_overlapped(c.kind == kKvInt8 ? kv_decode_kernel<kKvInt8> : kv_decode_kernel<kKvE4m3>, grid, 256, 0, stream, c,
                           pages, count, k_out, v_out);
}

}  // namespace se12
