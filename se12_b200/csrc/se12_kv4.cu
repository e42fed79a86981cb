// The paged 4-bit key/value cache: appending new tokens, normalised and
// rotated on the way, and reading pages back.
//
// Every token of a head is quantised by itself, in groups of 64 dimensions: a
// value is (u - 8) * scale + offset, u a code 0..15, with
//   scale = fp16((hi - lo) / 15), offset = fp16(lo + 8 scale),
//   u = clamp(rint((x - offset) / scale) + 8, 0, 15)
// of the group's largest and smallest value. (4.5 bits per key. One scale per
// 64 without the offset loses 1.4 times the squares on normal values and 2.5
// times on ones with a few large channels; groups of 32 with a scale alone, the
// same bits, 1.2 and 1.5 times.) Values have their power of two besides: scale
// and offset are those of x 2^-E, E = floor(log2 max |x|) - 3, -30 at least, so
// that attention's FP16 products of weights and scales keep their bits whatever
// the values' size. Nothing depends on the page's other tokens: no scale grows,
// no older code is touched, and a page is written by any number of warps.
//
// The order of a row's codes is the matrix instructions': words of 8 codes,
// word 8 g + r of the row at place r * groups + g, so that one 16-byte vector
// holds words of each group. Keys' scales lie token by token, values' as pairs
// of neighbouring tokens in cells of 16: [8 pairs][groups scales, groups
// offsets][2], then the 16 E.
//
// 13 prompt chunks of 301 to 2043 tokens, 16 query and 8 KV heads of 256, BF16,
// with norms: 118 us, 3.0 TB/s of what has to move; what bounds it is the issue of
// some 180 instructions per row at 2.5 of 4 a cycle (20 warps per SM). Their pages
// read back: 24 us, 6.2 TB/s. For few tokens both are bound by their latency (64
// tokens of 80 heads: 5 us).
#include "se12_kv.cuh"

#include <algorithm>
#include <cuda_fp16.h>

namespace se12 {

constexpr int kKv4Group = 64;
constexpr int kKv4MinExponent = -30;
constexpr float kKv4KeyLimit = 65000.f;         // larger keys do not fit FP16's scale and offset
constexpr float kKv4ValueLimit = 17179869184.f;  // 2^34: E is at most 30
constexpr int kKv4Threads = 128;

// How a head's row is spread over its team of DIM / 16 lanes. In order: lane l
// has the dimensions 8 l .. 8 l + 7 and DIM / 2 + 8 l .. + 7, a word of codes
// each. Read: the members of the pairs 8 l .. 8 l + 7 that are turned together,
// which are the same dimensions unless part of the row is turned in halves.
struct RowOrder {
  int mode;    // 0: not turned; 1: pairs (i, i + half); 2: neighbours
  int turned;  // pairs that are
  int half;    // distance in halves
  bool apart;  // read in another order than stored

  // The two dimensions of pair p.
  __device__ __forceinline__ void at(int p, int& a, int& b) const {
    if (p < half) {
      a = p;
      b = p + half;
    } else {
      a = 2 * p;
      b = 2 * p + 1;
    }
  }
};

template <int DIM>
__device__ __forceinline__ RowOrder row_order(const AppendArgs& a, bool turned) {
  RowOrder o;
  o.mode = !turned || !a.cos ? 0 : a.interleaved ? 2 : 1;
  o.turned = o.mode ? a.rotary / 2 : 0;
  o.half = o.mode == 1 ? o.turned : DIM / 2;
  o.apart = o.mode == 1 && a.rotary != DIM;
  return o;
}

// Eight values, two by two.
struct Eight {
  unsigned long long v[4];

  __device__ __forceinline__ void set(int j, float x) {  // (j known at compile time)
    float lo, hi;
    unpair(v[j >> 1], lo, hi);
    v[j >> 1] = j & 1 ? pair_of(lo, x) : pair_of(x, hi);
  }
  __device__ __forceinline__ float get(int j) const {
    float lo, hi;
    unpair(v[j >> 1], lo, hi);
    return j & 1 ? hi : lo;
  }
};

__device__ __forceinline__ unsigned long long both(float x) { return pair_of(x, x); }

// x + y and x - y, each rounded by itself also where x and y are products: of
// mul.rn.f32x2 and add.rn.f32x2 the assembler makes one fma, of this it does not.
__device__ __forceinline__ unsigned long long add_apart(unsigned long long x, unsigned long long y) {
  float a, b, c, d;
  unpair(x, a, b);
  unpair(y, c, d);
  return pair_of(__fadd_rn(a, c), __fadd_rn(b, d));
}
__device__ __forceinline__ unsigned long long sub_apart(unsigned long long x, unsigned long long y) {
  float a, b, c, d;
  unpair(x, a, b);
  unpair(y, c, d);
  return pair_of(__fsub_rn(a, c), __fsub_rn(b, d));
}

__device__ __forceinline__ void load_eight(Eight& x, const float* p) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float4 v = *reinterpret_cast<const float4*>(p + 4 * i);
    x.v[2 * i] = pair_of(v.x, v.y);
    x.v[2 * i + 1] = pair_of(v.z, v.w);
  }
}
__device__ __forceinline__ void load_eight(Eight& x, const __nv_bfloat16* p) {
  const uint4 v = *reinterpret_cast<const uint4*>(p);
#pragma unroll
  for (int i = 0; i < 4; ++i) x.v[i] = pair_of(__uint_as_float(word_of(v, i) << 16), __uint_as_float(word_of(v, i) & 0xFFFF0000u));
}

// A lane's part of a row.
struct RowPart16 {
  Eight a, b;
};

// How rows are read. kSimple: vectors of eight aligned elements, turned in halves
// as a whole or not at all; kVector: such vectors, halves multiples of eight or
// neighbours; kSingle: anything, element by element. us for 64 and 14000 tokens of 16
// query and 8 KV heads of 256, BF16 with norms: turned as a whole 4.0, 111;
// neighbours 4.0, 129; half of the row 5.2, 217; rows off alignment 5.4, 256; 12
// dimensions, whose halves are no vectors, 7.2, 406.
enum RowKind { kSimple, kVector, kSingle };

// Where in a row the two vectors of lane l begin.
template <int DIM, RowKind HOW>
__device__ __forceinline__ void vectors_at(const RowOrder& o, int l, int& ia, int& ib) {
  ia = 8 * l, ib = DIM / 2 + 8 * l;
  if (HOW == kVector && o.apart) {
    ia = 8 * l < o.half ? 8 * l : 16 * l;
    ib = 8 * l < o.half ? 8 * l + o.half : 16 * l + 8;
  }
}

template <int DIM, RowKind HOW, typename T>
__device__ __forceinline__ void load_row(RowPart16& r, const T* row, const RowOrder& o, int l) {
  if (HOW != kSingle) {
    int ia, ib;
    vectors_at<DIM, HOW>(o, l, ia, ib);
    load_eight(r.a, row + ia);
    load_eight(r.b, row + ib);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      int ia = 8 * l + j, ib = DIM / 2 + 8 * l + j;
      if (o.apart) o.at(8 * l + j, ia, ib);
      r.a.set(j, load_value(row + ia));
      r.b.set(j, load_value(row + ib));
    }
  }
}

// A row on its way: as it lies in memory, so that nothing is moved when it is taken.
template <typename T, int DIM, RowKind HOW>
struct RowAhead {
  static constexpr int kVectors = sizeof(T) / 2;  // of 16 bytes, of eight elements
  uint4 a[kVectors], b[kVectors];
  RowPart16 single;

  __device__ __forceinline__ void load(const T* row, const RowOrder& o, int l) {
    if (HOW == kSingle) {
      load_row<DIM, HOW>(single, row, o, l);
      return;
    }
    int ia, ib;
    vectors_at<DIM, HOW>(o, l, ia, ib);
#pragma unroll
    for (int i = 0; i < kVectors; ++i) {
      a[i] = reinterpret_cast<const uint4*>(row + ia)[i];
      b[i] = reinterpret_cast<const uint4*>(row + ib)[i];
    }
  }
  __device__ __forceinline__ static void eight_of(Eight& x, const uint4 (&v)[kVectors]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (sizeof(T) == 4)
        x.v[i] = pair_of(__uint_as_float(word_of(v[i / 2 % kVectors], 2 * (i & 1))), __uint_as_float(word_of(v[i / 2 % kVectors], 2 * (i & 1) + 1)));
      else
        x.v[i] = pair_of(__uint_as_float(word_of(v[0], i) << 16), __uint_as_float(word_of(v[0], i) & 0xFFFF0000u));
    }
  }
  __device__ __forceinline__ void take(RowPart16& r) const {
    if (HOW == kSingle) {
      r = single;
      return;
    }
    eight_of(r.a, a);
    eight_of(r.b, b);
  }
};

// The cosines and sines that a lane needs at one position: of the pairs 8 l ..
// 8 l + 7, or of the neighbours in its two vectors.
template <int DIM, RowKind HOW>
__device__ __forceinline__ void load_angles(RowPart16& t, const AppendArgs& a, const RowOrder& o, int pos, int l) {
  if (o.mode == 0) return;
  const float* cos = a.cos + pos * a.rope_stride;
  const float* sin = a.sin + pos * a.rope_stride;
  if (HOW == kSimple) {
    load_eight(t.a, cos + 8 * l);
    load_eight(t.b, sin + 8 * l);
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int p = o.mode == 1 ? 8 * l + j : (j < 4 ? 4 * l : DIM / 4 + 4 * l - 4) + j;
    t.a.set(j, p < o.turned ? cos[p] : 1.f);
    t.b.set(j, p < o.turned ? sin[p] : 0.f);
  }
}

template <int DIM, RowKind HOW>
__device__ __forceinline__ void load_weights_row(RowPart16& w, const RowNorm& norm, const RowOrder& o, int l) {
  if (norm.bf16)
    load_row<DIM, HOW>(w, static_cast<const __nv_bfloat16*>(norm.weight), o, l);
  else
    load_row<DIM, HOW>(w, static_cast<const float*>(norm.weight), o, l);
}

template <int DIM>
__device__ __forceinline__ void normalise_row(RowPart16& r, const RowPart16& w, double eps) {
  double sum[2] = {0.0, 0.0};
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const double x = r.a.get(j), y = r.b.get(j);
    sum[0] = fma(x, x, sum[0]);
    sum[1] = fma(y, y, sum[1]);
  }
  const unsigned long long f = both(norm_factor(team_sum(sum[0] + sum[1], DIM / 16), DIM, eps));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    r.a.v[i] = mul_pair(mul_pair(r.a.v[i], f), w.a.v[i]);
    r.b.v[i] = mul_pair(mul_pair(r.b.v[i], f), w.b.v[i]);
  }
}

template <int DIM, RowKind HOW>
__device__ __forceinline__ void rotate_row(RowPart16& r, const RowPart16& t, const RowOrder& o, int l) {
  if (o.mode == 0) return;
  if (HOW == kSimple) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // as turn(): each product and each sum rounded by itself
      const unsigned long long x = sub_apart(mul_pair(r.a.v[i], t.a.v[i]), mul_pair(r.b.v[i], t.b.v[i]));
      r.b.v[i] = add_apart(mul_pair(r.b.v[i], t.a.v[i]), mul_pair(r.a.v[i], t.b.v[i]));
      r.a.v[i] = x;
    }
  } else if (o.mode == 1) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float x = r.a.get(j), y = r.b.get(j);
      if (8 * l + j < o.turned) turn(x, y, t.a.get(j), t.b.get(j));
      r.a.set(j, x);
      r.b.set(j, y);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float x = r.a.get(2 * j), y = r.a.get(2 * j + 1);
      if (4 * l + j < o.turned) turn(x, y, t.a.get(j), t.b.get(j));
      r.a.set(2 * j, x);
      r.a.set(2 * j + 1, y);
      x = r.b.get(2 * j), y = r.b.get(2 * j + 1);
      if (DIM / 4 + 4 * l + j < o.turned) turn(x, y, t.a.get(4 + j), t.b.get(4 + j));
      r.b.set(2 * j, x);
      r.b.set(2 * j + 1, y);
    }
  }
}

// A row read apart put in order, through the team's row of shared memory.
template <int DIM, RowKind HOW>
__device__ __forceinline__ void reorder_row(RowPart16& r, float* staged, const RowOrder& o, int l) {
  __syncwarp();
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    int ia, ib;
    if (HOW == kVector) {
      ia = (8 * l < o.half ? 8 * l : 16 * l) + j;
      ib = (8 * l < o.half ? 8 * l + o.half : 16 * l + 8) + j;
    } else {
      o.at(8 * l + j, ia, ib);
    }
    staged[ia] = r.a.get(j);
    staged[ib] = r.b.get(j);
  }
  __syncwarp();
  load_eight(r.a, staged + 8 * l);
  load_eight(r.b, staged + DIM / 2 + 8 * l);
}

template <bool VEC>
__device__ __forceinline__ void store_eight(uint16_t* p, const Eight& x) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    w[i] = __bfloat16_as_ushort(__float2bfloat16_rn(x.get(2 * i))) |
           (static_cast<uint32_t>(__bfloat16_as_ushort(__float2bfloat16_rn(x.get(2 * i + 1)))) << 16);
  if (VEC) {
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      p[2 * i] = static_cast<uint16_t>(w[i]);
      p[2 * i + 1] = static_cast<uint16_t>(w[i] >> 16);
    }
  }
}

__device__ __forceinline__ void extremes(const Eight& x, float& lo, float& hi) {
  lo = hi = x.get(0);
#pragma unroll
  for (int j = 1; j < 8; ++j) {
    lo = min_nan(lo, x.get(j));
    hi = max_nan(hi, x.get(j));
  }
}

// A group's scale and offset, and the word of eight values' codes.
struct GroupLine {
  __half scale, offset;
  float middle, inverse;

  __device__ __forceinline__ void fit(float lo, float hi) {
    scale = __float2half_rn(__fmul_rn(__fsub_rn(hi, lo), 1.f / 15.f));
    const float s = __half2float(scale);
    offset = __float2half_rn(__fadd_rn(lo, 8.f * s));
    middle = __half2float(offset);
    inverse = s > 0.f ? __frcp_rn(s) : 0.f;
  }

  // Rounded to whole numbers by an addend of 1.5 2^23 (and 8, the zero point): the
  // code is in the last bits, under what eight of the addend's bits sum up to.
  __device__ __forceinline__ uint32_t word(const Eight& x) const {
    const unsigned long long m = both(middle), f = both(inverse), up = both(12582920.f);
    uint32_t w = 0;
#pragma unroll
    for (int i = 3; i >= 0; --i) {
      float lo, hi;
      unpair(mul_pair(sub_apart(x.v[i], m), f), lo, hi);
      lo = fminf(fmaxf(lo, -8.f), 7.f);  // (NaN: -8)
      hi = fminf(fmaxf(hi, -8.f), 7.f);
      unpair(add_pair(pair_of(lo, hi), up), lo, hi);
      w = (w * 16 + __float_as_uint(hi)) * 16 + __float_as_uint(lo);
    }
    return w - 0x4B400000u * 0x11111111u;
  }
};

// A lane's row quantised and stored as token `slot` of a block. All lanes of
// the warp take part; where `live` is false nothing is stored. (Keys and values
// by one piece of code: two, unrolled over four rows, were waiting for
// instructions most of the time, 13 prompt chunks 387 us.)
template <int DIM>
__device__ __forceinline__ void store_row(const AppendArgs& a, bool keys, RowPart16& r, long long block, int slot, int l, bool live) {
  constexpr int G = DIM / kKv4Group;
  constexpr int kSpan = DIM >= 128 ? 8 : 4;  // lanes of a group
  float lo_a, hi_a, lo_b, hi_b;
  extremes(r.a, lo_a, hi_a);
  extremes(r.b, lo_b, hi_b);
  if (DIM < 128) {
    lo_a = min_nan(lo_a, lo_b);
    hi_a = max_nan(hi_a, hi_b);
  }
#pragma unroll
  for (int d = 1; d < kSpan; d <<= 1) {
    lo_a = min_nan(lo_a, __shfl_xor_sync(0xFFFFFFFFu, lo_a, d));
    hi_a = max_nan(hi_a, __shfl_xor_sync(0xFFFFFFFFu, hi_a, d));
    if (DIM >= 128) {
      lo_b = min_nan(lo_b, __shfl_xor_sync(0xFFFFFFFFu, lo_b, d));
      hi_b = max_nan(hi_b, __shfl_xor_sync(0xFFFFFFFFu, hi_b, d));
    }
  }
  if (DIM < 128) lo_b = lo_a, hi_b = hi_a;
  const float size_a = max_nan(fabsf(lo_a), fabsf(hi_a)), size_b = max_nan(fabsf(lo_b), fabsf(hi_b));
  float exponent = 0.f;
  if (!keys) {
    float amax = max_nan(size_a, size_b);
    if (DIM == 256) amax = max_nan(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, 8));
    const bool fits = amax < kKv4ValueLimit;  // (otherwise, NaN too, the token is NaN through E alone: its line is 0)
    const int e = fits ? max(static_cast<int>(__float_as_uint(amax) >> 23) - 130, kKv4MinExponent) : 0;
    exponent = fits ? static_cast<float>(e) : __uint_as_float(0x7FC00000u);
    const float down = __uint_as_float(static_cast<unsigned>(127 - e) << 23);
    if (!fits) {
      lo_a = hi_a = lo_b = hi_b = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) r.a.v[i] = r.b.v[i] = 0;
    }
    lo_a *= down, hi_a *= down, lo_b *= down, hi_b *= down;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      r.a.v[i] = mul_pair(r.a.v[i], both(down));
      r.b.v[i] = mul_pair(r.b.v[i], both(down));
    }
  }
  GroupLine ga, gb;
  ga.fit(lo_a, hi_a);
  gb.fit(lo_b, hi_b);
  const uint32_t wa = ga.word(r.a), wb = gb.word(r.b);
  if (!live) return;
  const long long row = block * a.c.page_size + slot;
  uint32_t* words = reinterpret_cast<uint32_t*>((keys ? a.c.k_codes : a.c.v_codes) + row * (DIM / 2));
  const int n = DIM / 16 + l;
  words[(l & 7) * G + (l >> 3)] = wa;
  words[(n & 7) * G + (n >> 3)] = wb;
  // The lanes of span h hold group h of the first half (ga) and group G / 2 + h of the second.
  const int h = l / kSpan, k = l % kSpan;
  if (keys) {
    const bool second = k == 1;
    if (k == 0 || (DIM >= 128 && second)) {
      const bool fits = (second ? size_b : size_a) <= kKv4KeyLimit;
      const __half2 line = second ? __halves2half2(gb.scale, gb.offset) : __halves2half2(ga.scale, ga.offset);
      const __half2 nan = __half2half2(__ushort_as_half(0x7FFFu));
      reinterpret_cast<__half2*>(a.c.k_scales)[row * G + (second ? G / 2 + h : h)] = fits ? line : nan;
    }
  } else {
    __half* cell = reinterpret_cast<__half*>(a.c.v_scales) +
                   (block * (a.c.page_size >> 4) + (slot >> 4)) * (32 * G + 16);
    // lane k of a span: scale, offset of ga, of gb; the row's last lane: E
    const int at = ((slot & 15) >> 1) * (4 * G) + (slot & 1);
    const __half x = k == 0 ? ga.scale : k == 1 ? ga.offset : k == 2 ? gb.scale : gb.offset;
    if (k < (DIM >= 128 ? 4 : 2)) cell[at + 2 * ((k & 1 ? G : 0) + (k < 2 ? h : G / 2 + h))] = x;
    if (l == DIM / 16 - 1) cell[32 * G + (slot & 15)] = __float2half_rn(exponent);
  }
}

// The sequence that token t belongs to: the last one that starts at or before
// it (the first sequence where none does), found 32 at a time.
__device__ __forceinline__ int sequence_at(const TokenBatch& t, int token, int lane) {
  if (!t.query_start) return token;
  int low = 0, count = t.seqs;  // the answer is in low .. low + count - 1, starts[low] <= token or low = 0
  while (count > 1) {
    const int step = (count + 31) >> 5, i = low + lane * step;
    const bool before = lane > 0 && i < low + count && t.query_start[i] <= token;
    const int found = __popc(__ballot_sync(0xFFFFFFFFu, before)) * step;
    low += found;
    count = min(step, count - found);
  }
  return low;
}

// A warp takes a token's queries, keys or values, 32 / (DIM / 16) heads side by
// side and up to `turns` of those one after the other, the next on its way.
// `q_warps` and `kv_warps`: warps per token for its queries, and for its keys and
// for its values.
template <typename T, int DIM, RowKind HOW>
__global__ void __launch_bounds__(kKv4Threads, HOW == kSingle ? 3 : 5) kv4_append_kernel(const AppendArgs a, const int q_warps, const int kv_warps,
                                                                 const int turns) {
  constexpr int kTeam = DIM / 16, kTeams = 32 / kTeam;
  __shared__ float4 staged[HOW == kSimple ? 1 : kKv4Threads / 32][HOW == kSimple ? 1 : kTeams][HOW == kSimple ? 1 : DIM / 4];
  grid_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, l = lane % kTeam, team = lane / kTeam;
  const int per_token = q_warps + 2 * kv_warps;
  const long long item = static_cast<long long>(blockIdx.x) * (kKv4Threads / 32) + warp;
  grid_dependency_wait();
  if (item >= static_cast<long long>(a.t.tokens) * per_token) return;
  const int token = static_cast<int>(item / per_token);
  int part = static_cast<int>(item - static_cast<long long>(token) * per_token);
  const bool queries = part < q_warps, keys = !queries && part < q_warps + kv_warps;
  part -= queries ? 0 : keys ? q_warps : q_warps + kv_warps;
  const int heads = queries ? a.q_heads : a.c.heads, head0 = part * (turns * kTeams);
  const int end = min(head0 + turns * kTeams, heads);
  const T* src = static_cast<const T*>(queries ? a.q : keys ? a.k : a.v) + token * (queries ? a.q_ts : keys ? a.k_ts : a.v_ts);
  const long long hs = queries ? a.q_hs : keys ? a.k_hs : a.v_hs;
  const RowOrder order = row_order<DIM>(a, queries || keys);
  // (teams past the last head take the last one again, and store nothing)
  RowAhead<T, DIM, HOW> next;
  next.load(src + min(head0 + team, heads - 1) * hs, order, l);

  const ListSizes sizes{a.t.tokens, a.t.max_pages << a.c.page_shift, 1, 0};
  const int b = sequence_at(a.t, token, lane);
  const SeqRows s = a.t.rows_of(b, sizes);
  const int at = token - a.t.begin_of(b, sizes);
  int pos = at >= 0 && at < s.tokens ? s.first + at : -1;
  const bool off_table = a.cos && pos >= a.rope_rows;
  if (off_table) {  // queries are zeros, of keys and values neither is stored
    raise_status(kStatusBadArgument);
    pos = -1;
  }
  uint16_t* out = a.q_out + token * a.o_ts;
  if (pos < 0) {
    if (queries)
      for (int head = head0 + team; head < end; head += kTeams)
        for (int i = l; i < DIM; i += kTeam) out[head * a.o_hs + i] = 0;
    return;
  }
  const int page = queries ? 0 : page_of(a.t, a.c, b, pos);
  if (page < 0) return;
  RowPart16 angles;
  load_angles<DIM, HOW>(angles, a, order, pos, l);
  const RowNorm norm = queries ? a.q_norm : keys ? a.k_norm : RowNorm{};
  RowPart16 weight;
  if (norm.weight) load_weights_row<DIM, HOW>(weight, norm, order, l);
  const int slot = pos & (a.c.page_size - 1);
#pragma unroll 1
  for (int first = head0; first < end; first += kTeams) {
    const int head = first + team;
    const bool live = head < end;
    RowPart16 row;
    next.take(row);
    if (first + kTeams < end) next.load(src + min(head + kTeams, heads - 1) * hs, order, l);
    if (norm.weight) normalise_row<DIM>(row, weight, a.norm_eps);
    rotate_row<DIM, HOW>(row, angles, order, l);
    if (HOW != kSimple && order.apart) reorder_row<DIM, HOW>(row, reinterpret_cast<float*>(staged[warp][team]), order, l);
    if (!queries) {
      store_row<DIM>(a, keys, row, static_cast<long long>(page) * a.c.heads + head, slot, l, live);
    } else if (live) {
      uint16_t* to = out + head * a.o_hs;
      store_eight<HOW != kSingle>(to + 8 * l, row.a);
      store_eight<HOW != kSingle>(to + DIM / 2 + 8 * l, row.b);
    }
  }
}

// Pages read back as BF16, keys and values by blockIdx.y. A thread takes 16 bytes
// of codes of each of two neighbouring tokens, which share a cell's lines: 64
// values. (A thread per word of 8: 14000 tokens of 8 heads of 256 46 us.)
template <int DIM>
__global__ void __launch_bounds__(256) kv4_decode_kernel(const KvView c, const int32_t* pages, unsigned blocks, uint16_t* k_out,
                                                         uint16_t* v_out) {
  constexpr int G = DIM / kKv4Group, kParts = DIM / 32;  // 16 bytes of codes: words 4 part .. + 3
  grid_launch_dependents();
  grid_dependency_wait();
  const bool keys = blockIdx.y == 0;
  const int shift = c.page_shift - 1 + (DIM == 64 ? 1 : DIM == 128 ? 2 : 3);  // items of a block, a power of two
  const unsigned long long items = static_cast<unsigned long long>(blocks) << shift;
  for (unsigned long long at = blockIdx.x * 256ull + threadIdx.x; at < items; at += gridDim.x * 256ull) {
    const unsigned n = static_cast<unsigned>(at >> shift), nth = n / c.heads, head = n - nth * c.heads;
    const int item = static_cast<int>(at) & ((1 << shift) - 1), part = item % kParts, token = item / kParts * 2;
    const int page = pages ? pages[nth] : static_cast<int>(nth);
    uint16_t* out = (keys ? k_out : v_out) + (static_cast<unsigned long long>(n) * c.page_size + token) * DIM;
    // dimension where word w of the 16 bytes begins
    auto dim_of = [&](int w) { return (4 * part + w) % G * kKv4Group + (4 * part + w) / G * 8; };
    if (page < 0 || page >= c.pages) {
      raise_status(kStatusBadArgument);
#pragma unroll
      for (int w = 0; w < 8; ++w) *reinterpret_cast<uint4*>(out + (w >> 2) * DIM + dim_of(w & 3)) = make_uint4(0, 0, 0, 0);
      continue;
    }
    const long long row = (static_cast<long long>(page) * c.heads + head) * c.page_size + token;
    const uint4* codes = reinterpret_cast<const uint4*>((keys ? c.k_codes : c.v_codes) + row * (DIM / 2)) + part;
    const uint4 x[2] = {codes[0], codes[kParts]};
    float scale[2][G], offset[2][G], power[2] = {1.f, 1.f};
    if (keys) {
      const __half2* line = reinterpret_cast<const __half2*>(c.k_scales) + row * G;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int g = 0; g < G; ++g) {
          const float2 v = __half22float2(line[t * G + g]);
          scale[t][g] = v.x, offset[t][g] = v.y;
        }
    } else {
      const __half* cell = reinterpret_cast<const __half*>(c.v_scales) + (row >> 4) * (32 * G + 16);
      const __half2* pair = reinterpret_cast<const __half2*>(cell) + (token & 15) * G;
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const float2 s = __half22float2(pair[g]), o = __half22float2(pair[G + g]);
        scale[0][g] = s.x, scale[1][g] = s.y, offset[0][g] = o.x, offset[1][g] = o.y;
      }
      const float2 e = __half22float2(*reinterpret_cast<const __half2*>(cell + 32 * G + (token & 15)));  // whole numbers, or NaN
      power[0] = e.x == e.x ? __uint_as_float(static_cast<unsigned>(static_cast<int>(e.x) + 127) << 23) : e.x;
      power[1] = e.y == e.y ? __uint_as_float(static_cast<unsigned>(static_cast<int>(e.y) + 127) << 23) : e.y;
    }
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const int g = w % G;  // (four words, G of 1, 2 or 4)
        const uint32_t u = word_of(x[t], w);
        uint32_t o[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float v[2];
#pragma unroll
          for (int k = 0; k < 2; ++k)  // the code under 2^23's last bits is u + 2^23
            v[k] = fmaf(__uint_as_float(((u >> (8 * j + 4 * k)) & 15u) | 0x4B000000u) - 8388616.f, scale[t][g], offset[t][g]) * power[t];
          o[j] = __bfloat16_as_ushort(__float2bfloat16_rn(v[0])) |
                 (static_cast<uint32_t>(__bfloat16_as_ushort(__float2bfloat16_rn(v[1]))) << 16);
        }
        *reinterpret_cast<uint4*>(out + t * DIM + dim_of(w)) = make_uint4(o[0], o[1], o[2], o[3]);
      }
  }
}

// ------------------------------------------------------------------ launches

inline bool aligned_to(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

template <typename T, int DIM, RowKind HOW>
cudaError_t launch_append4_as(const AppendArgs& a, cudaStream_t stream) {
  constexpr int kTeams = 32 / (DIM / 16);
  // Few rows: a warp for every kTeams of a token; many: up to four times as many
  // in one, which finds the token's place and angles once for them. us for once and
  // four times, BF16 with norms: 64 query and 8 KV heads of 128 (20 rows per token) 64
  // tokens 4.1, 4.5; 200 6.0, 6.5; 600 11.9, 9.9; 1200 19.7, 14.6; 14000 205, 134. 16
  // and 8 of 256 (16): 4.0, 5.7; 6.0, 6.4; 10.7, 8.4; 17.6, 13.3; 175, 112. 32 and 8
  // of 64 (6): 3.3, 4.4; 3.7, 4.7; 5.4, 6.4; 7.8, 8.8; 63, 55; 2000 tokens 11.7, 11.9.
  const long long rows = static_cast<long long>(a.t.tokens) * (2 * a.c.heads + (a.q ? a.q_heads : 0)) / kTeams;
  const int turns = rows > 16384 ? 4 : 1;
  const int heads = turns * kTeams;  // of a warp
  const int q_warps = a.q ? (a.q_heads + heads - 1) / heads : 0, kv_warps = a.k ? (a.c.heads + heads - 1) / heads : 0;
  const long long warps = static_cast<long long>(a.t.tokens) * (q_warps + 2 * kv_warps);
  const long long ctas = (warps + kKv4Threads / 32 - 1) / (kKv4Threads / 32);
  if (ctas > INT32_MAX) return cudaErrorInvalidConfiguration;
  return launch_overlapped(kv4_append_kernel<T, DIM, HOW>, dim3(static_cast<unsigned>(ctas)), kKv4Threads, 0, stream, a, q_warps,
                           kv_warps, turns);
}

template <typename T, int DIM>
cudaError_t launch_append4_dim(const AppendArgs& a, cudaStream_t stream) {
  // vectors of eight elements: every row, angle and weight address 16-byte aligned
  const bool turned = a.cos != nullptr, simple = !turned || (!a.interleaved && a.rotary == DIM);
  bool vec = !turned || a.interleaved || a.rotary % 16 == 0;
  if (turned && simple) vec = vec && a.rope_stride % 4 == 0 && aligned_to(a.cos, 16) && aligned_to(a.sin, 16);
  constexpr int kElements = 16 / sizeof(T);
  const void* ptr[3] = {a.k, a.v, a.q};
  const long long stride[6] = {a.k_ts, a.k_hs, a.v_ts, a.v_hs, a.q_ts, a.q_hs};
  for (int i = 0; i < 3; ++i)
    if (ptr[i] && (!aligned_to(ptr[i], 16) || stride[2 * i] % kElements || stride[2 * i + 1] % kElements)) vec = false;
  if (a.q && (!aligned_to(a.q_out, 16) || a.o_ts % 8 || a.o_hs % 8)) vec = false;
  for (const RowNorm& n : {a.q_norm, a.k_norm})
    if (!aligned_to(n.weight, 16)) vec = false;
  if (!vec) return launch_append4_as<T, DIM, kSingle>(a, stream);
  return simple ? launch_append4_as<T, DIM, kSimple>(a, stream) : launch_append4_as<T, DIM, kVector>(a, stream);
}

// a.k null: the queries alone (for caches of any kind, head dimensions as here).
bool kv4_rows_take(int dim) { return dim == 64 || dim == 128 || dim == 256; }

cudaError_t launch_kv4_append(bool bf16, const AppendArgs& a, cudaStream_t stream) {
  switch (a.c.dim) {
    case 64: return bf16 ? launch_append4_dim<__nv_bfloat16, 64>(a, stream) : launch_append4_dim<float, 64>(a, stream);
    case 128: return bf16 ? launch_append4_dim<__nv_bfloat16, 128>(a, stream) : launch_append4_dim<float, 128>(a, stream);
    default: return bf16 ? launch_append4_dim<__nv_bfloat16, 256>(a, stream) : launch_append4_dim<float, 256>(a, stream);
  }
}

cudaError_t launch_kv4_decode(const KvView& c, const int32_t* pages, int count, uint16_t* k_out, uint16_t* v_out,
                              cudaStream_t stream) {
  const unsigned blocks = static_cast<unsigned>(count) * static_cast<unsigned>(c.heads);  // (their output has to fit the memory)
  const unsigned long long items = static_cast<unsigned long long>(blocks) * (c.page_size / 2) * (c.dim / 32);
  const dim3 grid(static_cast<unsigned>(std::min(items / 256 + 1, 1ull << 20)), 2);
  return launch_overlapped(c.dim == 64 ? kv4_decode_kernel<64> : c.dim == 128 ? kv4_decode_kernel<128> : kv4_decode_kernel<256>,
                           grid, 256, 0, stream, c, pages, blocks, k_out, v_out);
}

}  // namespace se12
