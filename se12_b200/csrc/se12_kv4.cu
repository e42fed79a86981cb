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
// Both kernels are bound by memory and, for few tokens, by their latency.
#include "se12_kv.cuh"

#include <cuda_fp16.h>

namespace se12 {

constexpr int kKv4Group = 64;
constexpr int kKv4MinExponent = -30;
constexpr float kKv4KeyLimit = 65000.f;         // larger keys do not fit FP16's scale and offset
constexpr float kKv4ValueLimit = 17179869184.f;  // 2^34: E is at most 30
constexpr int kKv4Threads = 128;

// How a head's row is spread over its team of DIM / 8 lanes. In order: lane l
// has the dimensions 4 l .. 4 l + 3 and DIM / 2 + 4 l .. + 3. Read: the members
// of the pairs 4 l .. 4 l + 3 that are turned together, which are the same
// dimensions unless part of the row is turned in halves.
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

// A lane's part of a row.
struct RowOf8 {
  float a[4], b[4];
};

// The cosines and sines that a lane needs at one position.
struct Angles {
  float c[4], s[4];
};

// VEC: every vector of four elements (and the angles' vectors) is aligned, and
// halves are multiples of four.
template <int DIM, bool VEC>
__device__ __forceinline__ void load_angles(Angles& t, const AppendArgs& a, const RowOrder& o, int pos, int l) {
#pragma unroll
  for (int j = 0; j < 4; ++j) t.c[j] = 1.f, t.s[j] = 0.f;
  if (o.mode == 0) return;
  const float* cos = a.cos + pos * a.rope_stride;
  const float* sin = a.sin + pos * a.rope_stride;
  if (o.mode == 1) {  // pairs 4 l .. 4 l + 3
    if (VEC) {
      if (4 * l < o.turned) {
        load_vector<4>(t.c, cos + 4 * l);
        load_vector<4>(t.s, sin + 4 * l);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (4 * l + j < o.turned) t.c[j] = cos[4 * l + j], t.s[j] = sin[4 * l + j];
    }
  } else {  // neighbours: two pairs in each of the lane's vectors
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int p = (j < 2 ? 2 * l : DIM / 4 + 2 * l - 2) + j;
      if (p < o.turned) t.c[j] = cos[p], t.s[j] = sin[p];
    }
  }
}

template <int DIM, bool VEC, typename T>
__device__ __forceinline__ void load_row(RowOf8& r, const T* row, const RowOrder& o, int l) {
  if (VEC) {
    int ia = 4 * l, ib = DIM / 2 + 4 * l;
    if (o.apart) {
      ia = 4 * l < o.half ? 4 * l : 8 * l;
      ib = 4 * l < o.half ? 4 * l + o.half : 8 * l + 4;
    }
    load_vector<4>(r.a, row + ia);
    load_vector<4>(r.b, row + ib);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      int ia = 4 * l + j, ib = DIM / 2 + 4 * l + j;
      if (o.apart) o.at(4 * l + j, ia, ib);
      r.a[j] = load_value(row + ia);
      r.b[j] = load_value(row + ib);
    }
  }
}

template <int DIM, bool VEC>
__device__ __forceinline__ void load_weight_row(RowOf8& w, const RowNorm& norm, const RowOrder& o, int l) {
  if (norm.bf16)
    load_row<DIM, VEC>(w, static_cast<const __nv_bfloat16*>(norm.weight), o, l);
  else
    load_row<DIM, VEC>(w, static_cast<const float*>(norm.weight), o, l);
}

template <int DIM>
__device__ __forceinline__ void normalise_row(RowOf8& r, const RowOf8& w, double eps) {
  const float f = norm_factor(team_sum(add_squares<4>(r.b, add_squares<4>(r.a, 0.0)), DIM / 8), DIM, eps);
  apply_norm<4>(r.a, f, w.a);
  apply_norm<4>(r.b, f, w.b);
}

__device__ __forceinline__ void rotate_row(RowOf8& r, const Angles& t, const RowOrder& o, int l, int quarter) {
  if (o.mode == 1) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (4 * l + j < o.turned) turn(r.a[j], r.b[j], t.c[j], t.s[j]);
  } else if (o.mode == 2) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      if (2 * l + j < o.turned) turn(r.a[2 * j], r.a[2 * j + 1], t.c[j], t.s[j]);
      if (quarter + 2 * l + j < o.turned) turn(r.b[2 * j], r.b[2 * j + 1], t.c[2 + j], t.s[2 + j]);
    }
  }
}

// A row read apart put in order, through the team's row of shared memory.
template <int DIM, bool VEC>
__device__ __forceinline__ void reorder_row(RowOf8& r, float* staged, const RowOrder& o, int l) {
  __syncwarp();
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    int ia, ib;
    if (VEC) {
      ia = (4 * l < o.half ? 4 * l : 8 * l) + j;
      ib = (4 * l < o.half ? 4 * l + o.half : 8 * l + 4) + j;
    } else {
      o.at(4 * l + j, ia, ib);
    }
    staged[ia] = r.a[j];
    staged[ib] = r.b[j];
  }
  __syncwarp();
  load_vector<4>(r.a, staged + 4 * l);
  load_vector<4>(r.b, staged + DIM / 2 + 4 * l);
}

// A group's scale and offset, and the codes of a lane's four values in 16 bits.
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

  __device__ __forceinline__ uint32_t codes(const float (&x)[4]) const {
    uint32_t w = 0;
#pragma unroll
    for (int j = 3; j >= 0; --j) {
      // rounded to a whole number by an addend of 1.5 2^23 (and 8, the zero point): the code is in the last bits
      const float u = fminf(fmaxf(__fmul_rn(__fsub_rn(x[j], middle), inverse), -8.f), 7.f);  // (NaN: -8)
      w = w * 16 + __float_as_uint(__fadd_rn(u, 12582920.f));
    }
    return w & 0xFFFFu;
  }
};

// A lane's row quantised and stored as token `slot` of a block. All lanes of
// the warp take part; where `live` is false nothing is stored. (Keys and values
// by one piece of code: two, unrolled over four rows, were waiting for
// instructions most of the time, 13 prompt chunks 387 us.)
template <int DIM>
__device__ __forceinline__ void store_row(const AppendArgs& a, bool keys, RowOf8& r, long long block, int slot, int l, bool live) {
  constexpr int G = DIM / kKv4Group;
  constexpr int kSpan = DIM >= 128 ? 16 : 8;  // lanes of a group
  float lo_a = min_nan(min_nan(r.a[0], r.a[1]), min_nan(r.a[2], r.a[3])), hi_a = max_nan(max_nan(r.a[0], r.a[1]), max_nan(r.a[2], r.a[3]));
  float lo_b = min_nan(min_nan(r.b[0], r.b[1]), min_nan(r.b[2], r.b[3])), hi_b = max_nan(max_nan(r.b[0], r.b[1]), max_nan(r.b[2], r.b[3]));
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
    if (DIM == 256) amax = max_nan(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, 16));
    const bool fits = amax < kKv4ValueLimit;  // (otherwise, NaN too, the token is NaN through E alone: its line is 0)
    const int e = fits ? max(static_cast<int>(__float_as_uint(amax) >> 23) - 130, kKv4MinExponent) : 0;
    exponent = fits ? static_cast<float>(e) : __uint_as_float(0x7FC00000u);
    const float down = __uint_as_float(static_cast<unsigned>(127 - e) << 23);
    auto scaled = [&](float x) { return fits ? x * down : 0.f; };
    lo_a = scaled(lo_a), hi_a = scaled(hi_a), lo_b = scaled(lo_b), hi_b = scaled(hi_b);
#pragma unroll
    for (int j = 0; j < 4; ++j) r.a[j] = scaled(r.a[j]), r.b[j] = scaled(r.b[j]);
  }
  GroupLine ga, gb;
  ga.fit(lo_a, hi_a);
  gb.fit(lo_b, hi_b);
  // Words of 8 codes: an even lane completes the first vector's, an odd one the second's.
  const uint32_t wa = ga.codes(r.a), wb = gb.codes(r.b);
  const uint32_t other = __shfl_xor_sync(0xFFFFFFFFu, l & 1 ? wa : wb, 1);
  const uint32_t word = l & 1 ? other | (wb << 16) : wa | (other << 16);
  if (!live) return;
  const int n = (l & 1 ? DIM / 16 : 0) + l / 2;  // the word in the row's order
  const long long row = block * a.c.page_size + slot;
  reinterpret_cast<uint32_t*>((keys ? a.c.k_codes : a.c.v_codes) + row * (DIM / 2))[(n & 7) * G + (n >> 3)] = word;
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
    // lane k of a span: scale, offset of ga, of gb; lane 4 of the row: E
    const int at = ((slot & 15) >> 1) * (4 * G) + (slot & 1);
    const __half x = k == 0 ? ga.scale : k == 1 ? ga.offset : k == 2 ? gb.scale : gb.offset;
    if (k < (DIM >= 128 ? 4 : 2)) cell[at + 2 * ((k & 1 ? G : 0) + (k < 2 ? h : G / 2 + h))] = x;
    if (l == 4) cell[32 * G + (slot & 15)] = __float2half_rn(exponent);
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

// A warp takes a token's queries, keys or values, 32 / (DIM / 8) heads side by
// side and up to `turns` of those one after the other, the next on its way.
// `q_warps` and `kv_warps`: warps per token for its queries, and for its keys and
// for its values.
template <typename T, int DIM, bool VEC>
__global__ void __launch_bounds__(kKv4Threads) kv4_append_kernel(const AppendArgs a, const int q_warps, const int kv_warps,
                                                                 const int turns) {
  constexpr int kTeam = DIM / 8, kTeams = 32 / kTeam;
  __shared__ float4 staged[kKv4Threads / 32][kTeams][DIM / 4];
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
  RowOf8 next;
  load_row<DIM, VEC>(next, src + min(head0 + team, heads - 1) * hs, order, l);

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
  Angles angles;
  load_angles<DIM, VEC>(angles, a, order, pos, l);
  const RowNorm norm = queries ? a.q_norm : keys ? a.k_norm : RowNorm{};
  RowOf8 weight;
  if (norm.weight) load_weight_row<DIM, VEC>(weight, norm, order, l);
  const int slot = pos & (a.c.page_size - 1);
#pragma unroll 1
  for (int first = head0; first < end; first += kTeams) {
    const int head = first + team;
    const bool live = head < end;
    RowOf8 row = next;
    if (first + kTeams < end) load_row<DIM, VEC>(next, src + min(head + kTeams, heads - 1) * hs, order, l);
    if (norm.weight) normalise_row<DIM>(row, weight, a.norm_eps);
    rotate_row(row, angles, order, l, DIM / 4);
    if (order.apart) reorder_row<DIM, VEC>(row, reinterpret_cast<float*>(staged[warp][team]), order, l);
    if (!queries) {
      store_row<DIM>(a, keys, row, static_cast<long long>(page) * a.c.heads + head, slot, l, live);
    } else if (live) {
      uint16_t* to = out + head * a.o_hs;
      if (VEC) {
        store_bf16<4>(to + 4 * l, row.a);
        store_bf16<4>(to + DIM / 2 + 4 * l, row.b);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          to[4 * l + j] = __bfloat16_as_ushort(__float2bfloat16_rn(row.a[j]));
          to[DIM / 2 + 4 * l + j] = __bfloat16_as_ushort(__float2bfloat16_rn(row.b[j]));
        }
      }
    }
  }
}

// Pages read back as BF16, a CTA per block (page of a head), keys and values by
// blockIdx.y, a thread per word of 8 values.
template <int DIM>
__global__ void __launch_bounds__(256) kv4_decode_kernel(const KvView c, const int32_t* pages, int count, uint16_t* k_out,
                                                         uint16_t* v_out) {
  constexpr int G = DIM / kKv4Group, kWords = DIM / 8;
  grid_launch_dependents();
  grid_dependency_wait();
  const bool keys = blockIdx.y == 0;
  const long long blocks = static_cast<long long>(count) * c.heads;
  const int words = c.page_size * kWords;
  for (long long n = blockIdx.x; n < blocks; n += gridDim.x) {
    const int nth = static_cast<int>(n / c.heads), head = static_cast<int>(n - static_cast<long long>(nth) * c.heads);
    const int page = pages ? pages[nth] : nth;
    uint4* out = reinterpret_cast<uint4*>((keys ? k_out : v_out) + n * (static_cast<long long>(c.page_size) * DIM));
    if (page < 0 || page >= c.pages) {
      raise_status(kStatusBadArgument);
      for (int i = threadIdx.x; i < words; i += 256) out[i] = make_uint4(0, 0, 0, 0);
      continue;
    }
    const long long block = static_cast<long long>(page) * c.heads + head;
    const uint32_t* codes = reinterpret_cast<const uint32_t*>((keys ? c.k_codes : c.v_codes) + block * c.page_size * (DIM / 2));
    const __half2* key_scales = reinterpret_cast<const __half2*>(c.k_scales) + block * c.page_size * G;
    const __half* value_scales = reinterpret_cast<const __half*>(c.v_scales) + block * (c.page_size >> 4) * (32 * G + 16);
#pragma unroll 4
    for (int i = threadIdx.x; i < words; i += 256) {
      const int token = i / kWords, w = i % kWords, g = w / 8;
      const uint32_t u = codes[token * kWords + (w & 7) * G + g];
      float scale, offset, power = 1.f;
      if (keys) {
        const float2 line = __half22float2(key_scales[token * G + g]);
        scale = line.x, offset = line.y;
      } else {
        const __half* cell = value_scales + (token >> 4) * (32 * G + 16);
        const __half* pair = cell + ((token & 15) >> 1) * (4 * G) + (token & 1);
        scale = __half2float(pair[2 * g]);
        offset = __half2float(pair[2 * (G + g)]);
        const float e = __half2float(cell[32 * G + (token & 15)]);  // a whole number, or NaN
        power = e == e ? __uint_as_float(static_cast<unsigned>(static_cast<int>(e) + 127) << 23) : e;
      }
      uint32_t o[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float x[2];
#pragma unroll
        for (int k = 0; k < 2; ++k)
          x[k] = fmaf(static_cast<float>(static_cast<int>((u >> (8 * j + 4 * k)) & 15u) - 8), scale, offset) * power;
        o[j] = __bfloat16_as_ushort(__float2bfloat16_rn(x[0])) |
               (static_cast<uint32_t>(__bfloat16_as_ushort(__float2bfloat16_rn(x[1]))) << 16);
      }
      out[i] = make_uint4(o[0], o[1], o[2], o[3]);
    }
  }
}

// ------------------------------------------------------------------ launches

template <typename T, int DIM, bool VEC>
cudaError_t launch_append4_as(const AppendArgs& a, cudaStream_t stream) {
  constexpr int kTeams = 32 / (DIM / 8);
  // Few rows: one after the other in as many warps; many: up to 8 in one, which
  // finds the token's place and angles once for them.
  const long long rows = static_cast<long long>(a.t.tokens) * (2 * a.c.heads + (a.q ? a.q_heads : 0)) / kTeams;
  const int turns = rows > 16384 ? 8 : 1;
  const int heads = turns * kTeams;  // of a warp
  const int q_warps = a.q ? (a.q_heads + heads - 1) / heads : 0, kv_warps = (a.c.heads + heads - 1) / heads;
  const long long warps = static_cast<long long>(a.t.tokens) * (q_warps + 2 * kv_warps);
  const long long ctas = (warps + kKv4Threads / 32 - 1) / (kKv4Threads / 32);
  if (ctas > INT32_MAX) return cudaErrorInvalidConfiguration;
  return launch_overlapped(kv4_append_kernel<T, DIM, VEC>, dim3(static_cast<unsigned>(ctas)), kKv4Threads, 0, stream, a, q_warps,
                           kv_warps, turns);
}

template <typename T, int DIM>
cudaError_t launch_append4_dim(const AppendArgs& a, cudaStream_t stream) {
  // vectors of four elements: every row, angle and weight address a multiple of four of its elements
  bool vec = !a.cos || (a.rotary % 8 == 0 && a.rope_stride % 4 == 0 && reinterpret_cast<uintptr_t>(a.cos) % 16 == 0 &&
                        reinterpret_cast<uintptr_t>(a.sin) % 16 == 0);
  const void* ptr[3] = {a.k, a.v, a.q};
  const long long stride[6] = {a.k_ts, a.k_hs, a.v_ts, a.v_hs, a.q_ts, a.q_hs};
  for (int i = 0; i < 3; ++i)
    if (ptr[i] && (reinterpret_cast<uintptr_t>(ptr[i]) % (4 * sizeof(T)) || stride[2 * i] % 4 || stride[2 * i + 1] % 4)) vec = false;
  if (a.q && (reinterpret_cast<uintptr_t>(a.q_out) % 8 || a.o_ts % 4 || a.o_hs % 4)) vec = false;
  for (const RowNorm& n : {a.q_norm, a.k_norm})
    if (reinterpret_cast<uintptr_t>(n.weight) % (n.bf16 ? 8 : 16)) vec = false;
  return vec ? launch_append4_as<T, DIM, true>(a, stream) : launch_append4_as<T, DIM, false>(a, stream);
}

cudaError_t launch_kv4_append(bool bf16, const AppendArgs& a, cudaStream_t stream) {
  switch (a.c.dim) {
    case 64: return bf16 ? launch_append4_dim<__nv_bfloat16, 64>(a, stream) : launch_append4_dim<float, 64>(a, stream);
    case 128: return bf16 ? launch_append4_dim<__nv_bfloat16, 128>(a, stream) : launch_append4_dim<float, 128>(a, stream);
    default: return bf16 ? launch_append4_dim<__nv_bfloat16, 256>(a, stream) : launch_append4_dim<float, 256>(a, stream);
  }
}

cudaError_t launch_kv4_decode(const KvView& c, const int32_t* pages, int count, uint16_t* k_out, uint16_t* v_out,
                              cudaStream_t stream) {
  const long long blocks = static_cast<long long>(count) * c.heads;
  const dim3 grid(static_cast<unsigned>(blocks < (1 << 20) ? blocks : (1 << 20)), 2);
  return launch_overlapped(c.dim == 64 ? kv4_decode_kernel<64> : c.dim == 128 ? kv4_decode_kernel<128> : kv4_decode_kernel<256>,
                           grid, 256, 0, stream, c, pages, count, k_out, v_out);
}

}  // namespace se12
