// What the kernels that append to the paged caches share: reading rows of
// queries, keys and values, their norms and the position rotation.
#pragma once

#include "se12_device.cuh"
#include "se12_serve.h"

#include <cuda_bf16.h>

namespace se12 {

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

// (a, b) turned by the angle whose cosine and sine are c and s; each product
// and each sum is rounded by itself, as elementary tensor operations do.
__device__ __forceinline__ void turn(float& a, float& b, float c, float s) {
  const float x = __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s));
  b = __fadd_rn(__fmul_rn(b, c), __fmul_rn(a, s));
  a = x;
}

template <int VP>
__device__ __forceinline__ unsigned magnitude_bits(const float (&x)[VP], unsigned m) {
#pragma unroll
  for (int j = 0; j < VP; ++j) m = max(m, __float_as_uint(x[j]) & 0x7FFFFFFFu);
  return m;
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

// VP weights of a norm from index `at` on.
template <int VP>
__device__ __forceinline__ void load_weights(float (&w)[VP], const RowNorm& n, int at) {
  if (n.bf16)
    load_vector<VP>(w, static_cast<const __nv_bfloat16*>(n.weight) + at);
  else
    load_vector<VP>(w, static_cast<const float*>(n.weight) + at);
}

// Squares are summed in 64 bits, so that the factor is the correctly rounded
// one in all but one row in 10^7 whatever the order of the sum: codes next to a
// rounding border are then those of the formula.
template <int VP>
__device__ __forceinline__ double add_squares(const float (&x)[VP], double sum) {
#pragma unroll
  for (int j = 0; j < VP; ++j) sum = fma(static_cast<double>(x[j]), static_cast<double>(x[j]), sum);
  return sum;
}

// What a row whose squares sum to `sum` is multiplied by.
__device__ __forceinline__ float norm_factor(double sum, int dim, double eps) {
  return static_cast<float>(rsqrt(sum / dim + eps));
}

template <int VP>
__device__ __forceinline__ void apply_norm(float (&x)[VP], float factor, const float (&w)[VP]) {
#pragma unroll
  for (int j = 0; j < VP; ++j) x[j] = __fmul_rn(__fmul_rn(x[j], factor), w[j]);
}

// The sum over the `lanes` (a power of two) neighbouring lanes of each team.
__device__ __forceinline__ double team_sum(double x, int lanes) {
  for (int d = 1; d < lanes; d <<= 1) x += __shfl_xor_sync(0xFFFFFFFFu, x, d);
  return x;
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

}  // namespace se12
