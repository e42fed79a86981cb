// What the two attention kernels share: codes as FP16, the softmax's
// references and the work list's sums on the device.
#pragma once

#include "se12_device.cuh"
#include "se12_serve.h"

#include <cuda_fp16.h>

namespace se12 {

constexpr float kAttendStart = -1.0e30f; // both references before the first token
constexpr float kAttendRaise = 8.f;      // weights up to 2^8 of the reference
constexpr float kAttendRaiseSum = 30.f;

__device__ __forceinline__ uint32_t half2_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }

// Four codes (bytes) as two FP16 pairs, bytes (0, 1) and (2, 3).
// int8: byte ^ 0x80 is code + 128; as the low byte of 0x6400 it makes the
// FP16 number 1024 + code + 128, from which 1152 is taken exactly.
template <int KIND>
__device__ __forceinline__ void widen(uint32_t codes, uint32_t& lo, uint32_t& hi) {
  if constexpr (KIND == kKvInt8) {
    const uint32_t u = codes ^ 0x80808080u;
    const uint32_t bias = 0x64806480u;
    asm("sub.f16x2 %0, %1, %2;" : "=r"(lo) : "r"(prmt(u, 0x64646464u, 0x4140u)), "r"(bias));
    asm("sub.f16x2 %0, %1, %2;" : "=r"(hi) : "r"(prmt(u, 0x64646464u, 0x4342u)), "r"(bias));
  } else {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(codes));
  }
}

__device__ __forceinline__ ListSizes list_sizes(const AttendArgs& a) {
  return {a.t.tokens, a.t.max_pages << a.c.page_shift, a.group, a.window};
}

// A sequence longer than its page table row: the tokens past it are skipped.
__device__ __forceinline__ void check_length(const AttendArgs& a, int b) {
  if (blockIdx.x == 0 && a.t.lens[b] > a.t.max_pages << a.c.page_shift) raise_status(kStatusBadArgument);
}

// Sums over the sequences, in place, by one warp: sums[i] of entries 1 .. i,
// at most `limit`.
__device__ __forceinline__ void sum_up_to(int* sums, int seqs, int limit, int lane) {
  int carry = 0;
  for (int i = 1; i <= seqs; i += 32) {
    int v = i + lane <= seqs ? sums[i + lane] : 0;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int u = __shfl_up_sync(0xFFFFFFFFu, v, d);
      if (lane >= d) v = add_work(v, u, limit);
    }
    v = add_work(v, carry, limit);
    if (i + lane <= seqs) sums[i + lane] = v;
    carry = __shfl_sync(0xFFFFFFFFu, v, 31);
  }
}

}  // namespace se12
