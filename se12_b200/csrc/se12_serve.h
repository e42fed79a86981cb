// Host/device parameter blocks of the decode-step operators around the GEMVs:
// the paged 8-bit key/value cache (se12_kv.cu), attention over it
// (se12_attend.cu) and token log probabilities (se12_logprobs.cu). Not part
// of the public interface (include/se12.h is).
#pragma once

#include <cstddef>
#include <cstdint>
#include <cuda.h>
#include <cuda_runtime.h>

#include "se12_worklist.h"

namespace se12 {

// Cache element kinds (SE12_KV_INT8, SE12_KV_E4M3).
constexpr int kKvInt8 = 0;
constexpr int kKvE4m3 = 1;

// One layer's cache on the device. A block is one page of one KV head:
// codes [pages][heads][page_size][dim], one fp32 scale per block.
struct KvView {
  uint8_t* k_codes;
  uint8_t* v_codes;
  float* k_scales;  // [pages][heads]
  float* v_scales;
  int pages, page_size, page_shift;
  int heads, dim;
  int kind;
};

// New tokens of a ragged batch. Sequence b's tokens are rows
// start(b) .. start(b + 1) - 1, at positions lens[b] - count .. lens[b] - 1.
struct TokenBatch {
  const int32_t* query_start;  // [seqs + 1], or null: one token per sequence
  const int32_t* lens;         // [seqs] tokens in the cache, the new ones included
  const int32_t* table;        // page ids, row b at table + b * table_stride
  long long table_stride;
  int max_pages;
  int seqs, tokens;

#if defined(__CUDACC__)
  // Sequence b's first row, and its rows and tokens; z.capacity is max_pages pages.
  __device__ __forceinline__ int begin_of(int b, const ListSizes& z) const {
    return first_row(query_start ? query_start[b] : b, z);
  }
  __device__ __forceinline__ SeqRows rows_of(int b, const ListSizes& z) const {
    return sequence_rows(query_start ? query_start[b] : b, query_start ? query_start[b + 1] : b + 1, lens[b], z);
  }
#endif
};

struct AppendArgs {
  KvView c;
  TokenBatch t;
  const void *q, *k, *v;  // fp32 or BF16; q may be null
  long long q_ts, q_hs, k_ts, k_hs, v_ts, v_hs;  // token and head strides, elements
  int q_heads;
  const float *cos, *sin;  // row p at p * rope_stride, or null: no rotation
  long long rope_stride;
  int rope_rows, rotary;   // rotated dimensions (even, <= dim)
  int interleaved;
  uint16_t* q_out;         // BF16
  long long o_ts, o_hs;
};

struct AttendArgs {
  KvView c;
  TokenBatch t;
  const uint16_t* q;  // BF16
  long long q_ts, q_hs;
  int q_vec;          // q rows are 16-byte aligned
  uint16_t* out;      // BF16
  long long o_ts, o_hs;
  int o_vec;          // and the output's
  int q_heads, group;
  float scale;        // of the logits
  float softcap;      // 0: none
  int window;         // 0: none
  float* partials;
  int* counters;
};

struct LogprobArgs {
  const void* logits;  // fp32 or BF16 [rows][ld]
  long long ld;
  int rows, vocab;
  const long long* tokens;
  int top;
  float softcap;
  float* logprob;
  float* entropy;
  long long* top_ids;
  float* top_logprobs;
  int vec;             // every row is 16-byte aligned
  int chunks_per_row;  // batches of a row
  int units_per_cta;
  unsigned char* partials;
  int* counters;
};

cudaError_t launch_kv_append(bool bf16, const AppendArgs& a, cudaStream_t stream);
cudaError_t launch_kv_decode(const KvView& c, const int32_t* pages, int count, uint16_t* k_out, uint16_t* v_out,
                             cudaStream_t stream);
cudaError_t launch_kv_attend(const CUtensorMap& kmap, const CUtensorMap& vmap, const AttendArgs& a, int max_query,
                             int sm_count, cudaStream_t stream);
size_t kv_attend_partial_bytes(int sm_count, bool tile);
bool kv_attend_takes_tiles(int max_query, int group, int dim);
cudaError_t launch_attend_tile(const AttendArgs& a, int sm_count, cudaStream_t stream);
size_t kv_attend_tile_partial_bytes(int sm_count);
cudaError_t launch_token_logprobs(bool bf16, LogprobArgs a, int sm_count, cudaStream_t stream);
size_t logprob_partial_bytes(int sm_count);

// A launch whose prologue may overlap the previous kernel's tail: the kernel
// waits (griddepcontrol.wait) before it touches memory other kernels write.
template <typename... Params, typename... Args>
inline cudaError_t launch_overlapped(void (*kernel)(Params...), dim3 grid, int threads, size_t smem, cudaStream_t stream,
                                     Args&&... args) {
  if (smem > 48 * 1024) {
    const cudaError_t err =
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (err != cudaSuccess) return err;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<Params>(args)...);
}

}  // namespace se12
