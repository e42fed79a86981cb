// C-ABI layer of the decode-step operators around the GEMVs: the paged 8-bit
// key/value cache, attention over it and token log probabilities (argument
// checks, TMA descriptors, launches). See include/se12.h.
#include "se12_serve.h"

#include <atomic>

struct se12_kv_cache {
  se12::KvView view;
  alignas(64) CUtensorMap k_map;
  alignas(64) CUtensorMap v_map;
  int sm_count;
};

namespace {

// A launch has at most kAttendMaxCtas CTAs per SM, each with a counter.
constexpr int kMaxSms = 160;
static_assert(kMaxSms * se12::kAttendMaxCtas * sizeof(int) <= SE12_COUNTER_BYTES, "the counters of a launch");

// Codes as [pages * heads * page_size rows][dim bytes], one box = 16 tokens x
// 128 bytes (a page is a multiple of 16 tokens, so a box never leaves it;
// columns past dim read as zero codes, which stand for zero).
int encode_kv_map(CUtensorMap* map, const void* codes, const se12::KvView& v) {
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(v.dim),
                              static_cast<cuuint64_t>(v.pages) * v.heads * v.page_size};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(v.dim)};
  const cuuint32_t box[2] = {128, 16};
  return encode_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, codes, dims, strides, box);
}

// SMs of the current device, at most kMaxSms; asked once per device.
int device_sm_count(int* sm_count) {
  constexpr int kDevices = 64;
  static std::atomic<int> known[kDevices];
  int device = 0;
  const cudaError_t err = cudaGetDevice(&device);
  if (err != cudaSuccess) return cuda_fail(err, "cudaGetDevice");
  if (device < kDevices && (*sm_count = known[device].load(std::memory_order_relaxed)) > 0) return SE12_OK;
  const int st = current_device_info(&device, sm_count);
  if (st != SE12_OK) return st;
  *sm_count = std::min(*sm_count, kMaxSms);
  if (device < kDevices) known[device].store(*sm_count, std::memory_order_relaxed);
  return SE12_OK;
}

int check_batch(const se12_kv_cache* cache, const se12_kv_batch* b, se12::TokenBatch* out) {
  if (!cache || !b) return fail(SE12_ERR_INVALID_ARGUMENT, "null argument");
  if (b->seqs < 1 || b->seqs > SE12_KV_MAX_SEQS)
    return fail(SE12_ERR_INVALID_ARGUMENT, "seqs must be in 1.." + std::to_string(SE12_KV_MAX_SEQS));
  if (b->tokens < 1) return fail(SE12_ERR_INVALID_ARGUMENT, "tokens must be positive");
  if (!b->query_start && b->tokens != b->seqs)
    return fail(SE12_ERR_INVALID_ARGUMENT, "without query_start there is one token per sequence");
  if (!b->lens || !b->block_table) return fail(SE12_ERR_INVALID_ARGUMENT, "null lens or block_table");
  if (b->max_pages < 1 || b->table_stride < 0)
    return fail(SE12_ERR_INVALID_ARGUMENT, "block_table needs a column, and a table_stride that is not negative");
  if (static_cast<long long>(b->max_pages) * cache->view.page_size > se12::kMaxPositions)
    return fail(SE12_ERR_INVALID_ARGUMENT, "positions must fit 31 bits");
  out->query_start = b->query_start;
  out->lens = b->lens;
  out->table = b->block_table;
  out->table_stride = b->table_stride;
  out->max_pages = b->max_pages;
  out->seqs = b->seqs;
  out->tokens = b->tokens;
  return SE12_OK;
}

// A cap below 1e-30 as 1e-30: its reciprocal stays finite, and either way the
// logits differ by nothing that an exponential shows.
float usable_cap(float softcap) { return softcap > 0.f && softcap < 1e-30f ? 1e-30f : softcap; }

}  // namespace

extern "C" {

int se12_kv_cache_create(const se12_kv_pages* p, se12_kv_cache** out) {
  if (!p || !out) return fail(SE12_ERR_INVALID_ARGUMENT, "null argument");
  *out = nullptr;
  if (p->pages < 1 || p->kv_heads < 1) return fail(SE12_ERR_INVALID_ARGUMENT, "pages and kv_heads must be positive");
  if (p->page_size < 16 || p->page_size > 256 || (p->page_size & (p->page_size - 1)))
    return fail(SE12_ERR_INVALID_ARGUMENT, "page_size must be 16, 32, 64, 128 or 256, got " + std::to_string(p->page_size));
  if (p->head_dim < 16 || p->head_dim > 256 || p->head_dim % 16)
    return fail(SE12_ERR_INVALID_ARGUMENT, "head_dim must be a multiple of 16 up to 256, got " + std::to_string(p->head_dim));
  if (p->kind != SE12_KV_INT8 && p->kind != SE12_KV_E4M3)
    return fail(SE12_ERR_UNSUPPORTED_FORMAT, "kind must be SE12_KV_INT8 or SE12_KV_E4M3");
  if (static_cast<long long>(p->pages) * p->kv_heads * p->page_size > INT32_MAX)
    return fail(SE12_ERR_INVALID_ARGUMENT, "pages * kv_heads * page_size must fit 31 bits");
  if (!p->k_codes || !p->v_codes || !p->k_scales || !p->v_scales)
    return fail(SE12_ERR_INVALID_ARGUMENT, "null cache pointer");
  if (!aligned16(p->k_codes) || !aligned16(p->v_codes))
    return fail(SE12_ERR_MISALIGNED, "cache codes must be 16-byte aligned");
  int device = 0, sm_count = 0;
  int st = current_device_info(&device, &sm_count);
  if (st != SE12_OK) return st;
  se12_kv_cache* c = new se12_kv_cache();
  se12::KvView& v = c->view;
  v.k_codes = static_cast<uint8_t*>(p->k_codes);
  v.v_codes = static_cast<uint8_t*>(p->v_codes);
  v.k_scales = p->k_scales;
  v.v_scales = p->v_scales;
  v.pages = p->pages;
  v.page_size = p->page_size;
  v.page_shift = 0;
  while ((1 << v.page_shift) < p->page_size) ++v.page_shift;
  v.heads = p->kv_heads;
  v.dim = p->head_dim;
  v.kind = p->kind;
  c->sm_count = std::min(sm_count, kMaxSms);
  st = encode_kv_map(&c->k_map, p->k_codes, v);
  if (st == SE12_OK) st = encode_kv_map(&c->v_map, p->v_codes, v);
  if (st != SE12_OK) {
    delete c;
    return st;
  }
  *out = c;
  return SE12_OK;
}

void se12_kv_cache_destroy(se12_kv_cache* c) { delete c; }

int se12_kv_append(const se12_kv_cache* cache, const se12_kv_batch* batch, const se12_kv_append_args* p, void* stream) {
  se12::AppendArgs a{};
  const int st = check_batch(cache, batch, &a.t);
  if (st != SE12_OK) return st;
  if (!p || !p->k || !p->v) return fail(SE12_ERR_INVALID_ARGUMENT, "null keys or values");
  if (p->q && (!p->q_out || p->q_heads < 1)) return fail(SE12_ERR_INVALID_ARGUMENT, "queries need q_out and q_heads");
  if (static_cast<long long>(batch->seqs) * (p->q ? p->q_heads : 0) > INT32_MAX)
    return fail(SE12_ERR_INVALID_ARGUMENT, "too many query heads");
  if (!p->cos != !p->sin) return fail(SE12_ERR_INVALID_ARGUMENT, "cos and sin go together");
  if (p->cos && (p->rotary_dim < 2 || p->rotary_dim % 2 || p->rotary_dim > cache->view.dim))
    return fail(SE12_ERR_INVALID_ARGUMENT, "rotary_dim must be even, in 2..head_dim");
  if (p->cos && (p->rope_rows < 1 || p->rope_stride < 0))
    return fail(SE12_ERR_INVALID_ARGUMENT, "the rotation table needs a row, and a rope_stride that is not negative");
  a.c = cache->view;
  a.q = p->q;
  a.k = p->k;
  a.v = p->v;
  a.q_ts = p->q_token_stride, a.q_hs = p->q_head_stride;
  a.k_ts = p->k_token_stride, a.k_hs = p->k_head_stride;
  a.v_ts = p->v_token_stride, a.v_hs = p->v_head_stride;
  a.q_heads = p->q_heads;
  a.cos = p->cos;
  a.sin = p->sin;
  a.rope_stride = p->rope_stride;
  a.rope_rows = p->rope_rows;
  a.rotary = p->rotary_dim;
  a.interleaved = p->interleaved;
  a.q_out = p->q_out;
  a.o_ts = p->q_out_token_stride, a.o_hs = p->q_out_head_stride;
  const cudaError_t err = se12::launch_kv_append(p->bf16 != 0, a, static_cast<cudaStream_t>(stream));
  if (err != cudaSuccess) return cuda_fail(err, "se12_kv_append launch");
  return SE12_OK;
}

// [arrival counters, zero between calls][partial sums]
size_t se12_kv_attend_workspace_bytes(const se12_kv_cache* c) {
  if (!c) return 0;
  return SE12_COUNTER_BYTES + std::max(se12::kv_attend_partial_bytes(c->sm_count, false),
                                       se12::kv_attend_partial_bytes(c->sm_count, true));
}

size_t se12_kv_attend_call_bytes(const se12_kv_cache* c, int q_heads, int max_query) {
  if (!c || q_heads < 1 || max_query < 1) return 0;
  const bool tiles = se12::kv_attend_takes_tiles(max_query, std::max(q_heads / c->view.heads, 1), c->view.dim);
  return SE12_COUNTER_BYTES + se12::kv_attend_partial_bytes(c->sm_count, tiles);
}

int se12_kv_attend(const se12_kv_cache* cache, const se12_kv_batch* batch, const se12_kv_attend_args* p, void* workspace,
                   size_t workspace_bytes, void* stream) {
  se12::AttendArgs a{};
  const int st = check_batch(cache, batch, &a.t);
  if (st != SE12_OK) return st;
  if (!p || !p->q || !p->out) return fail(SE12_ERR_INVALID_ARGUMENT, "null queries or output");
  const se12::KvView& v = cache->view;
  if (p->q_heads < 1 || p->q_heads % v.heads)
    return fail(SE12_ERR_INVALID_ARGUMENT, "q_heads must be a multiple of kv_heads");
  if (p->max_query < 1 || p->max_query > batch->tokens || (!batch->query_start && p->max_query != 1))
    return fail(SE12_ERR_INVALID_ARGUMENT, "max_query must be in 1..tokens, 1 without query_start");
  if (p->window < 0) return fail(SE12_ERR_INVALID_ARGUMENT, "window must not be negative");
  if (!(p->softcap >= 0.f) || !(p->softcap < 1e30f) || !(fabsf(p->scale) < 1e30f))
    return fail(SE12_ERR_INVALID_ARGUMENT, "scale and softcap must be finite, softcap not negative");
  const int group = p->q_heads / v.heads;
  // the kernel counts its work in 31 bits: chunks of 16 tokens or more, row
  // tiles of 8 rows or more, and what a pair of both costs besides its chunks
  const double work = static_cast<double>(v.heads) * batch->seqs *
                      (static_cast<double>(batch->max_pages) * v.page_size / 16 + 32) *
                      (static_cast<double>(p->max_query) * group / 8 + 1);
  if (work > 2.0e9 || static_cast<long long>(batch->tokens) * group > (1 << 30)) return fail(SE12_ERR_INVALID_ARGUMENT, "the batch is too large for one call: split it by sequences");
  const size_t need = se12_kv_attend_call_bytes(cache, p->q_heads, p->max_query);
  if (!workspace || workspace_bytes < need)
    return fail(SE12_ERR_WORKSPACE_TOO_SMALL, "workspace needs " + std::to_string(need) + " bytes");
  if (!aligned16(workspace)) return fail(SE12_ERR_MISALIGNED, "the workspace must be 16-byte aligned");
  a.c = v;
  a.q = p->q;
  a.q_ts = p->q_token_stride, a.q_hs = p->q_head_stride;
  a.q_vec = aligned16(p->q) && a.q_ts % 8 == 0 && a.q_hs % 8 == 0;
  a.out = p->out;
  a.o_ts = p->out_token_stride, a.o_hs = p->out_head_stride;
  a.o_vec = aligned16(p->out) && a.o_ts % 8 == 0 && a.o_hs % 8 == 0;
  a.q_heads = p->q_heads;
  a.group = group;
  a.scale = p->scale;
  a.softcap = usable_cap(p->softcap);
  // (a window as long as the page table hides nothing)
  a.window = p->window < batch->max_pages * v.page_size ? p->window : 0;
  a.counters = static_cast<int*>(workspace);
  a.partials = reinterpret_cast<float*>(static_cast<char*>(workspace) + SE12_COUNTER_BYTES);
  const cudaError_t err = se12::launch_kv_attend(cache->k_map, cache->v_map, a, p->max_query, cache->sm_count,
                                                 static_cast<cudaStream_t>(stream));
  if (err != cudaSuccess) return cuda_fail(err, "se12_kv_attend launch");
  return SE12_OK;
}

int se12_kv_decode(const se12_kv_cache* cache, const int32_t* pages, int count, uint16_t* k_out, uint16_t* v_out,
                   void* stream) {
  if (!cache || !k_out || !v_out) return fail(SE12_ERR_INVALID_ARGUMENT, "null argument");
  if (count < 1 || (!pages && count > cache->view.pages))
    return fail(SE12_ERR_INVALID_ARGUMENT, "count must be positive, and at most the cache's pages without page ids");
  if (!aligned16(k_out) || !aligned16(v_out)) return fail(SE12_ERR_MISALIGNED, "outputs must be 16-byte aligned");
  const cudaError_t err =
      se12::launch_kv_decode(cache->view, pages, count, k_out, v_out, static_cast<cudaStream_t>(stream));
  if (err != cudaSuccess) return cuda_fail(err, "se12_kv_decode launch");
  return SE12_OK;
}

// For any B200: 148 SMs, room for kMaxSms. [arrival counters][partial rows]
size_t se12_token_logprobs_workspace_bytes(void) {
  return SE12_COUNTER_BYTES + se12::logprob_partial_bytes(kMaxSms);
}

int se12_token_logprobs(const void* logits, int bf16, int rows, int vocab, int64_t ld, const int64_t* tokens, int top,
                        float softcap, float* logprob, float* entropy, int64_t* top_ids, float* top_logprobs,
                        void* workspace, size_t workspace_bytes, void* stream) {
  if (!logits || !tokens || !logprob || !entropy) return fail(SE12_ERR_INVALID_ARGUMENT, "null argument");
  if (rows < 1 || vocab < 1 || (ld < vocab && ld != 0))
    return fail(SE12_ERR_INVALID_ARGUMENT, "rows and vocab must be positive, ld 0 or at least vocab");
  if (top < 0 || top > SE12_LOGPROBS_MAX_TOP || top > vocab)
    return fail(SE12_ERR_INVALID_ARGUMENT, "top must be in 0.." + std::to_string(SE12_LOGPROBS_MAX_TOP) + " and at most vocab");
  if (top && (!top_ids || !top_logprobs)) return fail(SE12_ERR_INVALID_ARGUMENT, "null top outputs");
  if (!(softcap >= 0.f) || !(softcap < 1e30f)) return fail(SE12_ERR_INVALID_ARGUMENT, "softcap must be finite and not negative");
  const size_t need = se12_token_logprobs_workspace_bytes();
  if (!workspace || workspace_bytes < need)
    return fail(SE12_ERR_WORKSPACE_TOO_SMALL, "workspace needs " + std::to_string(need) + " bytes");
  if (!aligned16(workspace)) return fail(SE12_ERR_MISALIGNED, "the workspace must be 16-byte aligned");
  int sm_count = 0;
  const int st = device_sm_count(&sm_count);
  if (st != SE12_OK) return st;
  se12::LogprobArgs a{};
  a.logits = logits;
  a.ld = ld;
  a.rows = rows;
  a.vocab = vocab;
  a.tokens = reinterpret_cast<const long long*>(tokens);
  a.top = top;
  a.softcap = usable_cap(softcap);
  a.logprob = logprob;
  a.entropy = entropy;
  a.top_ids = reinterpret_cast<long long*>(top_ids);
  a.top_logprobs = top_logprobs;
  a.vec = aligned16(logits) && ld * (bf16 ? 2 : 4) % 16 == 0;
  a.counters = static_cast<int*>(workspace);
  a.partials = static_cast<unsigned char*>(workspace) + SE12_COUNTER_BYTES;
  const cudaError_t err = se12::launch_token_logprobs(bf16 != 0, a, sm_count, static_cast<cudaStream_t>(stream));
  if (err != cudaSuccess) return cuda_fail(err, "se12_token_logprobs launch");
  return SE12_OK;
}

}  // extern "C"
