// C entry points of the attention over the paged 8-bit KV cache. Part of the
// kvq_lib.cu unity build.
#pragma once
#include "kvq_paged_tile.cuh"

namespace kvq {
namespace paged {

inline size_t attention_bytes(int64_t D, int64_t max_new, int64_t group) {
  const int NT = row_tiles(max_new, group);
  if (NT == 0)
    return kTileParts * kUnitRows * (D + 4) * sizeof(float) + (kMaxSeqs + 1) * sizeof(int32_t);
  return (size_t)2 * kSms * kAttnWarps * part_floats((int)D, NT) * sizeof(float);
}

}  // namespace paged
}  // namespace kvq

extern "C" size_t kvq_paged_attention_workspace(int64_t head_dim, int64_t max_new, int64_t group) {
  if (head_dim < 0 || head_dim > 128 || max_new < 0 || group < 0) return 0;
  return kvq::paged::attention_bytes(head_dim, max_new, group);
}

extern "C" int kvq_paged_attention(const void* q, int64_t q_tok_stride, int64_t q_head_stride,
                                   int dtype, int64_t group, const uint8_t* pool, int kind,
                                   int64_t n_pages, int64_t n_heads, int64_t head_dim,
                                   int64_t page_tokens, const int32_t* table, int64_t n_slots,
                                   int64_t n_cols, const int32_t* lengths, const int32_t* slots,
                                   const int32_t* indptr, int64_t B, int64_t total,
                                   int64_t max_new, float scale, int64_t window, void* out,
                                   float* ml_out, void* workspace, size_t workspace_bytes,
                                   void* stream) {
  using namespace kvq;
  using namespace kvq::paged;
  clear_error();
  AttnArgs a;
  a.v = make_view(const_cast<uint8_t*>(pool), n_pages, n_heads, head_dim, page_tokens, table,
                  n_slots, n_cols, lengths, slots, indptr, B, total);
  int rc = check_view("paged_attention", a.v, kind, page_tokens);
  if (rc) return rc;
  if (dtype != 0 && dtype != 1) {
    set_error("paged_attention: dtype must be 0 (fp16) or 1 (bf16), got %d", dtype);
    return KVQ_ERR_UNSUPPORTED;
  }
  if (group < 1 || group > 64 || n_heads * group > 4096) {
    set_error("paged_attention: %lld query heads per KV head (1..64) of %lld", (long long)group,
              (long long)n_heads);
    return KVQ_ERR_UNSUPPORTED;
  }
  if (max_new < (total > 0) || max_new > 65536 || (!indptr && max_new < total / B) || window < 0 ||
      window > INT32_MAX) {
    set_error("paged_attention: max_new %lld (1..65536, at least the rows a sequence) or window "
              "%lld", (long long)max_new, (long long)window);
    return KVQ_ERR_INVALID;
  }
  if (total == 0) return KVQ_OK;
  if (!q || !out || !aligned16(q) || q_tok_stride % 8 || q_head_stride % 8 ||
      (reinterpret_cast<uintptr_t>(out) & 15) || (reinterpret_cast<uintptr_t>(ml_out) & 7)) {
    set_error("paged_attention: q rows and out must be 16-byte aligned (strides multiples of 8), "
              "ml_out 8-byte aligned");
    return KVQ_ERR_INVALID;
  }
  const size_t need = attention_bytes(head_dim, max_new, group);
  if (!workspace || !aligned16(workspace) || workspace_bytes < need) {
    set_error("paged_attention: workspace too small or unaligned (%zu < %zu)", workspace_bytes,
              need);
    return KVQ_ERR_INVALID;
  }
  a.q = q;
  a.q_tok = q_tok_stride;
  a.q_head = q_head_stride;
  a.group = (int)group;
  a.max_new = (int)max_new;
  a.window = (int)window;
  a.scale_log2 = scale * kLog2e;
  a.out = out;
  a.ml = reinterpret_cast<float2*>(ml_out);
  a.part = static_cast<float*>(workspace);
  const cudaStream_t st = as_stream(stream);
  const int NT = row_tiles(max_new, group);
  if (NT == 0) {
#define KVQ_TILE(D, T) \
  (kind == kInt8 ? launch_attend_tile<D, kInt8, T>(a, st) : launch_attend_tile<D, kE4m3, T>(a, st))
    if (head_dim == 64) return dtype == 0 ? KVQ_TILE(64, __half) : KVQ_TILE(64, __nv_bfloat16);
    return dtype == 0 ? KVQ_TILE(128, __half) : KVQ_TILE(128, __nv_bfloat16);
#undef KVQ_TILE
  }
#define KVQ_ATTEND3(D, KIND, T) \
  (NT == 1 ? launch_attend<D, KIND, 1, T>(a, st) : launch_attend<D, KIND, 2, T>(a, st))
#define KVQ_ATTEND2(D, T) (kind == kInt8 ? KVQ_ATTEND3(D, kInt8, T) : KVQ_ATTEND3(D, kE4m3, T))
  if (head_dim == 64)
    return dtype == 0 ? KVQ_ATTEND2(64, __half) : KVQ_ATTEND2(64, __nv_bfloat16);
  return dtype == 0 ? KVQ_ATTEND2(128, __half) : KVQ_ATTEND2(128, __nv_bfloat16);
#undef KVQ_ATTEND2
#undef KVQ_ATTEND3
}
