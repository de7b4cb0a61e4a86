// C entry points of the 8-bit paged cache with block scales and of the block tables: argument checks, then the launch.
#include <cmath>

#include "rpa_host.h"

namespace rpa {

namespace {

bool aligned_to(const void* ptr, uint32_t bytes) { return (reinterpret_cast<uintptr_t>(ptr) & (bytes - 1)) == 0; }
bool power_of_two(int32_t x) { return x > 0 && (x & (x - 1)) == 0; }

constexpr int32_t kMostCount = 1 << 30;  // of tokens, requests and places: sums of two and rounding up stay in 32 bits

// Shape of the pool; the same for the attention, the update and the read-back.
template <typename P>
int check_pool(const P& p) {
  if (p.total_tokens < 0 || p.num_kv_heads <= 0 || p.num_pages <= 0)
    return fail(RPA_ERR_INVALID_ARGUMENT, "non-positive dimension");
  if (p.total_tokens > kMostCount) return fail(RPA_ERR_UNSUPPORTED, "total_tokens=%d: at most 2^30", p.total_tokens);
  if (p.num_kv_heads > 16384) return fail(RPA_ERR_UNSUPPORTED, "num_kv_heads=%d: at most 16384", p.num_kv_heads);
  if (p.head_dim < 16 || p.head_dim > 256 || p.head_dim % 16 != 0)
    return fail(RPA_ERR_UNSUPPORTED, "head_dim=%d must be a multiple of 16 from 16 to 256", p.head_dim);
  if (!power_of_two(p.page_size) || p.page_size < 4 || p.page_size > 32768)
    return fail(RPA_ERR_UNSUPPORTED, "page_size=%d must be a power of two from 4 to 32768", p.page_size);
  if (!power_of_two(p.scale_block) || p.scale_block < 4 || p.scale_block > p.page_size)
    return fail(RPA_ERR_UNSUPPORTED, "scale_block=%d must be a power of two from 4 to page_size=%d", p.scale_block, p.page_size);
  if (static_cast<int64_t>(p.num_pages) * p.page_size > 0x7fffffff)
    return fail(RPA_ERR_UNSUPPORTED, "num_pages * page_size = %lld must be below 2^31", static_cast<long long>(p.num_pages) * p.page_size);
  if (2 * static_cast<int64_t>(p.num_kv_heads) * p.page_size * p.head_dim > 0x7fffffff)
    return fail(RPA_ERR_UNSUPPORTED, "a page of %lld bytes: it must be smaller than 2^31", 2 * static_cast<long long>(p.num_kv_heads) * p.page_size * p.head_dim);
  if (p.dtype != RPA_DTYPE_BF16 && p.dtype != RPA_DTYPE_F32)
    return fail(RPA_ERR_INVALID_ARGUMENT, "dtype=%d must be RPA_DTYPE_BF16 or RPA_DTYPE_F32", p.dtype);
  if (p.cache_dtype != RPA_DTYPE_INT8 && p.cache_dtype != RPA_DTYPE_FP8_E4M3 && p.cache_dtype != RPA_DTYPE_FP8_E5M2)
    return fail(RPA_ERR_INVALID_ARGUMENT, "cache_dtype=%d must be RPA_DTYPE_INT8, RPA_DTYPE_FP8_E4M3 or RPA_DTYPE_FP8_E5M2", p.cache_dtype);
  return RPA_OK;
}

bool strides_ok(int64_t token, int64_t head, int32_t dtype) {
  const int64_t unit = dtype == RPA_DTYPE_BF16 ? 8 : 4;  // 16 bytes
  return token >= 0 && head >= 0 && token % unit == 0 && head % unit == 0;
}

int check_attention(const RpaQuantParams& p) {
  const int rc = check_pool(p);
  if (rc != RPA_OK) return rc;
  if (p.num_q_heads <= 0 || p.max_num_seqs <= 0 || p.pages_per_seq <= 0 || p.num_sinks < 0)
    return fail(RPA_ERR_INVALID_ARGUMENT, "non-positive dimension in RpaQuantParams");
  if (p.max_num_seqs > kMostCount) return fail(RPA_ERR_UNSUPPORTED, "max_num_seqs=%d: at most 2^30", p.max_num_seqs);
  if (p.num_q_heads % p.num_kv_heads != 0)
    return fail(RPA_ERR_INVALID_ARGUMENT, "num_q_heads=%d must be divisible by num_kv_heads=%d", p.num_q_heads, p.num_kv_heads);
  if (static_cast<int64_t>(p.pages_per_seq) * p.page_size > (1 << 30))
    return fail(RPA_ERR_UNSUPPORTED, "pages_per_seq * page_size = %lld: a sequence holds at most 2^30 tokens", static_cast<long long>(p.pages_per_seq) * p.page_size);
  if (p.sliding_window < 0) return fail(RPA_ERR_INVALID_ARGUMENT, "sliding_window=%d must be positive", p.sliding_window);
  if (!std::isfinite(p.softmax_scale)) return fail(RPA_ERR_INVALID_ARGUMENT, "softmax_scale must be finite");
  if (!std::isfinite(p.logits_soft_cap)) return fail(RPA_ERR_INVALID_ARGUMENT, "logits_soft_cap must be finite");
  if (p.flags != 0) return fail(RPA_ERR_INVALID_ARGUMENT, "flags=%u: there are none", p.flags);
  return RPA_OK;
}

// Every entry point answers with a code whatever happens inside: no exception leaves the library.
template <typename F>
int guarded(F&& f) {
  try {
    return f();
  } catch (...) {
    return fail(RPA_ERR_LAUNCH, "unexpected exception");
  }
}

int launched(int rc) {
  if (rc == RPA_ERR_LAUNCH) return fail(rc, "kernel launch failed: %s", hipGetErrorString(hipGetLastError()));
  return rc;
}

}  // namespace

}  // namespace rpa

extern "C" {

uint64_t rpa_quant_workspace_bytes(const RpaQuantParams* dims) {
  if (dims == nullptr || rpa::check_attention(*dims) != RPA_OK) return 0;
  return rpa::quant_attention_workspace(*dims);
}

int rpa_quant_fwd_launch(const RpaQuantParams* params, void* hip_stream) {
  return rpa::guarded([&] {
    if (params == nullptr) return rpa::fail(RPA_ERR_INVALID_ARGUMENT, "params is null");
    const RpaQuantParams& p = *params;
    const int rc = rpa::check_attention(p);
    if (rc != RPA_OK) return rc;
    if (p.total_tokens == 0) return static_cast<int>(RPA_OK);
    if (!p.queries || !p.kv_cache || !p.kv_scales || !p.context_lens || !p.block_tables || !p.query_start_loc || !p.num_seqs || !p.out)
      return rpa::fail(RPA_ERR_INVALID_ARGUMENT, "null device pointer in RpaQuantParams");
    if (p.num_sinks > 0 && !p.sinks) return rpa::fail(RPA_ERR_INVALID_ARGUMENT, "num_sinks=%d but sinks is null", p.num_sinks);
    if (!rpa::strides_ok(p.query_token_stride, p.query_head_stride, p.dtype))
      return rpa::fail(RPA_ERR_INVALID_ARGUMENT, "the strides of queries must be multiples of 16 bytes and not negative");
    if (!rpa::aligned_to(p.queries, 16) || !rpa::aligned_to(p.kv_cache, 16) || !rpa::aligned_to(p.out, 16))
      return rpa::fail(RPA_ERR_INVALID_ARGUMENT, "queries, kv_cache and out must be aligned to 16 bytes");
    if (!rpa::aligned_to(p.kv_scales, 4) || !rpa::aligned_to(p.context_lens, 4) || !rpa::aligned_to(p.block_tables, 4) ||
        !rpa::aligned_to(p.query_start_loc, 4) || !rpa::aligned_to(p.num_seqs, 4) || !rpa::aligned_to(p.sinks, 4))
      return rpa::fail(RPA_ERR_INVALID_ARGUMENT, "int32 / fp32 arrays must be aligned to 4 bytes");
    const uint64_t need = rpa::quant_attention_workspace(p);
    if (p.workspace == nullptr || p.workspace_bytes < need || !rpa::aligned_to(p.workspace, 256))
      return rpa::fail(RPA_ERR_WORKSPACE, "workspace of %llu bytes is too small or not aligned to 256 bytes, rpa_quant_workspace_bytes() asks for %llu",
                       (unsigned long long)p.workspace_bytes, (unsigned long long)need);
    return rpa::launched(rpa::launch_quant_attention(p, static_cast<hipStream_t>(hip_stream)));
  });
}

int rpa_quant_update_launch(const RpaQuantUpdateParams* params, void* hip_stream) {
  return rpa::guarded([&] {
    if (params == nullptr) return rpa::fail(RPA_ERR_INVALID_ARGUMENT, "params is null");
    const RpaQuantUpdateParams& p = *params;
    const int rc = rpa::check_pool(p);
    if (rc != RPA_OK) return rc;
    if (p.total_tokens == 0) return static_cast<int>(RPA_OK);
    if (!p.keys || !p.values || !p.kv_cache || !p.kv_scales || !p.slot_mapping)
      return rpa::fail(RPA_ERR_INVALID_ARGUMENT, "null device pointer in RpaQuantUpdateParams");
    if (!rpa::strides_ok(p.key_token_stride, p.key_head_stride, p.dtype) || !rpa::strides_ok(p.value_token_stride, p.value_head_stride, p.dtype))
      return rpa::fail(RPA_ERR_INVALID_ARGUMENT, "the strides of keys and values must be multiples of 16 bytes and not negative");
    if (!rpa::aligned_to(p.keys, 16) || !rpa::aligned_to(p.values, 16) || !rpa::aligned_to(p.kv_cache, 16))
      return rpa::fail(RPA_ERR_INVALID_ARGUMENT, "keys, values and kv_cache must be aligned to 16 bytes");
    if (!rpa::aligned_to(p.kv_scales, 4) || !rpa::aligned_to(p.slot_mapping, 4))
      return rpa::fail(RPA_ERR_INVALID_ARGUMENT, "int32 / fp32 arrays must be aligned to 4 bytes");
    return rpa::launched(rpa::launch_quant_update(p, static_cast<hipStream_t>(hip_stream)));
  });
}

int rpa_quant_gather_launch(const RpaQuantGatherParams* params, void* hip_stream) {
  return rpa::guarded([&] {
    if (params == nullptr) return rpa::fail(RPA_ERR_INVALID_ARGUMENT, "params is null");
    const RpaQuantGatherParams& p = *params;
    const int rc = rpa::check_pool(p);
    if (rc != RPA_OK) return rc;
    if (p.total_tokens == 0) return static_cast<int>(RPA_OK);
    if (!p.keys || !p.values || !p.kv_cache || !p.kv_scales || !p.slot_mapping)
      return rpa::fail(RPA_ERR_INVALID_ARGUMENT, "null device pointer in RpaQuantGatherParams");
    if (!rpa::aligned_to(p.keys, 16) || !rpa::aligned_to(p.values, 16) || !rpa::aligned_to(p.kv_cache, 16))
      return rpa::fail(RPA_ERR_INVALID_ARGUMENT, "keys, values and kv_cache must be aligned to 16 bytes");
    if (!rpa::aligned_to(p.kv_scales, 4) || !rpa::aligned_to(p.slot_mapping, 4))
      return rpa::fail(RPA_ERR_INVALID_ARGUMENT, "int32 / fp32 arrays must be aligned to 4 bytes");
    return rpa::launched(rpa::launch_quant_gather(p, static_cast<hipStream_t>(hip_stream)));
  });
}

int rpa_block_tables_launch(const RpaBlockTablesParams* params, void* hip_stream) {
  return rpa::guarded([&] {
    if (params == nullptr) return rpa::fail(RPA_ERR_INVALID_ARGUMENT, "params is null");
    const RpaBlockTablesParams& p = *params;
    if (p.max_num_seqs <= 0 || p.pages_per_seq <= 0 || p.num_free_slots <= 0 || p.page_size <= 0 || p.total_tokens < 0)
      return rpa::fail(RPA_ERR_INVALID_ARGUMENT, "non-positive dimension in RpaBlockTablesParams");
    if (p.max_num_seqs > rpa::kMostCount || p.num_free_slots > rpa::kMostCount || p.total_tokens > rpa::kMostCount)
      return rpa::fail(RPA_ERR_UNSUPPORTED, "max_num_seqs=%d, num_free_slots=%d and total_tokens=%d: at most 2^30 each", p.max_num_seqs, p.num_free_slots, p.total_tokens);
    const void* ptrs[] = {p.query_lens, p.cached_lens, p.block_tables, p.free_pages, p.free_state, p.num_seqs, p.query_start_loc,
                          p.context_lens, p.admitted, p.cached_lens_out, p.free_state_out, p.scratch};
    for (const void* q : ptrs)
      if (q == nullptr || !rpa::aligned_to(q, 4)) return rpa::fail(RPA_ERR_INVALID_ARGUMENT, "null or misaligned device pointer in RpaBlockTablesParams");
    if (p.total_tokens > 0 && (!p.slot_mapping || !p.positions || !rpa::aligned_to(p.slot_mapping, 4) || !rpa::aligned_to(p.positions, 4)))
      return rpa::fail(RPA_ERR_INVALID_ARGUMENT, "null or misaligned slot_mapping / positions");
    if (!rpa::aligned_to(p.scratch, 16)) return rpa::fail(RPA_ERR_INVALID_ARGUMENT, "scratch must be aligned to 16 bytes");
    return rpa::launched(rpa::launch_block_tables(p, static_cast<hipStream_t>(hip_stream)));
  });
}

}  // extern "C"
