// Attention over the 8-bit paged cache with a scale per block of tokens and head.
#include "rpa_quant.h"

namespace rpa {

namespace {

// One wavefront per (token, query head): lanes are keys for the logits, then elements for the weighted sum.
template <int kCode, typename T>
__global__ __launch_bounds__(64) void quant_attention_kernel(RpaQuantParams p, int page_shift, int block_shift) {
  __shared__ float q_lds[256];
  const int t = blockIdx.x, h = blockIdx.y, lane = threadIdx.x, D = p.head_dim;
  T* out = static_cast<T*>(p.out) + (static_cast<size_t>(t) * p.num_q_heads + h) * D;
  const int n = min(max(p.num_seqs[0], 0), p.max_num_seqs);
  float acc[4] = {0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.f;
  const int end = min(max(p.query_start_loc[n], 0), p.total_tokens);
  if (t < end) {
    const int s = find_seq(p.query_start_loc, n, t);
    const int64_t room = static_cast<int64_t>(p.pages_per_seq) << page_shift;
    const int q0 = min(max(p.query_start_loc[s], 0), p.total_tokens), q1 = min(max(p.query_start_loc[s + 1], 0), p.total_tokens);
    const int len = static_cast<int>(min(static_cast<int64_t>(max(p.context_lens[s], 0)), room));
    const int pos = len - (q1 - q0) + (t - q0);
    const int first = p.sliding_window > 0 ? max(pos - p.sliding_window + 1, 0) : 0;
    const int kvh = h / (p.num_q_heads / p.num_kv_heads), heads = 2 * p.num_kv_heads;
    const T* q = static_cast<const T*>(p.queries) + t * p.query_token_stride + h * p.query_head_stride;
    for (int d = lane; d < D; d += 64) q_lds[d] = Elem<T>::load(q + d);
    __syncthreads();
    for (int k0 = first & ~63; k0 <= pos; k0 += 64) {
      const int k = k0 + lane;
      const bool seen = k >= first && k <= pos && k < len;
      float x = -INFINITY, vs = 0.f;
      size_t v_row = 0;
      if (seen) {
        const int page = clamp_page(p.block_tables[static_cast<size_t>(s) * p.pages_per_seq + (k >> page_shift)], p.num_pages);
        const int off = k & ((1 << page_shift) - 1);
        const size_t line = static_cast<size_t>(page) * heads + 2 * kvh;
        const uint32_t* row = reinterpret_cast<const uint32_t*>(static_cast<const char*>(p.kv_cache) + ((line << page_shift) + off) * D);
        v_row = (((line + 1) << page_shift) + off) * D;
        const float* sc = p.kv_scales + (line << (page_shift - block_shift)) + (off >> block_shift);
        vs = sc[static_cast<size_t>(1) << (page_shift - block_shift)];
        float a = 0.f;
        for (int d = 0; d < D; d += 4) {
          const uint32_t w = row[d / 4];
#pragma unroll
          for (int b = 0; b < 4; ++b) a = fmaf(q_lds[d + b], code_to_f32<kCode>(w, b), a);
        }
        x = a * sc[0] * p.softmax_scale;
        if (p.logits_soft_cap != 0.f) x = p.logits_soft_cap * tanhf(x / p.logits_soft_cap);
      }
      const float m_new = fmaxf(m, wave_max(x));
      const float pr = seen && x > -INFINITY ? expf(x - m_new) : 0.f;
      const float alpha = m_new == -INFINITY ? 1.f : expf(m - m_new);
      l = l * alpha + wave_sum(pr);
      m = m_new;
      for (int e = 0; e < 4; ++e) acc[e] *= alpha;
      for (int j = 0; j < 64; ++j) {
        const float w = __shfl(pr * vs, j);
        const size_t r = __shfl(static_cast<unsigned long long>(v_row), j);
        if (!__shfl(static_cast<int>(seen), j)) continue;
        for (int e = 0; e < 4; ++e) {
          const int d = lane + 64 * e;
          if (d < D) acc[e] = fmaf(w, code_to_f32<kCode>(static_cast<const uint8_t*>(p.kv_cache)[r + d], 0), acc[e]);
        }
      }
    }
    if (m > -INFINITY) {
      float top = m;
      for (int j = 0; j < p.num_sinks; ++j) top = fmaxf(top, p.sinks[static_cast<size_t>(h) * p.num_sinks + j]);
      const float w = expf(m - top);
      l *= w;
      for (int j = 0; j < p.num_sinks; ++j) l += expf(p.sinks[static_cast<size_t>(h) * p.num_sinks + j] - top);
      for (int e = 0; e < 4; ++e) acc[e] *= w / l;
    }
  }
  for (int e = 0; e < 4; ++e) {
    const int d = lane + 64 * e;
    if (d < D) Elem<T>::store(out + d, acc[e]);
  }
}

}  // namespace

uint64_t quant_attention_workspace(const RpaQuantParams& p) { return 256; }

int launch_quant_attention(const RpaQuantParams& p, hipStream_t stream) {
  const dim3 grid(p.total_tokens, p.num_q_heads);
  const int ps = __builtin_ctz(p.page_size), bs = __builtin_ctz(p.scale_block);
  auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(64), 0, stream, p, ps, bs); };
  const bool f32 = p.dtype == RPA_DTYPE_F32;
  switch (code_of_dtype(p.cache_dtype)) {
    case kCodeI8: f32 ? go(quant_attention_kernel<kCodeI8, float>) : go(quant_attention_kernel<kCodeI8, bf16_t>); break;
    case kCodeE4m3: f32 ? go(quant_attention_kernel<kCodeE4m3, float>) : go(quant_attention_kernel<kCodeE4m3, bf16_t>); break;
    default: f32 ? go(quant_attention_kernel<kCodeE5m2, float>) : go(quant_attention_kernel<kCodeE5m2, bf16_t>); break;
  }
  return hipGetLastError() == hipSuccess ? RPA_OK : RPA_ERR_LAUNCH;
}

}  // namespace rpa
