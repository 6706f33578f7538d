// Paged attention over a sliding window and a few first keys (sinks): token t with key count L
// sees keys j < L with j >= L - window or j < sinks.
//
//   out[t, h] = sum_j p_j V_j / sum_j p_j,  p_j = exp(scale q[t, h] . K_j - max)
//
// over the keys that it sees (zeros if none), online over chunks of 64 keys.
#include "attention_keys.hpp"

namespace nvf {

template <typename T>
int window_dispatch(AttnArgs<T> a, const WindowRule& rule, hipStream_t st) {
  a.nsplit = 1;
  launch_attn_any(a, rule, st);
  return launch_status("window_attention");
}

}  // namespace nvf

using namespace nvf;

extern "C" {

int64_t nvf_window_attention_workspace_size(int64_t tokens, int q_heads, int kv_heads, int head_dim, int block_size,
                                            int max_blocks, int64_t window, int64_t sinks, int64_t max_query_len) {
  return 0;
}

int nvf_window_attention_ws(const void* q, void* out, const void* k_cache, const void* v_cache,
                            const int32_t* query_seq, const int32_t* query_key_len, const int32_t* block_tables,
                            const int32_t* cu_seqlens_host, int num_seqs, int64_t tokens, int q_heads, int kv_heads,
                            int head_dim, int block_size, int max_blocks, int64_t num_blocks, float scale,
                            int64_t window, int64_t sinks, int64_t q_stride, int64_t max_query_len, void* workspace,
                            int64_t workspace_bytes, int dtype, void* stream) {
  const char* who = "nvf_window_attention";
  const int rc0 = check_attn(who, q, out, k_cache, v_cache, query_seq, query_key_len, block_tables, tokens, q_heads,
                             kv_heads, head_dim, block_size, max_blocks, num_seqs, num_blocks, q_stride, workspace,
                             dtype);
  if (rc0 != NVF_OK) return rc0;
  if (window < 0 || sinks < 0) return fail(NVF_ERR_INVALID, "%s: negative window or sinks", who);
  if (cu_seqlens_host) {
    if (cu_seqlens_host[0] != 0 || cu_seqlens_host[num_seqs] != tokens)
      return fail(NVF_ERR_INVALID, "%s: cu_seqlens must run from 0 to tokens=%lld", who, (long long)tokens);
    for (int s = 0; s < num_seqs; ++s)
      if (cu_seqlens_host[s + 1] < cu_seqlens_host[s])
        return fail(NVF_ERR_INVALID, "%s: cu_seqlens must not decrease", who);
  }
  if (tokens == 0) return NVF_OK;
  const WindowRule rule{(int)std::min<int64_t>(window, INT32_MAX), (int)std::min<int64_t>(sinks, INT32_MAX)};
  int rc = NVF_OK;
  NVF_DISPATCH_DTYPE(dtype, T, rc = window_dispatch<T>(
      attn_args<T>(q, out, k_cache, v_cache, query_seq, query_key_len, block_tables, tokens, q_heads, kv_heads,
                   head_dim, block_size, max_blocks, num_seqs, num_blocks, scale, q_stride),
      rule, as_stream(stream)));
  return rc;
}

}  // extern "C"
