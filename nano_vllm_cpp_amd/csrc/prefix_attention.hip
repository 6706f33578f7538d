// Paged attention of a batch whose sequences share long prefixes.  The tokens come in groups of
// consecutive ones; the sequences of a group hold the same first prefix_len keys.  The result is
// paged attention's: token t attends the first query_key_len[t] keys of its sequence.
#include "attention_keys.hpp"

namespace nvf {

template <typename T>
int prefix_dispatch(AttnArgs<T> a, const PrefixGroups& groups, hipStream_t st) {
  a.nsplit = 1;
  launch_attn_any(a, WindowRule{INT32_MAX, 0}, st);
  return launch_status("prefix_attention");
}

}  // namespace nvf

using namespace nvf;

extern "C" {

int64_t nvf_prefix_attention_workspace_size(const int32_t* group_start_host, const int32_t* prefix_len_host,
                                            int num_groups, int q_heads, int kv_heads, int head_dim, int block_size,
                                            int max_blocks) {
  return 0;
}

int nvf_prefix_attention_ws(const void* q, void* out, const void* k_cache, const void* v_cache,
                            const int32_t* query_seq, const int32_t* query_key_len, const int32_t* block_tables,
                            const int32_t* group_start_host, const int32_t* prefix_len_host, int num_groups,
                            int num_seqs, int64_t tokens, int q_heads, int kv_heads, int head_dim, int block_size,
                            int max_blocks, int64_t num_blocks, float scale, int64_t q_stride, void* workspace,
                            int64_t workspace_bytes, int dtype, void* stream) {
  const char* who = "nvf_prefix_attention";
  const int rc0 = check_attn(who, q, out, k_cache, v_cache, query_seq, query_key_len, block_tables, tokens, q_heads,
                             kv_heads, head_dim, block_size, max_blocks, num_seqs, num_blocks, q_stride, workspace,
                             dtype);
  if (rc0 != NVF_OK) return rc0;
  if (num_groups <= 0 || !group_start_host || !prefix_len_host)
    return fail(NVF_ERR_INVALID, "%s: group_start_host, prefix_len_host and num_groups > 0 are required", who);
  if (group_start_host[0] != 0 || group_start_host[num_groups] != tokens)
    return fail(NVF_ERR_INVALID, "%s: group_start must run from 0 to tokens=%lld", who, (long long)tokens);
  for (int g = 0; g < num_groups; ++g) {
    if (group_start_host[g + 1] < group_start_host[g])
      return fail(NVF_ERR_INVALID, "%s: group_start must not decrease", who);
    if (prefix_len_host[g] < 0 || prefix_len_host[g] > (int64_t)block_size * max_blocks)
      return fail(NVF_ERR_INVALID, "%s: prefix_len %d is outside the block tables", who, prefix_len_host[g]);
  }
  if (tokens == 0) return NVF_OK;
  int rc = NVF_OK;
  NVF_DISPATCH_DTYPE(dtype, T, rc = prefix_dispatch<T>(
      attn_args<T>(q, out, k_cache, v_cache, query_seq, query_key_len, block_tables, tokens, q_heads, kv_heads,
                   head_dim, block_size, max_blocks, num_seqs, num_blocks, scale, q_stride),
      PrefixGroups{}, as_stream(stream)));
  return rc;
}

}  // extern "C"
