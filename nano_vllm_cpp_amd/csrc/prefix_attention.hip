// Paged attention of a batch whose sequences share long prefixes.  The tokens come in groups of
// consecutive ones; the sequences of a group hold the same first prefix_len keys.  The result is
// paged attention's: token t attends the first query_key_len[t] keys of its sequence.
//
// softmax(s) V over all keys from the softmax states of disjoint parts (max m, sum l and O of each):
//   out = sum_i 2^(m_i - M) O_i / sum_i 2^(m_i - M) l_i,  M = max_i m_i
//
// * prefix_kernel: the prefix against all (token, head) rows of a group and kv head, 128 a workgroup, so
//   that its keys are read once for them, in key ranges that fill the GPU; and each token's own keys past
//   the prefix;
// * attn_join_kernel joins the states.
// Shapes that the matrix cores do not take run token by token over all keys (attn_any_kernel).
#include "attention_tiles.hpp"

#include <mutex>

namespace nvf {

// Workgroups: `tiles` x splits of the first kind, `tokens` x own splits of the second, in one launch, since
// the first are bound by the matrix units and the second by HBM.  Every 8th workgroup goes to one XCD: the even
// workgroups take the tiles, whose keys so stay in the L2 of half the XCDs, as far as prefix_level finds them no more
// than half of the work, and the tokens level the two.
//   tile x = (tile of the groups in turn, kv head), kv heads innermost; split x / tiles
//   token x = (token, kv head, 16 of its heads); split x / tokens, its states after the tiles'
struct PrefixWork {
  int tiles, splits, tokens, own_splits, tile_tokens;
  int even_tiles, odd_tokens;  // of all splits, at least half
};
template <typename T, int HD>
__global__ __launch_bounds__(kTileThreads<T>)
__attribute__((amdgpu_waves_per_eu(sizeof(T) == 4 && HD == 64 ? 4 : 2))) void prefix_kernel(
    const AttnArgs<T> a, const FastDiv div, const PrefixGroups groups, const PrefixWork work) {
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int i = (int)(blockIdx.x >> 1);
  const bool odd = (blockIdx.x & 1) != 0;
  const int all_tiles = work.tiles * work.splits, all_tokens = work.tokens * work.own_splits;
  const int tiles = odd ? all_tiles - work.even_tiles : work.even_tiles, k = i - tiles;
  const bool tile = i < tiles;
  const int alone = 2 * work.odd_tokens - all_tokens;  // the odd workgroups' first tokens; the rest go to both in turn
  const int x = tile ? (odd ? work.even_tiles + i : i) : odd ? (k < alone ? k : 2 * k - alone + 1) : alone + 2 * k;
  if (x >= (tile ? all_tiles : all_tokens)) return;  // past the shorter list
  if (tile) {
    const int wg = x % work.tiles, z = x / work.tiles;
    const TileAt at = tile_at(groups.start, groups.n, wg / a.kv_heads, work.tile_tokens);
    const TileJob job{at.t0, 0, at.n, -1, wg % a.kv_heads, groups.len[at.g], z, work.splits, z};
    tile_of<T, HD, kPrefixTile>(a, div, WindowRule{}, job, lds);
  } else {
    if (threadIdx.x >= 256) return;  // four waves a token; a barrier does not wait for waves that have ended
    const int parts = (a.q_heads / a.kv_heads + 15) / 16, per = a.kv_heads * parts;
    const int wg = x % work.tokens, z = x / work.tokens, rest = wg % per;
    token_of<T, HD>(a, div, SuffixRule{groups}, wg / per, rest / parts, rest % parts, z, work.own_splits,
                    work.splits + z, lds);
  }
}

// Whether tiles and tokens go into one launch and share the CUs, and so the GPU's time.  fp32 tiles of head size 128 take a
// CU's LDS each, which would leave the tokens one workgroup a CU: they come first, with the whole GPU.  (fp32, 14 / 2 heads
// of 64, 200 tokens over 6000 keys and 64 over 2000: 90 and 22 us in one launch, 88 and 32 in two.)
inline bool prefix_together(int hd, int dtype_bytes) { return !(dtype_bytes == 4 && hd == 128); }

// How a launch's groups are split: key ranges of the prefixes and of the tokens' own keys.
struct PrefixPlan {
  int tile_tokens = 0, tiles = 0, splits = 0, own_splits = 0;
};
// The time, in us, that a workgroup of each kind takes with two on a CU, measured at head size 128, by which 64 goes
// too: a tile's chunk 2.7 beside tokens (8 in fp32); a token's at 5.9 TB/s over all, 4 more.  The host does not know the tokens' own keys: half of those
// that the tables have past the prefix, and past a shorter prefix than the longest no more than twice as many as past
// that.
struct PrefixCost {
  double tile, token;
};
inline PrefixCost prefix_cost(const PrefixPlan& p, const PrefixGroups& groups, int hd, int64_t table_keys,
                              int dtype_bytes) {
  int64_t chunks = 0, longest = 0, own_keys = 0;
  for (int g = 0; g < groups.n; ++g) longest = std::max<int64_t>(longest, groups.len[g]);
  for (int g = 0; g < groups.n; ++g) {
    const int64_t n = groups.start[g + 1] - groups.start[g], tiles = (n + p.tile_tokens - 1) / p.tile_tokens;
    chunks += tiles * ((std::max<int64_t>(groups.len[g], 0) + kChunk - 1) / kChunk);
    own_keys += n * std::max<int64_t>(std::min(table_keys - groups.len[g], 2 * (table_keys - longest)), 0) / 2;
  }
  const double own = (double)own_keys / groups.start[groups.n] / kChunk / p.own_splits;  // chunks
  return PrefixCost{((double)chunks / (p.tiles * p.splits) + 2.0) * (dtype_bytes == 4 ? 8.0 : 2.7),
                    4.0 + own * (2.0 * kChunk * hd * dtype_bytes * 512 / 5.9e6)};
}
inline PrefixPlan prefix_plan(const PrefixGroups& groups, int q_heads, int kv_heads, int hd, int64_t table_keys,
                              int dtype_bytes) {
  PrefixPlan p;
  const int G = q_heads / kv_heads;
  p.tile_tokens = kTileRows / G;
  p.tiles = tiles_of(groups.start, groups.n, p.tile_tokens);
  int64_t longest = 0, shortest = INT32_MAX;
  for (int g = 0; g < groups.n; ++g) {
    longest = std::max<int64_t>(longest, groups.len[g]);
    shortest = std::min<int64_t>(shortest, groups.len[g]);
  }
  const int64_t rows = (int64_t)groups.start[groups.n] * q_heads;
  const int64_t tokens = (int64_t)groups.start[groups.n] * kv_heads * ((G + 15) / 16);
  p.splits = 1;
  p.own_splits = token_split(tokens, (table_keys - shortest) / kChunk + 1, rows, hd, true);
  // the tiles' part of the GPU
  const PrefixCost cost = prefix_cost(p, groups, hd, table_keys, dtype_bytes);
  const double tile_us = cost.tile * p.tiles * kv_heads, token_us = cost.token * (double)(tokens * p.own_splits);
  const double part = prefix_together(hd, dtype_bytes) ? std::max(0.5, tile_us / (tile_us + token_us)) : 1.0;
  p.splits = tile_split((int64_t)p.tiles * kv_heads, (longest + kChunk - 1) / kChunk, rows, hd, dtype_bytes, part, true);
  return p;
}
// Deals the work out to the even and the odd workgroups.  256 tokens over 8192 shared and up to 1024 own keys, bf16,
// 28 / 4 heads of 128: 119 us in two launches, 109 with both kinds on every XCD, 97 with the kinds in turn, 88 so (with
// P in one part; in two 94).
inline void prefix_level(PrefixWork& w, const PrefixCost& cost) {
  const int64_t tiles = (int64_t)w.tiles * w.splits, tokens = (int64_t)w.tokens * w.own_splits;
  const double half = (cost.tile * (double)tiles + cost.token * (double)tokens) / 2;
  w.even_tiles = (int)std::min<int64_t>(tiles, (int64_t)(half / cost.tile) + 1);
  w.odd_tokens = (int)std::min<int64_t>(tokens, (int64_t)(half / cost.token) + 1);
}

// Whether the tiles take a call (the other half of attn_mfma).
inline bool prefix_shape(int q_heads, int kv_heads, int hd, int bs) {
  return q_heads / kv_heads <= kTileRows / 2 && (hd == 64 || hd == 128) && bs % 16 == 0;
}

// Calls f(up to kMaxGroups groups, their first token) for all groups, empty ones left out.
template <typename F>
void by_groups(const int32_t* start, const int32_t* len, int n, F f) {
  for (int g = 0; g < n;) {
    PrefixGroups groups{};
    const int32_t first = start[g];
    for (; g < n && groups.n < kMaxGroups; ++g) {
      if (start[g] == start[g + 1]) continue;
      groups.start[groups.n] = start[g] - first;
      groups.len[groups.n++] = len[g];
      groups.start[groups.n] = start[g + 1] - first;
    }
    if (groups.n > 0) f(groups, first);
  }
}

template <typename T, int HD>
void prefix_mfma(const AttnArgs<T>& a, const PrefixGroups& groups, const PrefixPlan& p, hipStream_t st) {
  static constexpr int kTile = TileLds<T, HD>::kBytes, kToken = TokenLds<T, HD>::kBytes;
  static constexpr int kMost = kTile > kToken ? kTile : kToken;
  static std::once_flag lds_once;
  std::call_once(lds_once, [] {
    (void)hipFuncSetAttribute(reinterpret_cast<const void*>(&prefix_kernel<T, HD>),
                              hipFuncAttributeMaxDynamicSharedMemorySize, kMost);
  });
  const FastDiv div((uint32_t)a.bs);
  PrefixWork work{p.tiles * a.kv_heads, p.splits, (int)(a.tokens * a.kv_heads * ((a.q_heads / a.kv_heads + 15) / 16)),
                  p.own_splits, p.tile_tokens, 0, 0};
  const PrefixCost cost = prefix_cost(p, groups, HD, (int64_t)a.bs * a.max_blocks, (int)sizeof(T));
  const auto launch = [&](PrefixWork w, int threads, int lds) {
    prefix_level(w, cost);
    const int tiles = w.tiles * w.splits, tokens = w.tokens * w.own_splits;
    const int pairs = std::max(w.even_tiles + tokens - w.odd_tokens, w.odd_tokens + tiles - w.even_tiles);
    prefix_kernel<T, HD><<<dim3((unsigned)(2 * pairs)), threads, lds, st>>>(a, div, groups, w);
  };
  // (apart, all the same if there is a CU for each workgroup; and a launch has fewer than 2^32 threads, of which the
  // longer list's may be nearly half idle)
  const int64_t all = (int64_t)work.tiles * work.splits + (int64_t)work.tokens * work.own_splits;
  if (all <= (prefix_together(HD, (int)sizeof(T)) ? 1 << 21 : 256)) {
    launch(work, kTileThreads<T>, kMost);
  } else {
    PrefixWork tiles = work, tokens = work;
    tiles.tokens = 0;
    tokens.tiles = 0;
    launch(tiles, kTileThreads<T>, kTile);
    launch(tokens, 256, kToken);
  }
}

template <typename T>
int prefix_dispatch(AttnArgs<T> a, const int32_t* start, const int32_t* len, int n, void* ws, int64_t ws_bytes,
                    int64_t need, hipStream_t st) {
  int rc = NVF_OK;
  if (need > 0 && ws && ws_bytes >= need && attn_mfma(a)) {
    by_groups(start, len, n, [&](const PrefixGroups& groups, int32_t first) {
      if (rc != NVF_OK) return;
      AttnArgs<T> b = a;
      b.q += first * a.q_stride;
      b.out += (int64_t)first * a.q_heads * a.hd;
      b.qseq += first;
      b.qlen += first;
      b.tokens = groups.start[groups.n];
      const PrefixPlan p =
          prefix_plan(groups, a.q_heads, a.kv_heads, a.hd, (int64_t)a.bs * a.max_blocks, (int)sizeof(T));
      b.nsplit = p.splits + p.own_splits;
      b.part = static_cast<float*>(ws);
      if (a.hd == 64) prefix_mfma<T, 64>(b, groups, p, st);
      else prefix_mfma<T, 128>(b, groups, p, st);
      rc = launch_status("prefix_attention");
      if (rc == NVF_OK) rc = launch_attn_join(b, "prefix_attention(join)", st);
    });
    return rc;
  }
  launch_attn_any(a, WindowRule{INT32_MAX, 0}, st);
  return launch_status("prefix_attention");
}

}  // namespace nvf

using namespace nvf;

extern "C" {

int64_t nvf_prefix_attention_workspace_size(const int32_t* group_start_host, const int32_t* prefix_len_host,
                                            int num_groups, int q_heads, int kv_heads, int head_dim, int block_size,
                                            int max_blocks) {
  if (!group_start_host || !prefix_len_host || num_groups <= 0 || q_heads <= 0 || kv_heads <= 0 || block_size <= 0 ||
      max_blocks <= 0 || q_heads % kv_heads || !prefix_shape(q_heads, kv_heads, head_dim, block_size))
    return 0;
  for (int g = 0; g < num_groups; ++g)
    if (group_start_host[g] < 0 || group_start_host[g + 1] < group_start_host[g]) return 0;
  int64_t most = 0;
  by_groups(group_start_host, prefix_len_host, num_groups, [&](const PrefixGroups& groups, int32_t) {
    for (const int bytes : {2, 4}) {
      const PrefixPlan p = prefix_plan(groups, q_heads, kv_heads, head_dim, (int64_t)block_size * max_blocks, bytes);
      most = std::max(most, part_bytes(groups.start[groups.n], q_heads, head_dim, p.splits + p.own_splits));
    }
  });
  return most;
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
      group_start_host, prefix_len_host, num_groups, workspace, workspace_bytes,
      nvf_prefix_attention_workspace_size(group_start_host, prefix_len_host, num_groups, q_heads, kv_heads, head_dim,
                                          block_size, max_blocks),
      as_stream(stream)));
  return rc;
}

}  // extern "C"
