// Paged attention over a sliding window and a few first keys (sinks): token t with key count L
// sees keys j < L with j >= L - window or j < sinks.
//
//   out[t, h] = sum_j p_j V_j / sum_j p_j,  p_j = exp(scale q[t, h] . K_j - max)
//
// over the keys that it sees (zeros if none), online over chunks of 64 keys.
//
// * window_tile_kernel: prompts, 128 (token, head) rows of one kv head a workgroup;
// * window_token_kernel: single tokens, a workgroup each and kv head;
// * attn_any_kernel: every other shape.
// Calls with few workgroups over long windows are cut into key ranges and joined.
#include "attention_tiles.hpp"

#include <mutex>

namespace nvf {

// The sequences' first tokens, where the host knows the packing and there are few (n = 0: it does not): a tile
// then holds one sequence's tokens.  Otherwise tiles are cut from the batch as it is and walk their runs; a tile
// of two sequences takes twice as long as the others (fp32, 700 and 300 tokens, window 2048: 422 us, and
// 294 us with each sequence's own tiles).
constexpr int kMaxSeqs = 64;
struct SeqStarts {
  int n;
  int start[kMaxSeqs + 1];
};

// Tile x = (tile, kv head), kv heads innermost: with 8 (or 4, 2, 1) kv heads an XCD, which takes every 8th
// workgroup, keeps the keys of few heads in its L2.
template <typename T, int HD>
__global__ __launch_bounds__(kTileThreads<T>)
__attribute__((amdgpu_waves_per_eu(sizeof(T) == 4 && HD == 64 ? 4 : 2))) void window_tile_kernel(
    const AttnArgs<T> a, const FastDiv div, const WindowRule rule, int tile_tokens, int tiles, const SeqStarts seqs) {
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int tile = tiles - 1 - (int)(blockIdx.x / a.kv_heads), kvh = (int)(blockIdx.x % a.kv_heads);
  TileAt at{0, 0, (int64_t)tile * tile_tokens};
  if (seqs.n > 0) at = tile_at(seqs.start, seqs.n, tile, tile_tokens);
  else at.n = a.tokens - at.t0 < tile_tokens ? (int)(a.tokens - at.t0) : tile_tokens;
  const TileRuns runs(a.qseq, at.t0, at.n);
  if (runs.count() > kTileMaxRuns) return;  // the whole workgroup: window_token_kernel's
  int r0 = 0;
#pragma unroll 1
  while (true) {
    const int r1 = runs.end_after(r0, at.n);
    const TileJob job{at.t0,     r0, r1, __builtin_amdgcn_readfirstlane(a.qseq[at.t0 + r0]), kvh, INT32_MAX,
                      (int)blockIdx.z, a.nsplit, blockIdx.z};
    tile_of<T, HD, true>(a, div, rule, job, lds);
    r0 = r1;
    if (r0 >= at.n) break;
    __syncthreads();  // the next run's chunks reuse the LDS
  }
}

// tile_tokens == 0: workgroup x = (token - first, kv head, 16 heads).  Otherwise the tokens of tiles that
// window_tile_kernel leaves: walk: x = (tile, kv head, 16 heads), token by token; else as above, from
// token `first` on.
template <typename T, int HD>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) void window_token_kernel(
    const AttnArgs<T> a, const FastDiv div, const WindowRule rule, int64_t first, int tile_tokens, bool walk) {
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int parts = (a.q_heads / a.kv_heads + 15) / 16;
  const int rest = (int)(blockIdx.x % (a.kv_heads * parts));
  const int64_t x = blockIdx.x / (a.kv_heads * parts);
  int64_t t = walk ? x * tile_tokens : first + x, t1 = t + 1;
  if (tile_tokens > 0) {
    const int64_t t0 = t / tile_tokens * tile_tokens;
    const int n = a.tokens - t0 < tile_tokens ? (int)(a.tokens - t0) : tile_tokens;
    if (TileRuns(a.qseq, t0, n).count() <= kTileMaxRuns) return;
    if (walk) t1 = t0 + n;
  }
#pragma unroll 1
  for (; t < t1; ++t) {
    token_of<T, HD>(a, div, rule, t, rest / parts, rest % parts, (int)blockIdx.z, a.nsplit, blockIdx.z, lds);
    if (t + 1 < t1) __syncthreads();  // the next token's keys reuse the LDS
  }
}

// Tiles unless the caller promised single tokens, or there are no more rows than one token's MFMAs take.
inline int window_tile_tokens(int64_t tokens, int q_heads, int kv_heads, int64_t max_query_len) {
  const int G = q_heads / kv_heads;
  return max_query_len != 1 && G <= kTileRows / 2 && tokens * G > 16 ? kTileRows / G : 0;
}
// Key ranges for a call with few workgroups.
inline int window_split(int64_t tokens, int q_heads, int kv_heads, int hd, int bs, int max_blocks, int64_t window,
                        int64_t sinks, int64_t max_query_len, int dtype_bytes) {
  if ((hd != 64 && hd != 128) || bs % 16) return 1;
  const int tq = window_tile_tokens(tokens, q_heads, kv_heads, max_query_len);
  const int64_t most = INT32_MAX;
  const int64_t keys = std::min<int64_t>((int64_t)bs * max_blocks, std::min(window, most) + tq + std::min(sinks, most));
  const int64_t chunks = (keys + kChunk - 1) / kChunk + 1;
  if (tq) return tile_split((tokens + tq - 1) / tq * kv_heads, chunks, tokens * q_heads, hd, dtype_bytes);
  return token_split(tokens * kv_heads * ((q_heads / kv_heads + 15) / 16), chunks, tokens * q_heads, hd);
}

// What the packing on the host says: the sequences, if they are few; else the tokens [first, end) of the tiles that
// window_tile_kernel leaves.
struct TilePlan {
  bool known = false;
  int64_t first = 0, end = 0;
  SeqStarts seqs{};
};
inline TilePlan tile_plan(const int32_t* cu, int num_seqs, int tile_tokens) {
  TilePlan plan;
  plan.known = true;
  int n = 0;
  for (int s = 0; s < num_seqs && n <= kMaxSeqs; ++s) {
    if (cu[s] == cu[s + 1]) continue;
    if (n < kMaxSeqs) {
      plan.seqs.start[n] = cu[s];
      plan.seqs.start[n + 1] = cu[s + 1];
    }
    ++n;
  }
  if (n <= kMaxSeqs) {
    plan.seqs.n = n;
    return plan;
  }
  plan.seqs = SeqStarts{};
  int64_t tile = -1;
  int runs = 0;
  const auto close = [&] {
    if (tile < 0 || runs <= kTileMaxRuns) return;
    if (plan.end == 0) plan.first = tile * tile_tokens;
    plan.end = (tile + 1) * tile_tokens;
  };
  for (int s = 0; s < num_seqs; ++s) {
    if (cu[s] == cu[s + 1]) continue;
    const int64_t b = cu[s] / tile_tokens, e = (cu[s + 1] - 1) / tile_tokens;  // its first and last tile
    if (b != tile) {
      close();
      tile = b;
      runs = 0;
    }
    ++runs;
    if (e != tile) {
      close();
      tile = e;
      runs = 1;
    }
  }
  close();
  plan.end = std::min<int64_t>(plan.end, cu[num_seqs]);
  return plan;
}

template <typename T, int HD>
int window_mfma(AttnArgs<T> a, const WindowRule& rule, int tile_tokens, const TilePlan& plan, hipStream_t st) {
  static std::once_flag lds_once;
  std::call_once(lds_once, [] {
    (void)hipFuncSetAttribute(reinterpret_cast<const void*>(&window_tile_kernel<T, HD>),
                              hipFuncAttributeMaxDynamicSharedMemorySize, TileLds<T, HD>::kBytes);
    (void)hipFuncSetAttribute(reinterpret_cast<const void*>(&window_token_kernel<T, HD>),
                              hipFuncAttributeMaxDynamicSharedMemorySize, TokenLds<T, HD>::kBytes);
  });
  const FastDiv div((uint32_t)a.bs);
  const int parts = (a.q_heads / a.kv_heads + 15) / 16;
  const unsigned nz = (unsigned)a.nsplit;
  if (tile_tokens) {
    const int tiles = plan.seqs.n > 0 ? tiles_of(plan.seqs.start, plan.seqs.n, tile_tokens)
                                      : (int)((a.tokens + tile_tokens - 1) / tile_tokens);
    window_tile_kernel<T, HD><<<dim3((unsigned)(tiles * a.kv_heads), 1, nz), kTileThreads<T>, TileLds<T, HD>::kBytes, st>>>(
        a, div, rule, tile_tokens, tiles, plan.seqs);
    const int64_t items = plan.known ? plan.end - plan.first : tiles;
    if (items > 0)
      window_token_kernel<T, HD><<<dim3((unsigned)(items * a.kv_heads * parts), 1, nz), 256, TokenLds<T, HD>::kBytes, st>>>(
          a, div, rule, plan.first, tile_tokens, !plan.known);
  } else {
    window_token_kernel<T, HD><<<dim3((unsigned)(a.tokens * a.kv_heads * parts), 1, nz), 256, TokenLds<T, HD>::kBytes, st>>>(
        a, div, rule, 0, 0, false);
  }
  return launch_status("window_attention");
}

template <typename T>
int window_dispatch(AttnArgs<T> a, const WindowRule& rule, int64_t max_query_len, const int32_t* cu, void* ws,
                    int64_t ws_bytes, hipStream_t st) {
  const int nsplit = window_split(a.tokens, a.q_heads, a.kv_heads, a.hd, a.bs, a.max_blocks, rule.window, rule.sinks,
                                  max_query_len, (int)sizeof(T));
  a.part = static_cast<float*>(ws);
  a.nsplit = ws && ws_bytes >= part_bytes(a.tokens, a.q_heads, a.hd, nsplit) ? nsplit : 1;
  int rc;
  if (attn_mfma(a)) {
    const int tq = window_tile_tokens(a.tokens, a.q_heads, a.kv_heads, max_query_len);
    const TilePlan plan = tq && cu ? tile_plan(cu, a.num_seqs, tq) : TilePlan{};
    rc = a.hd == 64 ? window_mfma<T, 64>(a, rule, tq, plan, st) : window_mfma<T, 128>(a, rule, tq, plan, st);
  } else {
    launch_attn_any(a, rule, st);
    rc = launch_status("window_attention");
  }
  return rc == NVF_OK && a.nsplit > 1 ? launch_attn_join(a, "window_attention(join)", st) : rc;
}

}  // namespace nvf

using namespace nvf;

extern "C" {

int64_t nvf_window_attention_workspace_size(int64_t tokens, int q_heads, int kv_heads, int head_dim, int block_size,
                                            int max_blocks, int64_t window, int64_t sinks, int64_t max_query_len) {
  if (tokens <= 0 || q_heads <= 0 || kv_heads <= 0 || head_dim <= 0 || block_size <= 0 || max_blocks <= 0 ||
      q_heads % kv_heads || window < 0 || sinks < 0)
    return 0;
  const auto split = [&](int dtype_bytes) {
    return window_split(tokens, q_heads, kv_heads, head_dim, block_size, max_blocks, window, sinks, max_query_len,
                        dtype_bytes);
  };
  return part_bytes(tokens, q_heads, head_dim, std::max(split(2), split(4)));
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
      rule, max_query_len, cu_seqlens_host, workspace, workspace_bytes, as_stream(stream)));
  return rc;
}

}  // extern "C"
