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

// Tile x = (tile, kv head), kv heads innermost: with 8 (or 4, 2, 1) kv heads an XCD, which takes every 8th
// workgroup, keeps the keys of few heads in its L2.
template <typename T, int HD>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) void window_tile_kernel(
    const AttnArgs<T> a, const FastDiv div, const WindowRule rule, int tile_tokens, int64_t tiles) {
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int64_t tile = tiles - 1 - blockIdx.x / a.kv_heads, t0 = tile * tile_tokens;
  const int kvh = (int)(blockIdx.x % a.kv_heads);
  const int end = a.tokens - t0 < tile_tokens ? (int)(a.tokens - t0) : tile_tokens;
  const TileRuns runs(a.qseq, t0, end);
  if (runs.count() > kTileMaxRuns) return;  // the whole workgroup: window_token_kernel's
  int r0 = 0;
#pragma unroll 1
  while (true) {
    const int r1 = runs.end_after(r0, end);
    const TileJob job{t0,        r0, r1, __builtin_amdgcn_readfirstlane(a.qseq[t0 + r0]), kvh, INT32_MAX,
                      (int)blockIdx.z, a.nsplit, blockIdx.z};
    tile_of<T, HD, true>(a, div, rule, job, lds);
    r0 = r1;
    if (r0 >= end) break;
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
// Key ranges for a call with few workgroups: enough to fill the GPU, each of some chunks.
inline int window_split(int64_t tokens, int q_heads, int kv_heads, int hd, int bs, int max_blocks, int64_t window,
                        int64_t sinks, int64_t max_query_len) {
  if ((hd != 64 && hd != 128) || bs % 16) return 1;
  const int tq = window_tile_tokens(tokens, q_heads, kv_heads, max_query_len);
  const int64_t wgs = tq ? (tokens + tq - 1) / tq * kv_heads : tokens * kv_heads * ((q_heads / kv_heads + 15) / 16);
  const int64_t keys = std::min<int64_t>((int64_t)bs * max_blocks, std::min<int64_t>(window, INT32_MAX) + tq + std::min<int64_t>(sinks, INT32_MAX));
  const int64_t chunks = keys / kChunk + 2;
  const int64_t want = tq ? 768 : 512, least = tq ? 8 : 4;  // workgroups; chunks of a range
  if (wgs * 2 > want) return 1;
  return (int)std::max<int64_t>(1, std::min<int64_t>({want / wgs, chunks / least, 64}));
}

// Whether the host knows the tiles that window_tile_kernel leaves, and their tokens [first, end).
struct LeftTokens {
  bool known = false;
  int64_t first = 0, end = 0;
};
inline LeftTokens left_tokens(const int32_t* cu, int num_seqs, int tile_tokens) {
  LeftTokens left;
  left.known = true;
  int64_t tile = -1;
  int runs = 0;
  const auto close = [&] {
    if (tile < 0 || runs <= kTileMaxRuns) return;
    if (left.end == 0) left.first = tile * tile_tokens;
    left.end = (tile + 1) * tile_tokens;
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
  left.end = std::min<int64_t>(left.end, cu[num_seqs]);
  return left;
}

template <typename T, int HD>
int window_mfma(AttnArgs<T> a, const WindowRule& rule, int tile_tokens, const LeftTokens& left, hipStream_t st) {
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
    const int64_t tiles = (a.tokens + tile_tokens - 1) / tile_tokens;
    window_tile_kernel<T, HD><<<dim3((unsigned)(tiles * a.kv_heads), 1, nz), 256, TileLds<T, HD>::kBytes, st>>>(
        a, div, rule, tile_tokens, tiles);
    const int64_t items = left.known ? left.end - left.first : tiles;
    if (items > 0)
      window_token_kernel<T, HD><<<dim3((unsigned)(items * a.kv_heads * parts), 1, nz), 256, TokenLds<T, HD>::kBytes, st>>>(
          a, div, rule, left.first, tile_tokens, !left.known);
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
                                  max_query_len);
  a.part = static_cast<float*>(ws);
  a.nsplit = ws && ws_bytes >= part_bytes(a.tokens, a.q_heads, a.hd, nsplit) ? nsplit : 1;
  int rc;
  if (attn_mfma(a)) {
    const int tq = window_tile_tokens(a.tokens, a.q_heads, a.kv_heads, max_query_len);
    const LeftTokens left = tq && cu ? left_tokens(cu, a.num_seqs, tq) : LeftTokens{};
    rc = a.hd == 64 ? window_mfma<T, 64>(a, rule, tq, left, st) : window_mfma<T, 128>(a, rule, tq, left, st);
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
  return part_bytes(tokens, q_heads, head_dim,
                    window_split(tokens, q_heads, kv_heads, head_dim, block_size, max_blocks, window, sinks,
                                 max_query_len));
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
