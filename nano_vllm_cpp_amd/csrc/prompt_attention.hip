// Causal attention of packed prompts over their own keys and values: rows of q, k and v, no pages.  Tokens
// cu[s] .. cu[s + 1] - 1 are sequence s; token t of it sees the rows cu[s] .. t.
//
//   out[t, h] = sum_j p_j V_j / sum_j p_j,  p_j = exp(scale q[t, h] . K_j - max)
//
// online over chunks of 64 keys.  The packing lies on the device, so a captured call follows what later
// replays find there; entries are taken into [0, tokens], and tokens of no sequence are left as they are.
#include "attention_tiles.hpp"

#include <mutex>

namespace nvf {

struct PromptRows {
  const int32_t* cu;
  int num_seqs;
};

// The first token of t's sequence, -1 where it has none: the last sequence that begins at or before t.
__device__ __forceinline__ int64_t prompt_start(const PromptRows& p, int64_t t, int64_t tokens) {
  int lo = 0, hi = p.num_seqs;  // cu[lo] <= t < cu[hi], where t lies in a sequence
  if (t < p.cu[0] || t >= p.cu[hi]) return -1;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (p.cu[mid] <= t) lo = mid;
    else hi = mid;
  }
  return max(p.cu[lo], 0);
}

// ---------------------------------------------------------------------------
// Any head size up to 256, type, stride, alignment and head group, as attn_any_kernel.
template <typename T, int GH, int DPL>
__global__ __launch_bounds__(kGenWaves * 64) void prompt_any_kernel(const AttnArgs<T> a, const PromptRows rows) {
  constexpr int N = Pack<T>::N;
  __shared__ GenLds<T, GH, DPL> s;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int G = a.q_heads / a.kv_heads, parts = (G + GH - 1) / GH;
  const int64_t t = blockIdx.x / (a.kv_heads * parts);
  const int rest = (int)(blockIdx.x % (a.kv_heads * parts));
  const int kvh = rest / parts, h0 = kvh * G + rest % parts * GH;
  const int heads = min(GH, (kvh + 1) * G - h0);
  const int64_t start = prompt_start(rows, t, a.tokens);
  if (start < 0) return;  // the whole workgroup: no sequence's token
  const int L = (int)(t - start) + 1;
  for (int i = threadIdx.x; i < GH * 64 * DPL; i += kGenWaves * 64) {
    const int g = i / (64 * DPL), d = i % (64 * DPL);
    s.q[g][d] = g < heads && d < a.hd ? to_f32(a.q[t * a.q_stride + (int64_t)(h0 + g) * a.hd + d]) : 0.0f;
  }
  __syncthreads();

  float m[GH], l[GH], acc[GH][DPL];
#pragma unroll
  for (int g = 0; g < GH; ++g) {
    m[g] = -INFINITY;
    l[g] = 0.0f;
#pragma unroll
    for (int i = 0; i < DPL; ++i) acc[g][i] = 0.0f;
  }
  const T* k = a.kc + start * a.k_stride + (int64_t)kvh * a.hd;
  const T* v = a.vc + start * a.v_stride + (int64_t)kvh * a.hd;
  for (int c = w; c < (L + kChunk - 1) / kChunk; c += kGenWaves) {
    const int key = c * kChunk + lane;
    const bool seen = key < L;
    float sc[GH];
#pragma unroll
    for (int g = 0; g < GH; ++g) sc[g] = 0.0f;
    if (seen) {
      const T* kp = k + key * a.k_stride;
      if (a.vec) {
        for (int d0 = 0; d0 < a.hd; d0 += N) {
          float kv[N];
          Pack<T>::unpack(ld16(kp + d0), kv);
#pragma unroll
          for (int g = 0; g < GH; ++g)
#pragma unroll
            for (int e = 0; e < N; ++e) sc[g] = fmaf(s.q[g][d0 + e], kv[e], sc[g]);
        }
      } else {
        for (int d = 0; d < a.hd; ++d) {
          const float kv = to_f32(kp[d]);
#pragma unroll
          for (int g = 0; g < GH; ++g) sc[g] = fmaf(s.q[g][d], kv, sc[g]);
        }
      }
    }
#pragma unroll
    for (int g = 0; g < GH; ++g) {
      const float x = seen ? sc[g] * a.scale_log2 : -INFINITY;
      const float m_new = fmaxf(m[g], wave_max(x));
      const float m_use = m_new == -INFINITY ? 0.0f : m_new;
      const float alpha = __builtin_amdgcn_exp2f(m[g] - m_use);
      const float p = __builtin_amdgcn_exp2f(x - m_use);
      l[g] = l[g] * alpha + wave_sum(p);
      m[g] = m_new;
      s.p[w][g][lane] = p;
#pragma unroll
      for (int i = 0; i < DPL; ++i) acc[g][i] *= alpha;
    }
    __builtin_amdgcn_wave_barrier();  // wave-private LDS: other lanes read what this wave wrote
    const int n = min(kChunk, L - c * kChunk);
    for (int j = 0; j < n; ++j) {
      const T* vp = v + (int64_t)(c * kChunk + j) * a.v_stride;
#pragma unroll
      for (int i = 0; i < DPL; ++i) {
        const int d = lane + 64 * i;
        const float x = d < a.hd ? to_f32(vp[d]) : 0.0f;
#pragma unroll
        for (int g = 0; g < GH; ++g) acc[g][i] = fmaf(s.p[w][g][j], x, acc[g][i]);
      }
    }
    __builtin_amdgcn_wave_barrier();  // the chunk's reads before the next one's writes
  }

#pragma unroll
  for (int g = 0; g < GH; ++g) {
#pragma unroll
    for (int i = 0; i < DPL; ++i) s.acc[w][g][lane + 64 * i] = acc[g][i];
    if (lane == 0) {
      s.m[w][g] = m[g];
      s.l[w][g] = l[g];
    }
  }
  __syncthreads();
  gen_join(a, s, t, h0, heads);
}

template <typename T>
void launch_prompt_any(const AttnArgs<T>& a, const PromptRows& rows, hipStream_t st) {
  const int G = a.q_heads / a.kv_heads;
  const auto by_group = [&](auto dpl) {
    constexpr int DPL = decltype(dpl)::value;
    const auto launch = [&](auto gh) {
      constexpr int GH = decltype(gh)::value;
      const dim3 grid((unsigned)(a.tokens * a.kv_heads * ((G + GH - 1) / GH)));
      prompt_any_kernel<T, GH, DPL><<<grid, kGenWaves * 64, 0, st>>>(a, rows);
    };
    if (G == 1) launch(std::integral_constant<int, 1>{});
    else if (G <= 4) launch(std::integral_constant<int, 4>{});
    else launch(std::integral_constant<int, 8>{});
  };
  if (a.hd <= 64) by_group(std::integral_constant<int, 1>{});
  else if (a.hd <= 128) by_group(std::integral_constant<int, 2>{});
  else by_group(std::integral_constant<int, 4>{});
}

// ---------------------------------------------------------------------------
// Tile x of the packing: a sequence's first token, and tokens t0 + [0, n) of it.  n = 0: there are fewer tiles.
// Up to 64 sequences: in the order of the tiles' places in their sequences, the last ones first, so that the work of
// a tile falls from first to last and the last workgroups are short: prompts of 4096, 1500, 777, 64 and 1 tokens 158
// us, sequence after sequence 162.  More: sequence after sequence, of each the last tile first.
struct PromptTile {
  int64_t start, t0;
  int n;
};
__device__ __forceinline__ PromptTile prompt_tile(const PromptRows& p, int x, int tile_tokens, int64_t tokens) {
  const int lane = threadIdx.x & 63;
  int first = 0, end = 0;
  const auto tiles_of_lane = [&](int s) {  // a lane a sequence
    first = end = 0;
    if (s >= 0 && s < p.num_seqs) {
      first = (int)min(max((int64_t)p.cu[s], (int64_t)0), tokens);
      end = (int)min(max((int64_t)p.cu[s + 1], (int64_t)first), tokens);
    }
    return (end - first + tile_tokens - 1) / tile_tokens;
  };
  const auto pick = [&](int j, int tile) {
    const int a = __builtin_amdgcn_readlane(first, j), b = __builtin_amdgcn_readlane(end, j);
    return PromptTile{a, a + (int64_t)tile * tile_tokens, min(tile_tokens, b - a - tile * tile_tokens)};
  };
  if (p.num_seqs <= 64) {
    const int tiles = tiles_of_lane(lane);
    // how many tiles have a place from j on
    const auto from = [&](int j) {
      int n = 0;
      for (int s = 0; s < p.num_seqs; ++s) n += max(__builtin_amdgcn_readlane(tiles, s) - j, 0);
      return n;
    };
    int lo = 0, hi = __builtin_amdgcn_readfirstlane(wave_max_int(tiles));
    if (from(0) <= x) return PromptTile{0, 0, 0};
    while (hi - lo > 1) {  // from(lo) > x >= from(hi); 64 places between them at a time
      const int step = (hi - lo + 63) / 64, past = __popcll(__ballot(from(lo + step * lane) > x));
      hi = min(hi, lo + step * past);
      lo += step * (past - 1);
    }
    const uint64_t here = __ballot(tiles > lo);
    const int rank = x - from(lo + 1);
    return pick(__builtin_ctzll(__ballot(tiles > lo && __popcll(here & ((uint64_t(1) << lane) - 1)) == rank)), lo);
  }
  for (int s0 = p.num_seqs; s0 > 0; s0 -= 64) {
    const int tiles = tiles_of_lane(s0 - 1 - lane);
    int sum = tiles;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int up = __shfl_up(sum, d);
      if (lane >= d) sum += up;
    }
    const uint64_t past = __ballot(sum > x);
    if (past) {
      const int j = __builtin_ctzll(past);
      return pick(j, __builtin_amdgcn_readlane(sum, j) - 1 - x);
    }
    x -= __builtin_amdgcn_readlane(sum, 63);
  }
  return PromptTile{0, 0, 0};
}

// Workgroup x = (tile, kv head), kv heads innermost: with 8 (or 4, 2, 1) kv heads an XCD, which takes every 8th
// workgroup, keeps the keys of few heads in its L2.
// Bound as the window's tiles are, by matrix units and vector instructions that overlap in part: a prompt of 8192
// tokens, 32 / 8 heads of 128, fp16, 555 us, 0.99 PFLOP/s of the keys that are seen; fp32 by its matrix units and few
// tiles, 1429 tokens 125 us.
template <typename T, int HD>
__global__ __launch_bounds__(kTileThreads<T>)
__attribute__((amdgpu_waves_per_eu(sizeof(T) == 4 && HD == 64 ? 4 : 2))) void prompt_tile_kernel(
    const AttnArgs<T> a, const PromptRows rows, int tile_tokens) {
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const PromptTile at = prompt_tile(rows, (int)(blockIdx.x / a.kv_heads), tile_tokens, a.tokens);
  if (at.n == 0) return;  // the whole workgroup
  const TileJob job{at.t0, 0, at.n, 0, (int)(blockIdx.x % a.kv_heads), INT32_MAX, (int)blockIdx.z, a.nsplit, blockIdx.z,
                    at.start};
  tile_of<T, HD, kPromptTile>(a, FastDiv{}, WindowRule{}, job, lds);
}

// (token, head) rows that lie in a sequence
struct PromptJoin {
  PromptRows rows;
  int64_t tokens;
  FastDiv heads;
  __device__ __forceinline__ bool has(int64_t r) const {
    return prompt_start(rows, heads.div((uint32_t)__builtin_amdgcn_readfirstlane((int)r)), tokens) >= 0;
  }
};

// Tokens of a tile; 0: its 128 rows do not hold two tokens' heads.
inline int prompt_tile_tokens(int q_heads, int kv_heads) {
  const int G = q_heads / kv_heads;
  return G <= kTileRows / 2 ? kTileRows / G : 0;
}
// No packing of num_seqs sequences has more tiles.
inline int64_t prompt_tiles(int num_seqs, int64_t tokens, int tile_tokens) {
  return std::min<int64_t>(tokens, (tokens + (int64_t)num_seqs * (tile_tokens - 1)) / tile_tokens);
}
// Key ranges for a call with few tiles.  The host does not know the lengths: the longest sequence is taken to be
// twice the mean.
inline int prompt_split(int num_seqs, int64_t tokens, int q_heads, int kv_heads, int hd, int dtype_bytes) {
  const int tq = prompt_tile_tokens(q_heads, kv_heads);
  if ((hd != 64 && hd != 128) || tq == 0) return 1;
  const int64_t longest = std::min(tokens, 2 * tokens / num_seqs + 1);
  return tile_split(prompt_tiles(num_seqs, tokens, tq) * kv_heads, (longest + kChunk - 1) / kChunk, tokens * q_heads, hd,
                    dtype_bytes);
}

template <typename T, int HD>
int prompt_mfma(const AttnArgs<T>& a, const PromptRows& rows, int tile_tokens, hipStream_t st) {
  static std::once_flag lds_once;
  std::call_once(lds_once, [] {
    (void)hipFuncSetAttribute(reinterpret_cast<const void*>(&prompt_tile_kernel<T, HD>),
                              hipFuncAttributeMaxDynamicSharedMemorySize, TileLds<T, HD>::kBytes);
  });
  const int64_t tiles = prompt_tiles(rows.num_seqs, a.tokens, tile_tokens);
  prompt_tile_kernel<T, HD><<<dim3((unsigned)(tiles * a.kv_heads), 1, (unsigned)a.nsplit), kTileThreads<T>,
                              TileLds<T, HD>::kBytes, st>>>(a, rows, tile_tokens);
  return launch_status("prompt_attention");
}

template <typename T>
int prompt_dispatch(AttnArgs<T> a, const PromptRows& rows, void* ws, int64_t ws_bytes, hipStream_t st) {
  const int tq = prompt_tile_tokens(a.q_heads, a.kv_heads);
  const int64_t most = INT32_MAX / 64 / (int64_t)sizeof(T);  // (16 rows' bytes are a buffer's)
  const bool tiles = (a.hd == 64 || a.hd == 128) && tq > 0 && a.scale_log2 > 0.0f && aligned16(a.q) && aligned16(a.out) &&
                     aligned16(a.kc) && aligned16(a.vc) && a.q_stride % Pack<T>::N == 0 && a.k_stride % Pack<T>::N == 0 &&
                     a.v_stride % Pack<T>::N == 0 && a.k_stride < most && a.v_stride < most;
  if (!tiles) {
    launch_prompt_any(a, rows, st);
    return launch_status("prompt_attention");
  }
  const int nsplit = prompt_split(rows.num_seqs, a.tokens, a.q_heads, a.kv_heads, a.hd, (int)sizeof(T));
  a.part = static_cast<float*>(ws);
  a.nsplit = ws && ws_bytes >= part_bytes(a.tokens, a.q_heads, a.hd, nsplit) ? nsplit : 1;
  const int rc = a.hd == 64 ? prompt_mfma<T, 64>(a, rows, tq, st) : prompt_mfma<T, 128>(a, rows, tq, st);
  if (rc != NVF_OK || a.nsplit == 1) return rc;
  return launch_attn_join(a, "prompt_attention(join)", st, PromptJoin{rows, a.tokens, FastDiv((uint32_t)a.q_heads)});
}

}  // namespace nvf

using namespace nvf;

extern "C" {

int64_t nvf_prompt_attention_workspace_size(int num_seqs, int64_t tokens, int q_heads, int kv_heads, int head_dim) {
  if (num_seqs <= 0 || tokens <= 0 || q_heads <= 0 || kv_heads <= 0 || head_dim <= 0 || q_heads % kv_heads) return 0;
  return part_bytes(tokens, q_heads, head_dim,
                    std::max(prompt_split(num_seqs, tokens, q_heads, kv_heads, head_dim, 2),
                             prompt_split(num_seqs, tokens, q_heads, kv_heads, head_dim, 4)));
}

int nvf_prompt_attention_ws(const void* q, const void* k, const void* v, void* out, const int32_t* cu_seqlens,
                            int num_seqs, int64_t tokens, int q_heads, int kv_heads, int head_dim, float scale,
                            int64_t q_stride, int64_t k_stride, int64_t v_stride, void* workspace,
                            int64_t workspace_bytes, int dtype, void* stream) {
  const char* who = "nvf_prompt_attention";
  if (!dtype_ok(dtype)) return fail(NVF_ERR_INVALID, "%s: bad dtype %d", who, dtype);
  if (num_seqs < 0 || tokens < 0 || q_heads <= 0 || kv_heads <= 0 || head_dim <= 0)
    return fail(NVF_ERR_INVALID, "%s: bad shape", who);
  if (q_heads % kv_heads != 0)
    return fail(NVF_ERR_INVALID, "%s: q_heads=%d is not a multiple of kv_heads=%d", who, q_heads, kv_heads);
  if (head_dim > 256) return fail(NVF_ERR_INVALID, "%s: head_dim=%d exceeds 256", who, head_dim);
  if (q_stride < (int64_t)q_heads * head_dim || k_stride < (int64_t)kv_heads * head_dim ||
      v_stride < (int64_t)kv_heads * head_dim)
    return fail(NVF_ERR_INVALID, "%s: a stride is shorter than its row", who);
  if (workspace && !aligned16(workspace)) return fail(NVF_ERR_INVALID, "%s: workspace must be 16-byte aligned", who);
  if (tokens == 0 || num_seqs == 0) return NVF_OK;
  if (!q || !k || !v || !out || !cu_seqlens) return fail(NVF_ERR_INVALID, "%s: NULL pointer", who);
  if (tokens * q_heads > INT32_MAX) return fail(NVF_ERR_INVALID, "%s: too many (token, head) pairs", who);
  const int64_t e = dtype_bytes(dtype), kn = (int64_t)kv_heads * head_dim, qn = (int64_t)q_heads * head_dim;
  const int64_t out_bytes = tokens * qn * e;
  if (bytes_overlap(out, out_bytes, q, ((tokens - 1) * q_stride + qn) * e) ||
      bytes_overlap(out, out_bytes, k, ((tokens - 1) * k_stride + kn) * e) ||
      bytes_overlap(out, out_bytes, v, ((tokens - 1) * v_stride + kn) * e))
    return fail(NVF_ERR_INVALID, "%s: out overlaps q, k or v", who);
  const PromptRows rows{cu_seqlens, num_seqs};
  int rc = NVF_OK;
  NVF_DISPATCH_DTYPE(dtype, T, {
    AttnArgs<T> a = attn_args<T>(q, out, k, v, nullptr, nullptr, nullptr, tokens, q_heads, kv_heads, head_dim, 16, 1,
                                 num_seqs, 0, scale, q_stride);
    a.vec = a.vec && k_stride % Pack<T>::N == 0;
    a.k_stride = k_stride;
    a.v_stride = v_stride;
    rc = prompt_dispatch<T>(a, rows, workspace, workspace_bytes, as_stream(stream));
  });
  return rc;
}

}  // extern "C"
