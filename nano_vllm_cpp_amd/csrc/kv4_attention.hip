// Paged attention over a 4-bit cache (kv4.hpp): token t with key count L sees the first L keys of its sequence.
//
//   out[t, h] = sum_j p_j V_j / sum_j p_j,  p_j = exp(scale q[t, h] . K_j - max)
//
// over the cached values d (n - z) (zeros if there are no keys), online over chunks of 64 keys.
#include "attention_tiles.hpp"
#include "kv4.hpp"

#include <mutex>

namespace nvf {

template <typename T>
struct Kv4Args : AttnArgs<T> {
  const uint8_t *k, *v;  // the caches
  int64_t row_bytes;
  int words;  // where a row's words begin
};

// ---------------------------------------------------------------------------
// Any head size, block size and head group, as attn_any_kernel: a workgroup is GH query heads of one (token, kv head), its 4
// waves take the chunks in turn; a lane is a key in the scores and head dimensions lane + 64 i in P . V; fp32 math.
template <typename T, int GH, int DPL>
__global__ __launch_bounds__(kGenWaves * 64) void kv4_any_kernel(const Kv4Args<T> a) {
  __shared__ GenLds<T, GH, DPL> s;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int G = a.q_heads / a.kv_heads, parts = (G + GH - 1) / GH;
  const int64_t t = blockIdx.x / (a.kv_heads * parts);
  const int rest = (int)(blockIdx.x % (a.kv_heads * parts));
  const int kvh = rest / parts, h0 = kvh * G + rest % parts * GH;
  const int heads = min(GH, (kvh + 1) * G - h0);
  const int L = key_count(a, t), seq = a.qseq[t], groups = a.hd / kKv4Group;
  const int code_at = kvh * (a.hd / 2), word_at = a.words + kvh * (a.hd / 16);
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
  const ChunkList list(0, L, 0);
  const int c1 = list.split_begin((int)blockIdx.z + 1, a.nsplit);
  for (int c = list.split_begin((int)blockIdx.z, a.nsplit) + w; c < c1; c += kGenWaves) {
    const int key = c * kChunk + lane;
    const bool seen = key < L;
    const uint64_t seen_mask = __ballot(seen);
    const int block = seen ? key_block(a, seq, key) : -1;
    const int64_t row = block >= 0 ? (int64_t)block * a.bs + key % a.bs : 0;
    float sc[GH];
#pragma unroll
    for (int g = 0; g < GH; ++g) sc[g] = block >= 0 ? 0.0f : __builtin_nanf("");
    if (block >= 0) {
      const uint8_t* kp = a.k + row * a.row_bytes;
      for (int gr = 0; gr < groups; ++gr) {
        const u32x4 codes = ld16(kp + code_at + 16 * gr);
        const uint32_t word = *reinterpret_cast<const uint16_t*>(kp + word_at + 2 * gr);
        const float scale = kv4_scale(word);
        const int z = (int)(word & 15u);
#pragma unroll
        for (int e = 0; e < kKv4Group; ++e) {
          const float kv = scale * (float)((int)(codes[e / 8] >> (4 * (e % 8)) & 15u) - z);
#pragma unroll
          for (int g = 0; g < GH; ++g) sc[g] = fmaf(s.q[g][kKv4Group * gr + e], kv, sc[g]);
        }
      }
    }
    s.row[w][lane] = row;
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
    for (uint64_t left = seen_mask; left; left &= left - 1) {
      const int j = __builtin_ctzll(left);
      const uint8_t* vp = a.v + s.row[w][j] * a.row_bytes;
#pragma unroll
      for (int i = 0; i < DPL; ++i) {
        const int d = lane + 64 * i;
        float v = 0.0f;
        if (d < a.hd)
          v = kv4_value(*reinterpret_cast<const uint16_t*>(vp + word_at + 2 * (d / kKv4Group)),
                        (uint32_t)vp[code_at + d / 2] >> (4 * (d & 1)) & 15u);
#pragma unroll
        for (int g = 0; g < GH; ++g) acc[g][i] = fmaf(s.p[w][g][j], v, acc[g][i]);
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
void launch_kv4_any(const Kv4Args<T>& a, hipStream_t st) {
  const int G = a.q_heads / a.kv_heads;
  const auto by_group = [&](auto dpl) {
    constexpr int DPL = decltype(dpl)::value;
    const auto launch = [&](auto gh) {
      constexpr int GH = decltype(gh)::value;
      const dim3 grid((unsigned)(a.tokens * a.kv_heads * ((G + GH - 1) / GH)), 1, (unsigned)a.nsplit);
      kv4_any_kernel<T, GH, DPL><<<grid, kGenWaves * 64, 0, st>>>(a);
    };
    if (G == 1) launch(std::integral_constant<int, 1>{});
    else if (G <= 4) launch(std::integral_constant<int, 4>{});
    else launch(std::integral_constant<int, 8>{});
  };
  if (a.hd <= 64) by_group(std::integral_constant<int, 1>{});
  else if (a.hd <= 128) by_group(std::integral_constant<int, 2>{});
  else by_group(std::integral_constant<int, 4>{});
}

template <typename T>
int kv4_dispatch(const Kv4Args<T>& a, hipStream_t st) {
  launch_kv4_any(a, st);
  return launch_status("paged_attention_kv4");
}

}  // namespace nvf

using namespace nvf;

extern "C" {

int64_t nvf_paged_attention_kv4_workspace_size(int64_t tokens, int q_heads, int kv_heads, int head_dim, int block_size,
                                               int max_blocks, int64_t max_query_len) {
  return 0;
}

int nvf_paged_attention_kv4_ws(const void* q, void* out, const void* k_cache, const void* v_cache,
                               const int32_t* query_seq, const int32_t* query_key_len, const int32_t* block_tables,
                               const int32_t* cu_seqlens_host, int num_seqs, int64_t tokens, int q_heads, int kv_heads,
                               int head_dim, int block_size, int max_blocks, int64_t num_blocks, float scale,
                               int64_t q_stride, int64_t max_query_len, void* workspace, int64_t workspace_bytes,
                               int dtype, void* stream) {
  const char* who = "nvf_paged_attention_kv4";
  const int rc0 = check_attn(who, q, out, k_cache, v_cache, query_seq, query_key_len, block_tables, tokens, q_heads,
                             kv_heads, head_dim, block_size, max_blocks, num_seqs, num_blocks, q_stride, workspace,
                             dtype);
  if (rc0 != NVF_OK) return rc0;
  if (!kv4_head_dim_ok(head_dim))
    return fail(NVF_ERR_INVALID, "%s: head_dim=%d is not a multiple of %d", who, head_dim, kKv4Group);
  if (cu_seqlens_host) {
    const int rc1 = check_packing(who, cu_seqlens_host, num_seqs, tokens);
    if (rc1 != NVF_OK) return rc1;
  }
  if (tokens == 0) return NVF_OK;
  if (!aligned16(k_cache) || !aligned16(v_cache))
    return fail(NVF_ERR_INVALID, "%s: the caches must be 16-byte aligned", who);
  int rc = NVF_OK;
  NVF_DISPATCH_DTYPE(dtype, T, {
    Kv4Args<T> a;
    static_cast<AttnArgs<T>&>(a) =
        attn_args<T>(q, out, nullptr, nullptr, query_seq, query_key_len, block_tables, tokens, q_heads, kv_heads,
                     head_dim, block_size, max_blocks, num_seqs, num_blocks, scale, q_stride);
    a.k = static_cast<const uint8_t*>(k_cache);
    a.v = static_cast<const uint8_t*>(v_cache);
    a.row_bytes = kv4_row_bytes(kv_heads, head_dim);
    a.words = kv_heads * (head_dim / 2);
    rc = kv4_dispatch<T>(a, as_stream(stream));
  });
  return rc;
}

}  // extern "C"
