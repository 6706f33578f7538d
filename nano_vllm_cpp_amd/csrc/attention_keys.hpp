// What the window and prefix attention kernels share: which keys a token sees, where they
// lie in the paged cache, the kernel that takes any shape, and the merge of split softmax
// states.
//
// The keys that a token sees are [lo, L) and [0, sinks), L its key count.  Kernels walk them
// in chunks of 64: the sinks' chunks, then those from lo's on; a chunk holds each key once, so
// a sink that lies in or past lo's chunk comes with that one.  Key j of sequence s lies in
// cache row table[s][j / bs] * bs + j % bs.  A key whose table entry is not a block of the
// cache (or whose sequence is no row of the tables) is never read: its score is NaN, so the
// rows that see it are NaN, and the entries of keys that no token sees may hold anything.
#pragma once

#include <hip/hip_runtime.h>
#include <math.h>

#include <algorithm>

#include "nvf_device.hpp"
#include "nvf_host.hpp"

namespace nvf {

constexpr int kChunk = 64;  // keys

template <typename T>
struct AttnArgs {
  const T* q;
  T* out;
  const T* kc;
  const T* vc;
  const int32_t* qseq;
  const int32_t* qlen;
  const int32_t* tables;
  int64_t tokens, num_blocks, q_stride;
  int q_heads, kv_heads, hd, bs, max_blocks, num_seqs;
  int most_keys;     // one more than the block tables hold
  float scale_log2;  // scale * log2(e): scores in exp2 units
  bool vec;          // 16-byte K rows
  int nsplit;        // key ranges, each a softmax state in `part`
  float* part;       // [tokens][q_heads][nsplit][hd] unnormalised O, then [tokens][q_heads][nsplit][2] max, sum
};

// Token t's key count.  (Keys past the tables have no block, so one of them stands for all; counts below zero are none,
// and as they are would overflow in the masks' differences.)
template <typename T>
__device__ __forceinline__ int key_count(const AttnArgs<T>& a, int64_t t) {
  return max(min(a.qlen[t], a.most_keys), 0);
}

// The rules: the keys that token t with key count L sees are [lo, L) and [0, sinks).
struct WindowRule {
  int window, sinks;
  __device__ __forceinline__ int lo(int64_t, int L) const { return L > window ? L - window : 0; }
};

// Groups of consecutive tokens that share their first len keys; the rule leaves those out.
constexpr int kMaxGroups = 64;
struct PrefixGroups {
  int n;
  int start[kMaxGroups + 1];  // tokens
  int len[kMaxGroups];
};
struct SuffixRule {
  static constexpr int sinks = 0;
  PrefixGroups groups;
  __device__ __forceinline__ int lo(int64_t t, int) const {
    int len = 0;
    for (int g = 0; g < groups.n; ++g)  // uniform: scalar loads of the kernel's arguments
      if (t >= groups.start[g]) len = groups.len[g];
    return len;
  }
};

struct ChunkList {
  int ns, cw, n;  // sink chunks 0 .. ns - 1, then chunks from cw on; n in all
  __device__ __forceinline__ ChunkList(int lo, int L, int sinks) {
    cw = lo / kChunk;
    const int s = sinks < L ? sinks : L;
    ns = s > 0 ? (s - 1) / kChunk + 1 : 0;
    n = ns;
    if (L > lo) {
      ns = min(ns, cw);
      n = ns + (L - 1) / kChunk + 1 - cw;
    }
  }
  __device__ __forceinline__ int chunk(int i) const { return i < ns ? i : cw + i - ns; }
  // the list's part of split z
  __device__ __forceinline__ int split_begin(int z, int nsplit) const { return (int)((int64_t)n * z / nsplit); }
};

// The cache block of key j, -1 where there is none.
template <typename T>
__device__ __forceinline__ int key_block(const AttnArgs<T>& a, int seq, int j) {
  const int b = j / a.bs;
  if ((unsigned)seq >= (unsigned)a.num_seqs || b >= a.max_blocks) return -1;
  const int32_t e = a.tables[(int64_t)seq * a.max_blocks + b];
  return e >= 0 && e < a.num_blocks ? e : -1;
}

// ---------------------------------------------------------------------------
// Any head size up to 256, type, block size and head group: a workgroup is GH query heads of
// one (token, kv head), its 4 waves take the chunks in turn.  A lane is a key in the scores
// (its K row read once for the GH heads) and head dimensions lane + 64 i in P . V; fp32 math.
// Only keys that the token sees are read.
constexpr int kGenWaves = 4;

template <typename T, int GH, int DPL>
struct GenLds {
  float q[GH][64 * DPL];
  float p[kGenWaves][GH][kChunk];
  int64_t row[kGenWaves][kChunk];
  float acc[kGenWaves][GH][64 * DPL];
  float m[kGenWaves][GH], l[kGenWaves][GH];
};

template <typename T, int GH, int DPL, typename Rule>
__global__ __launch_bounds__(kGenWaves * 64) void attn_any_kernel(const AttnArgs<T> a, const Rule rule) {
  constexpr int N = Pack<T>::N;
  __shared__ GenLds<T, GH, DPL> s;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int G = a.q_heads / a.kv_heads, parts = (G + GH - 1) / GH;
  const int64_t t = blockIdx.x / (a.kv_heads * parts);
  const int rest = (int)(blockIdx.x % (a.kv_heads * parts));
  const int kvh = rest / parts, h0 = kvh * G + rest % parts * GH;
  const int heads = min(GH, (kvh + 1) * G - h0);
  const int L = key_count(a, t), lo = rule.lo(t, L), seq = a.qseq[t];
  const int64_t row_len = (int64_t)a.kv_heads * a.hd;
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
  const ChunkList list(lo, L, rule.sinks);
  const int c1 = list.split_begin((int)blockIdx.z + 1, a.nsplit);
  for (int c = list.split_begin((int)blockIdx.z, a.nsplit) + w; c < c1; c += kGenWaves) {
    const int key = list.chunk(c) * kChunk + lane;
    const bool seen = key < L && (key >= lo || key < rule.sinks);
    const uint64_t seen_mask = __ballot(seen);
    const int block = seen ? key_block(a, seq, key) : -1;
    const int64_t row = block >= 0 ? (int64_t)block * a.bs + key % a.bs : 0;
    float sc[GH];
#pragma unroll
    for (int g = 0; g < GH; ++g) sc[g] = block >= 0 ? 0.0f : __builtin_nanf("");
    if (block >= 0) {
      const T* kp = a.kc + row * row_len + (int64_t)kvh * a.hd;
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
      const T* vp = a.vc + s.row[w][j] * row_len + (int64_t)kvh * a.hd;
#pragma unroll
      for (int i = 0; i < DPL; ++i) {
        const int d = lane + 64 * i;
        const float v = d < a.hd ? to_f32(vp[d]) : 0.0f;
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
  for (int i = threadIdx.x; i < heads * a.hd; i += kGenWaves * 64) {
    const int g = i / a.hd, d = i % a.hd;
    float mx = -INFINITY, den = 0.0f, o = 0.0f;
#pragma unroll
    for (int k = 0; k < kGenWaves; ++k) mx = fmaxf(mx, s.m[k][g]);
#pragma unroll
    for (int k = 0; k < kGenWaves; ++k) {
      // (a wave without keys: m = -inf, l = O = 0; one whose scores were all NaN has m = -inf, l = NaN)
      const float sk = s.m[k][g] == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(s.m[k][g] - mx);
      den += s.l[k][g] * sk;
      o += s.acc[k][g][d] * sk;
    }
    const int64_t th = t * a.q_heads + h0 + g;
    if (a.nsplit > 1) {
      const int64_t pi = th * a.nsplit + blockIdx.z;
      a.part[pi * a.hd + d] = o;
      if (d == 0) {
        float* ml = a.part + a.tokens * a.q_heads * a.nsplit * a.hd + 2 * pi;
        ml[0] = mx;
        ml[1] = den;
      }
    } else {
      a.out[th * a.hd + d] = from_f32<T>(den == 0.0f ? 0.0f : o / den);
    }
  }
}

// out = sum_z 2^(m_z - M) O_z / sum_z 2^(m_z - M) l_z over a (token, head)'s split states
// (m_z = -inf: no keys, O_z = l_z = 0, or NaN scores alone, l_z = NaN).  LANES lanes of 4 dims a row, the
// others of the wave at every (64 / LANES)-th state; a state's max, sum and O are read together and
// joined online, four ahead.  A wave per (token, head).
template <typename T, int LANES>
__global__ __launch_bounds__(256) void attn_join_kernel(const float* __restrict__ part, T* __restrict__ out,
                                                        int64_t rows, int hd, int nsplit) {
  typedef float f4 __attribute__((ext_vector_type(4)));
  typedef float f2 __attribute__((ext_vector_type(2)));
  const int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, d = 4 * (lane % LANES);
  if (r >= rows || d >= hd) return;  // (no lane that stays asks one that left: the same LANES in every group leave)
  const float* ml = part + rows * nsplit * hd + 2 * r * nsplit;
  const float* po = part + r * nsplit * hd + d;
  const bool vec = hd % 4 == 0;
  float m = -INFINITY, den = 0.0f;
  f4 o = {0.0f, 0.0f, 0.0f, 0.0f};
  const auto add = [&](float mz, float lz, f4 oz) {
    const float mn = fmaxf(m, mz);
    const float so = m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
    const float sz = mz == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(mz - mn);
    den = den * so + lz * sz;
    o = o * so + oz * sz;
    m = mn;
  };
#pragma unroll 4
  for (int z = lane / LANES; z < nsplit; z += 64 / LANES) {
    const f2 s = *reinterpret_cast<const f2*>(ml + 2 * z);
    f4 v;
    if (vec) {
      v = *reinterpret_cast<const f4*>(po + (int64_t)z * hd);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = d + e < hd ? po[(int64_t)z * hd + e] : 0.0f;
    }
    add(s[0], s[1], v);
  }
#pragma unroll
  for (int step = LANES; step < 64; step <<= 1) {
    const float mz = __shfl_xor(m, step), lz = __shfl_xor(den, step);
    f4 oz;
#pragma unroll
    for (int e = 0; e < 4; ++e) oz[e] = __shfl_xor(o[e], step);
    add(mz, lz, oz);
  }
  if (lane >= LANES) return;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (d + e < hd) out[r * hd + d + e] = from_f32<T>(den == 0.0f ? 0.0f : o[e] / den);
}

// Bytes of `nsplit` softmax states for each (token, head).
inline int64_t part_bytes(int64_t tokens, int q_heads, int hd, int nsplit) {
  return nsplit > 1 ? tokens * q_heads * nsplit * (hd + 2) * (int64_t)sizeof(float) : 0;
}

template <typename T, int GH, int DPL, typename Rule>
void launch_any(const AttnArgs<T>& a, const Rule& rule, hipStream_t st) {
  const int G = a.q_heads / a.kv_heads;
  const dim3 grid((unsigned)(a.tokens * a.kv_heads * ((G + GH - 1) / GH)), 1, (unsigned)a.nsplit);
  attn_any_kernel<T, GH, DPL, Rule><<<grid, kGenWaves * 64, 0, st>>>(a, rule);
}

// attn_any_kernel at the call's head size and group
template <typename T, typename Rule>
void launch_attn_any(const AttnArgs<T>& a, const Rule& rule, hipStream_t st) {
  const int G = a.q_heads / a.kv_heads;
  const auto by_group = [&](auto dpl) {
    constexpr int DPL = decltype(dpl)::value;
    if (G == 1) launch_any<T, 1, DPL>(a, rule, st);
    else if (G <= 4) launch_any<T, 4, DPL>(a, rule, st);
    else launch_any<T, 8, DPL>(a, rule, st);
  };
  if (a.hd <= 64) by_group(std::integral_constant<int, 1>{});
  else if (a.hd <= 128) by_group(std::integral_constant<int, 2>{});
  else by_group(std::integral_constant<int, 4>{});
}

template <typename T>
int launch_attn_join(const AttnArgs<T>& a, const char* what, hipStream_t st) {
  const int64_t rows = a.tokens * a.q_heads;
  const dim3 grid((unsigned)((rows + 3) / 4));
  if (a.hd <= 64) attn_join_kernel<T, 16><<<grid, 256, 0, st>>>(a.part, a.out, rows, a.hd, a.nsplit);
  else if (a.hd <= 128) attn_join_kernel<T, 32><<<grid, 256, 0, st>>>(a.part, a.out, rows, a.hd, a.nsplit);
  else attn_join_kernel<T, 64><<<grid, 256, 0, st>>>(a.part, a.out, rows, a.hd, a.nsplit);
  return launch_status(what);
}

// An entry point's arguments as a kernel takes them.
template <typename T>
AttnArgs<T> attn_args(const void* q, void* out, const void* kc, const void* vc, const int32_t* qseq,
                      const int32_t* qlen, const int32_t* tables, int64_t tokens, int q_heads, int kv_heads, int hd,
                      int bs, int max_blocks, int num_seqs, int64_t num_blocks, float scale, int64_t q_stride) {
  AttnArgs<T> a{};
  a.q = static_cast<const T*>(q);
  a.out = static_cast<T*>(out);
  a.kc = static_cast<const T*>(kc);
  a.vc = static_cast<const T*>(vc);
  a.qseq = qseq;
  a.qlen = qlen;
  a.tables = tables;
  a.tokens = tokens;
  a.num_blocks = num_blocks;
  a.q_stride = q_stride;
  a.q_heads = q_heads;
  a.kv_heads = kv_heads;
  a.hd = hd;
  a.bs = bs;
  a.max_blocks = max_blocks;
  a.num_seqs = num_seqs;
  a.most_keys = bs * max_blocks + 1;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.vec = hd % Pack<T>::N == 0 && aligned16(kc);
  a.nsplit = 1;
  return a;
}

// The checks that the two entry points share; NVF_OK with tokens > 0 means that a launch may follow.
inline int check_attn(const char* who, const void* q, const void* out, const void* kc, const void* vc,
                      const int32_t* qseq, const int32_t* qlen, const int32_t* tables, int64_t tokens, int q_heads,
                      int kv_heads, int head_dim, int block_size, int max_blocks, int num_seqs, int64_t num_blocks,
                      int64_t q_stride, const void* workspace, int dtype) {
  if (!dtype_ok(dtype)) return fail(NVF_ERR_INVALID, "%s: bad dtype %d", who, dtype);
  if (tokens < 0 || q_heads <= 0 || kv_heads <= 0 || head_dim <= 0 || block_size <= 0 || max_blocks <= 0 ||
      num_seqs < 0 || num_blocks < 0 || (tokens > 0 && num_blocks == 0))
    return fail(NVF_ERR_INVALID, "%s: bad shape", who);
  if (q_heads % kv_heads != 0)
    return fail(NVF_ERR_INVALID, "%s: q_heads=%d is not a multiple of kv_heads=%d", who, q_heads, kv_heads);
  if (head_dim > 256) return fail(NVF_ERR_INVALID, "%s: head_dim=%d exceeds 256", who, head_dim);
  if ((int64_t)block_size * max_blocks > INT32_MAX - 1024)
    return fail(NVF_ERR_INVALID, "%s: block tables of over 2^31 keys", who);
  if (q_stride < (int64_t)q_heads * head_dim)
    return fail(NVF_ERR_INVALID, "%s: q_stride must be >= q_heads * head_dim", who);
  if (workspace && !aligned16(workspace)) return fail(NVF_ERR_INVALID, "%s: workspace must be 16-byte aligned", who);
  if (tokens == 0) return NVF_OK;
  if (!q || !out || !kc || !vc || !qseq || !qlen || !tables) return fail(NVF_ERR_INVALID, "%s: NULL pointer", who);
  if (tokens * q_heads > INT32_MAX) return fail(NVF_ERR_INVALID, "%s: too many (token, head) pairs", who);
  return NVF_OK;
}

}  // namespace nvf
