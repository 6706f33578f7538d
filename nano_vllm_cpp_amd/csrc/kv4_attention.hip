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

// The cache blocks of a sequence's keys, as for other caches.
struct Kv4Slabs : SlabTable {
  template <typename T>
  __device__ __forceinline__ Kv4Slabs(const Kv4Args<T>& a, const FastDiv& d, int seq, int keys_end)
      : SlabTable(a, d, seq, keys_end) {
    row_b = (uint32_t)a.row_bytes;
  }
};

// ---------------------------------------------------------------------------
// Codes as fp16: a nibble at bits 0 .. 3 of a half word, or'ed with 0x6400, is the number 1024 + n, at bits 4 .. 7 with 0x5400
// 64 + n (their last places are 1 and 1/16).  Adding -(1024 + z) or -(64 + z) and multiplying by d are exact in
// fp16: n - z has four bits and a sign, d seven.
struct Kv4Half {       // a pair of groups' (or one group's, twice) scale and offsets
  f16x2 d, z_low, z_high;
};
__device__ __forceinline__ Kv4Half kv4_half(uint32_t words) {  // a word in each half
  return {__builtin_bit_cast(f16x2, words & 0xFFF0FFF0u), __builtin_bit_cast(f16x2, (words & 0x000F000Fu) | 0xE400E400u),
          __builtin_bit_cast(f16x2, (words << 4 & 0x00F000F0u) | 0xD400D400u)};
}
// The nibbles of x at bits 0 .. 3 and 16 .. 19, and those at 4 .. 7 and 20 .. 23, as values.
__device__ __forceinline__ uint32_t kv4_low(uint32_t x, const Kv4Half& h) {
  return __builtin_bit_cast(uint32_t, (__builtin_bit_cast(f16x2, (x & 0x000F000Fu) | 0x64006400u) + h.z_low) * h.d);
}
__device__ __forceinline__ uint32_t kv4_high(uint32_t x, const Kv4Half& h) {
  return __builtin_bit_cast(uint32_t, (__builtin_bit_cast(f16x2, (x & 0x00F000F0u) | 0x54005400u) + h.z_high) * h.d);
}
// Eight dimensions (a dword of codes) in the order 0 4 1 5 2 6 3 7.
__device__ __forceinline__ u32x4 kv4_eight(uint32_t codes, const Kv4Half& h) {
  const uint32_t up = codes >> 8;
  return u32x4{kv4_low(codes, h), kv4_high(codes, h), kv4_low(up, h), kv4_high(up, h)};
}

// A row of q as operands of the fp16 matrix cores: times 2^shift, so that its largest value lies in [2^10, 2^11), which fp16
// holds to 2^-24 beside it.  q of 16 bits is exact so (but for what lies 2^34 below the largest), fp32 takes two
// operands, what is left of each value in the second.
template <typename T>
constexpr int kQParts = sizeof(T) == 4 ? 2 : 1;
__device__ __forceinline__ int q_shift(float largest) {
  const int e = (int)(__builtin_bit_cast(uint32_t, largest) >> 23);  // biased; subnormal ones stay small
  return e == 0 || e == 255 ? 0 : 137 - e;
}

using Kv4Mma = AttnMma<_Float16>;
typedef Kv4Mma::v8 h8;

// One token: a wave is (token, kv head, 16 of its heads) and takes 32 keys at a time on its own:
//   S^T = K . Q^T     16x16x32 MFMAs: lane (row of 16 keys, quarter of the head) loads its codes in one go and turns them
//                     into the operand, one scale a lane (head size 256: two)
//   O^T += V^T . P^T  a lane holds head dimensions HD / 16 r .. of eight keys; byte b of two keys' codes side by side
//                     (one v_perm) is the low nibbles' operand of tile 2 b and the high ones' of 2 b + 1, so V needs no
//                     transpose; B = S^T's registers, P in two parts
// Waves of a workgroup take as many kv heads as fit side by side, so that each row's bytes are read together, and share out
// the keys where the heads are few.  Keys in flight lie in registers, the next unit's while this one is worked on.
template <int HD>
struct Kv4Lds {
  static constexpr int kState = HD * 16 + 32;  // O^T [HD][16], m [16], l [16] of a wave
  static constexpr int kBytes = 4 * kState * (int)sizeof(float);
};

template <typename T, int HD, int HEADS>
__global__ __launch_bounds__(256) void kv4_token_kernel(const Kv4Args<T> a, const FastDiv div) {
  constexpr int kWays = 4 / HEADS;              // waves that share a head's keys
  constexpr int kTiles = HD / 16, kSteps = HD / 32;
  constexpr int kKDwords = HD / 32;             // codes of a lane in K: HD / 4 dimensions
  constexpr int kKGroups = HD > 128 ? HD / 128 : 1;
  constexpr int kVBytes = HD / 32;              // of a lane in V: HD / 16 dimensions
  extern __shared__ __attribute__((aligned(16))) float state[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int col = lane & 15, g = lane >> 4;
  const int G = a.q_heads / a.kv_heads, parts = (G + 15) / 16, blocks = a.kv_heads / HEADS;
  const int rest = (int)(blockIdx.x % (blocks * parts));
  const int64_t t = blockIdx.x / (blocks * parts);
  const int kvh = rest / parts * HEADS + wave % HEADS, part = rest % parts, way = wave / HEADS;
  const int h0 = kvh * G + 16 * part, heads = min(16, (kvh + 1) * G - h0);
  const int L = __builtin_amdgcn_readfirstlane(key_count(a, t)), seq = __builtin_amdgcn_readfirstlane(a.qseq[t]);
  const uint32_t row_b = (uint32_t)a.row_bytes;

  // q: operand element j of step s is dimension HD / 4 g + 8 s + {0, 4, 1, 5, 2, 6, 3, 7}[j]
  h8 qf[kQParts<T>][kSteps];
  float to_exp2;
  {
    float x[kSteps][8], most = 0.0f;
    const T* q = a.q + t * a.q_stride + (int64_t)(h0 + col) * HD + HD / 4 * g;
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
#pragma unroll
      for (int e = 0; e < 8; e += Pack<T>::N) {
        if (col < heads) Pack<T>::unpack(ld16(q + 8 * s + e), x[s] + e);
        else
#pragma unroll
          for (int i = 0; i < Pack<T>::N; ++i) x[s][e + i] = 0.0f;
      }
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
#pragma unroll
      for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(x[s][e]));
    most = fmaxf(most, __shfl_xor(most, 16));
    most = fmaxf(most, __shfl_xor(most, 32));
    const int shift = q_shift(most);
    to_exp2 = ldexpf(a.scale_log2, -shift);
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float v = ldexpf(x[s][(j >> 1) + 4 * (j & 1)], shift);
        qf[0][s][j] = (_Float16)v;
        if constexpr (kQParts<T> == 2) qf[1][s][j] = rest_of(v, qf[0][s][j]);
      }
  }

  f32x4 o[kTiles];
#pragma unroll
  for (int d = 0; d < kTiles; ++d) o[d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  float m = -INFINITY, l = 0.0f;

  const int units = (L + 31) / 32;
  const int u0 = (int)((int64_t)units * blockIdx.z / a.nsplit) + way;
  const int u1 = (int)((int64_t)units * (blockIdx.z + 1) / a.nsplit);
  const Kv4Slabs table(a, div, seq, L);
  const uint32_t code = (uint32_t)(kvh * (HD / 2)), word = (uint32_t)(a.words + kvh * (HD / 16));
  const uint32_t k_off = (uint32_t)col * row_b + code + HD / 8 * g;
  const uint32_t kw_off = (uint32_t)col * row_b + word + 2 * (HD / 4 * g / kKv4Group);
  uint32_t v_off[4], vw_off[4];  // key 4 g + i of a slab
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v_off[i] = (uint32_t)(4 * g + i) * row_b + code + kVBytes * col;
    vw_off[i] = (uint32_t)(4 * g + i) * row_b + word + 2 * (HD / 16 * col / kKv4Group);
  }
  struct Keys {
    uint32_t k[2][kKDwords], kw[2];
    uint32_t v[2][4][(kVBytes + 3) / 4], vw[2][4];
  };
  const auto load = [&](const SlabEntry (&entry)[2], Keys& x) {
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      const SlabEntry& e = entry[kt];
      const uint64_t at = table.at(e);
      const int bytes = table.bytes(e);
      const __amdgpu_buffer_rsrc_t rk = rows_rsrc(a.k + at, bytes), rv = rows_rsrc(a.v + at, bytes);
      if constexpr (kKDwords == 2) {
        const u32x2 w = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(rk, k_off, 0, 0));
        x.k[kt][0] = w[0];
        x.k[kt][1] = w[1];
      } else {
#pragma unroll
        for (int i = 0; i < kKDwords / 4; ++i) {
          const u32x4 w = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rk, k_off + 16 * i, 0, 0));
#pragma unroll
          for (int j = 0; j < 4; ++j) x.k[kt][4 * i + j] = w[j];
        }
      }
      if constexpr (kKGroups == 2) x.kw[kt] = __builtin_amdgcn_raw_buffer_load_b32(rk, kw_off, 0, 0);
      else x.kw[kt] = __builtin_amdgcn_raw_buffer_load_b16(rk, kw_off, 0, 0);
      if (table.bad(e)) x.kw[kt] = kKv4NotANumber | kKv4NotANumber << 16;  // keys without a block: NaN where they are seen
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (kVBytes == 2) x.v[kt][i][0] = __builtin_amdgcn_raw_buffer_load_b16(rv, v_off[i], 0, 0);
        else if constexpr (kVBytes == 4) x.v[kt][i][0] = __builtin_amdgcn_raw_buffer_load_b32(rv, v_off[i], 0, 0);
        else {
          const u32x2 w = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(rv, v_off[i], 0, 0));
          x.v[kt][i][0] = w[0];
          x.v[kt][i][1] = w[1];
        }
        x.vw[kt][i] = __builtin_amdgcn_raw_buffer_load_b16(rv, vw_off[i], 0, 0);
      }
    }
  };
  const auto entries = [&](int u, SlabEntry (&e)[2]) {
    e[0] = table.entry(32 * u);
    e[1] = table.entry(32 * u + 16);
  };
  const auto add = [&](const Keys& x, int u) {
    f32x4 st[2];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      st[kt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int gr = 0; gr < kKGroups; ++gr) {
        const uint32_t w = kKGroups == 1 ? x.kw[kt] : gr == 0 ? x.kw[kt] & 0xFFFFu : x.kw[kt] >> 16;
        const Kv4Half h = kv4_half((w & 0xFFFFu) | w << 16);
#pragma unroll
        for (int i = 0; i < kSteps / kKGroups; ++i) {
          const int s = kSteps / kKGroups * gr + i;
          const h8 k = __builtin_bit_cast(h8, kv4_eight(x.k[kt][s], h));
#pragma unroll
          for (int p = 0; p < kQParts<T>; ++p) st[kt] = Kv4Mma::mma(k, qf[p][s], st[kt]);
        }
      }
    }
    // element j of tile kt is key 32 u + 16 kt + 4 g + j
    float mx = -INFINITY;
    const bool whole = 32 * u + 32 <= L;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (!whole && 32 * u + 16 * kt + 4 * g + j >= L) st[kt][j] = -INFINITY;
        mx = fmaxf(mx, st[kt][j]);
      }
    if (__any(fmaxf(m, mx * to_exp2) > m + kLazyMax)) {  // as in attend_token
      mx = fmaxf(mx, __shfl_xor(mx, 16));
      mx = fmaxf(mx, __shfl_xor(mx, 32));
      const float m_new = fmaxf(m, mx * to_exp2);
      const float alpha = __builtin_amdgcn_exp2f(m - (m_new == -INFINITY ? 0.0f : m_new));
      l *= alpha;
#pragma unroll
      for (int d = 0; d < kTiles; ++d) o[d] *= alpha;
      m = m_new;
    }
    const float m_use = m == -INFINITY ? 0.0f : m;
    h8 ph, pl;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float p = __builtin_amdgcn_exp2f(fmaf(st[kt][j], to_exp2, -m_use));
        l += p;
        ph[4 * kt + j] = (_Float16)p;
        pl[4 * kt + j] = rest_of(p, ph[4 * kt + j]);
      }
    Kv4Half h[4];
#pragma unroll
    for (int p = 0; p < 4; ++p) h[p] = kv4_half(x.vw[p / 2][2 * (p % 2)] | x.vw[p / 2][2 * (p % 2) + 1] << 16);
#pragma unroll
    for (int b = 0; b < kVBytes; ++b) {
      u32x4 low, high;
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        const uint32_t pair = __builtin_amdgcn_perm(x.v[p / 2][2 * (p % 2) + 1][b / 4], x.v[p / 2][2 * (p % 2)][b / 4],
                                                    0x0C040C00u + 0x00010001u * (b % 4));
        low[p] = kv4_low(pair, h[p]);
        high[p] = kv4_high(pair, h[p]);
      }
      o[2 * b] = Kv4Mma::mma(__builtin_bit_cast(h8, low), ph, o[2 * b]);
      o[2 * b] = Kv4Mma::mma(__builtin_bit_cast(h8, low), pl, o[2 * b]);
      o[2 * b + 1] = Kv4Mma::mma(__builtin_bit_cast(h8, high), ph, o[2 * b + 1]);
      o[2 * b + 1] = Kv4Mma::mma(__builtin_bit_cast(h8, high), pl, o[2 * b + 1]);
    }
  };
  // two units a trip, the register sets trading places; the block-table entries another one ahead
  Keys x, y;
  SlabEntry e[2] = {};
  if (u0 < u1) {
    entries(u0, e);
    load(e, x);
    if (u0 + kWays < u1) entries(u0 + kWays, e);
  }
#pragma unroll 1
  for (int u = u0; u < u1; u += 2 * kWays) {
    if (u + kWays < u1) {
      load(e, y);
      if (u + 2 * kWays < u1) entries(u + 2 * kWays, e);
    }
    add(x, u);
    if (u + kWays >= u1) break;
    if (u + 2 * kWays < u1) {
      load(e, x);
      if (u + 3 * kWays < u1) entries(u + 3 * kWays, e);
    }
    add(y, u + kWays);
  }
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);

  // O^T: lane column = head, element i of tile j dimension kTiles (4 g + i) + j
  if constexpr (kWays > 1) {
    float* own = state + wave * Kv4Lds<HD>::kState;
#pragma unroll
    for (int j = 0; j < kTiles; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) own[(kTiles * (4 * g + i) + j) * 16 + col] = o[j][i];
    if (g == 0) {
      own[HD * 16 + col] = m;
      own[HD * 16 + 16 + col] = l;
    }
    __syncthreads();
    if (way > 0) return;
    // the first wave of a head joins its ways
    float mall = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWays; ++w) mall = fmaxf(mall, state[(wave + w * HEADS) * Kv4Lds<HD>::kState + HD * 16 + col]);
    l = 0.0f;
#pragma unroll
    for (int j = 0; j < kTiles; ++j) o[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < kWays; ++w) {
      const float* of = state + (wave + w * HEADS) * Kv4Lds<HD>::kState;
      const float mw = of[HD * 16 + col], sc = mw == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(mw - mall);
      l += sc * of[HD * 16 + 16 + col];  // (no keys: O = l = 0, or NaN)
#pragma unroll
      for (int j = 0; j < kTiles; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[j][i] += sc * of[(kTiles * (4 * g + i) + j) * 16 + col];
    }
    m = mall;
  }
  if (col >= heads) return;
  const int64_t th = t * a.q_heads + h0 + col;
  if (a.nsplit > 1) {
    const int64_t pi = th * a.nsplit + blockIdx.z;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < kTiles; j += 4)
        st16(a.part + pi * HD + kTiles * (4 * g + i) + j,
             __builtin_bit_cast(u32x4, f32x4{o[j][i], o[j + 1][i], o[j + 2][i], o[j + 3][i]}));
    if (g == 0) {
      float* ml = a.part + a.tokens * a.q_heads * a.nsplit * HD + 2 * pi;
      ml[0] = m;
      ml[1] = l;
    }
  } else {
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    typedef T t4 __attribute__((ext_vector_type(4)));
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < kTiles; j += 4) {
        t4 v;
#pragma unroll
        for (int e2 = 0; e2 < 4; ++e2) v[e2] = (T)(o[j + e2][i] * inv);
        *reinterpret_cast<t4*>(a.out + th * HD + kTiles * (4 * g + i) + j) = v;
      }
  }
}

// Key ranges of a call of single tokens (kv4_token_kernel's workgroups, units of 32 keys).
inline int kv4_token_split(int64_t wgs, int64_t units, int64_t rows, int hd) {
  int best = 1;
  double least = 0.0;
  for (int n = 1; n <= 64 && (n == 1 || (n * 4 <= units && wgs * n <= 4096)); ++n) {
    const double t =
        (double)((wgs * n + 767) / 768) * ((double)((units + n - 1) / n) + 4) * 0.7 + split_us(n, rows, hd, false);
    if (n == 1 || t < least) {
      best = n;
      least = t;
    }
  }
  return best;
}
// The kv heads that a workgroup takes side by side.
inline int kv4_heads_side_by_side(int kv_heads) { return kv_heads % 4 == 0 ? 4 : kv_heads % 2 == 0 ? 2 : 1; }
inline int64_t kv4_token_wgs(int64_t tokens, int q_heads, int kv_heads) {
  return tokens * (kv_heads / kv4_heads_side_by_side(kv_heads)) * ((q_heads / kv_heads + 15) / 16);
}

template <typename T, int HD>
int launch_kv4_token(const Kv4Args<T>& a, hipStream_t st) {
  const FastDiv div((uint32_t)a.bs);
  const dim3 grid((unsigned)kv4_token_wgs(a.tokens, a.q_heads, a.kv_heads), 1, (unsigned)a.nsplit);
  const int side = kv4_heads_side_by_side(a.kv_heads);
  static std::once_flag lds_once;
  std::call_once(lds_once, [] {
    (void)hipFuncSetAttribute(reinterpret_cast<const void*>(&kv4_token_kernel<T, HD, 1>),
                              hipFuncAttributeMaxDynamicSharedMemorySize, Kv4Lds<HD>::kBytes);
    (void)hipFuncSetAttribute(reinterpret_cast<const void*>(&kv4_token_kernel<T, HD, 2>),
                              hipFuncAttributeMaxDynamicSharedMemorySize, Kv4Lds<HD>::kBytes);
  });
  if (side == 4) kv4_token_kernel<T, HD, 4><<<grid, 256, 0, st>>>(a, div);
  else if (side == 2) kv4_token_kernel<T, HD, 2><<<grid, 256, Kv4Lds<HD>::kBytes, st>>>(a, div);
  else kv4_token_kernel<T, HD, 1><<<grid, 256, Kv4Lds<HD>::kBytes, st>>>(a, div);
  return launch_status("paged_attention_kv4");
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

// The matrix cores' kernels take head sizes 64, 128 and 256 and blocks of a multiple of 16 keys.
inline bool kv4_mfma_shape(int hd, int bs) { return (hd == 64 || hd == 128 || hd == 256) && bs % 16 == 0; }
inline int kv4_split(int64_t tokens, int q_heads, int kv_heads, int hd, int bs, int max_blocks, int64_t max_query_len) {
  if (!kv4_mfma_shape(hd, bs)) return 1;
  return kv4_token_split(kv4_token_wgs(tokens, q_heads, kv_heads), ((int64_t)bs * max_blocks + 31) / 32, tokens * q_heads,
                         hd);
}

template <typename T>
int kv4_dispatch(Kv4Args<T> a, int64_t max_query_len, void* ws, int64_t ws_bytes, hipStream_t st) {
  const bool mfma = kv4_mfma_shape(a.hd, a.bs) && aligned16(a.q) && aligned16(a.out) && a.q_stride % Pack<T>::N == 0 &&
                    a.scale_log2 > 0.0f && a.row_bytes < INT32_MAX / 64 && a.num_blocks <= INT32_MAX / a.bs;
  if (!mfma) {
    launch_kv4_any(a, st);
    return launch_status("paged_attention_kv4");
  }
  const int nsplit = kv4_split(a.tokens, a.q_heads, a.kv_heads, a.hd, a.bs, a.max_blocks, max_query_len);
  a.part = static_cast<float*>(ws);
  a.nsplit = ws && ws_bytes >= part_bytes(a.tokens, a.q_heads, a.hd, nsplit) ? nsplit : 1;
  const int rc = a.hd == 64    ? launch_kv4_token<T, 64>(a, st)
                 : a.hd == 128 ? launch_kv4_token<T, 128>(a, st)
                               : launch_kv4_token<T, 256>(a, st);
  return rc == NVF_OK && a.nsplit > 1 ? launch_attn_join(a, "paged_attention_kv4(join)", st) : rc;
}

}  // namespace nvf

using namespace nvf;

extern "C" {

int64_t nvf_paged_attention_kv4_workspace_size(int64_t tokens, int q_heads, int kv_heads, int head_dim, int block_size,
                                               int max_blocks, int64_t max_query_len) {
  if (tokens <= 0 || q_heads <= 0 || kv_heads <= 0 || !kv4_head_dim_ok(head_dim) || block_size <= 0 || max_blocks <= 0 ||
      q_heads % kv_heads)
    return 0;
  return part_bytes(tokens, q_heads, head_dim,
                    kv4_split(tokens, q_heads, kv_heads, head_dim, block_size, max_blocks, max_query_len));
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
    rc = kv4_dispatch<T>(a, max_query_len, workspace, workspace_bytes, as_stream(stream));
  });
  return rc;
}

}  // extern "C"
